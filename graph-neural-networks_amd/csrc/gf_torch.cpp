// gf_torch.cpp -- the autograd nodes of the sequence and output operators, in C++: linear_recurrence, token_log_probs, distill_top.
//
// At the reference's own sizes these operators are a few microseconds of GPU work, so what a call costs is the host: a node written in Python
// pays for the interpreter twice (the backward pass runs on the autograd engine's thread) and for the conversion of seventeen arguments.  A
// training pass of distill_top on 100 x 5 logits takes 56 us here and took 87 us there (38 us of either are the engine's own), a call without
// gradients 10 us instead of 17.  The arithmetic is libgfhip.so's, reached through its C ABI;
// torch supplies memory, streams and the graph.  Arguments are checked here; what is refused is explained by the Python layer.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include "gfhip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// libgfhip.so as the Python layer has loaded it (bind)
struct Api {
    decltype(&gf_last_error) last_error;
    decltype(&gf_recurrence_checkpoint_floats) recurrence_checkpoint_floats;
    decltype(&gf_recurrence_workspace_bytes) recurrence_workspace_bytes;
    decltype(&gf_recurrence_forward) recurrence_forward;
    decltype(&gf_recurrence_backward) recurrence_backward;
    decltype(&gf_token_logp_workspace_bytes) token_workspace_bytes;
    decltype(&gf_token_logp_forward) token_forward;
    decltype(&gf_token_logp_backward) token_backward;
    decltype(&gf_distill_top_workspace_bytes) distill_workspace_bytes;
    decltype(&gf_distill_top_forward) distill_forward;
    decltype(&gf_distill_top_backward) distill_backward;
} api;

struct Refused : std::exception {};                             // arguments that are not served: the Python layer says which and why
struct ShapeError : std::runtime_error { using std::runtime_error::runtime_error; };      // GF_ERR_SHAPE: AssertionError, as everywhere in the package

void check(int rc, const char* what) {
    if (rc == GF_OK) return;
    const std::string msg = std::string(what) + ": " + api.last_error();
    if (rc == GF_ERR_SHAPE) throw ShapeError(msg);
    TORCH_CHECK(false, msg, " (status ", rc, ")");
}
void want(bool ok) {
    if (!ok) throw Refused();
}

// Forward-mode derivatives: a dual tensor does not require a gradient, so the direct path would answer without its tangent.
void no_tangent(std::initializer_list<Tensor> inputs) {
    for (const Tensor& t : inputs) want(!t.defined() || !t._fw_grad(/*level=*/0).defined());
}

int dtype_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return GF_F32;
        case at::kBFloat16: return GF_BF16;
        case at::kHalf: return GF_F16;
        default: return -1;
    }
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
int64_t* iptr(const Tensor& t) { return static_cast<int64_t*>(ptr(t)); }
Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }
Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }
// contiguous and aligned to 16 bytes (the recurrence's vector loads): a view that starts at an odd element is copied
Tensor dense(const Tensor& t) {
    if (!t.defined()) return t;
    Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
// gradients of a node that has no second derivative: under create_graph they refuse to be differentiated
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    auto error = std::make_shared<torch::autograd::DelayedError>("this operator is differentiable once only", (int64_t)grads.size());
    return error->apply(std::move(grads));
}

// ---- linear_recurrence -------------------------------------------------------------------------------------------------------
int gate_kind(const Tensor& q, const Tensor& u) {
    want(q.dim() == 4 && q.size(1) == u.size(1));
    int kind = 0;
    for (const auto& [axis, bit] : {std::pair<int, int>(0, GF_GATE_B), std::pair<int, int>(2, GF_GATE_H), std::pair<int, int>(3, GF_GATE_N)}) {
        want(q.size(axis) == 1 || q.size(axis) == u.size(axis));
        if (q.size(axis) == u.size(axis)) kind |= bit;
    }
    return kind;
}

struct Kinds {
    int check, hat;
    bool has_hat;
};

std::tuple<Tensor, Tensor, Tensor> recurrence_forward(const Tensor& u, const Tensor& qc, const Tensor& qh, const Tensor& z0, const Tensor& lengths, Kinds k,
                                                      bool keep) {
    const int64_t B = u.size(0), T = u.size(1), H = u.size(2), N = u.size(3);
    const c10::DeviceGuard guard(u.device());
    Tensor z = at::empty(u.sizes(), u.options()), zT = floats({B, H, N}, u), ckpt;
    if (B * H * N == 0) return {z, zT, ckpt};
    if (keep) ckpt = floats({(int64_t)api.recurrence_checkpoint_floats(B, T, H, N, k.check, k.has_hat, k.hat)}, u);
    const size_t nb = api.recurrence_workspace_bytes(B, T, H, N, k.check, k.has_hat, k.hat, 0);
    Tensor ws;
    if (nb) ws = bytes(nb, u);
    check(api.recurrence_forward(ptr(u), ptr(qc), k.check, ptr(qh), k.hat, fptr(z0), static_cast<int32_t*>(ptr(lengths)), ptr(z), fptr(zT), fptr(ckpt), ptr(ws),
                                 nb, dtype_of(u), B, T, H, N, stream_of(u)),
          "gf_recurrence_forward");
    return {z, zT, ckpt};
}

struct Recurrence : torch::autograd::Function<Recurrence> {
    static variable_list forward(AutogradContext* ctx, Tensor u, Tensor qc, std::optional<Tensor> qh_, std::optional<Tensor> z0_,
                                 std::optional<Tensor> lengths_, int64_t kc, int64_t kh) {
        Tensor qh = qh_.value_or(Tensor()), z0 = z0_.value_or(Tensor());
        const Tensor lengths = lengths_.value_or(Tensor());
        const bool keep = qc.requires_grad();
        ctx->saved_data["state"] = z0.defined();
        const Kinds k{(int)kc, (int)kh, qh.defined()};
        u = dense(u), qc = dense(qc), qh = dense(qh), z0 = dense(z0);
        auto [z, zT, ckpt] = recurrence_forward(u, qc, qh, z0, lengths, k, keep);
        ctx->save_for_backward({u, qc, qh, lengths, ckpt});
        ctx->saved_data["kinds"] = std::vector<int64_t>{kc, kh};
        ctx->set_materialize_grads(false);
        return {z, zT};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &u = saved[0], &qc = saved[1], &qh = saved[2], &lengths = saved[3], &ckpt = saved[4];
        const auto kinds = ctx->saved_data["kinds"].toIntVector();
        const Kinds k{(int)kinds[0], (int)kinds[1], qh.defined()};
        variable_list out(7);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const Tensor dz = dense(grads[0]), dzT = dense(grads[1]);
        const int64_t B = u.size(0), T = u.size(1), H = u.size(2), N = u.size(3);
        const c10::DeviceGuard guard(u.device());
        const bool empty = B * H * N == 0;
        if (ctx->needs_input_grad(0)) out[0] = at::empty_like(u);
        if (ctx->needs_input_grad(1)) out[1] = empty ? at::zeros_like(qc) : at::empty_like(qc);
        // (edges are numbered over the tensors that were given)
        if (k.has_hat && ctx->needs_input_grad(2)) out[2] = empty ? at::zeros_like(qh) : at::empty_like(qh);
        if (ctx->saved_data["state"].toBool() && ctx->needs_input_grad(k.has_hat ? 3 : 2)) out[3] = floats({B, H, N}, u);
        if (!empty) {
            const size_t nb = api.recurrence_workspace_bytes(B, T, H, N, k.check, k.has_hat, k.hat, 1);
            Tensor ws;
            if (nb) ws = bytes(nb, u);
            check(api.recurrence_backward(ptr(u), ptr(qc), k.check, ptr(qh), k.hat, static_cast<int32_t*>(ptr(lengths)), fptr(ckpt), ptr(dz), fptr(dzT),
                                          ptr(out[0]), ptr(out[1]), ptr(out[2]), fptr(out[3]), ptr(ws), nb, dtype_of(u), B, T, H, N, stream_of(u)),
                  "gf_recurrence_backward");
        }
        return once(std::move(out));
    }
};

std::tuple<Tensor, Tensor> linear_recurrence(const Tensor& u, const Tensor& qc, const std::optional<Tensor>& qh_, const std::optional<Tensor>& z0_,
                                             const std::optional<Tensor>& lengths_) {
    const Tensor qh = qh_.value_or(Tensor()), z0 = z0_.value_or(Tensor());
    Tensor lengths = lengths_.value_or(Tensor());
    no_tangent({u, qc, qh, z0});
    want(u.dim() == 4 && u.is_cuda() && dtype_of(u) >= 0);
    for (const int64_t n : u.sizes()) want(n <= (1ll << 31) - (1ll << 17));
    Kinds k{0, 0, qh.defined()};
    const auto gate = [&](const Tensor& q) {
        const int kind = gate_kind(q, u);
        want(q.device() == u.device() && q.scalar_type() == u.scalar_type());
        return kind;
    };
    k.check = gate(qc);
    if (k.has_hat) k.hat = gate(qh);
    if (z0.defined()) {
        want(z0.dim() == 3 && z0.size(0) == u.size(0) && z0.size(1) == u.size(2) && z0.size(2) == u.size(3));
        want(z0.device() == u.device() && z0.scalar_type() == at::kFloat);
    }
    if (lengths.defined()) {
        want(lengths.dim() == 1 && lengths.size(0) == u.size(0) && lengths.device() == u.device() && lengths.scalar_type() == at::kInt);
        lengths = lengths.contiguous();
    }
    if (at::GradMode::is_enabled() &&
        (u.requires_grad() || qc.requires_grad() || (qh.defined() && qh.requires_grad()) || (z0.defined() && z0.requires_grad()))) {
        const auto given = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
        auto out = Recurrence::apply(u, qc, given(qh), given(z0), given(lengths), (int64_t)k.check, (int64_t)k.hat);
        return {out[0], out[1]};
    }
    auto [z, zT, ckpt] = recurrence_forward(dense(u), dense(qc), dense(qh), dense(z0), lengths, k, false);
    return {z, zT};
}

// ---- rows of logits ------------------------------------------------------------------------------------------------------------
// [R, V] with unit stride inside a row (a view where the strides allow it) of logits with the classes along `dim`
Tensor rows_of(Tensor logits, int64_t dim, std::vector<int64_t>& lead) {
    const int64_t n = logits.dim();
    want(n >= 1 && dim >= -n && dim < n && logits.is_cuda() && dtype_of(logits) >= 0);
    if (dim < 0) dim += n;
    if (dim != n - 1) logits = logits.movedim(dim, -1);
    const int64_t V = logits.size(-1);
    want(V > 0 && V < (1ll << 31) - (1ll << 16));
    lead.assign(logits.sizes().begin(), logits.sizes().end() - 1);
    Tensor x = n == 2 ? logits : logits.reshape({-1, V});
    return V > 1 && x.stride(1) != 1 ? x.contiguous() : x;
}
bool usable(double temperature) { return temperature >= 1e-30 && temperature <= 1e30; }

// ---- token_log_probs -----------------------------------------------------------------------------------------------------------
struct TokenArgs {
    int64_t top, ignore;
    double temperature;
    bool entropy;
};

variable_list token_forward(const Tensor& x, const Tensor& tokens, const TokenArgs& a, Tensor* stats) {
    const int64_t R = x.size(0), V = x.size(1);
    const int dt = dtype_of(x);
    const c10::DeviceGuard guard(x.device());
    Tensor logp = floats({R}, x), ent, tl, ti;
    if (a.entropy) ent = floats({R}, x);
    if (a.top) {
        tl = floats({R, a.top}, x);
        ti = at::empty({R, a.top}, x.options().dtype(at::kLong));
    }
    if (stats) *stats = floats({R, 3}, x);
    if (R) {
        const size_t nb = api.token_workspace_bytes(R, V, a.top, dt);
        const Tensor ws = bytes(nb, x);
        check(api.token_forward(ptr(x), x.stride(0), iptr(tokens), (float)a.temperature, a.ignore, fptr(logp), fptr(ent), fptr(tl), iptr(ti), a.top,
                                stats ? fptr(*stats) : nullptr, ptr(ws), nb, dt, R, V, stream_of(x)),
              "gf_token_logp_forward");
    }
    return {logp, ent, tl, ti};
}

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
    static variable_list forward(AutogradContext* ctx, Tensor x, Tensor tokens, int64_t top, int64_t ignore, double temperature, bool entropy) {
        Tensor stats;
        variable_list out = token_forward(x, tokens, TokenArgs{top, ignore, temperature, entropy}, &stats);
        ctx->save_for_backward({x, tokens, stats, out[3]});
        ctx->saved_data["top"] = top;
        ctx->saved_data["ignore"] = ignore;
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["entropy"] = entropy;
        ctx->set_materialize_grads(false);
        if (top) ctx->mark_non_differentiable({out[3]});
        variable_list asked;                                    // a node's outputs are defined tensors: those that were asked for
        for (const auto& t : out)
            if (t.defined()) asked.push_back(t);
        return asked;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &tokens = saved[1], &stats = saved[2], &ti = saved[3];
        const int64_t top = ctx->saved_data["top"].toInt(), ent = ctx->saved_data["entropy"].toBool() ? 1 : 0;
        variable_list out(6);
        Tensor g[3];                                            // of logp, entropy, top_logp
        if (grads[0].defined()) g[0] = grads[0].contiguous();
        if (ent && grads[1].defined()) g[1] = grads[1].contiguous();
        if (top && grads[1 + ent].defined()) g[2] = grads[1 + ent].contiguous();
        if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return out;
        const int64_t R = x.size(0), V = x.size(1);
        const c10::DeviceGuard guard(x.device());
        out[0] = at::empty({R, V}, x.options());
        if (R)
            check(api.token_backward(ptr(x), x.stride(0), iptr(tokens), (float)ctx->saved_data["temperature"].toDouble(), ctx->saved_data["ignore"].toInt(),
                                     fptr(stats), iptr(ti), top, fptr(g[0]), fptr(g[1]), fptr(g[2]), ptr(out[0]), dtype_of(x), R, V,
                                     stream_of(x)),
                  "gf_token_logp_backward");
        return once(std::move(out));
    }
};

py::tuple token_log_probs(const Tensor& logits, Tensor tokens, int64_t top, double temperature, int64_t ignore, bool entropy, int64_t dim) {
    std::vector<int64_t> lead;
    no_tangent({logits});
    const Tensor x = rows_of(logits, dim, lead);
    want(usable(temperature) && top >= 0 && top <= 64 && top <= x.size(1));
    want(tokens.sizes() == at::IntArrayRef(lead) && tokens.scalar_type() == at::kLong && tokens.device() == x.device());
    tokens = lead.size() == 1 ? tokens.contiguous() : tokens.reshape({-1}).contiguous();
    variable_list out;
    if (at::GradMode::is_enabled() && x.requires_grad()) {
        const variable_list asked = TokenLogProbs::apply(x, tokens, top, ignore, temperature, entropy);
        out = {asked[0], entropy ? asked[1] : Tensor(), top ? asked[1 + entropy] : Tensor(), top ? asked[2 + entropy] : Tensor()};
    } else {
        out = token_forward(x, tokens, TokenArgs{top, ignore, temperature, entropy}, nullptr);
    }
    if (lead.size() != 1) {
        std::vector<int64_t> wide = lead;
        wide.push_back(top);
        for (int i = 0; i < 4; ++i)
            if (out[i].defined()) out[i] = out[i].view(i < 2 ? lead : wide);
    }
    const auto give = [](const Tensor& t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
    return py::make_tuple(give(out[0]), give(out[1]), give(out[2]), give(out[3]));
}

// ---- distill_top -----------------------------------------------------------------------------------------------------------------
// the loss [R]; *kept = stats [R, 3], then the named outputs' coefficients [R, K]
Tensor distill_forward(const Tensor& x, const Tensor& indices, const Tensor& values, double temperature, bool tail, Tensor* kept) {
    const int64_t R = x.size(0), V = x.size(1), K = indices.size(1);
    const int dt = dtype_of(x);
    const c10::DeviceGuard guard(x.device());
    Tensor loss = floats({R}, x);
    *kept = floats({R * (3 + K)}, x);
    if (R) {
        const size_t nb = api.distill_workspace_bytes(R, V, K, dt);
        const Tensor ws = bytes(nb, x);
        check(api.distill_forward(ptr(x), x.stride(0), iptr(indices), fptr(values), (float)temperature, tail, fptr(loss), fptr(*kept), fptr(*kept) + 3 * R,
                                  ptr(ws), nb, dt, R, V, K, stream_of(x)),
              "gf_distill_top_forward");
    }
    return loss;
}

struct DistillTop : torch::autograd::Function<DistillTop> {
    static Tensor forward(AutogradContext* ctx, Tensor x, Tensor indices, Tensor values, double temperature, bool tail) {
        Tensor kept, loss = distill_forward(x, indices, values, temperature, tail, &kept);
        ctx->save_for_backward({x, indices, kept});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["tail"] = tail;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &indices = saved[1], &kept = saved[2];
        const Tensor dloss = grads[0].contiguous();
        const int64_t R = x.size(0), V = x.size(1), K = indices.size(1);
        const c10::DeviceGuard guard(x.device());
        variable_list out(5);
        out[0] = at::empty({R, V}, x.options());
        if (R)
            check(api.distill_backward(ptr(x), x.stride(0), iptr(indices), fptr(kept) + 3 * R, fptr(kept), (float)ctx->saved_data["temperature"].toDouble(),
                                       ctx->saved_data["tail"].toBool(), fptr(dloss), ptr(out[0]), dtype_of(x), R, V, K, stream_of(x)),
                  "gf_distill_top_backward");
        return once(std::move(out));
    }
};

Tensor distill_top(const Tensor& logits, Tensor indices, Tensor values, double temperature, bool tail, int64_t dim) {
    std::vector<int64_t> lead;
    no_tangent({logits, values});
    const Tensor x = rows_of(logits, dim, lead);
    want(usable(temperature) && indices.dim() == (int64_t)lead.size() + 1);
    const int64_t K = indices.size(-1);
    want(K >= 1 && K <= 64 && indices.sizes().slice(0, lead.size()) == at::IntArrayRef(lead) && values.sizes() == indices.sizes());
    want(indices.scalar_type() == at::kLong && dtype_of(values) >= 0 && indices.device() == x.device() && values.device() == x.device());
    want(!(values.requires_grad() && at::GradMode::is_enabled()));
    if (indices.dim() != 2) indices = indices.reshape({-1, K}), values = values.reshape({-1, K});
    indices = indices.contiguous();
    values = values.to(at::kFloat).contiguous();
    Tensor kept;
    const Tensor loss = at::GradMode::is_enabled() && x.requires_grad() ? DistillTop::apply(x, indices, values, temperature, tail)
                                                                        : distill_forward(x, indices, values, temperature, tail, &kept);
    return lead.size() == 1 ? loss : loss.view(lead);
}

template <typename F> void take(F& f, const py::dict& addresses, const char* name) { f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>()); }

void bind(const py::dict& a) {                                  // {symbol: address} of the loaded library
    take(api.last_error, a, "gf_last_error");
    take(api.recurrence_checkpoint_floats, a, "gf_recurrence_checkpoint_floats");
    take(api.recurrence_workspace_bytes, a, "gf_recurrence_workspace_bytes");
    take(api.recurrence_forward, a, "gf_recurrence_forward");
    take(api.recurrence_backward, a, "gf_recurrence_backward");
    take(api.token_workspace_bytes, a, "gf_token_logp_workspace_bytes");
    take(api.token_forward, a, "gf_token_logp_forward");
    take(api.token_backward, a, "gf_token_logp_backward");
    take(api.distill_workspace_bytes, a, "gf_distill_top_workspace_bytes");
    take(api.distill_forward, a, "gf_distill_top_forward");
    take(api.distill_backward, a, "gf_distill_top_backward");
}

}  // namespace

PYBIND11_MODULE(_gf_torch, m) {
    py::register_exception<Refused>(m, "Refused");
    py::register_exception<ShapeError>(m, "ShapeError", PyExc_AssertionError);
    m.def("bind", &bind);
    m.def("linear_recurrence", &linear_recurrence);
    m.def("token_log_probs", &token_log_probs);
    m.def("distill_top", &distill_top);
}
