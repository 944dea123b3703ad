"""Autograd boundary of what a classifier answers and learns from (csrc/gf_output.hip), over rows of logits:

    logp, entropy, top_logp, top_tokens = token_log_probs(logits, tokens, top=K)
    loss = distill_top(logits, indices, values)

The reference feeds its readouts to torch losses and reduces them to an error rate (examples/sourceLocGNN.py:167,
alegnn/modules/evaluation.py:58-71); here an answer is a probability with its alternatives, and those alternatives are what a second network
can be trained on."""
from __future__ import annotations

import torch

from . import _lib
from .functional import _ptr
from .functional_seq import _DTYPES, _FLOATS, _on, _once, _require_cuda, _stream

TOP_MAX = 64
_I64 = (torch.int64,)


def _rows(who, logits, dim):
    """(rows as [R, V] with unit stride inside a row, leading shape): a view where the strides allow it, a copy otherwise."""
    assert logits.dim() >= 1 and -logits.dim() <= dim < logits.dim(), f"{who}: dim {dim} of logits with shape {tuple(logits.shape)}"
    _require_cuda(who, "logits", logits, _FLOATS)
    if dim % logits.dim() != logits.dim() - 1:
        logits = logits.movedim(dim, -1)
    V = logits.shape[-1]
    assert V > 0, f"{who}: logits have shape {tuple(logits.shape)}: no outputs to choose from"
    assert V < 2 ** 31 - 2 ** 16, f"{who}: {V} outputs (fewer than 2^31 - 2^16 are supported)"
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)
    if V > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x, logits.shape[:-1]


def _check_temperature(who, temperature):
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"alegnn_amd.{who}: temperature {temperature} (want a number between 1e-30 and 1e30)")
    return temperature


def _same_device(who, name, t, x):
    if t.device != x.device:
        raise RuntimeError(f"alegnn_amd.{who}: `{name}` is on '{t.device}', the logits on '{x.device}'")


def _tokens_forward(x, tokens, top, temperature, ignore_index, entropy, keep):
    L = _lib.lib()
    R, V = x.shape
    dev, dt = x.device, _DTYPES[x.dtype]
    with _on(dev):
        logp = torch.empty(R, dtype=torch.float32, device=dev)
        ent = torch.empty(R, dtype=torch.float32, device=dev) if entropy else None
        tl = torch.empty((R, top), dtype=torch.float32, device=dev) if top else None
        ti = torch.empty((R, top), dtype=torch.int64, device=dev) if top else None
        stats = torch.empty((R, 3), dtype=torch.float32, device=dev) if keep else None
        if R:
            nb = L.gf_token_logp_workspace_bytes(R, V, top, dt)
            ws = torch.empty(nb, dtype=torch.uint8, device=dev)
            _lib.check(L.gf_token_logp_forward(x.data_ptr(), x.stride(0), tokens.data_ptr(), temperature, ignore_index, logp.data_ptr(), _ptr(ent),
                                               _ptr(tl), _ptr(ti), top, _ptr(stats), ws.data_ptr(), nb, dt, R, V, _stream(dev)),
                       "gf_token_logp_forward")
    return logp, ent, tl, ti, stats


def _tokens_backward(ctx, dlogp, dent, dtop, _):
    L = _lib.lib()
    x, tokens, stats, ti = ctx.saved_tensors
    top, temperature, ignore_index = ctx.args
    R, V = x.shape
    dev = x.device
    if dlogp is None and dent is None and dtop is None:
        return (None,) * 6
    dlogp, dent, dtop = (None if g is None else g.contiguous() for g in (dlogp, dent, dtop))
    with _on(dev):
        dx = torch.empty((R, V), dtype=x.dtype, device=dev)
        if R:
            _lib.check(L.gf_token_logp_backward(x.data_ptr(), x.stride(0), tokens.data_ptr(), temperature, ignore_index, stats.data_ptr(), _ptr(ti),
                                                top, _ptr(dlogp), _ptr(dent), _ptr(dtop), dx.data_ptr(), _DTYPES[x.dtype], R, V, _stream(dev)),
                       "gf_token_logp_backward")
    return dx, None, None, None, None, None


class _TokenLogProbsFunction(torch.autograd.Function):
    """gf_token_logp_forward / gf_token_logp_backward (include/gfhip.h)."""

    @staticmethod
    def forward(ctx, x, tokens, top, temperature, ignore_index, entropy):
        logp, ent, tl, ti, stats = _tokens_forward(x, tokens, top, temperature, ignore_index, entropy, True)
        ctx.args = (top, temperature, ignore_index)
        ctx.save_for_backward(x, tokens, stats, ti)
        ctx.set_materialize_grads(False)
        if ti is not None:
            ctx.mark_non_differentiable(ti)
        return logp, ent, tl, ti

    @staticmethod
    def backward(ctx, *grads):
        return _once(_tokens_backward, ctx, *grads)


def token_log_probs(logits, tokens, top=0, temperature=1.0, ignore_index=-100, entropy=True, dim=-1):
    """Log probabilities of the given outputs under softmax(logits / temperature), with the entropy and the `top` best alternatives.

    logits [..., V] in float32, bfloat16 or float16 (the classes along `dim`: 1 for a LocalGNN's B x C x N; another axis than the last
    is copied); tokens [...] int64: the given output of each row.  Returns (logp, entropy, top_logp, top_tokens): float32 [...], float32 [...]
    (None with entropy=False), float32 [..., top] and int64 [..., top] (None with top=0), alternatives in descending order, equal logits
    in ascending index order.
    A row whose token is `ignore_index` has logp 0 (its entropy and alternatives are answered all the same); any other token outside [0, V)
    gives NaN.  -inf marks an output that is ruled out; a row of nothing else has logp -inf, entropy 0 and gradient 0.  A NaN or +inf logit
    makes its row's values NaN.  0 <= top <= min(V, 64).  Differentiable (once) in logits through logp, entropy and top_logp."""
    who = "token_log_probs"
    x, lead = _rows(who, logits, dim)
    temperature = _check_temperature(who, temperature)
    top = int(top)
    assert 0 <= top <= min(x.shape[1], TOP_MAX), f"{who}: top={top} for {x.shape[1]} outputs (want 0..min(V, {TOP_MAX}))"
    assert tokens.shape == lead, f"{who}: tokens have shape {tuple(tokens.shape)}, logits {tuple(logits.shape)} with the classes along {dim}"
    _require_cuda(who, "tokens", tokens, _I64)
    _same_device(who, "tokens", tokens, x)
    tokens = tokens.reshape(-1).contiguous()
    args = (x, tokens, top, temperature, int(ignore_index), bool(entropy))
    if torch.is_grad_enabled() and x.requires_grad:
        logp, ent, tl, ti = _TokenLogProbsFunction.apply(*args)
    else:
        logp, ent, tl, ti, _ = _tokens_forward(*args, False)
    if len(lead) == 1:
        return logp, ent, tl, ti
    return (logp.view(lead), None if ent is None else ent.view(lead), None if tl is None else tl.view(*lead, top),
            None if ti is None else ti.view(*lead, top))


def _distill_forward(x, indices, values, temperature, tail):
    L = _lib.lib()
    (R, V), K = x.shape, indices.shape[1]
    dev, dt = x.device, _DTYPES[x.dtype]
    with _on(dev):
        loss = torch.empty(R, dtype=torch.float32, device=dev)
        kept = torch.empty(R * (3 + K), dtype=torch.float32, device=dev)            # stats [R, 3], then the named outputs' coefficients [R, K]
        if R:
            nb = L.gf_distill_top_workspace_bytes(R, V, K, dt)
            ws = torch.empty(nb, dtype=torch.uint8, device=dev)
            at = kept.data_ptr()
            _lib.check(L.gf_distill_top_forward(x.data_ptr(), x.stride(0), indices.data_ptr(), values.data_ptr(), temperature, tail, loss.data_ptr(),
                                                at, at + 12 * R, ws.data_ptr(), nb, dt, R, V, K, _stream(dev)), "gf_distill_top_forward")
    return loss, kept


def _distill_backward(ctx, dloss):
    L = _lib.lib()
    x, indices, kept = ctx.saved_tensors
    temperature, tail = ctx.args
    (R, V), K = x.shape, indices.shape[1]
    dev = x.device
    dloss = dloss.contiguous()
    with _on(dev):
        dx = torch.empty((R, V), dtype=x.dtype, device=dev)
        if R:
            at = kept.data_ptr()
            _lib.check(L.gf_distill_top_backward(x.data_ptr(), x.stride(0), indices.data_ptr(), at + 12 * R, at, temperature, tail, dloss.data_ptr(),
                                                 dx.data_ptr(), _DTYPES[x.dtype], R, V, K, _stream(dev)), "gf_distill_top_backward")
    return dx, None, None, None, None


class _DistillTopFunction(torch.autograd.Function):
    """gf_distill_top_forward / gf_distill_top_backward (include/gfhip.h)."""

    @staticmethod
    def forward(ctx, x, indices, values, temperature, tail):
        loss, kept = _distill_forward(x, indices, values, temperature, tail)
        ctx.args = (temperature, tail)
        ctx.save_for_backward(x, indices, kept)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        return _once(_distill_backward, ctx, dloss)


def distill_top(logits, indices, values, temperature=1.0, tail=False, dim=-1):
    """Distillation loss of every row of logits against a teacher's K best outputs, with q = softmax(logits / temperature).

    logits [..., V] in float32, bfloat16 or float16 (classes along `dim`, as in token_log_probs); indices [..., K] int64 and values [..., K]
    floating point: the teacher's outputs, 1 <= K <= 64.  An index outside [0, V) (say -1) is padding.  Returns the loss [...] in float32.
      tail=False: values are logits (or log probabilities), p = softmax(values / temperature) over the row's entries;
                  loss = sum_k p_k (log p_k - log q[i_k]).
      tail=True:  values are log probabilities (at this temperature), p_k = exp(values_k), and what is left to one is one more outcome:
                  loss = sum_k p_k (log p_k - log q[i_k]) + p_r (log p_r - log q_r), q_r = the mass of the outputs that are not named.
                  (With every output named there are none: the loss is inf if the values leave any mass.)
    A row without entries (tail=False: without mass) has loss 0 and gradient 0; an index that is named twice counts as two entries.  No factor
    temperature^2 is applied.  Differentiable (once) in logits; the teacher's values are constants."""
    who = "distill_top"
    x, lead = _rows(who, logits, dim)
    temperature = _check_temperature(who, temperature)
    K = indices.shape[-1] if indices.dim() else 0
    assert 1 <= K <= TOP_MAX, f"{who}: indices have shape {tuple(indices.shape)} (want [..., K] with 1 <= K <= {TOP_MAX})"
    assert indices.shape == (*lead, K) and values.shape == indices.shape, (
        f"{who}: indices {tuple(indices.shape)} and values {tuple(values.shape)} for logits {tuple(logits.shape)} with the classes along {dim}")
    _require_cuda(who, "indices", indices, _I64)
    _require_cuda(who, "values", values, _FLOATS)
    _same_device(who, "indices", indices, x)
    _same_device(who, "values", values, x)
    if values.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("distill_top: values.requires_grad is not supported (the teacher's outputs are constants); detach them")
    if indices.dim() != 2:
        indices, values = indices.reshape(-1, K), values.reshape(-1, K)
    args = (x, indices.contiguous(), values.float().contiguous(), temperature, int(bool(tail)))
    if torch.is_grad_enabled() and x.requires_grad:
        loss = _DistillTopFunction.apply(*args)
    else:
        loss = _distill_forward(*args)[0]
    return loss if len(lead) == 1 else loss.view(lead)
