// gf_recur.hip -- gated linear recurrence  z_t = qc_t z_{t-1} + qh_t u_t  over [B, T, H, N], forward and backward.
//
// The recursion of GatedGRNN (reference graphML.py:1421-1462) with B(S) = identity and sigma = identity: linear in the state, so a
// stretch of steps is one pair (A, h) with z_out = A z_in + h, and stretches compose: (A2, h2) o (A1, h1) = (A2 A1, A2 h1 + h2).
// The channels c = h N + n are contiguous and independent; time is cut into tiles:
//   thread     kL steps x V channels, all loads issued before the first use
//   wave       its rows of 16 lanes hold consecutive stretches (GW = 4), joined by row swaps, or all lanes are channels (GW = 1)
//   workgroup  WT waves along time (joined through LDS, one barrier per slab) or 4 waves side by side along the channels (no barrier)
//   slab       GW WT kL steps, walked in order with the state in registers
//   split      few channels and a long T: the time axis is cut into S splits, recur_split_kernel reads the inputs for each split's (A, h),
//              the main kernel starts from the composition of the splits before its own (inputs are read twice).  There A has an exponent of its
//              own: a product over thousands of gates may leave the range of a float32 where no state does
// Backward: with r_t = qc_t g_t the adjoint  g_t = dz_t + r_{t+1}  is the same recurrence run backwards with the same coefficients, and
// needs the states z_{t-1} in fp32 for the gate's gradient: they are recomputed from the inputs (which qh's gradient reads anyway) and one
// fp32 checkpoint per slab instead of being read back rounded.  Bound by HBM: forward reads u, qc, qh and writes z, backward reads u, qc,
// qh, dz and writes du, dqc, dqh.
//
// State and products are fp32, the gate sums over a launch's partial ones fp64; outputs are rounded once.  Steps at or behind a sequence's length leave the state as it is (A = 1,
// h = 0), whatever they hold (their values are replaced behind the load), and their outputs and gradients are zero.
#include "gf_num.h"

#include <type_traits>

namespace {

// Chosen by measurement (GPU time, forward and backward):
constexpr int kL = 4;              // steps per thread and slab: 4 / 8: 1.37 / 1.52 ms for 32 x 257 x 53824 bf16 (twice the registers), 221 / 208 us for 65537 x 808
constexpr int kGW = 4;             // time groups of a wave.  Timed before the joins by row swaps, which are for 4: backward of 32 x 257 x 53824 with 4 / 8 / 2
                                   // (of 8 steps each) 0.89 / 1.02 / 0.97 ms
constexpr int kMaxSplit = 128;     // splits of a long time axis: 64 / 128 / 256: 238 / 221 / 210 us for 65537 x 808 bf16 (on an earlier form 344 / 307 / 323)

// What the kernels reach now: 32 x 257 x 53824 bf16 with lengths 0 .. 257: forward 0.47 ms, backward 0.90 ms = 4.9 TB/s of the rows they touch (a large
// copy: 4.7); 65537 x 808 bf16 with a gate per step: split 20 + forward 50, split 33 + backward 111 us: the instructions per element (30 forward,
// 50 backward in a join of 16 steps) weigh as much as the bytes there; 20 x 100 x 1600 fp32: forward 11, backward 20, gate sums 6 us.
// What costs more than its bytes: gates that lack one of the channel axes (their products go through memory in fp32: 32 x 257 x 32 x 1682 bf16 with two
// node / feature gates: forward 0.77 / 0.57, backward 1.75 / 1.46, sums 0.73 / 1.29 ms, full gates 0.70 + 1.25), and odd channel counts (one channel
// per thread: 32 x 257 x 31 x 1681 with full gates 1.46 + 2.76 ms in bf16, 2.09 + 4.27 in fp32, against 1.42 + 2.49 for 32 x 1682 in fp32).
struct Gate {                      // a gate of shape [B|1, T, H|1, N|1]: element (b, t, h, n) at b sb + t st + channel offset
    const void* p;
    int64_t sb;
    int32_t st;
    int32_t kind;                  // GF_GATE_H | GF_GATE_N
};

struct Dims {
    int32_t B, T, H, N, C;         // C = H N
    int32_t chunks;                // channel chunks of a workgroup
    int32_t splits, split_len;     // steps per split (a multiple of the slab)
    int32_t every;                 // steps per checkpoint
    int32_t nck;                   // checkpoints per sequence
};

// What a wave reads or writes of a tensor in a slab: `base` is the same for the whole wave (sequence, wave's first row), `off` is the lane's byte
// offset in it (its row group's first row, its channel), so the address of step l is one scalar and one 32-bit vector register.
struct Stream {
    char* base;
    int64_t step;                  // bytes per time step
    uint32_t off;
    int32_t row;                   // the lane's first row at ts = 0
    __device__ __forceinline__ char* at(int t) const { return base + (int64_t)t * step + off; }             // t = ts + l
};
template <typename D> __device__ __forceinline__ Stream stream(const void* p, int64_t first, int wrow, int lrow, int st, int coff) {
    Stream s;
    s.base = const_cast<char*>(static_cast<const char*>(p)) + (first + (int64_t)wrow * st) * (int64_t)sizeof(D);
    s.step = (int64_t)st * (int64_t)sizeof(D);
    s.off = ((uint32_t)lrow * (uint32_t)st + (uint32_t)coff) * (uint32_t)sizeof(D);
    s.row = wrow + lrow;
    return s;
}
// The loads of a slab are straight-line code: all of them are in flight before the first one is waited for.  VEC: V elements per step, else one value
// for the thread's V channels (a gate without the node axis; V > 1 only where they share the feature).  Rows behind the last step of the tensor
// are clamped to the last live one (only in a tensor's last slab: the lane's address is then computed the long way).
template <typename D, int V, bool VEC> __device__ __forceinline__ void load_one(const char* p, gf_vec<D, V>& raw) {
    if constexpr (VEC) raw = *reinterpret_cast<const gf_vec<D, V>*>(p);
    else raw.e[0] = *reinterpret_cast<const D*>(p);
}
template <typename D, int V, bool VEC>
__device__ __forceinline__ void load_slab(const Stream& s, int ts, bool inside, int last, gf_vec<D, V> (&raw)[kL]) {
    if (inside) {
#pragma unroll
        for (int l = 0; l < kL; ++l) load_one<D, V, VEC>(s.at(ts + l), raw[l]);
    } else {
#pragma unroll
        for (int l = 0; l < kL; ++l) load_one<D, V, VEC>(s.base + s.off + (int64_t)(min(ts + s.row + l, last) - s.row) * s.step, raw[l]);
    }
}
template <typename D, int V, bool VEC> __device__ __forceinline__ float pick(const gf_vec<D, V>& raw, int i) { return gf_to_f<D>(raw.e[VEC ? i : 0]); }

__device__ __forceinline__ int gate_coff(const Gate& g, int c, int N) {
    if (g.kind == (GF_GATE_H | GF_GATE_N)) return c;
    if (g.kind == GF_GATE_N) return c % N;
    if (g.kind == GF_GATE_H) return c / N;
    return 0;
}

// where a thread works: channel c (V of them), time group tg of its workgroup
template <int V, int WT, int GW>
struct Place {
    static constexpr int CX = 64 / GW;                          // channel threads of a wave
    static constexpr int NW = WT == 1 ? 4 : WT;                 // waves of a workgroup
    static constexpr int CW = (WT == 1 ? NW * CX : CX) * V;     // channels of a workgroup
    static constexpr int SLAB = WT * GW * kL;
    int lane, wave, cx, tg, c, b, split, column;
    bool on, work;                  // channel inside the row; (uniform) workgroup has work
    __device__ __forceinline__ Place(const Dims& d) {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
        cx = lane % CX;
        tg = (WT == 1 ? 0 : wave * GW) + lane / CX;
        unsigned blk = blockIdx.x;
        if (d.splits > 1) {
            // Workgroups go to the 8 XCDs in turn.  Long runs put all chunks of a (sequence, split) on one XCD: a chunk's row segments (128 bytes,
            // starting at any multiple of V elements) share their cache lines with its neighbours' (65537 x 808 bf16, forward and backward: 248 ->
            // 233 us).  Without splits there is work enough to stream, and sequences of unlike lengths are better spread over the XCDs
            // (32 x 257 x 53824, lengths 0 .. 257: 1361 us spread, 1513 us with a sequence per XCD).
            const unsigned x = blk & 7u, k = blk >> 3;
            blk = (x + 8u * (k / (unsigned)d.chunks)) * (unsigned)d.chunks + k % (unsigned)d.chunks;
        }
        const unsigned chunk = blk % (unsigned)d.chunks, rest = blk / (unsigned)d.chunks;
        work = rest < (unsigned)d.splits * (unsigned)d.B;
        column = (int)chunk;
        split = (int)(rest % (unsigned)d.splits);
        b = (int)(rest / (unsigned)d.splits);
        c = (int)chunk * CW + (WT == 1 ? wave * CX : 0) * V + cx * V;
        on = c < d.C;
    }
};

// Rows of 16 lanes moved inside the vector unit (no LDS traffic): of x's rows (0, 1, 2, 3), lo16 = (0, 0, 2, 2), hi16 = (1, 1, 3, 3),
// lo32 = (0, 1, 0, 1), hi32 = (2, 3, 2, 3).
__device__ __forceinline__ float lo16(float x) { return __uint_as_float(__builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false)[0]); }
__device__ __forceinline__ float hi16(float x) { return __uint_as_float(__builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false)[1]); }
__device__ __forceinline__ float lo32(float x) { return __uint_as_float(__builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false)[0]); }
__device__ __forceinline__ float hi32(float x) { return __uint_as_float(__builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false)[1]); }

// exclusive composition of the stretches before (FWD) / behind (!FWD) this thread's own, and of the whole slab.  GW = 4: the wave's rows of 16
// lanes are the stretches (pairs first, then the halves); WT > 1: the waves' compositions through LDS.  SAME: the thread's V channels share their gate,
// so their products are one (lane swaps are no common subexpressions to the compiler; 65537 x 808 bf16, a gate per
// step: forward 53 -> 49, backward 118 -> 110 us).
template <int V, int WT, int GW, bool FWD, bool SAME>
__device__ __forceinline__ void join(const float (&A)[V], const float (&S)[V], float (&Ae)[V], float (&Se)[V], float (&At)[V], float (&St)[V],
                                     int lane, int wave, float* lds) {
    static_assert(GW == 1 || GW == 4, "a wave's stretches are its rows of 16 lanes, or one");
    constexpr int CX = 64 / GW;
    const int row = lane >> 4;
    const bool odd = row & 1, upper = row & 2;
    const bool second = FWD ? odd : !odd, later = FWD ? upper : !upper;     // second of its pair, of the second pair, in walking order
    float a = 1.f, a1 = 1.f, a2 = 1.f, a3 = 1.f, ap = 1.f, ea = 1.f;        // products: channel i's, or all channels' (SAME)
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const bool own = !SAME || i == 0;
        float s = S[i];
        if (own) a = ap = A[i];
        Ae[i] = 1.f, Se[i] = 0.f;
        if constexpr (GW == 4) {
            // step 1: within pairs of rows; step 2: the other pair's composition, which both its rows hand over
            if (own) {
                a = A[i];
                a1 = FWD ? lo16(a) : hi16(a);
                ap = second ? a * a1 : a;
                const float pa = FWD ? hi16(ap) : lo16(ap);                 // a pair's composition, in both its rows
                a2 = FWD ? lo32(pa) : hi32(pa);                             // the first pair's, everywhere
                a3 = FWD ? hi32(pa) : lo32(pa);                             // the second pair's
                ea = second ? a1 : 1.f;                                     // before my row, inside its pair
            }
            const float s1 = FWD ? lo16(s) : hi16(s);
            s = second ? fmaf(a, s1, s) : s;
            const float ps = FWD ? hi16(s) : lo16(s);
            const float s2 = FWD ? lo32(ps) : hi32(ps);
            const float es = second ? s1 : 0.f;
            Ae[i] = later ? ea * a2 : ea;
            Se[i] = later ? fmaf(ea, s2, es) : es;
            if constexpr (WT == 1) {                            // all four rows: second pair after the first
                const float s3 = FWD ? hi32(ps) : lo32(ps);
                At[i] = a2 * a3;
                St[i] = fmaf(a3, s2, s3);
            } else {
                s = later ? fmaf(ap, s2, s) : s;
            }
        } else if constexpr (WT == 1) {
            At[i] = a, St[i] = s;
        }
        if constexpr (WT > 1) {
            if (lane / CX == (FWD ? GW - 1 : 0)) {              // last row in walking order: the wave's composition
                lds[((wave * CX + lane % CX) * V + i) * 2] = later ? ap * a2 : ap;
                lds[((wave * CX + lane % CX) * V + i) * 2 + 1] = s;
            }
        }
    }
    if constexpr (WT > 1) {
        __syncthreads();
        float pa[V], ps[V];
#pragma unroll
        for (int i = 0; i < V; ++i) At[i] = 1.f, St[i] = 0.f, pa[i] = 1.f, ps[i] = 0.f;
#pragma unroll
        for (int k = 0; k < WT; ++k) {
            const int w = FWD ? k : WT - 1 - k;
            if (w == wave) {
#pragma unroll
                for (int i = 0; i < V; ++i) pa[i] = At[i], ps[i] = St[i];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float wa = lds[((w * CX + lane % CX) * V + (SAME ? 0 : i)) * 2], ws = lds[((w * CX + lane % CX) * V + i) * 2 + 1];
                St[i] = fmaf(wa, St[i], ws);
                At[i] *= wa;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {                           // waves before mine, then the groups before mine
            Se[i] = fmaf(Ae[i], ps[i], Se[i]);
            Ae[i] *= pa[i];
        }
    }
}

// A stretch longer than a slab: z_out = m 2^e z_in + s.  The product of its gates has an exponent of its own, so that it may leave the range of a
// float32 where the states do not (gates above one while the state is zero, say): a stretch's s is in range whenever the step by step walk is,
// and m 2^e only ever meets the state it is applied to.  e stays within 2^29 (a thread's stretch is at most 2^31 / 144 steps of |e| <= 150 / 8 each).
struct Span {
    float m;
    int e;
    float s;
};
__device__ __forceinline__ float span_apply(const Span& x, float z) { return ldexpf(x.m * z, x.e) + x.s; }
__device__ __forceinline__ void span_norm(float& m, int& e) {
    e += __builtin_amdgcn_frexp_expf(m);                        // (0 for 0, inf and NaN, which the mantissa keeps)
    m = __builtin_amdgcn_frexp_mantf(m);
}
__device__ __forceinline__ Span span_after(const Span& x, const Span& y) {      // x behind y
    Span r;
    r.m = x.m * y.m, r.e = x.e + y.e, r.s = span_apply(x, y.s);
    span_norm(r.m, r.e);
    r.e = min(max(r.e, -(1 << 29)), 1 << 29);
    return r;
}
// LDS of a workgroup's spans: [m, e, s][time group][channel of the workgroup]
template <int V, int WT, int GW> constexpr int span_floats() { return 3 * WT * GW * (64 / GW) * V; }

// The time groups' spans, joined in walking order: thread k < CX V answers channel k.  SAME: the V channels of a group share m and e.
template <int V, int WT, int GW, bool FWD, bool SAME>
__device__ __forceinline__ Span join_groups(const float (&m)[V], const int (&e)[V], const float (&s)[V], const Place<V, WT, GW>& p, float* lds) {
    constexpr int TG = WT * GW, CW = 64 / GW * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int at = p.tg * CW + p.cx * V + i;
        lds[at] = m[SAME ? 0 : i];
        lds[TG * CW + at] = __int_as_float(e[SAME ? 0 : i]);
        lds[2 * TG * CW + at] = s[i];
    }
    __syncthreads();
    Span r{1.f, 0, 0.f};
    if (p.wave == 0) {
        static_assert(CW <= 64, "a channel per lane of the first wave");
#pragma unroll
        for (int g = 0; g < TG; ++g) {
            const int at = (FWD ? g : TG - 1 - g) * CW + p.lane % CW;
            r = span_after(Span{lds[at], __float_as_int(lds[TG * CW + at]), lds[2 * TG * CW + at]}, r);
        }
    }
    return r;
}

// carry becomes the state behind the splits [s0, s1) of the thread's channels, whose spans are shared out over the time groups (walked forwards or
// backwards).  agg: per split three planes m, e, s of `all` channels.
template <int V, int WT, int GW, bool FWD, bool SAME>
__device__ __forceinline__ void join_splits(const float* __restrict__ agg, int64_t all, int64_t chan, int s0, int s1, const Place<V, WT, GW>& p,
                                            float (&carry)[V], float* lds) {
    constexpr int TG = WT * GW, CW = 64 / GW * V;
    const int q = (s1 - s0 + TG - 1) / TG, lo = min(s1, s0 + p.tg * q), hi = min(s1, lo + q);
    float m[V], s[V];
    int e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) m[i] = 1.f, e[i] = 0, s[i] = 0.f;
#pragma unroll 4
    for (int k = lo; k < hi; ++k) {
        const float* g = agg + 3 * (int64_t)(FWD ? k : lo + hi - 1 - k) * all + chan;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int o = SAME ? 0 : i;
            const Span r = span_after(Span{g[o], __float_as_int(g[all + o]), g[2 * all + i]}, Span{m[i], e[i], s[i]});
            m[i] = r.m, e[i] = r.e, s[i] = r.s;
        }
    }
    const Span r = join_groups<V, WT, GW, FWD, SAME>(m, e, s, p, lds);
    __syncthreads();
    if (threadIdx.x < CW) lds[threadIdx.x] = r.m, lds[CW + threadIdx.x] = __int_as_float(r.e), lds[2 * CW + threadIdx.x] = r.s;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int at = p.cx * V + i;
        carry[i] = span_apply(Span{lds[at], __float_as_int(lds[CW + at]), lds[2 * CW + at]}, carry[i]);
    }
    __syncthreads();                                            // (the slabs' joins use the same memory)
}

// ---- splits: each one's span, forwards or backwards ---------------------------------------------------------------------------
// Every thread walks a stretch of its own (split_len / 16 steps) and the workgroup joins once, so this pass is loads and three operations per element
// (the product's exponent is taken out every eight steps).
// CN / HAT: how q_check / q_hat are loaded (CN: V elements or one; HAT: 0 no q_hat, 1 V elements, 2 one).
template <typename D, int V, bool FWD, bool CN, int HAT>
__global__ __launch_bounds__(256) void recur_split_kernel(const D* __restrict__ in, Gate gc, Gate gh, const int32_t* __restrict__ lengths,
                                                          float* __restrict__ agg, Dims d) {
    constexpr int WT = 4, GW = 4, kU = 8;
    using P = Place<V, WT, GW>;
    __shared__ float s_span[span_floats<V, WT, GW>()];
    const P p(d);
    if (!p.work) return;
    if (p.split == (FWD ? d.splits - 1 : 0)) return;            // (uniform) nothing starts behind the last split
    int len = d.T;
    if (lengths) len = min(max(lengths[p.b], 0), d.T);
    const int pc = p.on ? p.c : d.C - V;
    const int64_t all = (int64_t)d.B * d.C;
    const int q = d.split_len / (WT * GW), lo = p.split * d.split_len + p.tg * q, hi = min(lo + q, len);
    const int64_t C = d.C;
    const D* pi = in ? in + ((int64_t)p.b * d.T + lo) * C + pc : nullptr;
    const D* pg = static_cast<const D*>(gc.p) + p.b * gc.sb + (int64_t)lo * gc.st + gate_coff(gc, pc, d.N);
    const D* ph = HAT ? static_cast<const D*>(gh.p) + p.b * gh.sb + (int64_t)lo * gh.st + gate_coff(gh, pc, d.N) : nullptr;
    float A[V], S[V];                                           // (one product for channels that share their gate)
    int E[V];
#pragma unroll
    for (int i = 0; i < V; ++i) A[i] = 1.f, E[i] = 0, S[i] = 0.f;
    auto norm = [&] {
#pragma unroll
        for (int i = 0; i < (CN ? V : 1); ++i) span_norm(A[i], E[i]);
    };
    auto take = [&](const gf_vec<D, V>& ra, const gf_vec<D, V>& rb, const gf_vec<D, V>& rq) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float a = pick<D, V, CN>(ra, i);
            float b = gf_to_f<D>(rb.e[i]);
            if (HAT) b *= pick<D, V, HAT == 1>(rq, i);
            S[i] = FWD ? fmaf(a, S[i], b) : a * (b + S[i]);
            if (CN || i == 0) A[i] *= a;
        }
    };
    const int n = max(hi - lo, 0), whole = in ? n / kU * kU : 0;
    // forwards: eight steps at a time, then the rest; backwards: the rest first
    auto eight = [&](int k) {
        gf_vec<D, V> ra[kU], rb[kU], rq[kU];
#pragma unroll
        for (int l = 0; l < kU; ++l) {
            load_one<D, V, true>(reinterpret_cast<const char*>(pi + (k + l) * C), rb[l]);
            load_one<D, V, CN>(reinterpret_cast<const char*>(pg + (int64_t)(k + l) * gc.st), ra[l]);
            if (HAT) load_one<D, V, HAT == 1>(reinterpret_cast<const char*>(ph + (int64_t)(k + l) * gh.st), rq[l]);
        }
#pragma unroll
        for (int e = 0; e < kU; ++e) take(ra[FWD ? e : kU - 1 - e], rb[FWD ? e : kU - 1 - e], rq[FWD ? e : kU - 1 - e]);
        norm();
    };
    auto one = [&](int k) {
        gf_vec<D, V> ra, rb, rq;
#pragma unroll
        for (int i = 0; i < V; ++i) rb.e[i] = gf_from_f<D>(0.f);
        if (in) load_one<D, V, true>(reinterpret_cast<const char*>(pi + k * C), rb);
        load_one<D, V, CN>(reinterpret_cast<const char*>(pg + (int64_t)k * gc.st), ra);
        if (HAT) load_one<D, V, HAT == 1>(reinterpret_cast<const char*>(ph + (int64_t)k * gh.st), rq);
        take(ra, rb, rq);
        norm();
    };
    if (FWD) {
        for (int k = 0; k < whole; k += kU) eight(k);
        for (int k = whole; k < n; ++k) one(k);
    } else {
        for (int k = n - 1; k >= whole; --k) one(k);
        for (int k = whole - kU; k >= 0; k -= kU) eight(k);
    }
    const Span r = join_groups<V, WT, GW, FWD, !CN>(A, E, S, p, s_span);
    const int c = p.column * P::CW + (int)threadIdx.x;
    if (threadIdx.x < P::CW && c < d.C) {
        float* g = agg + 3 * (int64_t)p.split * all + (int64_t)p.b * d.C + c;
        g[0] = r.m, g[all] = __int_as_float(r.e), g[2 * all] = r.s;
    }
}

// ---- forward -------------------------------------------------------------------------------------------------------------
template <typename D, int V, int WT, int GW, bool CN, int HAT>
__global__ __launch_bounds__(64 * (WT == 1 ? 4 : WT)) void recur_fwd_kernel(const D* __restrict__ u, Gate gc, Gate gh, const float* __restrict__ z0,
                                                                            const int32_t* __restrict__ lengths, D* __restrict__ z,
                                                                            float* __restrict__ zT, float* __restrict__ ckpt,
                                                                            float* __restrict__ agg, Dims d) {
    using P = Place<V, WT, GW>;
    constexpr int JOIN = WT == 1 ? 1 : WT * P::CX * V * 2;
    __shared__ float s_mem[WT == 1 ? 1 : span_floats<V, WT, GW>()];        // the splits' spans, then two joins' buffers
    const P p(d);
    if (!p.work) return;
    int len = d.T;
    if (lengths) len = min(max(lengths[p.b], 0), d.T);
    const int pc = p.on ? p.c : d.C - V;                        // lanes behind the last channel read its values and store nothing
    const int64_t chan = (int64_t)p.b * d.C + pc, all = (int64_t)d.B * d.C;
    const int wrow = WT == 1 ? 0 : p.wave * GW * kL, lrow = p.lane / P::CX * kL;
    const Stream su = stream<D>(u, (int64_t)p.b * d.T * d.C, wrow, lrow, d.C, pc), sz = stream<D>(z, (int64_t)p.b * d.T * d.C, wrow, lrow, d.C, pc);
    const Stream sc = stream<D>(gc.p, p.b * gc.sb, wrow, lrow, gc.st, gate_coff(gc, pc, d.N));
    const Stream sh = stream<D>(gh.p, p.b * gh.sb, wrow, lrow, gh.st, gate_coff(gh, pc, d.N));
    float carry[V];
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = 0.f;
    if (z0) {
#pragma unroll
        for (int i = 0; i < V; ++i) carry[i] = z0[chan + i];
    }
    if constexpr (WT > 1) {
        if (p.split > 0) join_splits<V, WT, GW, true, !CN>(agg, all, chan, 0, p.split, p, carry, s_mem);     // (uniform) the splits before this one
    }
    const int tbeg = p.split * d.split_len, tend = min(d.T, tbeg + d.split_len);
    const int live_end = min(tend, len);
    gf_vec<D, V> ra[kL], rb[kL], rq[kL];
    auto fetch = [&](int ts) {
        const bool inside = ts + P::SLAB <= d.T;                // (uniform)
        load_slab<D, V, true>(su, ts, inside, len - 1, rb);
        load_slab<D, V, CN>(sc, ts, inside, len - 1, ra);
        if (HAT) load_slab<D, V, HAT == 1>(sh, ts, inside, len - 1, rq);
    };
    if (tbeg < live_end) fetch(tbeg);
    int flip = 0;
    for (int ts = tbeg; ts < tend; ts += P::SLAB, flip ^= 1) {
        const int t0 = ts + p.tg * kL;
        if (ts >= len) {                                        // (uniform) behind the sequence: the state stays, the output is zero
            if (p.on) {
                const float zero[V] = {};
                for (int l = 0; l < kL; ++l)
                    if (t0 + l < d.T) gf_store<D, V>(reinterpret_cast<D*>(sz.at(ts + l)), zero);
            }
            continue;
        }
        float a[kL][V], b[kL][V], A[V], S[V];
#pragma unroll
        for (int l = 0; l < kL; ++l)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                a[l][i] = pick<D, V, CN>(ra[l], i);
                b[l][i] = gf_to_f<D>(rb[l].e[i]);
                if (HAT) b[l][i] *= pick<D, V, HAT == 1>(rq[l], i);
            }
        if (ts + P::SLAB < live_end) fetch(ts + P::SLAB);       // (into the registers just read: the next slab loads while this one is joined)
        if (ts + P::SLAB > len) {                               // (uniform) the sequence ends in this slab
#pragma unroll
            for (int l = 0; l < kL; ++l)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (t0 + l >= len) a[l][i] = 1.f, b[l][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) A[i] = 1.f, S[i] = 0.f;
#pragma unroll
        for (int l = 0; l < kL; ++l)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                S[i] = fmaf(a[l][i], S[i], b[l][i]);
                A[i] *= a[l][i];
            }
        float Ae[V], Se[V], At[V], St[V], h[V];
        join<V, WT, GW, true, !CN>(A, S, Ae, Se, At, St, p.lane, p.wave, s_mem + (WT == 1 ? 0 : flip * JOIN));
#pragma unroll
        for (int i = 0; i < V; ++i) {
            h[i] = fmaf(Ae[i], carry[i], Se[i]);
            carry[i] = fmaf(At[i], carry[i], St[i]);
        }
        if (p.on) {
            if (ckpt && t0 < d.T && t0 % d.every == 0) {
                float* k = ckpt + ((int64_t)p.b * d.nck + t0 / d.every) * d.C + pc;
#pragma unroll
                for (int i = 0; i < V; ++i) k[i] = h[i];
            }
            if (ts + P::SLAB <= len) {
#pragma unroll
                for (int l = 0; l < kL; ++l) {
#pragma unroll
                    for (int i = 0; i < V; ++i) h[i] = fmaf(a[l][i], h[i], b[l][i]);
                    gf_store<D, V>(reinterpret_cast<D*>(sz.at(ts + l)), h);
                }
            } else {
#pragma unroll
                for (int l = 0; l < kL; ++l) {
                    if (t0 + l < d.T) {
                        float o[V];
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            h[i] = fmaf(a[l][i], h[i], b[l][i]);
                            o[i] = t0 + l < len ? h[i] : 0.f;
                        }
                        gf_store<D, V>(reinterpret_cast<D*>(sz.at(ts + l)), o);
                    }
                }
            }
        }
    }
    if (p.on && p.tg == 0) {
        if (p.split == d.splits - 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) zT[chan + i] = carry[i];
        }
    }
}

// ---- backward ------------------------------------------------------------------------------------------------------------
enum { kOutNone = 0, kOutDirect = 1, kOutProduct = 2, kOutTime = 3 };   // a gate's gradient: not wanted | its own element | fp32 product, summed
                                                                       // by recur_fold_kernel | sum over the wave's channels, then likewise
struct GateOut {
    void* p;
    int32_t mode;
};

template <int CTRL> __device__ __forceinline__ float row_shift(float v) {       // the lane that many below in the row, 0 at its start
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, false));
}

template <typename D, int V, int CX>
__device__ __forceinline__ void put_gate(const GateOut& g, const float (&v)[V], char* direct, int64_t off, int64_t toff, bool on, bool live, int lane) {
    if (g.mode == kOutDirect) {
        if (on && live) gf_store<D, V>(reinterpret_cast<D*>(direct), v);
    } else if (g.mode == kOutProduct) {
        if (on && live) gf_store<float, V>(static_cast<float*>(g.p) + off, v);
    } else if (g.mode == kOutTime) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) s += on ? v[i] : 0.f;
        s += row_shift<0x111>(s);                               // over the row of 16 lanes: its last lane has the sum
        s += row_shift<0x112>(s);
        s += row_shift<0x114>(s);
        s += row_shift<0x118>(s);
        if constexpr (CX == 64) {
            s += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(s), 0x142, 0xa, 0xf, false));
            s += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(s), 0x143, 0xc, 0xf, false));
        }
        if (live && lane % CX == CX - 1) static_cast<float*>(g.p)[toff] = s;
    }
}

template <typename D, int V, int WT, int GW, bool CN, int HAT>
__global__ __launch_bounds__(64 * (WT == 1 ? 4 : WT)) void recur_bwd_kernel(const D* __restrict__ u, Gate gc, Gate gh, const int32_t* __restrict__ lengths,
                                                                            const D* __restrict__ dz, const float* __restrict__ dzT,
                                                                            const float* __restrict__ ckpt, D* __restrict__ du, GateOut oc, GateOut oh,
                                                                            float* __restrict__ dz0, float* __restrict__ agg, Dims d) {
    using P = Place<V, WT, GW>;
    constexpr int JOIN = WT == 1 ? 1 : WT * P::CX * V * 2;
    static_assert(WT == 1 || 4 * JOIN <= span_floats<V, WT, GW>(), "four joins' buffers in the memory of the splits' spans");
    __shared__ float s_mem[WT == 1 ? 1 : span_floats<V, WT, GW>()];
    const P p(d);
    if (!p.work) return;
    int len = d.T;
    if (lengths) len = min(max(lengths[p.b], 0), d.T);
    const int pc = p.on ? p.c : d.C - V;
    const int64_t ub = (int64_t)p.b * d.T * d.C + pc, chan = (int64_t)p.b * d.C + pc, all = (int64_t)d.B * d.C;
    const int wrow = WT == 1 ? 0 : p.wave * GW * kL, lrow = p.lane / P::CX * kL;
    const int64_t first = (int64_t)p.b * d.T * d.C;
    const Stream su = stream<D>(u, first, wrow, lrow, d.C, pc), sg = stream<D>(dz, first, wrow, lrow, d.C, pc), so = stream<D>(du, first, wrow, lrow, d.C, pc);
    const Stream soc = stream<D>(oc.p, first, wrow, lrow, d.C, pc), soh = stream<D>(oh.p, first, wrow, lrow, d.C, pc);
    const Stream sc = stream<D>(gc.p, p.b * gc.sb, wrow, lrow, gc.st, gate_coff(gc, pc, d.N));
    const Stream sh = stream<D>(gh.p, p.b * gh.sb, wrow, lrow, gh.st, gate_coff(gh, pc, d.N));
    // sums over a wave's channels (time gates): one row of [B, T] per wave column
    const int64_t cols = (int64_t)p.column * (WT == 1 ? P::NW : 1) + (WT == 1 ? p.wave : 0);
    const int64_t tbase = (cols * d.B + p.b) * d.T;
    float carry[V];
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = 0.f;
    if (dzT) {
#pragma unroll
        for (int i = 0; i < V; ++i) carry[i] = dzT[chan + i];
    }
    if constexpr (WT > 1) {                             // (uniform) the splits behind this one
        if (p.split + 1 < d.splits) join_splits<V, WT, GW, false, !CN>(agg, all, chan, p.split + 1, d.splits, p, carry, s_mem);
    }
    const int tbeg = p.split * d.split_len, tend = min(d.T, tbeg + d.split_len);
    const int slabs = tend > tbeg ? (tend - tbeg + P::SLAB - 1) / P::SLAB : 0;
    gf_vec<D, V> ra[kL], rx[kL], rq[kL], rg[kL];
    auto fetch = [&](int ts) {
        const bool inside = ts + P::SLAB <= d.T;                // (uniform)
        if (dz) load_slab<D, V, true>(sg, ts, inside, len - 1, rg);
        load_slab<D, V, true>(su, ts, inside, len - 1, rx);
        load_slab<D, V, CN>(sc, ts, inside, len - 1, ra);
        if (HAT) load_slab<D, V, HAT == 1>(sh, ts, inside, len - 1, rq);
    };
    if (tbeg < min(tend, len)) fetch(tbeg + (min(tend, len) - tbeg - 1) / P::SLAB * P::SLAB);     // the last slab with a live step
    int flip = 0;
    for (int sl = slabs - 1; sl >= 0; --sl) {
        const int ts = tbeg + sl * P::SLAB, t0 = ts + p.tg * kL;
        if (ts >= len) {                                        // (uniform) behind the sequence: nothing flows, the gradients are zero
            const float zero[V] = {};
            for (int l = 0; l < kL; ++l) {
                const int64_t off = ub + (int64_t)(t0 + l) * d.C;
                const bool in = t0 + l < d.T;
                if (du && p.on && in) gf_store<D, V>(reinterpret_cast<D*>(so.at(ts + l)), zero);
                if (oc.mode) put_gate<D, V, P::CX>(oc, zero, soc.at(ts + l), off, tbase + t0 + l, p.on, in, p.lane);
                if (HAT && oh.mode) put_gate<D, V, P::CX>(oh, zero, soh.at(ts + l), off, tbase + t0 + l, p.on, in, p.lane);
            }
            continue;
        }
        const bool ends = ts + P::SLAB > len;                   // (uniform) the sequence ends in this slab
        float a[kL][V], x[kL][V], q[kL][V], g[kL][V], A[V], R[V];
#pragma unroll
        for (int l = 0; l < kL; ++l)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                a[l][i] = pick<D, V, CN>(ra[l], i);
                x[l][i] = gf_to_f<D>(rx[l].e[i]);
                q[l][i] = HAT ? pick<D, V, HAT == 1>(rq[l], i) : 1.f;
                g[l][i] = dz ? gf_to_f<D>(rg[l].e[i]) : 0.f;
            }
        if (sl > 0) fetch(ts - P::SLAB);                        // (into the registers just read: the next slab loads while this one is joined)
        if (ends) {
#pragma unroll
            for (int l = 0; l < kL; ++l)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (t0 + l >= len) a[l][i] = 1.f, x[l][i] = 0.f, q[l][i] = 1.f, g[l][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) A[i] = 1.f, R[i] = 0.f;
#pragma unroll
        for (int l = kL - 1; l >= 0; --l)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                R[i] = a[l][i] * (g[l][i] + R[i]);
                A[i] *= a[l][i];
            }
        float Ae[V], Re[V], At[V], Rt[V], r[V];
        join<V, WT, GW, false, !CN>(A, R, Ae, Re, At, Rt, p.lane, p.wave, s_mem + (WT == 1 ? 0 : flip * JOIN));
#pragma unroll
        for (int i = 0; i < V; ++i) {
            r[i] = fmaf(Ae[i], carry[i], Re[i]);
            carry[i] = fmaf(At[i], carry[i], Rt[i]);
        }
        {
            float zp[kL][V];
            if (oc.mode != kOutNone) {                          // the states z_{t-1} of this slab, from its checkpoint
                float S[V], h[V], Se[V], St[V];
#pragma unroll
                for (int i = 0; i < V; ++i) S[i] = 0.f;
#pragma unroll
                for (int l = 0; l < kL; ++l)
#pragma unroll
                    for (int i = 0; i < V; ++i) S[i] = fmaf(a[l][i], S[i], HAT ? x[l][i] * q[l][i] : x[l][i]);
                join<V, WT, GW, true, !CN>(A, S, Ae, Se, At, St, p.lane, p.wave, s_mem + (WT == 1 ? 0 : (flip + 1) * JOIN));
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float start = ckpt[((int64_t)p.b * d.nck + ts / d.every) * d.C + pc + i];
                    h[i] = fmaf(Ae[i], start, Se[i]);
                }
#pragma unroll
                for (int l = 0; l < kL; ++l)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        zp[l][i] = h[i];
                        h[i] = fmaf(a[l][i], h[i], HAT ? x[l][i] * q[l][i] : x[l][i]);
                    }
            }
#pragma unroll
            for (int l = kL - 1; l >= 0; --l) {
                float o[V], oq[V], ox[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float gt = g[l][i] + r[i];            // dL/dz_t
                    o[i] = gt * zp[l][i];
                    oq[i] = gt * x[l][i];
                    ox[i] = HAT ? gt * q[l][i] : gt;
                    r[i] = a[l][i] * gt;
                }
                bool in = true;
                if (ends) {                                     // padded steps pass the state's gradient on and have none of their own
                    in = t0 + l < d.T;
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (t0 + l >= len) o[i] = oq[i] = ox[i] = 0.f;
                }
                const int64_t off = ub + (int64_t)(t0 + l) * d.C;
                if (du && p.on && in) gf_store<D, V>(reinterpret_cast<D*>(so.at(ts + l)), ox);
                if (oc.mode) put_gate<D, V, P::CX>(oc, o, soc.at(ts + l), off, tbase + t0 + l, p.on, in, p.lane);
                if (HAT && oh.mode) put_gate<D, V, P::CX>(oh, oq, soh.at(ts + l), off, tbase + t0 + l, p.on, in, p.lane);
            }
        }
        flip ^= 2;
    }
    if (p.on && p.tg == 0) {
        if (p.split == 0 && dz0) {
#pragma unroll
            for (int i = 0; i < V; ++i) dz0[chan + i] = carry[i];
        }
    }
}

// Sum of the fp32 products [rows, T, inner, H, N] ... over the axes a gate does not have, in a fixed order: out[b, t, h, n] (gate shape).
// src [nb, B, T, Hs, Ns] : nb partial rows; axes: nb always, B if !GF_GATE_B, Hs if !(kind & H), Ns if !(kind & N).
// One wave per output element where the node axis is summed, one thread per element otherwise (coalesced over nodes).  The sums are fp64 and rounded
// once: a gate per step of an odd number of channels has thousands of partial ones (one after the other in fp32 they were off by 6e-7 of the result).
__device__ __forceinline__ double sum_strided(const float* __restrict__ p, int n, int64_t stride, double s) {   // in order, eight loads in flight
    int i = 0;
    for (; i + 8 <= n; i += 8) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = p[(i + e) * stride];
#pragma unroll
        for (int e = 0; e < 8; ++e) s += v[e];
    }
    for (; i < n; ++i) s += p[i * stride];
    return s;
}

struct Fold {                      // src [nb, B, T, Hs, Ns] -> out in the gate's shape
    const float* src;
    void* out;
    int32_t nb, Hs, Ns, kind;
    int64_t total;
};

// blockIdx.y: q_check's and q_hat's gradient in one launch
template <typename D>
__global__ __launch_bounds__(256) void recur_fold_kernel(Fold f0, Fold f1, int B, int T) {
    const Fold f = blockIdx.y ? f1 : f0;
    const float* __restrict__ src = f.src;
    D* __restrict__ out = static_cast<D*>(f.out);
    const int nb = f.nb, Hs = f.Hs, Ns = f.Ns, kind = f.kind;
    const int64_t total = f.total;
    const bool byN = !(kind & GF_GATE_N) && Ns > 1;
    const int Ho = (kind & GF_GATE_H) ? Hs : 1, No = (kind & GF_GATE_N) ? Ns : 1, Bo = (kind & GF_GATE_B) ? B : 1;
    const int lane = threadIdx.x & 63;
    const int64_t stride = byN ? (int64_t)gridDim.x * 4 : (int64_t)gridDim.x * 256, row = (int64_t)Hs * Ns;
    for (int64_t o = byN ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x * 256 + threadIdx.x; o < total; o += stride) {
        const int n = (int)(o % No);
        const int64_t o1 = o / No;
        const int h = (int)(o1 % Ho);
        const int64_t o2 = o1 / Ho;
        const int t = (int)(o2 % T), b = (int)(o2 / T);
        const float* p = src + ((int64_t)b * T + t) * row + (int64_t)h * Ns + n;
        const int hs = Ho == 1 ? Hs : 1, bs = Bo == 1 ? B : 1;
        double s = 0.0;
        if (byN) {
            for (int k = 0; k < nb * bs; ++k)                   // (nb > 1 only with Hs = Ns = 1)
                for (int hh = 0; hh < hs; ++hh)
                    for (int m = lane; m < Ns; m += 64) s += p[(int64_t)k * T * row + (int64_t)hh * Ns + m];
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) s += __shfl_xor(s, off);
            if (lane == 0) out[o] = gf_from_f<D>((float)s);
        } else {
            if (hs > 1) {
                for (int bb = 0; bb < bs; ++bb) s = sum_strided(p + (int64_t)bb * T * row, hs, Ns, s);
            } else if (bs > 1) {
                s = sum_strided(p, nb * bs, T * row, s);        // (partial rows of all sequences: [nb][B] is one axis)
            } else {
                s = sum_strided(p, nb, (int64_t)B * T * row, s);
            }
            out[o] = gf_from_f<D>((float)s);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
struct Shape {                     // what the kernels are chosen by: a function of the sizes alone, so forward and backward agree
    int V, WT, GW, slab, splits, split_len;
};

Shape choose(int B, int T, int64_t C, int N, int kinds) {
    Shape s;
    const bool within = kinds != 0;                             // some gate is shared along one of the two channel axes
    const int64_t by = within ? N : C;                          // (C is a multiple of N)
    s.V = by % 4 == 0 ? 4 : by % 2 == 0 ? 2 : 1;
    const int64_t lanes = (int64_t)B * ((C + s.V - 1) / s.V);
    const int need = (T + kL - 1) / kL;                         // time groups that have work
    // enough threads to keep the memory busy (128k with 8 vector loads each), no more groups than there is time
    s.WT = 1, s.GW = 1;
    if (need > 1) s.GW = kGW;
    if (need > 8 && lanes * 8 < 131072) s.WT = 4;
    s.slab = s.WT * s.GW * kL;
    const int64_t blocks = (int64_t)B * ((C + (int64_t)(s.WT == 1 ? 4 : 1) * (64 / s.GW) * s.V - 1) / ((int64_t)(s.WT == 1 ? 4 : 1) * (64 / s.GW) * s.V));
    const int slabs = (T + s.slab - 1) / s.slab;
    s.splits = 1;
    if (s.WT == 4 && blocks < 256 && slabs >= 8) {                           // fewer workgroups than compute units and a long way to walk
        int64_t want = (2048 + blocks - 1) / blocks;
        if (want > slabs / 4) want = slabs / 4;
        if (want > kMaxSplit) want = kMaxSplit;
        s.splits = want < 1 ? 1 : (int)want;
    }
    const int per = (slabs + s.splits - 1) / s.splits;
    s.split_len = per * s.slab;
    if (slabs > 0) s.splits = (slabs + per - 1) / per;
    return s;
}

bool aligned(const void* p, size_t bytes) { return p == nullptr || reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int kind_bits(int kind_c, bool has_h, int kind_h) {             // which channel axes some gate lacks
    int m = 0;
    for (int k : {kind_c, has_h ? kind_h : (GF_GATE_H | GF_GATE_N)}) {
        if ((k & GF_GATE_H) && !(k & GF_GATE_N)) m |= 1;
        if (!(k & GF_GATE_H) && (k & GF_GATE_N)) m |= 2;
    }
    return m;
}

Gate make_gate(const void* p, int kind, int T, int H, int N) {
    Gate g;
    g.p = p;
    g.kind = kind & (GF_GATE_H | GF_GATE_N);
    g.st = ((kind & GF_GATE_H) ? H : 1) * ((kind & GF_GATE_N) ? N : 1);
    g.sb = (kind & GF_GATE_B) ? (int64_t)T * g.st : 0;
    return g;
}

int check_dims(const char* who, int B, int T, int H, int N, int dtype, int kc, int kh) {
    GF_REQUIRE_ARG(gf_dtype_ok(dtype), "%s: dtype %d", who, dtype);
    GF_REQUIRE_ARG((kc & ~7) == 0 && (kh & ~7) == 0, "%s: gate kinds %d, %d", who, kc, kh);
    GF_REQUIRE_SHAPE(B > 0 && T >= 0 && H > 0 && N > 0, "%s: bad shape B=%d T=%d H=%d N=%d", who, B, T, H, N);
    GF_REQUIRE_SHAPE((int64_t)H * N < (1ll << 26), "%s: H * N = %lld channels", who, (long long)H * N);   // (a lane's byte offset is 32 bits: 13 rows)
    GF_REQUIRE_SHAPE(T <= INT32_MAX - (1 << 16), "%s: T = %d steps", who, T);                 // (a slab's end stays an int32)
    return GF_OK;
}

Dims make_dims(const Shape& s, int B, int T, int H, int N) {
    Dims d;
    d.B = B, d.T = T, d.H = H, d.N = N, d.C = H * N;
    const int cw = (s.WT == 1 ? 4 : 1) * (64 / s.GW) * s.V;
    d.chunks = (d.C + cw - 1) / cw;
    d.splits = s.splits, d.split_len = s.split_len;
    d.every = s.slab;
    d.nck = (T + s.slab - 1) / s.slab;
    return d;
}

template <int V, int WT, int GW, typename F>
int by_gates(bool cn, int hat, F&& f) {
    using std::bool_constant;
    using std::integral_constant;
    const integral_constant<int, V> v;
    const integral_constant<int, WT> wt;
    const integral_constant<int, GW> gw;
    if constexpr (V == 1) {                                     // one element per thread either way
        return hat ? f(v, wt, gw, bool_constant<true>(), integral_constant<int, 1>()) : f(v, wt, gw, bool_constant<true>(), integral_constant<int, 0>());
    } else if (cn) {
        return hat == 0 ? f(v, wt, gw, bool_constant<true>(), integral_constant<int, 0>())
             : hat == 1 ? f(v, wt, gw, bool_constant<true>(), integral_constant<int, 1>()) : f(v, wt, gw, bool_constant<true>(), integral_constant<int, 2>());
    } else {
        return hat == 0 ? f(v, wt, gw, bool_constant<false>(), integral_constant<int, 0>())
             : hat == 1 ? f(v, wt, gw, bool_constant<false>(), integral_constant<int, 1>()) : f(v, wt, gw, bool_constant<false>(), integral_constant<int, 2>());
    }
}
template <int V, typename F>
int by_time(const Shape& s, bool cn, int hat, F&& f) {
    if (s.GW == 1) return by_gates<V, 1, 1>(cn, hat, f);
    return s.WT == 1 ? by_gates<V, 1, kGW>(cn, hat, f) : by_gates<V, 4, kGW>(cn, hat, f);
}
// f(V, WT, GW, CN, HAT) as compile-time constants
template <typename F>
int by_shape(const Shape& s, const Gate& gc, const Gate& gh, F&& f) {
    const bool cn = gc.kind & GF_GATE_N;
    const int hat = !gh.p ? 0 : (gh.kind & GF_GATE_N) ? 1 : 2;
    return s.V == 4 ? by_time<4>(s, cn, hat, f) : s.V == 2 ? by_time<2>(s, cn, hat, f) : by_time<1>(s, cn, hat, f);
}

int wave_columns(const Dims& d, const Shape& s) { return d.chunks * (s.WT == 1 ? 4 : 1); }

int out_mode(int kind) {
    if ((kind & 7) == (GF_GATE_B | GF_GATE_H | GF_GATE_N)) return kOutDirect;
    return (kind & (GF_GATE_H | GF_GATE_N)) == 0 ? kOutTime : kOutProduct;
}
size_t out_floats(int kind, const Dims& d, const Shape& s) {
    const int m = out_mode(kind);
    if (m == kOutDirect) return 0;
    const size_t f = m == kOutTime ? (size_t)wave_columns(d, s) * d.B * d.T : (size_t)d.B * d.T * d.C;
    return (f + 3) / 4 * 4;                                     // the next region starts 16-byte aligned
}
size_t agg_floats(const Dims& d) { return d.splits > 1 ? ((size_t)3 * d.splits * d.B * d.C + 3) / 4 * 4 : 0; }

template <typename D>
int forward_t(const Shape& s, const Dims& d, const void* u, Gate gc, Gate gh, const float* z0, const int32_t* lengths, void* z, float* zT, float* ckpt,
              float* agg, hipStream_t st) {
    return by_shape(s, gc, gh, [&](auto v, auto wt, auto gw, auto cn, auto hat) -> int {
        constexpr int V = decltype(v)::value, WT = decltype(wt)::value, GW = decltype(gw)::value, HAT = decltype(hat)::value;
        constexpr bool CN = decltype(cn)::value;
        const dim3 grid((unsigned)((int64_t)d.chunks * (d.splits > 1 ? ((int64_t)d.splits * d.B + 7) / 8 * 8 : d.B))), block(64 * (WT == 1 ? 4 : WT));
        const D* up = static_cast<const D*>(u);
        D* zp = static_cast<D*>(z);
        if (d.splits > 1) {
            if constexpr (WT == 4) recur_split_kernel<D, V, true, CN, HAT><<<grid, 256, 0, st>>>(up, gc, gh, lengths, agg, d);
            GF_LAUNCH_CHECK("recur_split_kernel");
        }
        recur_fwd_kernel<D, V, WT, GW, CN, HAT><<<grid, block, 0, st>>>(up, gc, gh, z0, lengths, zp, zT, ckpt, agg, d);
        GF_LAUNCH_CHECK("recur_fwd_kernel");
        return GF_OK;
    });
}

Fold make_fold(const float* src, void* out, int kind, int mode, const Dims& d, const Shape& s) {
    Fold f;
    f.src = src, f.out = out, f.kind = kind;
    f.nb = mode == kOutTime ? wave_columns(d, s) : 1, f.Hs = mode == kOutTime ? 1 : d.H, f.Ns = mode == kOutTime ? 1 : d.N;
    f.total = (int64_t)((kind & GF_GATE_B) ? d.B : 1) * d.T * ((kind & GF_GATE_H) ? d.H : 1) * ((kind & GF_GATE_N) ? d.N : 1);
    return f;
}
int64_t fold_blocks(const Fold& f) {
    const int64_t per = (!(f.kind & GF_GATE_N) && f.Ns > 1) ? 4 : 256, blocks = (f.total + per - 1) / per;
    return blocks > 256 * 32 ? 256 * 32 : blocks;
}

template <typename D>
int backward_t(const Shape& s, const Dims& d, const void* u, Gate gc, Gate gh, const int32_t* lengths, const void* dz, const float* dzT, const float* ckpt,
               void* du, void* dqc, int kc, void* dqh, int kh, float* dz0, float* ws, hipStream_t st) {
    float* agg = ws;
    float* pc = agg + agg_floats(d);
    float* ph = pc + (dqc ? out_floats(kc, d, s) : 0);
    GateOut oc{nullptr, kOutNone}, oh{nullptr, kOutNone};
    if (dqc) oc.mode = out_mode(kc), oc.p = oc.mode == kOutDirect ? dqc : pc;
    if (dqh) oh.mode = out_mode(kh), oh.p = oh.mode == kOutDirect ? dqh : ph;
    const int rc = by_shape(s, gc, gh, [&](auto v, auto wt, auto gw, auto cn, auto hat) -> int {
        constexpr int V = decltype(v)::value, WT = decltype(wt)::value, GW = decltype(gw)::value, HAT = decltype(hat)::value;
        constexpr bool CN = decltype(cn)::value;
        const dim3 grid((unsigned)((int64_t)d.chunks * (d.splits > 1 ? ((int64_t)d.splits * d.B + 7) / 8 * 8 : d.B))), block(64 * (WT == 1 ? 4 : WT));
        const D *up = static_cast<const D*>(u), *dzp = static_cast<const D*>(dz);
        D* dup = static_cast<D*>(du);
        if (d.splits > 1) {
            if constexpr (WT == 4) recur_split_kernel<D, V, false, CN, 0><<<grid, 256, 0, st>>>(dzp, gc, gh, lengths, agg, d);
            GF_LAUNCH_CHECK("recur_split_kernel");
        }
        recur_bwd_kernel<D, V, WT, GW, CN, HAT><<<grid, block, 0, st>>>(up, gc, gh, lengths, dzp, dzT, ckpt, dup, oc, oh, dz0, agg, d);
        GF_LAUNCH_CHECK("recur_bwd_kernel");
        return GF_OK;
    });
    if (rc != GF_OK) return rc;
    Fold f[2];
    int n = 0;
    if (d.T > 0 && dqc && oc.mode != kOutDirect) f[n++] = make_fold(pc, dqc, kc, oc.mode, d, s);
    if (d.T > 0 && dqh && oh.mode != kOutDirect) f[n++] = make_fold(ph, dqh, kh, oh.mode, d, s);
    if (n) {
        if (n == 1) f[1] = f[0];
        const int64_t a = fold_blocks(f[0]), b = fold_blocks(f[1]);
        recur_fold_kernel<D><<<dim3((unsigned)(a > b ? a : b), (unsigned)n), dim3(256), 0, st>>>(f[0], f[1], d.B, d.T);
        GF_LAUNCH_CHECK("recur_fold_kernel");
    }
    return GF_OK;
}

// the kernels' shape may not depend on pointers (forward and backward see different ones): V = 4 needs every tensor 4-element aligned,
// which the callers below check and refuse otherwise
Shape shape_of(int B, int T, int H, int N, int kc, bool has_h, int kh) { return choose(B, T, (int64_t)H * N, N, kind_bits(kc, has_h, kh)); }

}  // namespace

extern "C" size_t gf_recurrence_checkpoint_floats(int32_t B, int32_t T, int32_t H, int32_t N, int32_t kind_check, int32_t has_hat, int32_t kind_hat) {
    if (B <= 0 || T <= 0 || H <= 0 || N <= 0) return 0;
    const Shape s = shape_of(B, T, H, N, kind_check, has_hat != 0, kind_hat);
    return (size_t)B * ((T + s.slab - 1) / s.slab) * H * N;
}

extern "C" size_t gf_recurrence_workspace_bytes(int32_t B, int32_t T, int32_t H, int32_t N, int32_t kind_check, int32_t has_hat, int32_t kind_hat,
                                                int32_t backward) {
    if (B <= 0 || T <= 0 || H <= 0 || N <= 0) return 0;
    const Shape s = shape_of(B, T, H, N, kind_check, has_hat != 0, kind_hat);
    const Dims d = make_dims(s, B, T, H, N);
    size_t f = agg_floats(d);
    if (backward) f += out_floats(kind_check, d, s) + (has_hat ? out_floats(kind_hat, d, s) : 0);
    return f * 4;
}

extern "C" int gf_recurrence_forward(const void* u, const void* q_check, int32_t kind_check, const void* q_hat, int32_t kind_hat, const float* z0,
                                     const int32_t* lengths, void* z, float* zT, float* checkpoints, void* workspace, size_t workspace_bytes,
                                     int32_t dtype, int32_t B, int32_t T, int32_t H, int32_t N, void* stream) {
    const int rc = check_dims("gf_recurrence_forward", B, T, H, N, dtype, kind_check, kind_hat);
    if (rc != GF_OK) return rc;
    GF_REQUIRE_ARG(zT && (T == 0 || (u && q_check && z)), "gf_recurrence_forward: NULL tensor");
    const Shape s = shape_of(B, T, H, N, kind_check, q_hat != nullptr, kind_hat);
    const Dims d = make_dims(s, B, T, H, N);
    const size_t el = gf_dtype_bytes(dtype);
    GF_REQUIRE_ARG(workspace_bytes >= agg_floats(d) * 4 && (workspace || agg_floats(d) == 0), "gf_recurrence_forward: workspace of %zu bytes, needs %zu",
                   workspace_bytes, agg_floats(d) * 4);
    GF_REQUIRE_ARG(s.V == 1 || (aligned(u, 4 * el) && aligned(q_check, 4 * el) && aligned(q_hat, 4 * el) && aligned(z, 4 * el)),
                   "gf_recurrence_forward: a tensor is not aligned to four elements");
    // (256 threads per workgroup, and a launch's threads are counted in 32 bits)
    GF_REQUIRE_SHAPE((int64_t)d.chunks * d.splits * B < (1ll << 24), "gf_recurrence_forward: too many workgroups (B=%d, H*N=%d)", B, d.C);
    const Gate gc = make_gate(q_check, kind_check, T, H, N), gh = make_gate(q_hat, kind_hat, T, H, N);
    float* ws = static_cast<float*>(workspace);
    hipStream_t st = gf_stream(stream);
    if (dtype == GF_F32) return forward_t<float>(s, d, u, gc, gh, z0, lengths, z, zT, checkpoints, ws, st);
    if (dtype == GF_BF16) return forward_t<gf_bf16>(s, d, u, gc, gh, z0, lengths, z, zT, checkpoints, ws, st);
    return forward_t<gf_f16>(s, d, u, gc, gh, z0, lengths, z, zT, checkpoints, ws, st);
}

extern "C" int gf_recurrence_backward(const void* u, const void* q_check, int32_t kind_check, const void* q_hat, int32_t kind_hat, const int32_t* lengths,
                                      const float* checkpoints, const void* dz, const float* dzT, void* du, void* dq_check, void* dq_hat, float* dz0,
                                      void* workspace, size_t workspace_bytes, int32_t dtype, int32_t B, int32_t T, int32_t H, int32_t N, void* stream) {
    const int rc = check_dims("gf_recurrence_backward", B, T, H, N, dtype, kind_check, kind_hat);
    if (rc != GF_OK) return rc;
    GF_REQUIRE_ARG(T == 0 || (u && q_check), "gf_recurrence_backward: NULL tensor");
    GF_REQUIRE_ARG(!dq_check || T == 0 || checkpoints, "gf_recurrence_backward: the gradient of q_check needs the forward's checkpoints");
    GF_REQUIRE_ARG(!dq_hat || q_hat, "gf_recurrence_backward: a gradient of q_hat without q_hat");
    const Shape s = shape_of(B, T, H, N, kind_check, q_hat != nullptr, kind_hat);
    const Dims d = make_dims(s, B, T, H, N);
    const size_t el = gf_dtype_bytes(dtype);
    const size_t need = 4 * (agg_floats(d) + (dq_check ? out_floats(kind_check, d, s) : 0) + (dq_hat ? out_floats(kind_hat, d, s) : 0));
    GF_REQUIRE_ARG(workspace_bytes >= need && (workspace || need == 0), "gf_recurrence_backward: workspace of %zu bytes, needs %zu", workspace_bytes, need);
    GF_REQUIRE_ARG(s.V == 1 || (aligned(u, 4 * el) && aligned(q_check, 4 * el) && aligned(q_hat, 4 * el) && aligned(dz, 4 * el) && aligned(du, 4 * el) &&
                                aligned(dq_check, 4 * el) && aligned(dq_hat, 4 * el) && aligned(workspace, 16)),
                   "gf_recurrence_backward: a tensor is not aligned to four elements");
    GF_REQUIRE_SHAPE((int64_t)d.chunks * d.splits * B < (1ll << 24), "gf_recurrence_backward: too many workgroups (B=%d, H*N=%d)", B, d.C);
    const Gate gc = make_gate(q_check, kind_check, T, H, N), gh = make_gate(q_hat, kind_hat, T, H, N);
    float* ws = static_cast<float*>(workspace);
    hipStream_t st = gf_stream(stream);
    if (dtype == GF_F32) return backward_t<float>(s, d, u, gc, gh, lengths, dz, dzT, checkpoints, du, dq_check, kind_check, dq_hat, kind_hat, dz0, ws, st);
    if (dtype == GF_BF16) return backward_t<gf_bf16>(s, d, u, gc, gh, lengths, dz, dzT, checkpoints, du, dq_check, kind_check, dq_hat, kind_hat, dz0, ws, st);
    return backward_t<gf_f16>(s, d, u, gc, gh, lengths, dz, dzT, checkpoints, du, dq_check, kind_check, dq_hat, kind_hat, dz0, ws, st);
}
