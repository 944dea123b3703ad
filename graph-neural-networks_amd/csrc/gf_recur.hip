// gf_recur.hip -- gated linear recurrence  z_t = qc_t z_{t-1} + qh_t u_t  over [B, T, H, N], forward and backward.
//
// The recursion of GatedGRNN (reference graphML.py:1421-1462) with B(S) = identity and sigma = identity: linear in the state, so a
// stretch of steps is one pair (A, h) with z_out = A z_in + h, and stretches compose: (A2, h2) o (A1, h1) = (A2 A1, A2 h1 + h2).
// The channels c = h N + n are contiguous and independent; time is cut into tiles:
//   thread     kL steps x V channels, all loads issued before the first use
//   wave       GW groups of 64 / GW lanes; the groups hold consecutive stretches, joined by a shuffle scan
//   workgroup  WT waves along time (joined through LDS, one barrier per slab) or 4 waves side by side along the channels (no barrier)
//   slab       GW WT kL steps, walked in order with the state in registers
//   split      few channels and a long T: the time axis is cut into S splits, a first kernel reads the inputs for each split's (A, h),
//              the second one starts from the composition of the splits before its own (inputs are read twice)
// Backward: with r_t = qc_t g_t the adjoint  g_t = dz_t + r_{t+1}  is the same recurrence run backwards with the same coefficients, and
// needs the states z_{t-1} in fp32 for the gate's gradient: they are recomputed from the inputs (which qh's gradient reads anyway) and one
// fp32 checkpoint per slab instead of being read back rounded.  Bound by HBM: forward reads u, qc, qh and writes z, backward reads u, qc,
// qh, dz and writes du, dqc, dqh.
//
// State, products and sums are fp32; outputs are rounded once.  Steps at or behind a sequence's length leave the state as it is (A = 1,
// h = 0), are not read, and their outputs and gradients are zero.
#include "gf_num.h"

#include <type_traits>

namespace {

constexpr int kL = 4;              // steps per thread and slab.  8 steps need twice the registers and lose: backward of 32 x 257 x 53824 bf16 in 1.32 ms
                                   // against 1.69 ms, of 65537 x 808 in 301 us against 416 us (both before the straight-line loads)
constexpr int kGW = 4;             // time groups of a wave: 4 (rows of 16 lanes) against 8: 0.89 / 1.02 ms, against 2 with 8 steps: 0.89 / 0.97 ms
constexpr int kMaxSplit = 128;     // splits of a long time axis: 128 / 64 / 256 give 307 / 344 / 323 us for 65537 x 808 bf16, forward and backward

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

// The loads of a slab are straight-line code (addresses clamped to the last live step, values replaced afterwards): all of them are in
// flight before the first one is waited for.  A gate without the node axis has one value for the thread's V channels (V > 1 only where they
// share the feature); it is spread after the other loads have been issued.
template <typename D, int V>
__device__ __forceinline__ void load_gate(const Gate& g, int64_t at, const int (&t)[kL], gf_vec<D, V> (&raw)[kL]) {
    const D* p = static_cast<const D*>(g.p) + at;
    if (V > 1 && (g.kind & GF_GATE_N)) {
#pragma unroll
        for (int l = 0; l < kL; ++l) raw[l] = *reinterpret_cast<const gf_vec<D, V>*>(p + (int64_t)t[l] * g.st);
    } else {
#pragma unroll
        for (int l = 0; l < kL; ++l) raw[l].e[0] = p[(int64_t)t[l] * g.st];
    }
}
template <typename D, int V> __device__ __forceinline__ void spread_gate(const Gate& g, gf_vec<D, V> (&raw)[kL]) {
    if (V > 1 && !(g.kind & GF_GATE_N)) {
#pragma unroll
        for (int l = 0; l < kL; ++l)
#pragma unroll
            for (int i = 1; i < V; ++i) raw[l].e[i] = raw[l].e[0];
    }
}
template <typename D, int V>
__device__ __forceinline__ void load_rows(const D* __restrict__ p, int64_t C, const int (&t)[kL], gf_vec<D, V> (&raw)[kL]) {
#pragma unroll
    for (int l = 0; l < kL; ++l) raw[l] = *reinterpret_cast<const gf_vec<D, V>*>(p + t[l] * C);
}
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
    int lane, wave, cx, tg, c, b, split;
    bool on;
    __device__ __forceinline__ Place(const Dims& d) {
        lane = threadIdx.x & 63;
        wave = threadIdx.x >> 6;
        cx = lane % CX;
        tg = (WT == 1 ? 0 : wave * GW) + lane / CX;
        const unsigned blk = blockIdx.x;
        const unsigned chunk = blk % (unsigned)d.chunks, rest = blk / (unsigned)d.chunks;
        split = (int)(rest % (unsigned)d.splits);
        b = (int)(rest / (unsigned)d.splits);
        c = (int)chunk * CW + (WT == 1 ? wave * CX : 0) * V + cx * V;
        on = c < d.C;
    }
};

// exclusive composition of the stretches before (FWD) / behind (!FWD) this thread's own, and of the whole slab
template <int V, int WT, int GW, bool FWD>
__device__ __forceinline__ void join(const float (&A)[V], const float (&S)[V], float (&Ae)[V], float (&Se)[V], float (&At)[V], float (&St)[V],
                                     int lane, int wave, float* lds) {
    constexpr int CX = 64 / GW;
    float a[V], s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = A[i], s[i] = S[i];
#pragma unroll
    for (int off = CX; off < 64; off <<= 1) {
        const bool take = FWD ? lane >= off : lane < 64 - off;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float ao = FWD ? __shfl_up(a[i], off) : __shfl_down(a[i], off);
            const float so = FWD ? __shfl_up(s[i], off) : __shfl_down(s[i], off);
            if (take) {
                s[i] = fmaf(a[i], so, s[i]);
                a[i] *= ao;
            }
        }
    }
    const bool edge = FWD ? lane < CX : lane >= 64 - CX;        // first group in walking order
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float ao = FWD ? __shfl_up(a[i], CX) : __shfl_down(a[i], CX);
        const float so = FWD ? __shfl_up(s[i], CX) : __shfl_down(s[i], CX);
        Ae[i] = (GW == 1 || edge) ? 1.f : ao;
        Se[i] = (GW == 1 || edge) ? 0.f : so;
    }
    const int last = FWD ? 64 - CX + lane % CX : lane % CX;     // lane with the wave's composition
    if constexpr (WT == 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) At[i] = __shfl(a[i], last), St[i] = __shfl(s[i], last);
    } else {
        if (lane == last) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                lds[((wave * CX + lane % CX) * V + i) * 2] = a[i];
                lds[((wave * CX + lane % CX) * V + i) * 2 + 1] = s[i];
            }
        }
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
                const float wa = lds[((w * CX + lane % CX) * V + i) * 2], ws = lds[((w * CX + lane % CX) * V + i) * 2 + 1];
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

// composition of the splits [s0, s1) of the thread's channels, shared out over the time groups (walked forwards or backwards)
template <int V, int WT, int GW, bool FWD>
__device__ __forceinline__ void join_splits(const float* __restrict__ agg, int64_t all, int64_t chan, int s0, int s1, const Place<V, WT, GW>& p,
                                            float (&At)[V], float (&St)[V], float* lds) {
    constexpr int TG = WT * GW;
    const int q = (s1 - s0 + TG - 1) / TG, lo = min(s1, s0 + p.tg * q), hi = min(s1, lo + q);
    float A[V], S[V], Ae[V], Se[V];
#pragma unroll
    for (int i = 0; i < V; ++i) A[i] = 1.f, S[i] = 0.f;
#pragma unroll 4
    for (int k = lo; k < hi; ++k) {
        const float* g = agg + 2 * (int64_t)(FWD ? k : lo + hi - 1 - k) * all + chan;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float ak = g[i];
            S[i] = fmaf(ak, S[i], g[all + i]);
            A[i] *= ak;
        }
    }
    join<V, WT, GW, FWD>(A, S, Ae, Se, At, St, p.lane, p.wave, lds);
}

// ---- forward -------------------------------------------------------------------------------------------------------------
// AGG: the first kernel of a split run -- no outputs but each split's (A, h)
template <typename D, int V, int WT, int GW, bool AGG>
__global__ __launch_bounds__(64 * (WT == 1 ? 4 : WT)) void recur_fwd_kernel(const D* __restrict__ u, Gate gc, Gate gh, const float* __restrict__ z0,
                                                                            const int32_t* __restrict__ lengths, D* __restrict__ z,
                                                                            float* __restrict__ zT, float* __restrict__ ckpt,
                                                                            float* __restrict__ agg, Dims d) {
    using P = Place<V, WT, GW>;
    __shared__ float s_join[WT == 1 ? 1 : 2][WT == 1 ? 1 : WT * P::CX * V * 2];
    const P p(d);
    if (AGG && p.split == d.splits - 1) return;                 // nothing starts behind the last split
    int len = d.T;
    if (lengths) len = min(max(lengths[p.b], 0), d.T);
    const int pc = p.on ? p.c : d.C - V;                        // lanes behind the last channel read its values and store nothing
    const int64_t ub = (int64_t)p.b * d.T * d.C + pc, chan = (int64_t)p.b * d.C + pc, all = (int64_t)d.B * d.C;
    const int64_t cb = p.b * gc.sb + gate_coff(gc, pc, d.N), hb = p.b * gh.sb + gate_coff(gh, pc, d.N);
    float carry[V], Asum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = 0.f, Asum[i] = 1.f;
    if (!AGG) {
        if (z0) {
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = z0[chan + i];
        }
    }
    if (!AGG && p.split > 0) {                                  // (uniform) the splits before this one
        float At[V], St[V];
        join_splits<V, WT, GW, true>(agg, all, chan, 0, p.split, p, At, St, s_join[WT == 1 ? 0 : 1]);
#pragma unroll
        for (int i = 0; i < V; ++i) carry[i] = fmaf(At[i], carry[i], St[i]);
    }
    const int tbeg = p.split * d.split_len, tend = min(d.T, tbeg + d.split_len);
    const int live_end = min(tend, len);
    gf_vec<D, V> ra[kL], rb[kL], rq[kL];
    auto fetch = [&](int ts) {
        int t[kL];
#pragma unroll
        for (int l = 0; l < kL; ++l) t[l] = min(ts + p.tg * kL + l, len - 1);
        load_rows<D, V>(u + ub, d.C, t, rb);
        load_gate<D, V>(gc, cb, t, ra);
        if (gh.p) load_gate<D, V>(gh, hb, t, rq);
    };
    if (tbeg < live_end) fetch(tbeg);
    int flip = 0;
    for (int ts = tbeg; ts < tend; ts += P::SLAB, flip ^= 1) {
        const int t0 = ts + p.tg * kL;
        if (ts >= len) {                                        // (uniform) behind the sequence: the state stays, the output is zero
            if (!AGG && p.on) {
                const float zero[V] = {};
                for (int l = 0; l < kL; ++l)
                    if (t0 + l < d.T) gf_store<D, V>(z + ub + (int64_t)(t0 + l) * d.C, zero);
            }
            continue;
        }
        float a[kL][V], b[kL][V], A[V], S[V];
        spread_gate<D, V>(gc, ra);
#pragma unroll
        for (int l = 0; l < kL; ++l)
#pragma unroll
            for (int i = 0; i < V; ++i) a[l][i] = gf_to_f<D>(ra[l].e[i]), b[l][i] = gf_to_f<D>(rb[l].e[i]);
        if (gh.p) {
            spread_gate<D, V>(gh, rq);
#pragma unroll
            for (int l = 0; l < kL; ++l)
#pragma unroll
                for (int i = 0; i < V; ++i) b[l][i] *= gf_to_f<D>(rq[l].e[i]);
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
        join<V, WT, GW, true>(A, S, Ae, Se, At, St, p.lane, p.wave, s_join[WT == 1 ? 0 : flip]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            h[i] = fmaf(Ae[i], carry[i], Se[i]);
            carry[i] = fmaf(At[i], carry[i], St[i]);
            Asum[i] *= At[i];
        }
        if (!AGG && p.on) {
            if (ckpt && t0 < d.T && t0 % d.every == 0) {
                float* k = ckpt + ((int64_t)p.b * d.nck + t0 / d.every) * d.C + pc;
#pragma unroll
                for (int i = 0; i < V; ++i) k[i] = h[i];
            }
#pragma unroll
            for (int l = 0; l < kL; ++l) {
                if (t0 + l < d.T) {
                    float o[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        h[i] = fmaf(a[l][i], h[i], b[l][i]);
                        o[i] = t0 + l < len ? h[i] : 0.f;
                    }
                    gf_store<D, V>(z + ub + (int64_t)(t0 + l) * d.C, o);
                }
            }
        }
    }
    if (p.on && p.tg == 0) {
        if (AGG) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                agg[(2 * (int64_t)p.split) * all + chan + i] = Asum[i];
                agg[(2 * (int64_t)p.split + 1) * all + chan + i] = carry[i];
            }
        } else if (p.split == d.splits - 1) {
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

template <typename D, int V, int CX>
__device__ __forceinline__ void put_gate(const GateOut& g, const float (&v)[V], int64_t off, int64_t toff, bool on, bool live, int lane) {
    if (g.mode == kOutDirect) {
        if (on && live) gf_store<D, V>(static_cast<D*>(g.p) + off, v);
    } else if (g.mode == kOutProduct) {
        if (on && live) gf_store<float, V>(static_cast<float*>(g.p) + off, v);
    } else if (g.mode == kOutTime) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) s += on ? v[i] : 0.f;
#pragma unroll
        for (int off2 = 1; off2 < CX; off2 <<= 1) s += __shfl_xor(s, off2);
        if (live && lane % CX == 0) static_cast<float*>(g.p)[toff] = s;
    }
}

template <typename D, int V, int WT, int GW, bool AGG>
__global__ __launch_bounds__(64 * (WT == 1 ? 4 : WT)) void recur_bwd_kernel(const D* __restrict__ u, Gate gc, Gate gh, const int32_t* __restrict__ lengths,
                                                                            const D* __restrict__ dz, const float* __restrict__ dzT,
                                                                            const float* __restrict__ ckpt, D* __restrict__ du, GateOut oc, GateOut oh,
                                                                            float* __restrict__ dz0, float* __restrict__ agg, Dims d) {
    using P = Place<V, WT, GW>;
    __shared__ float s_join[WT == 1 ? 1 : 4][WT == 1 ? 1 : WT * P::CX * V * 2];
    const P p(d);
    if (AGG && p.split == 0) return;
    int len = d.T;
    if (lengths) len = min(max(lengths[p.b], 0), d.T);
    const int pc = p.on ? p.c : d.C - V;
    const int64_t ub = (int64_t)p.b * d.T * d.C + pc, chan = (int64_t)p.b * d.C + pc, all = (int64_t)d.B * d.C;
    const int64_t cb = p.b * gc.sb + gate_coff(gc, pc, d.N), hb = p.b * gh.sb + gate_coff(gh, pc, d.N);
    // sums over a wave's channels (time gates): one row of [B, T] per wave column
    const int64_t cols = (int64_t)(blockIdx.x % (unsigned)d.chunks) * (WT == 1 ? P::NW : 1) + (WT == 1 ? p.wave : 0);
    const int64_t tbase = (cols * d.B + p.b) * d.T;
    float carry[V], Asum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = 0.f, Asum[i] = 1.f;
    if (!AGG) {
        if (dzT) {
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = dzT[chan + i];
        }
    }
    if (!AGG && p.split + 1 < d.splits) {                       // (uniform) the splits behind this one
        float At[V], St[V];
        join_splits<V, WT, GW, false>(agg, all, chan, p.split + 1, d.splits, p, At, St, s_join[WT == 1 ? 0 : 2]);
#pragma unroll
        for (int i = 0; i < V; ++i) carry[i] = fmaf(At[i], carry[i], St[i]);
    }
    const int tbeg = p.split * d.split_len, tend = min(d.T, tbeg + d.split_len);
    const int slabs = tend > tbeg ? (tend - tbeg + P::SLAB - 1) / P::SLAB : 0;
    gf_vec<D, V> ra[kL], rx[kL], rq[kL], rg[kL];
    auto fetch = [&](int ts) {
        int t[kL];
#pragma unroll
        for (int l = 0; l < kL; ++l) t[l] = min(ts + p.tg * kL + l, len - 1);
        if (dz) load_rows<D, V>(dz + ub, d.C, t, rg);
        load_gate<D, V>(gc, cb, t, ra);
        if (!AGG) {
            load_rows<D, V>(u + ub, d.C, t, rx);
            if (gh.p) load_gate<D, V>(gh, hb, t, rq);
        }
    };
    if (tbeg < min(tend, len)) fetch(tbeg + (min(tend, len) - tbeg - 1) / P::SLAB * P::SLAB);     // the last slab with a live step
    int flip = 0;
    for (int sl = slabs - 1; sl >= 0; --sl, flip ^= 2) {
        const int ts = tbeg + sl * P::SLAB, t0 = ts + p.tg * kL;
        if (ts >= len) {                                        // (uniform) behind the sequence: nothing flows, the gradients are zero
            if (!AGG) {
                const float zero[V] = {};
                for (int l = 0; l < kL; ++l) {
                    const int64_t off = ub + (int64_t)(t0 + l) * d.C;
                    if (du && p.on && t0 + l < d.T) gf_store<D, V>(du + off, zero);
                    if (oc.mode) put_gate<D, V, P::CX>(oc, zero, off, tbase + t0 + l, p.on, t0 + l < d.T, p.lane);
                    if (oh.mode) put_gate<D, V, P::CX>(oh, zero, off, tbase + t0 + l, p.on, t0 + l < d.T, p.lane);
                }
            }
            continue;
        }
        const bool ends = ts + P::SLAB > len;                   // (uniform) the sequence ends in this slab
        float a[kL][V], x[kL][V], q[kL][V], g[kL][V], A[V], R[V];
        spread_gate<D, V>(gc, ra);
#pragma unroll
        for (int l = 0; l < kL; ++l)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                a[l][i] = gf_to_f<D>(ra[l].e[i]);
                g[l][i] = 0.f;
                x[l][i] = AGG ? 0.f : gf_to_f<D>(rx[l].e[i]);
                q[l][i] = 1.f;
            }
        if (dz) {
#pragma unroll
            for (int l = 0; l < kL; ++l)
#pragma unroll
                for (int i = 0; i < V; ++i) g[l][i] = gf_to_f<D>(rg[l].e[i]);
        }
        if (!AGG && gh.p) {
            spread_gate<D, V>(gh, rq);
#pragma unroll
            for (int l = 0; l < kL; ++l)
#pragma unroll
                for (int i = 0; i < V; ++i) q[l][i] = gf_to_f<D>(rq[l].e[i]);
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
        join<V, WT, GW, false>(A, R, Ae, Re, At, Rt, p.lane, p.wave, s_join[WT == 1 ? 0 : flip]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            r[i] = fmaf(Ae[i], carry[i], Re[i]);
            carry[i] = fmaf(At[i], carry[i], Rt[i]);
            Asum[i] *= At[i];
        }
        if (!AGG) {
            float zp[kL][V];
            if (oc.mode != kOutNone) {                          // the states z_{t-1} of this slab, from its checkpoint
                float S[V], h[V], Se[V], St[V];
#pragma unroll
                for (int i = 0; i < V; ++i) S[i] = 0.f;
#pragma unroll
                for (int l = 0; l < kL; ++l)
#pragma unroll
                    for (int i = 0; i < V; ++i) S[i] = fmaf(a[l][i], S[i], x[l][i] * q[l][i]);
                join<V, WT, GW, true>(A, S, Ae, Se, At, St, p.lane, p.wave, s_join[WT == 1 ? 0 : flip + 1]);
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
                        h[i] = fmaf(a[l][i], h[i], x[l][i] * q[l][i]);
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
                    ox[i] = gt * q[l][i];
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
                if (du && p.on && in) gf_store<D, V>(du + off, ox);
                if (oc.mode) put_gate<D, V, P::CX>(oc, o, off, tbase + t0 + l, p.on, in, p.lane);
                if (oh.mode) put_gate<D, V, P::CX>(oh, oq, off, tbase + t0 + l, p.on, in, p.lane);
            }
        }
    }
    if (p.on && p.tg == 0) {
        if (AGG) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                agg[(2 * (int64_t)p.split) * all + chan + i] = Asum[i];
                agg[(2 * (int64_t)p.split + 1) * all + chan + i] = carry[i];
            }
        } else if (p.split == 0 && dz0) {
#pragma unroll
            for (int i = 0; i < V; ++i) dz0[chan + i] = carry[i];
        }
    }
}

// Sum of the fp32 products [rows, T, inner, H, N] ... over the axes a gate does not have, in a fixed order: out[b, t, h, n] (gate shape).
// src [nb, B, T, Hs, Ns] : nb partial rows; axes: nb always, B if !GF_GATE_B, Hs if !(kind & H), Ns if !(kind & N).
// One wave per output element where the node axis is summed, one thread per element otherwise (coalesced over nodes).
__device__ __forceinline__ float sum_strided(const float* __restrict__ p, int n, int64_t stride, float s) {   // in order, eight loads in flight
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

template <typename D>
__global__ __launch_bounds__(256) void recur_fold_kernel(const float* __restrict__ src, D* __restrict__ out, int nb, int B, int T, int Hs, int Ns,
                                                         int kind, int64_t total) {
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
        float s = 0.f;
        if (byN) {
            for (int k = 0; k < nb * bs; ++k)                   // (nb > 1 only with Hs = Ns = 1)
                for (int hh = 0; hh < hs; ++hh)
                    for (int m = lane; m < Ns; m += 64) s += p[(int64_t)k * T * row + (int64_t)hh * Ns + m];
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) s += __shfl_xor(s, off);
            if (lane == 0) out[o] = gf_from_f<D>(s);
        } else {
            if (hs > 1) {
                for (int bb = 0; bb < bs; ++bb) s = sum_strided(p + (int64_t)bb * T * row, hs, Ns, s);
            } else if (bs > 1) {
                s = sum_strided(p, nb * bs, T * row, s);        // (partial rows of all sequences: [nb][B] is one axis)
            } else {
                s = sum_strided(p, nb, (int64_t)B * T * row, s);
            }
            out[o] = gf_from_f<D>(s);
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
    if (blocks < 256 && slabs >= 8) {                           // fewer workgroups than compute units and a long way to walk
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
    GF_REQUIRE_SHAPE((int64_t)H * N < (1ll << 30), "%s: H * N = %lld channels", who, (long long)H * N);
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

template <int V, typename F>
int by_time(const Shape& s, F&& f) {
    using std::integral_constant;
    if (s.GW == 1) return f(integral_constant<int, V>(), integral_constant<int, 1>(), integral_constant<int, 1>());
    if (s.WT == 1) return f(integral_constant<int, V>(), integral_constant<int, 1>(), integral_constant<int, kGW>());
    return f(integral_constant<int, V>(), integral_constant<int, 4>(), integral_constant<int, kGW>());
}
template <typename F>
int by_shape(const Shape& s, F&& f) {
    return s.V == 4 ? by_time<4>(s, f) : s.V == 2 ? by_time<2>(s, f) : by_time<1>(s, f);
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
size_t agg_floats(const Dims& d) { return d.splits > 1 ? ((size_t)2 * d.splits * d.B * d.C + 3) / 4 * 4 : 0; }

template <typename D>
int forward_t(const Shape& s, const Dims& d, const void* u, Gate gc, Gate gh, const float* z0, const int32_t* lengths, void* z, float* zT, float* ckpt,
              float* agg, hipStream_t st) {
    return by_shape(s, [&](auto v, auto wt, auto gw) -> int {
        constexpr int V = decltype(v)::value, WT = decltype(wt)::value, GW = decltype(gw)::value;
        const dim3 grid((unsigned)((int64_t)d.chunks * d.splits * d.B)), block(64 * (WT == 1 ? 4 : WT));
        const D* up = static_cast<const D*>(u);
        D* zp = static_cast<D*>(z);
        if (d.splits > 1) {
            recur_fwd_kernel<D, V, WT, GW, true><<<grid, block, 0, st>>>(up, gc, gh, z0, lengths, zp, zT, nullptr, agg, d);
            GF_LAUNCH_CHECK("recur_fwd_kernel (splits)");
        }
        recur_fwd_kernel<D, V, WT, GW, false><<<grid, block, 0, st>>>(up, gc, gh, z0, lengths, zp, zT, ckpt, agg, d);
        GF_LAUNCH_CHECK("recur_fwd_kernel");
        return GF_OK;
    });
}

template <typename D>
int fold_t(const float* src, void* out, int kind, int mode, const Dims& d, const Shape& s, hipStream_t st) {
    const int nb = mode == kOutTime ? wave_columns(d, s) : 1, Hs = mode == kOutTime ? 1 : d.H, Ns = mode == kOutTime ? 1 : d.N;
    const int64_t total = (int64_t)((kind & GF_GATE_B) ? d.B : 1) * d.T * ((kind & GF_GATE_H) ? d.H : 1) * ((kind & GF_GATE_N) ? d.N : 1);
    if (total == 0) return GF_OK;
    const int64_t per = (!(kind & GF_GATE_N) && Ns > 1) ? 4 : 256;
    int64_t blocks = (total + per - 1) / per;
    if (blocks > 256 * 32) blocks = 256 * 32;
    recur_fold_kernel<D><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(src, static_cast<D*>(out), nb, d.B, d.T, Hs, Ns, kind, total);
    GF_LAUNCH_CHECK("recur_fold_kernel");
    return GF_OK;
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
    const int rc = by_shape(s, [&](auto v, auto wt, auto gw) -> int {
        constexpr int V = decltype(v)::value, WT = decltype(wt)::value, GW = decltype(gw)::value;
        const dim3 grid((unsigned)((int64_t)d.chunks * d.splits * d.B)), block(64 * (WT == 1 ? 4 : WT));
        const D *up = static_cast<const D*>(u), *dzp = static_cast<const D*>(dz);
        D* dup = static_cast<D*>(du);
        if (d.splits > 1) {
            recur_bwd_kernel<D, V, WT, GW, true><<<grid, block, 0, st>>>(up, gc, gh, lengths, dzp, dzT, ckpt, dup, oc, oh, dz0, agg, d);
            GF_LAUNCH_CHECK("recur_bwd_kernel (splits)");
        }
        recur_bwd_kernel<D, V, WT, GW, false><<<grid, block, 0, st>>>(up, gc, gh, lengths, dzp, dzT, ckpt, dup, oc, oh, dz0, agg, d);
        GF_LAUNCH_CHECK("recur_bwd_kernel");
        return GF_OK;
    });
    if (rc != GF_OK) return rc;
    if (dqc && oc.mode != kOutDirect) {
        const int r = fold_t<D>(pc, dqc, kc, oc.mode, d, s, st);
        if (r != GF_OK) return r;
    }
    if (dqh && oh.mode != kOutDirect) return fold_t<D>(ph, dqh, kh, oh.mode, d, s, st);
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
