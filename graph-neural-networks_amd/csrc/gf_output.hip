// gf_output.hip -- what a classifier answers and learns from, over rows of V logits (V = classes, or nodes of the graph):
//   gf_token_logp_*     log probabilities of given tokens, entropy, the best alternatives; their gradient
//   gf_distill_top_*    distillation loss against a teacher's K best outputs; its gradient
// (the reference hands its readouts to torch losses and reduces them to an error rate: sourceLocGNN.py:167, evaluation.py:58-71).
//
// Forward: a row is cut into tiles that a workgroup holds in registers, so the logits are read once.  With m the tile's maximum, c = 1 / T:
//   s = sum e^{c (x - m)},   t = sum e^{c (x - m)} c (x - m);    tiles join by rescaling to the common maximum M:
//   log q_j = c (x_j - M) - log S,    entropy = log S - t / S
// Best alternatives: the thread maxima give a lower bound of the tile's k-th largest value (the k-th largest of one wave's 64 maxima, or the
// smallest of the four waves' (k / 4)-th largest ones); the few elements at or above it are collected in LDS and ranked by counting, as 64-bit
// keys {ordered value, ~index}: distinct, so the order of collection does not matter and equal values come in index order.
// Backward: one more read of the logits and one write; the few outputs that are named (token, alternatives, teacher's entries) are then
// written over by the same workgroup.
// Bound by HBM for fp32; for 16-bit logits the exponential (a quarter-rate instruction) and the conversions weigh about as much.
// Sums are fp32 and in a fixed order; the K-wide part of the distillation loss is fp64 (a small difference of masses near one).
#include "gf_num.h"

#include <type_traits>

namespace {

constexpr int kThr = 256;
constexpr int kTopMax = 64;
constexpr int kCand = 1024;        // candidates that are ranked in LDS; more (heavy ties) take the extraction loop
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

typedef unsigned long long u64;

__device__ __forceinline__ unsigned ord32(float x) {            // order of floats as unsigned; -0 = +0, any NaN above everything
    if (x != x) return 0xfffffffeu;              // (the all-ones key is kept free: "nothing taken yet")
    const unsigned b = __float_as_uint(x + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unord32(unsigned o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ u64 make_key(float x, int64_t j) { return ((u64)ord32(x) << 32) | (unsigned)~(unsigned)j; }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
template <typename T> __device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// A row's elements as 16-byte groups: group g holds elements g VE .. g VE + VE.  Rows of odd length start at any element: the group loads and stores
// are marked unaligned (one instruction all the same, and the grouping -- the order of the sums -- does not depend on the address).  The
// group that sticks out of the row is handled element by element.
template <typename D> struct Row {
    static constexpr int VE = 16 / sizeof(D);
    const D* p;
    int V;
    __device__ __forceinline__ Row(const D* row, int V_) : p(row), V(V_) {}
    __device__ __forceinline__ int64_t first(int64_t g) const { return g * VE; }
    __device__ __forceinline__ bool load(int64_t g, float (&x)[VE], float fill) const {
        const int64_t j = first(g);
        if (j + VE <= V) {
            gf_load_any<D, VE>(p + j, x);
            return true;
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) x[e] = j + e < V ? gf_to_f<D>(p[j + e]) : fill;
        return false;
    }
};
template <typename D> __host__ __device__ inline int64_t row_groups(int64_t V) { return (V + 16 / (int64_t)sizeof(D) - 1) / (16 / (int64_t)sizeof(D)); }

struct Parts {                     // per (row, tile): maximum, sums, and the tile's best keys
    float *m, *s, *t;
    u64* keys;
};

// k-th largest of the wave's 64 values (as ordered unsigned), by bits from the top; 16-bit types have no more than 16 significant ones
template <int BITS> __device__ __forceinline__ unsigned kth_of_wave(unsigned v, int k) {
    unsigned thr = 0;
#pragma unroll
    for (int b = 31; b >= 32 - BITS; --b) {
        const unsigned c = thr | (1u << b);
        if (__popcll(__ballot(v >= c)) >= k) thr = c;
    }
    return thr;
}

// ---- tile statistics (and best keys) -----------------------------------------------------------------------------------
// MASK: the outputs named by indices[row][0..K) are left out
template <typename D, int NV, bool TOP, bool MASK>
__global__ __launch_bounds__(kThr) void tile_kernel(const D* __restrict__ logits, int64_t row_stride, int V, int tiles, float c2, int top,
                                                    const int64_t* __restrict__ indices, int K, Parts out) {
    constexpr int VE = Row<D>::VE, TE = NV * kThr * VE;
    __shared__ float s_m[4], s_s[4], s_t[4];
    __shared__ unsigned s_thr[8];
    __shared__ int s_n;
    __shared__ u64 s_cand[TOP ? kCand : 1];
    __shared__ unsigned s_bits[MASK ? TE / 32 : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x / (unsigned)tiles;
    const int tile = (int)(blockIdx.x % (unsigned)tiles);
    const Row<D> row(logits + r * row_stride, V);
    const int64_t g0 = (int64_t)tile * NV * kThr;
    float x[NV][VE];
#pragma unroll
    for (int v = 0; v < NV; ++v) row.load(g0 + v * kThr + tid, x[v], -INFINITY);
    if constexpr (MASK) {
        for (int i = tid; i < TE / 32; i += kThr) s_bits[i] = 0u;
        __syncthreads();
        if (tid < K) {
            const int64_t j = indices[r * K + tid], q = j - row.first(g0);
            if (j >= 0 && j < V && q >= 0 && q < TE) atomicOr(&s_bits[q >> 5], 1u << (q & 31));
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int q = (v * kThr + tid) * VE;
            const unsigned w = s_bits[q >> 5] >> (q & 31);
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (w >> e & 1u) x[v][e] = -INFINITY;
        }
    }
    float tm = -INFINITY, vm[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        vm[v] = x[v][0];
#pragma unroll
        for (int e = 1; e < VE; ++e) vm[v] = fmaxf(vm[v], x[v][e]);
        tm = fmaxf(tm, vm[v]);
    }
    const float wm = wave_max(tm);
    if (lane == 0) s_m[wave] = wm;
    if constexpr (TOP) {
        constexpr int BITS = sizeof(D) == 2 && std::is_same<D, gf_bf16>::value ? 16 : 32;
        const unsigned o = ord32(tm);
        const unsigned a = kth_of_wave<BITS>(o, (top + 3) / 4), b = kth_of_wave<BITS>(o, top);
        if (lane == 0) s_thr[wave] = a, s_thr[4 + wave] = b;
        if (tid == 0) s_n = 0;
    }
    __syncthreads();
    const float m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    const float ref = m == -INFINITY ? 0.f : m;                 // a tile with nothing in it: all exponentials are zero
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float y = (x[v][e] - ref) * c2;               // base-2 exponent
            const float p = exp2f(y);
            s += p;
            t = fmaf(p, fmaxf(y, -3e38f), t);                   // p = 0 where y = -inf
        }
    s = wave_sum(s);
    t = wave_sum(t);
    if (lane == 0) s_s[wave] = s, s_t[wave] = t;
    __syncthreads();
    s = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
    t = (s_t[0] + s_t[1]) + (s_t[2] + s_t[3]);
    const int64_t at = r * tiles + tile;
    if (tid == 0) {
        out.m[at] = m;
        out.s[at] = s;
        out.t[at] = t * kLn2;
    }
    if constexpr (TOP) {
        u64* keys = out.keys + at * top;
        const int64_t jend = V;
        bool ranked = false;
        if (s == s) {                                           // no NaN in the tile: the maxima above are the values' own order
            unsigned ua = s_thr[0], ub = s_thr[4];
#pragma unroll
            for (int w = 1; w < 4; ++w) ua = min(ua, s_thr[w]), ub = max(ub, s_thr[4 + w]);
            const unsigned u = max(ua, ub);
            const float thr = u < 0x00800000u ? -INFINITY : unord32(u);   // (bits below the ordered -inf = negative NaNs)
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (vm[v] >= thr) {
                    const int64_t j0 = row.first(g0 + v * kThr + tid);
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        if (x[v][e] >= thr && j0 + e < jend) {
                            const int at2 = atomicAdd(&s_n, 1);
                            if (at2 < kCand) s_cand[at2] = make_key(x[v][e], j0 + e);
                        }
                    }
                }
            }
            __syncthreads();
            const int n = s_n;
            ranked = n <= kCand;
            if (ranked) {
                for (int i = tid; i < n; i += kThr) {
                    const u64 key = s_cand[i];
                    int rank = 0;
                    for (int q = 0; q < n; ++q) rank += s_cand[q] > key;
                    if (rank < top) keys[rank] = key;
                }
                for (int i = n + tid; i < top; i += kThr) keys[i] = 0ull;
            }
        }
        if (!ranked) {                                          // (uniform) heavy ties or NaN: extract the largest key below the last one, `top` times
            u64 last = ~0ull;
            for (int k = 0; k < top; ++k) {
                u64 best = 0ull;
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    const int64_t j0 = row.first(g0 + v * kThr + tid);
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        if (j0 + e < jend) {
                            const u64 key = make_key(x[v][e], j0 + e);
                            if (key < last && key > best) best = key;
                        }
                    }
                }
#pragma unroll
                for (int o = 32; o; o >>= 1) {
                    const u64 other = __shfl_xor(best, o);
                    best = other > best ? other : best;
                }
                __syncthreads();
                if (lane == 0) s_cand[wave] = best;
                __syncthreads();
                best = s_cand[0];
#pragma unroll
                for (int w = 1; w < 4; ++w) best = s_cand[w] > best ? s_cand[w] : best;
                if (tid == 0) keys[k] = best;
                last = best;                                    // 0 once the tile is used up: nothing is below it
            }
        }
    }
}

// the tiles' statistics of a row, joined (every lane of the wave gets them): maximum, sum, weighted sum
__device__ __forceinline__ void join_tiles(const Parts& in, int64_t r, int tiles, float c, int lane, float& M, float& S, float& Tw) {
    float m = -INFINITY;
    for (int i = lane; i < tiles; i += 64) m = fmaxf(m, in.m[r * tiles + i]);
    M = wave_max(m);
    float s = 0.f, t = 0.f;
    for (int i = lane; i < tiles; i += 64) {
        const float mi = in.m[r * tiles + i], si = in.s[r * tiles + i];
        if (mi == -INFINITY && si == 0.f) continue;             // nothing in this tile
        const float y = (mi - M) * c, w = exp2f(y * kLog2e);
        s = fmaf(si, w, s);
        if (w > 0.f) t = fmaf(fmaf(si, y, in.t[r * tiles + i]), w, t);
        if (w != w) t = w;
    }
    S = wave_sum(s);
    Tw = wave_sum(t);
}

// ---- tokens: join the tiles of a row, answer --------------------------------------------------------------------------------
template <typename D>
__global__ __launch_bounds__(kThr) void token_finish_kernel(const D* __restrict__ logits, int64_t row_stride, const int64_t* __restrict__ tokens, float c,
                                                            int64_t ignore_index, Parts in, int tiles, int V, int top, float* __restrict__ logp,
                                                            float* __restrict__ entropy, float* __restrict__ top_logp, int64_t* __restrict__ top_tokens,
                                                            float* __restrict__ stats) {
    __shared__ float s_row[2];
    __shared__ u64 s_key[2048 + kTopMax], s_best[kTopMax];
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t r = blockIdx.x;
    if (tid < 64) {
        float M, S, Tw;
        join_tiles(in, r, tiles, c, lane, M, S, Tw);
        if (lane == 0) {
            const bool empty = M == -INFINITY && S == 0.f;
            const float ls = empty ? 0.f : logf(S);
            const float H = empty ? 0.f : ls - Tw / S;
            const int64_t y = tokens[r];
            float lp = 0.f;
            if (y != ignore_index)
                lp = (y < 0 || y >= V) ? NAN : empty ? -INFINITY : (gf_to_f<D>(logits[r * row_stride + y]) - M) * c - ls;
            logp[r] = lp;
            if (entropy) entropy[r] = H;
            if (stats) stats[r * 3] = M, stats[r * 3 + 1] = ls, stats[r * 3 + 2] = H;
            s_row[0] = M;
            s_row[1] = ls;
        }
    }
    if (top == 0) return;
    if (tid < top) s_best[tid] = 0ull;
    __syncthreads();
    const int64_t total = (int64_t)tiles * top;
    for (int64_t k0 = 0; k0 < total; k0 += 2048) {              // the tiles' best keys in pieces, with the best ones so far
        const int n0 = (int)(total - k0 < 2048 ? total - k0 : 2048), n = n0 + top;
        for (int i = tid; i < n; i += kThr) s_key[i] = i < top ? s_best[i] : in.keys[r * total + k0 + i - top];
        __syncthreads();
        if (tid < top) s_best[tid] = 0ull;
        __syncthreads();
        for (int i = tid; i < n; i += kThr) {
            const u64 key = s_key[i];
            if (key == 0ull) continue;
            int rank = 0;
            for (int q = 0; q < n; ++q) rank += s_key[q] > key;
            if (rank < top) s_best[rank] = key;
        }
        __syncthreads();
    }
    if (tid < top) {
        const u64 key = s_best[tid];
        const int64_t j = (unsigned)~(unsigned)key;
        const unsigned o = (unsigned)(key >> 32);
        const float x = o == 0xfffffffeu ? NAN : unord32(o), M = s_row[0];
        top_tokens[r * top + tid] = j;
        top_logp[r * top + tid] = (M == -INFINITY && s_row[1] == 0.f) ? -INFINITY : (x - M) * c - s_row[1];
    }
}

// ---- gradients: dlogits = f(x) for every output, then the named ones over it ------------------------------------------------
template <typename D, typename F>
__device__ __forceinline__ void for_tile(const Row<D>& row, D* __restrict__ drow, int64_t g0, int groups, F&& f) {
    constexpr int VE = Row<D>::VE;
    for (int g = threadIdx.x; g < groups; g += kThr) {
        float x[VE], d[VE];
        const int64_t j = row.first(g0 + g);
        const bool whole = row.load(g0 + g, x, 0.f);
#pragma unroll
        for (int e = 0; e < VE; ++e) d[e] = f(x[e]);
        if (whole) {
            gf_store_any<D, VE>(drow + j, d);
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (j + e < row.V) drow[j + e] = gf_from_f<D>(d[e]);
        }
    }
}

template <typename D>
__global__ __launch_bounds__(kThr) void token_bwd_kernel(const D* __restrict__ logits, int64_t row_stride, const int64_t* __restrict__ tokens, float c,
                                                         int64_t ignore_index, const float* __restrict__ stats, const int64_t* __restrict__ top_tokens,
                                                         int top, const float* __restrict__ dlogp, const float* __restrict__ dentropy,
                                                         const float* __restrict__ dtop, D* __restrict__ dlogits, int V, int tiles, int groups) {
    __shared__ float s_w[kTopMax + 1];
    __shared__ int64_t s_j[kTopMax + 1];
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x / (unsigned)tiles;
    const int64_t g0 = (int64_t)(blockIdx.x % (unsigned)tiles) * groups;
    const float m = stats[r * 3], ls = stats[r * 3 + 1], H = stats[r * 3 + 2];
    const int64_t y = tokens[r];
    const bool empty = m == -INFINITY && ls == 0.f;             // nothing but ruled-out outputs
    if (tid <= top) {                                           // the named outputs and their weights
        float w = 0.f;
        int64_t j = -1;
        if (tid == top) {
            if (y != ignore_index && dlogp) {
                w = dlogp[r];
                j = y;
                if ((y < 0 || y >= V) && w != 0.f) w = NAN;     // its log probability is NaN
            }
        } else if (dtop) {
            w = dtop[r * top + tid];
            j = top_tokens[r * top + tid];
        }
        s_w[tid] = empty ? 0.f : w;
        s_j[tid] = j;
    }
    __syncthreads();
    float A = 0.f;
    for (int k = 0; k <= top; ++k) A += s_w[k];
    const float gH = (dentropy && !empty) ? dentropy[r] : 0.f;
    const Row<D> row(logits + r * row_stride, V);
    D* drow = dlogits + r * V;
    const bool none = A == 0.f && gH == 0.f;
    auto base = [&](float x) {
        const float lp = (x - m) * c - ls, p = exp2f(lp * kLog2e);
        return (none || p == 0.f) ? 0.f : -c * p * fmaf(gH, lp + H, A);
    };
    for_tile<D>(row, drow, g0, groups, base);
    __syncthreads();                                            // (the workgroup's own stores are done: the named outputs follow them)
    if (tid <= top) {
        const int64_t j = s_j[tid], q = j - row.first(g0);
        if (j >= 0 && j < V && q >= 0 && q < (int64_t)groups * Row<D>::VE) {
            float w = 0.f;
            for (int k = 0; k <= top; ++k) w += s_j[k] == j ? s_w[k] : 0.f;
            if (w != 0.f) drow[j] = gf_from_f<D>(base(gf_to_f<D>(row.p[j])) + c * w);
        }
    }
}

// ---- distillation: one wave per row joins the tiles and does the K-wide part ------------------------------------------------------
template <typename D>
__global__ __launch_bounds__(kThr) void distill_finish_kernel(const D* __restrict__ logits, int64_t row_stride, const int64_t* __restrict__ indices,
                                                              const float* __restrict__ values, float c, int tail, Parts in, int tiles, int64_t R, int V,
                                                              int K, float* __restrict__ loss, float* __restrict__ stats, float* __restrict__ probs) {
    const int lane = threadIdx.x & 63;
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= R) return;
    float M, S, Tw;
    join_tiles(in, r, tiles, c, lane, M, S, Tw);
    int64_t j = -1;
    double v = -INFINITY, x = 0.0;
    if (lane < K) {
        j = indices[r * K + lane];
        if (j < 0 || j >= V) j = -1;
    }
    if (j >= 0) {
        v = values[r * K + lane];
        x = gf_to_f<D>(logits[r * row_stride + j]);
    }
    const bool on = j >= 0;
    double G = 0.0, L = 0.0;
    float coef = 0.f;
    bool some = __ballot(on && !(v == -INFINITY)) != 0ull;      // an entry with mass (or NaN)
    // entries with my index: their mass belongs to the same output; the first one stands for it
    const double cd = c;
    double p;
    if (tail) {
        p = on ? exp(v) : 0.0;
    } else {
        double vm = on && v == v ? v : -INFINITY;
#pragma unroll
        for (int o = 32; o; o >>= 1) vm = fmax(vm, __shfl_xor(vm, o));
        p = on ? exp((v - vm) * cd) : 0.0;
        if (v == -INFINITY) p = 0.0;
        p /= wave_sum(p);
    }
    some = tail ? __ballot(on) != 0ull : some;
    double mine = 0.0;                                          // mass of my output
    bool first = true;
    for (int k = 0; k < K; ++k) {
        const int64_t jk = __shfl(j, k);
        const double pk = __shfl(p, k);
        if (jk == j) mine += pk;
        if (jk == j && k < lane) first = false;
    }
    if (!tail) {
        const double ls = log((double)S);
        const double lq = (M == -INFINITY && S == 0.f) ? -INFINITY : (x - (double)M) * cd - ls;
        if (on && p != 0.0) L = p * (log(p) - lq);
        G = on ? exp(lq) - mine : 0.0;
        L = wave_sum(L);
        coef = 1.f;
        if (lane == 0 && some) stats[r * 3] = M, stats[r * 3 + 1] = (float)ls;
    } else {
        // rest: outputs not named (M, S are theirs); all = rest and named ones, joined at the larger maximum
        const bool rest = M != -INFINITY || S != 0.f;
        double xm = (on && x == x) ? x : -INFINITY;
#pragma unroll
        for (int o = 32; o; o >>= 1) xm = fmax(xm, __shfl_xor(xm, o));
        const double Ma = fmax(xm, rest ? (double)M : -INFINITY);
        const double near = on ? (x - Ma) * cd : 0.0;
        const double named = wave_sum(on && first ? (Ma == -INFINITY ? 0.0 : exp(near)) : 0.0);
        const double lrest = rest ? log((double)S) + ((double)M - Ma) * cd : -INFINITY;      // log of the rest's sum, at Ma
        const double srest = exp(lrest);
        const double lall = log(named + srest);
        const double psum = wave_sum(p), pr = fmax(1.0 - psum, 0.0);
        const double lq = Ma == -INFINITY ? -INFINITY : near - lall;
        const double q = on ? exp(lq) : 0.0;
        // sum p f(log(q / p)) + corrections, f(d) = e^d - 1 - d >= 0: no cancellation where both masses are near one
        double term = q;
        if (p != 0.0) {
            const double d = lq - v;
            term = p * (expm1(d) - d);
        }
        L = wave_sum(on ? term - (first ? 0.0 : q) : 0.0);
        // log q_r = log(srest / (srest + named)), exact where the named mass is small
        const double lqr = lrest == -INFINITY ? -INFINITY : (named <= srest ? -log1p(named / srest) : lrest - lall);
        const double W = pr > 0.0 ? 1.0 : psum;
        double cr;
        if (pr > 0.0) {
            const double dr = lqr - log(pr);
            L += pr * (expm1(dr) - dr);
            cr = pr * expm1(dr);                                // q_r - p_r
        } else {
            L += (psum - 1.0) + exp(lqr);
            cr = psum * exp(lqr);
        }
        if (pr != pr || psum != psum) L = cr = NAN;
        coef = (float)cr;
        G = on ? W * q - mine : 0.0;
        if (lane == 0 && some) stats[r * 3] = M, stats[r * 3 + 1] = (float)log((double)S);
    }
    if (lane == 0) {
        loss[r] = some ? (float)L : 0.f;
        stats[r * 3 + 2] = some ? coef : 0.f;
        if (!some) stats[r * 3] = 0.f, stats[r * 3 + 1] = 0.f;
    }
    if (lane < K) probs[r * K + lane] = some && on ? (float)G : 0.f;
}

template <typename D>
__global__ __launch_bounds__(kThr) void distill_bwd_kernel(const D* __restrict__ logits, int64_t row_stride, const int64_t* __restrict__ indices,
                                                           const float* __restrict__ probs, const float* __restrict__ stats, float c,
                                                           const float* __restrict__ dloss, D* __restrict__ dlogits, int V, int K, int tiles, int groups) {
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x / (unsigned)tiles;
    const int64_t g0 = (int64_t)(blockIdx.x % (unsigned)tiles) * groups;
    const float m = stats[r * 3], ls = stats[r * 3 + 1], g = c * dloss[r], w = g * stats[r * 3 + 2];
    const Row<D> row(logits + r * row_stride, V);
    D* drow = dlogits + r * V;
    const bool none = g == 0.f || w == 0.f || (m == -INFINITY && ls == -INFINITY);   // (the second: every output named or ruled out)
    for_tile<D>(row, drow, g0, groups, [&](float x) {
        const float p = exp2f(((x - m) * c - ls) * kLog2e);
        return none ? 0.f : w * p;
    });
    __syncthreads();                                            // (the workgroup's own stores are done: the named outputs follow them)
    if (tid < K) {
        const int64_t j = indices[r * K + tid], q = j - row.first(g0);
        if (j >= 0 && j < V && q >= 0 && q < (int64_t)groups * Row<D>::VE) drow[j] = gf_from_f<D>(g == 0.f ? 0.f : g * probs[r * K + tid]);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// groups (16-byte vectors) per thread of a tile: as large as the registers hold (8) once that gives the chip enough workgroups
template <typename D> int pick_nv(int64_t R, int64_t V) {
    const int64_t groups = row_groups<D>(V);
    for (int nv = 8; nv > 1; nv >>= 1) {
        const int64_t tiles = (groups + (int64_t)nv * kThr - 1) / ((int64_t)nv * kThr);
        if (R * tiles >= 2048 && groups > (int64_t)(nv / 2) * kThr) return nv;
    }
    int nv = 1;                                                 // few rows: small tiles; a single one where it suffices
    while (nv < 8 && (groups + (int64_t)nv * kThr - 1) / ((int64_t)nv * kThr) * R > 4096) nv <<= 1;
    return nv;
}
template <typename D> int64_t tiles_of(int64_t V, int nv) { return (row_groups<D>(V) + (int64_t)nv * kThr - 1) / ((int64_t)nv * kThr); }

int64_t tiles_for(int64_t R, int64_t V, int dtype) {
    return dtype == GF_F32 ? tiles_of<float>(V, pick_nv<float>(R, V)) : tiles_of<gf_bf16>(V, pick_nv<gf_bf16>(R, V));
}
size_t parts_bytes(int64_t R, int64_t tiles, int top) { return (size_t)R * tiles * ((size_t)top * 8 + 12); }

Parts make_parts(void* ws, int64_t R, int64_t tiles, int top) {
    Parts p;
    p.keys = static_cast<u64*>(ws);
    p.m = reinterpret_cast<float*>(p.keys + R * tiles * top);
    p.s = p.m + R * tiles;
    p.t = p.s + R * tiles;
    return p;
}

template <typename D, bool TOP, bool MASK>
int run_tiles(const void* logits, int64_t row_stride, int64_t R, int V, float c, int top, const int64_t* indices, int K, const Parts& parts,
              hipStream_t st) {
    const int nv = pick_nv<D>(R, V);
    const int tiles = (int)tiles_of<D>(V, nv);
    const dim3 grid((unsigned)(R * tiles));
    const D* x = static_cast<const D*>(logits);
    const float c2 = c * kLog2e;
    if (nv == 8) tile_kernel<D, 8, TOP, MASK><<<grid, kThr, 0, st>>>(x, row_stride, V, tiles, c2, top, indices, K, parts);
    else if (nv == 4) tile_kernel<D, 4, TOP, MASK><<<grid, kThr, 0, st>>>(x, row_stride, V, tiles, c2, top, indices, K, parts);
    else if (nv == 2) tile_kernel<D, 2, TOP, MASK><<<grid, kThr, 0, st>>>(x, row_stride, V, tiles, c2, top, indices, K, parts);
    else tile_kernel<D, 1, TOP, MASK><<<grid, kThr, 0, st>>>(x, row_stride, V, tiles, c2, top, indices, K, parts);
    GF_LAUNCH_CHECK("tile_kernel");
    return GF_OK;
}

int check_rows(const char* who, int64_t R, int64_t V, int64_t row_stride, int dtype, float temperature) {
    GF_REQUIRE_ARG(gf_dtype_ok(dtype), "%s: dtype %d", who, dtype);
    GF_REQUIRE_SHAPE(R > 0 && V > 0 && row_stride >= 0, "%s: bad shape R=%lld V=%lld row stride %lld", who, (long long)R, (long long)V, (long long)row_stride);
    GF_REQUIRE_ARG(temperature > 0.f && temperature < INFINITY, "%s: temperature %g", who, (double)temperature);
    // one workgroup per (row, tile of at least 1024 elements): the launch grid is 32 bits wide
    GF_REQUIRE_SHAPE(V < (1ll << 31) - 64 && R < (1ll << 31) && (double)R * ((double)V / 1024.0 + 2.0) < 2147483000.0, "%s: R=%lld rows of V=%lld are too many", who,
                     (long long)R, (long long)V);
    return GF_OK;
}

// tiles of a gradient kernel: 16 KiB of logits per workgroup where that gives enough workgroups, fewer otherwise
template <typename D> void bwd_tiles(int64_t R, int64_t V, int& tiles, int& groups) {
    const int64_t all = row_groups<D>(V);
    int64_t per = 4 * kThr;
    while (per > kThr && R * ((all + per - 1) / per) < 2048) per >>= 1;
    groups = (int)per;
    tiles = (int)((all + per - 1) / per);
}

template <typename D>
int token_forward_t(const void* logits, int64_t row_stride, const int64_t* tokens, float c, int64_t ignore, float* logp, float* entropy, float* top_logp,
                    int64_t* top_tokens, int top, float* stats, void* ws, int64_t R, int V, hipStream_t st) {
    const int tiles = (int)tiles_of<D>(V, pick_nv<D>(R, V));
    const Parts p = make_parts(ws, R, tiles, top);
    const int rc = top ? run_tiles<D, true, false>(logits, row_stride, R, V, c, top, nullptr, 0, p, st)
                       : run_tiles<D, false, false>(logits, row_stride, R, V, c, 0, nullptr, 0, p, st);
    if (rc != GF_OK) return rc;
    token_finish_kernel<D><<<dim3((unsigned)R), dim3(top ? kThr : 64), 0, st>>>(static_cast<const D*>(logits), row_stride, tokens, c, ignore, p, tiles, V,
                                                                                top, logp, entropy, top_logp, top_tokens, stats);
    GF_LAUNCH_CHECK("token_finish_kernel");
    return GF_OK;
}

template <typename D>
int token_backward_t(const void* logits, int64_t row_stride, const int64_t* tokens, float c, int64_t ignore, const float* stats, const int64_t* top_tokens,
                     int top, const float* dlogp, const float* dentropy, const float* dtop, void* dlogits, int64_t R, int V, hipStream_t st) {
    int tiles, groups;
    bwd_tiles<D>(R, V, tiles, groups);
    token_bwd_kernel<D><<<dim3((unsigned)(R * tiles)), kThr, 0, st>>>(static_cast<const D*>(logits), row_stride, tokens, c, ignore, stats, top_tokens, top,
                                                                      dlogp, dentropy, dtop, static_cast<D*>(dlogits), V, tiles, groups);
    GF_LAUNCH_CHECK("token_bwd_kernel");
    return GF_OK;
}

template <typename D>
int distill_forward_t(const void* logits, int64_t row_stride, const int64_t* indices, const float* values, float c, int tail, float* loss, float* stats,
                      float* probs, void* ws, int64_t R, int V, int K, hipStream_t st) {
    const int tiles = (int)tiles_of<D>(V, pick_nv<D>(R, V));
    const Parts p = make_parts(ws, R, tiles, 0);
    const int rc = tail ? run_tiles<D, false, true>(logits, row_stride, R, V, c, 0, indices, K, p, st)
                        : run_tiles<D, false, false>(logits, row_stride, R, V, c, 0, nullptr, 0, p, st);
    if (rc != GF_OK) return rc;
    distill_finish_kernel<D><<<dim3((unsigned)((R + 3) / 4)), kThr, 0, st>>>(static_cast<const D*>(logits), row_stride, indices, values, c, tail, p, tiles,
                                                                             R, V, K, loss, stats, probs);
    GF_LAUNCH_CHECK("distill_finish_kernel");
    return GF_OK;
}

template <typename D>
int distill_backward_t(const void* logits, int64_t row_stride, const int64_t* indices, const float* probs, const float* stats, float c,
                       const float* dloss, void* dlogits, int64_t R, int V, int K, hipStream_t st) {
    int tiles, groups;
    bwd_tiles<D>(R, V, tiles, groups);
    distill_bwd_kernel<D><<<dim3((unsigned)(R * tiles)), kThr, 0, st>>>(static_cast<const D*>(logits), row_stride, indices, probs, stats, c, dloss,
                                                                        static_cast<D*>(dlogits), V, K, tiles, groups);
    GF_LAUNCH_CHECK("distill_bwd_kernel");
    return GF_OK;
}

template <typename F> int by_dtype(int dtype, F&& f) {
    if (dtype == GF_F32) return f(float());
    if (dtype == GF_BF16) return f(gf_bf16());
    return f(gf_f16());
}

}  // namespace

extern "C" size_t gf_token_logp_workspace_bytes(int64_t R, int32_t V, int32_t top, int32_t dtype) {
    if (R <= 0 || V <= 0 || top < 0 || !gf_dtype_ok(dtype)) return 0;
    return parts_bytes(R, tiles_for(R, V, dtype), top);
}

extern "C" int gf_token_logp_forward(const void* logits, int64_t row_stride, const int64_t* tokens, float temperature, int64_t ignore_index, float* logp,
                                     float* entropy, float* top_logp, int64_t* top_tokens, int32_t top, float* stats, void* workspace,
                                     size_t workspace_bytes, int32_t dtype, int64_t R, int32_t V, void* stream) {
    const int rc = check_rows("gf_token_logp_forward", R, V, row_stride, dtype, temperature);
    if (rc != GF_OK) return rc;
    GF_REQUIRE_SHAPE(top >= 0 && top <= kTopMax && top <= V, "gf_token_logp_forward: top=%d (0..min(V, %d))", top, kTopMax);
    GF_REQUIRE_ARG(logits && tokens && logp && (top == 0 || (top_logp && top_tokens)), "gf_token_logp_forward: NULL tensor");
    const size_t need = gf_token_logp_workspace_bytes(R, V, top, dtype);
    GF_REQUIRE_ARG(workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 8 == 0,
                   "gf_token_logp_forward: workspace of %zu bytes, needs %zu, 8-byte aligned", workspace_bytes, need);
    return by_dtype(dtype, [&](auto d) -> int {
        return token_forward_t<decltype(d)>(logits, row_stride, tokens, 1.f / temperature, ignore_index, logp, entropy, top_logp, top_tokens, top, stats,
                                            workspace, R, V, gf_stream(stream));
    });
}

extern "C" int gf_token_logp_backward(const void* logits, int64_t row_stride, const int64_t* tokens, float temperature, int64_t ignore_index,
                                      const float* stats, const int64_t* top_tokens, int32_t top, const float* dlogp, const float* dentropy,
                                      const float* dtop, void* dlogits, int32_t dtype, int64_t R, int32_t V, void* stream) {
    const int rc = check_rows("gf_token_logp_backward", R, V, row_stride, dtype, temperature);
    if (rc != GF_OK) return rc;
    GF_REQUIRE_SHAPE(top >= 0 && top <= kTopMax && top <= V, "gf_token_logp_backward: top=%d (0..min(V, %d))", top, kTopMax);
    GF_REQUIRE_ARG(logits && tokens && stats && dlogits && (top == 0 || top_tokens), "gf_token_logp_backward: NULL tensor");
    return by_dtype(dtype, [&](auto d) -> int {
        return token_backward_t<decltype(d)>(logits, row_stride, tokens, 1.f / temperature, ignore_index, stats, top_tokens, top, dlogp, dentropy, dtop,
                                             dlogits, R, V, gf_stream(stream));
    });
}

extern "C" size_t gf_distill_top_workspace_bytes(int64_t R, int32_t V, int32_t K, int32_t dtype) {
    if (R <= 0 || V <= 0 || K <= 0 || !gf_dtype_ok(dtype)) return 0;
    return parts_bytes(R, tiles_for(R, V, dtype), 0);
}

extern "C" int gf_distill_top_forward(const void* logits, int64_t row_stride, const int64_t* indices, const float* values, float temperature, int32_t tail,
                                      float* loss, float* stats, float* probs, void* workspace, size_t workspace_bytes, int32_t dtype, int64_t R,
                                      int32_t V, int32_t K, void* stream) {
    const int rc = check_rows("gf_distill_top_forward", R, V, row_stride, dtype, temperature);
    if (rc != GF_OK) return rc;
    GF_REQUIRE_SHAPE(K >= 1 && K <= kTopMax, "gf_distill_top_forward: K=%d (1..%d)", K, kTopMax);
    GF_REQUIRE_ARG(logits && indices && values && loss && stats && probs, "gf_distill_top_forward: NULL tensor");
    const size_t need = gf_distill_top_workspace_bytes(R, V, K, dtype);
    GF_REQUIRE_ARG(workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 8 == 0,
                   "gf_distill_top_forward: workspace of %zu bytes, needs %zu, 8-byte aligned", workspace_bytes, need);
    return by_dtype(dtype, [&](auto d) -> int {
        return distill_forward_t<decltype(d)>(logits, row_stride, indices, values, 1.f / temperature, tail, loss, stats, probs, workspace, R, V, K,
                                              gf_stream(stream));
    });
}

extern "C" int gf_distill_top_backward(const void* logits, int64_t row_stride, const int64_t* indices, const float* probs, const float* stats,
                                       float temperature, int32_t tail, const float* dloss, void* dlogits, int32_t dtype, int64_t R, int32_t V, int32_t K,
                                       void* stream) {
    const int rc = check_rows("gf_distill_top_backward", R, V, row_stride, dtype, temperature);
    if (rc != GF_OK) return rc;
    GF_REQUIRE_SHAPE(K >= 1 && K <= kTopMax, "gf_distill_top_backward: K=%d (1..%d)", K, kTopMax);
    GF_REQUIRE_ARG(logits && indices && probs && stats && dloss && dlogits, "gf_distill_top_backward: NULL tensor");
    (void)tail;
    return by_dtype(dtype, [&](auto d) -> int {
        return distill_backward_t<decltype(d)>(logits, row_stride, indices, probs, stats, 1.f / temperature, dloss, dlogits, R, V, K, gf_stream(stream));
    });
}
