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
// Bound by HBM; for 16-bit logits the exponential (a quarter-rate instruction) and the conversions weigh about as much.  Reached: forward over
// 2048 x 100k bf16 104 + 8 us (tiles, join; 3.9 TB/s in the tiles), with entropy and 8 alternatives over 4096 x 50001 117 + 14 us (3.5); gradients
// 131-139 us (5.9-6.2 TB/s read and written; a copy of 4 GiB 4.7, of 128 MiB 7.2); 2000 x 10k fp32: 16 + 4 and 26 us; 1M rows of 5: 43 us with 3 alternatives.
// exp2_fast gives zero below 2^-126: a probability is off by less than that.
// Sums are fp32 and in a fixed order; the K-wide part of the distillation loss is fp64 (a small difference of masses near one).
#include "gf_num.h"

#include <type_traits>

namespace {

constexpr int kThr = 256;
constexpr int kTopMax = 64;
constexpr int kPackMax = 64;       // rows of up to so many outputs are packed into waves
constexpr int kMaxNV = 4;          // 16-byte groups per thread and tile: 4 / 2: 117 / 155 us for 4096 x 50001 bf16 with 8 alternatives, 104 / 103 without (8 would
                                   // need a 64-bit hit mask; timed before there was one at all: 189 against 162 us)
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

// reductions over the wave by lane shifts inside the vector unit (no LDS traffic); every lane gets the result.  Fixed order.
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp(float old, float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(old), __float_as_uint(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float last_lane(float v) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63)); }
__device__ __forceinline__ float wave_max(float v) {
    const float n = -INFINITY;
    v = fmaxf(v, dpp<0x111, 0xf>(n, v));                        // rows of 16: shifted by 1, 2, 4, 8
    v = fmaxf(v, dpp<0x112, 0xf>(n, v));
    v = fmaxf(v, dpp<0x114, 0xf>(n, v));
    v = fmaxf(v, dpp<0x118, 0xf>(n, v));
    v = fmaxf(v, dpp<0x142, 0xa>(n, v));                        // last lane of a row to the next row, rows 1 and 3
    v = fmaxf(v, dpp<0x143, 0xc>(n, v));                        // lane 31 to rows 2 and 3
    return last_lane(v);
}
__device__ __forceinline__ float wave_sum(float v) {
    v += dpp<0x111, 0xf>(0.f, v);
    v += dpp<0x112, 0xf>(0.f, v);
    v += dpp<0x114, 0xf>(0.f, v);
    v += dpp<0x118, 0xf>(0.f, v);
    v += dpp<0x142, 0xa>(0.f, v);
    v += dpp<0x143, 0xc>(0.f, v);
    return last_lane(v);
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ double lane_value(double v, int k) {  // lane k's value (k uniform)
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), k), __builtin_amdgcn_readlane(__double2loint(v), k));
}
__device__ __forceinline__ float exp2_fast(float y) { return __builtin_amdgcn_exp2f(y); }   // one instruction; results below 2^-126 are zero

// how many of the n keys are larger than `key`, eight LDS reads in flight
__device__ __forceinline__ int rank_of(const u64* keys, int n, u64 key) {
    int rank = 0, q = 0;
    for (; q + 8 <= n; q += 8) {
        u64 k[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = keys[q + e];
#pragma unroll
        for (int e = 0; e < 8; ++e) rank += k[e] > key;
    }
    for (; q < n; ++q) rank += keys[q] > key;
    return rank;
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

// Lower bound of the k-th largest of the wave's 64 values (as ordered unsigned): its bits from LOW up, found one by one.  LOW = 16: exact for bf16,
// and for the other types a few values more pass (half the steps of the exact search, LOW = 0).
template <int LOW = 16> __device__ __forceinline__ unsigned kth_of_wave(unsigned v, int k) {
    unsigned thr = 0;
#pragma unroll
    for (int b = 31; b >= LOW; --b) {
        const unsigned c = thr | (1u << b);
        if (__popcll(__ballot(v >= c)) >= k) thr = c;
    }
    return thr;
}

struct TokenOut {                  // what a row of token_log_probs is answered with
    const int64_t* tokens;
    int64_t ignore;
    float *logp, *entropy, *top_logp;
    int64_t* top_tokens;
    float* stats;
};
// one thread: the row's statistics (maximum M, sum S, weighted sum T in natural units)
template <typename D>
__device__ __forceinline__ void answer_row(const TokenOut& o, int64_t r, const D* row, int V, float c, float M, float S, float T, float& ls) {
    const bool empty = M == -INFINITY && S == 0.f;              // nothing but ruled-out outputs
    ls = empty ? 0.f : logf(S);
    const float H = empty ? 0.f : ls - T / S;
    const int64_t y = o.tokens[r];
    float lp = 0.f;
    if (y != o.ignore) lp = (y < 0 || y >= V) ? NAN : empty ? -INFINITY : (gf_to_f<D>(row[y]) - M) * c - ls;
    o.logp[r] = lp;
    if (o.entropy) o.entropy[r] = H;
    if (o.stats) o.stats[r * 3] = M, o.stats[r * 3 + 1] = ls, o.stats[r * 3 + 2] = H;
}
__device__ __forceinline__ void answer_top(const TokenOut& o, int64_t at, u64 key, float c, float M, float ls) {
    const unsigned v = (unsigned)(key >> 32);
    const float x = v == 0xfffffffeu ? NAN : unord32(v);
    o.top_tokens[at] = (unsigned)~(unsigned)key;
    o.top_logp[at] = (M == -INFINITY && ls == 0.f) ? -INFINITY : (x - M) * c - ls;
}

// A tile with more than kCand elements at or above its threshold: equal values, as rows of outputs that are ruled out (-inf) or all alike have them.  With
// the threshold u exact (the k-th largest of the same maxima, all bits) every element above it is a candidate, and of those equal to it the first
// ones in index order, counted by a scan over the threads per row of groups.  Returns the number of candidates in s_cand (more than kCand: does
// not fit).  The tile is read again, so that the usual case keeps no registers for this.
// (4096 x 50001 bf16 but for 20 outputs ruled out, 8 / 64 alternatives: 984 / 4971 us with the extraction loop below alone,
// 531 / 550 us with this; 134 / 197 us without the mask.)
// Not for rows that rise or fall with the index: a full tile's threshold is the smallest of the waves' (k / 4)-th maxima, the wave with the low
// values decides it, 1500-1800 of 8192 values pass, above the exact threshold too, and the loop is taken (4096 x 50001 bf16 sorted, 8 / 64
// alternatives: 0.82 / 4.9 ms; values that fall as a power law of the index 0.21 / 0.40 ms).
template <typename D, int NV>
__device__ __forceinline__ int collect_ties(const Row<D>& row, int64_t g0, float tm, bool full, int top, unsigned* s_thr, int* s_n, u64* s_cand) {
    constexpr int VE = Row<D>::VE;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __syncthreads();                                            // s_thr and s_n have been read
    {
        const unsigned o = ord32(tm), a = kth_of_wave<0>(o, (top + 3) / 4), b = full ? 0u : kth_of_wave<0>(o, top);
        if (lane == 0) s_thr[wave] = a, s_thr[4 + wave] = b;
        if (tid == 0) *s_n = 0;
    }
    __syncthreads();
    unsigned ua = s_thr[0], ub = s_thr[4];
#pragma unroll
    for (int w = 1; w < 4; ++w) ua = min(ua, s_thr[w]), ub = max(ub, s_thr[4 + w]);
    const unsigned u = max(ua, ub);
    int nothing = 0;                                            // (an address that looks new to the compiler: nothing is kept from the first read)
    asm volatile("" : "+v"(nothing));
    const Row<D> again(row.p + nothing, row.V);
    auto each = [&](int v, auto&& f) {                          // f(e, ordered value, index) of the thread's elements of group row v
        float y[VE];
        const int64_t j0 = row.first(g0 + v * kThr + tid);
        again.load(g0 + v * kThr + tid, y, -INFINITY);
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (j0 + e < row.V) f(e, ord32(y[e]), j0 + e);
    };
#pragma unroll 1
    for (int v = 0; v < NV; ++v)
        each(v, [&](int, unsigned o, int64_t j) {
            if (o > u) {
                const int k = atomicAdd(s_n, 1);
                if (k < kCand) s_cand[k] = ((u64)o << 32) | (unsigned)~(unsigned)j;
            }
        });
    __syncthreads();
    const int above = *s_n;
    if (above >= top) return above;
    int taken = 0;                                              // of the equal ones, so far
#pragma unroll 1
    for (int v = 0; v < NV && taken < top - above; ++v) {       // (uniform)
        unsigned equal = 0u;
        each(v, [&](int e, unsigned o, int64_t) { equal |= o == u ? 1u << e : 0u; });
        int before = __popc(equal);                             // inclusive scan of the counts over the workgroup
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int below = __shfl_up(before, o);
            if (lane >= o) before += below;
        }
        __syncthreads();
        if (lane == 63) s_thr[wave] = (unsigned)before;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w == wave) before += all;
            all += (int)s_thr[w];
        }
        int at = taken + before - __popc(equal);
        const int64_t j0 = row.first(g0 + v * kThr + tid);
        while (equal && at < top - above) {
            const int e = __ffs(equal) - 1;
            equal &= equal - 1u;
            s_cand[above + at++] = ((u64)u << 32) | (unsigned)~(unsigned)(j0 + e);
        }
        taken += all;
    }
    __syncthreads();
    return above + min(taken, top - above);
}

// ---- tile statistics (and best keys) -----------------------------------------------------------------------------------
// TOP: the tile's best keys too; ENT: the weighted sum t; MASK: the outputs named by indices[row][0..K) are left out; ONE: a tile is a whole row and
// answered here (tokens).  Each wave has a maximum of its own, so the sums need no workgroup barrier; the four waves join at the end.
// The exponent is the difference first, then the scale (one fma of c2 x - c2 m overflows on masks of the type's lowest value).
template <typename D, int NV, bool TOP, bool ENT, bool MASK, bool ONE>
__global__ __launch_bounds__(kThr) void tile_kernel(const D* __restrict__ logits, int64_t row_stride, int V, int tiles, float c, int top,
                                                    const int64_t* __restrict__ indices, int K, Parts out, TokenOut ans) {
    constexpr int VE = Row<D>::VE, TE = NV * kThr * VE;
    __shared__ float s_m[4], s_s[4], s_t[4], s_row[2];
    __shared__ unsigned s_thr[8];
    __shared__ int s_n;
    __shared__ u64 s_cand[TOP ? kCand : 1];
    __shared__ unsigned s_bits[MASK ? TE / 32 : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = ONE ? blockIdx.x : blockIdx.x / (unsigned)tiles;
    const int tile = ONE ? 0 : (int)(blockIdx.x % (unsigned)tiles);
    const Row<D> row(logits + r * row_stride, V);
    const int64_t g0 = (int64_t)tile * NV * kThr;
    float x[NV][VE];
    const bool full = row.first(g0 + NV * kThr) <= V;
    if (full) {                                                 // (uniform) a tile inside the row: plain loads
        gf_vec_any<D, VE> raw[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) raw[v] = *reinterpret_cast<const gf_vec_any<D, VE>*>(row.p + row.first(g0 + v * kThr + tid));
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < VE; ++e) x[v][e] = gf_to_f<D>(raw[v].e[e]);
    } else {
#pragma unroll
        for (int v = 0; v < NV; ++v) row.load(g0 + v * kThr + tid, x[v], -INFINITY);
    }
    if constexpr (TOP) {
        if (tid == 0) s_n = 0;
    }
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
            const unsigned w = (s_bits[q >> 5] >> (q & 31)) & ((1u << VE) - 1u);
            if (w) {
#pragma unroll
                for (int e = 0; e < VE; ++e)
                    if (w >> e & 1u) x[v][e] = -INFINITY;
            }
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
    if constexpr (TOP) {
        const unsigned o = ord32(tm);
        // (a tile the row does not fill has waves without enough values: their own k-th largest then decides)
        const unsigned a = kth_of_wave(o, (top + 3) / 4), b = full ? 0u : kth_of_wave(o, top);
        if (lane == 0) s_thr[wave] = a, s_thr[4 + wave] = b;
    }
    const float c2 = c * kLog2e, ref = wm == -INFINITY ? 0.f : wm;         // a wave with nothing in it: all exponentials are zero
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float y = (x[v][e] - ref) * c2;               // base-2 exponent
            const float p = exp2_fast(y);
            s += p;
            if (ENT) t = fmaf(p, fmaxf(y, -3e38f), t);          // p = 0 where y = -inf
        }
    s = wave_sum(s);
    if (ENT) t = wave_sum(t) * kLn2;
    if (lane == 0) {
        s_m[wave] = wm;
        s_s[wave] = s;
        s_t[wave] = t;
    }
    __syncthreads();
    float m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    s = t = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float sw = s_s[w], mw = s_m[w];
        if (mw == -INFINITY && sw == 0.f) continue;
        const float y = (mw - m) * c, f = exp2_fast(y * kLog2e);
        s = fmaf(sw, f, s);
        if (ENT && f > 0.f) t = fmaf(fmaf(sw, y, s_t[w]), f, t);
        if (f != f) s = t = f;
    }
    const int64_t at = r * tiles + tile;
    float ls = 0.f;
    if (tid == 0) {
        if constexpr (ONE) {
            answer_row<D>(ans, r, row.p, V, c, m, s, t, ls);
            s_row[0] = ls;
        } else {
            out.m[at] = m;
            out.s[at] = s;
            if (ENT) out.t[at] = t;
        }
    }
    if constexpr (TOP) {
        u64* keys = ONE ? nullptr : out.keys + at * top;
        auto put = [&](int k, u64 key) {
            if constexpr (ONE) answer_top(ans, r * top + k, key, c, m, s_row[0]);
            else keys[k] = key;
        };
        bool ranked = false;
        int n = 0;
        const bool plain = s == s;                              // no NaN in the tile: the maxima above are the values' own order
        if (plain) {
            unsigned ua = s_thr[0], ub = s_thr[4];
#pragma unroll
            for (int w = 1; w < 4; ++w) ua = min(ua, s_thr[w]), ub = max(ub, s_thr[4 + w]);
            const unsigned u = max(ua, ub);
            const float thr = u < 0x00800000u ? -INFINITY : unord32(u);   // (bits below the ordered -inf = negative NaNs)
            static_assert(NV * VE <= 32, "a thread's elements are the bits of a mask");
            unsigned hits = 0u;                                 // (the few hits are read again: no code per element for them)
            if (tm >= thr) {
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    if (vm[v] >= thr) {
#pragma unroll
                        for (int e = 0; e < VE; ++e) hits |= x[v][e] >= thr ? 1u << (v * VE + e) : 0u;
                    }
                }
            }
            while (hits) {
                const int at2 = __ffs(hits) - 1;
                hits &= hits - 1u;
                const int64_t j = row.first(g0 + at2 / VE * kThr + tid) + at2 % VE;
                if (j < V) {
                    const int k = atomicAdd(&s_n, 1);
                    if (k < kCand) s_cand[k] = make_key(gf_to_f<D>(row.p[j]), j);
                }
            }
        }
        __syncthreads();
        if (plain) {
            n = s_n;
            if (n > kCand) n = collect_ties<D, NV>(row, g0, tm, full, top, s_thr, &s_n, s_cand);
            ranked = n <= kCand;
            if (ranked) {
                for (int i = tid; i < n; i += kThr) {
                    const u64 key = s_cand[i];
                    const int rank = rank_of(s_cand, n, key);
                    if (rank < top) put(rank, key);
                }
                if constexpr (!ONE)
                    for (int i = n + tid; i < top; i += kThr) keys[i] = 0ull;
            }
        }
        if (!ranked) {                                          // (uniform) NaN, +inf, or too many above an exact threshold: extract the largest key below the last one, `top` times
            u64 last = ~0ull;
            for (int k = 0; k < top; ++k) {
                u64 best = 0ull;
                int nothing = 0;                                // (rare: the tile is read again rather than kept in registers for this,
                asm volatile("" : "+v"(nothing));               //  so the address must look new to the compiler)
                const Row<D> row2(row.p + nothing, V);
#pragma unroll 1
                for (int v = 0; v < NV; ++v) {
                    float y[VE];
                    const int64_t j0 = row.first(g0 + v * kThr + tid);
                    row2.load(g0 + v * kThr + tid, y, -INFINITY);
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        if (j0 + e < V) {
                            const u64 key = make_key(y[e], j0 + e);
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
                if (tid == 0) put(k, best);
                last = best;                                    // 0 once the tile is used up: nothing is below it
            }
        }
    }
}

// the tiles' statistics of a row, joined (every lane of the wave gets them): maximum, sum, weighted sum
__device__ __forceinline__ void join_tiles(const Parts& in, int64_t r, int tiles, float c, int lane, bool ent, float& M, float& S, float& Tw) {
    float m = -INFINITY;
    for (int i = lane; i < tiles; i += 64) m = fmaxf(m, in.m[r * tiles + i]);
    M = wave_max(m);
    float s = 0.f, t = 0.f;
    for (int i = lane; i < tiles; i += 64) {
        const float mi = in.m[r * tiles + i], si = in.s[r * tiles + i];
        if (mi == -INFINITY && si == 0.f) continue;             // nothing in this tile
        const float y = (mi - M) * c, w = exp2_fast(y * kLog2e);
        s = fmaf(si, w, s);
        if (ent && w > 0.f) t = fmaf(fmaf(si, y, in.t[r * tiles + i]), w, t);
        if (w != w) t = w;
    }
    S = wave_sum(s);
    Tw = wave_sum(t);
}

// ---- tokens: join the tiles of a row, answer --------------------------------------------------------------------------------
template <typename D>
__global__ __launch_bounds__(kThr) void token_finish_kernel(const D* __restrict__ logits, int64_t row_stride, float c, Parts in, int tiles, int V, int top,
                                                            TokenOut ans) {
    constexpr int kPer = 8;                                     // keys per thread and piece
    __shared__ float s_row[2];
    __shared__ u64 s_cand[kPer * kThr + kTopMax], s_best[kTopMax];
    __shared__ unsigned s_thr[8];
    __shared__ int s_n;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x;
    if (tid < 64) {
        float M, S, Tw, ls;
        join_tiles(in, r, tiles, c, lane, true, M, S, Tw);
        if (lane == 0) {
            answer_row<D>(ans, r, logits + r * row_stride, V, c, M, S, Tw, ls);
            s_row[0] = M;
            s_row[1] = ls;
        }
    }
    if (top == 0) return;
    if (tid < top) s_best[tid] = 0ull;
    const int64_t total = (int64_t)tiles * top;
    const u64* keys = in.keys + r * total;
    for (int64_t k0 = 0; k0 < total; k0 += kPer * kThr) {       // the tiles' best keys in pieces, with the best ones so far; chosen as in a tile
        u64 key[kPer + 1], best = 0ull;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int64_t k = k0 + i * kThr + tid;
            key[i] = k < total ? keys[k] : 0ull;
        }
        if (tid == 0) s_n = 0;
        __syncthreads();
        key[kPer] = tid < top ? s_best[tid] : 0ull;
#pragma unroll
        for (int i = 0; i <= kPer; ++i) best = key[i] > best ? key[i] : best;
        const unsigned o = (unsigned)(best >> 32);
        const unsigned a = kth_of_wave(o, (top + 3) / 4), b = kth_of_wave(o, top);
        if (lane == 0) s_thr[wave] = a, s_thr[4 + wave] = b;
        __syncthreads();
        unsigned ua = s_thr[0], ub = s_thr[4];
#pragma unroll
        for (int w = 1; w < 4; ++w) ua = min(ua, s_thr[w]), ub = max(ub, s_thr[4 + w]);
        const unsigned u = max(ua, ub);
        if (tid < top) s_best[tid] = 0ull;
#pragma unroll
        for (int i = 0; i <= kPer; ++i)
            if (key[i] != 0ull && (unsigned)(key[i] >> 32) >= u) s_cand[atomicAdd(&s_n, 1)] = key[i];
        __syncthreads();
        const int n = s_n;
        for (int i = tid; i < n; i += kThr) {
            const u64 k = s_cand[i];
            const int rank = rank_of(s_cand, n, k);
            if (rank < top) s_best[rank] = k;
        }
        __syncthreads();
    }
    if (tid < top) answer_top(ans, r * top + tid, s_best[tid], c, s_row[0], s_row[1]);
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
        const float lp = (x - m) * c - ls, p = exp2_fast(lp * kLog2e);
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
    join_tiles(in, r, tiles, c, lane, false, M, S, Tw);
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
    const int ji = (int)j;                                      // (V < 2^31)
    for (int k = 0; k < K; ++k) {
        const int jk = __builtin_amdgcn_readlane(ji, k);
        const double pk = lane_value(p, k);
        if (jk == ji) mine += pk;
        if (jk == ji && k < lane) first = false;
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
        const float p = exp2_fast(((x - m) * c - ls) * kLog2e);
        return none ? 0.f : w * p;
    });
    __syncthreads();                                            // (the workgroup's own stores are done: the named outputs follow them)
    if (tid < K) {
        const int64_t j = indices[r * K + tid], q = j - row.first(g0);
        if (j >= 0 && j < V && q >= 0 && q < (int64_t)groups * Row<D>::VE) drow[j] = gf_from_f<D>(g == 0.f ? 0.f : g * probs[r * K + tid]);
    }
}

// ---- few outputs (V <= 64): G = 8 .. 64 lanes per row, one output per lane, 64 / G rows per wave ----------------------------------
// A workgroup per row would be idle but for V of its 256 threads; with the rows packed, 1M rows of 5 classes move at the memory's rate.
template <int G> struct Pack {
    int i;                         // output
    int64_t r;                     // row (clamped to the last one: lanes behind it compute on it and store nothing)
    bool row_on, on;
    __device__ __forceinline__ Pack(int64_t R, int V) {
        const int lane = threadIdx.x & 63;
        i = lane % G;
        const int64_t q = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * (64 / G) + lane / G;
        row_on = q < R;
        r = row_on ? q : R - 1;
        on = row_on && i < V;
    }
};
template <int G> __device__ __forceinline__ float pack_max(float v) {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
template <int G> __device__ __forceinline__ float pack_sum(float v) {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

template <typename D, int G>
__global__ __launch_bounds__(kThr) void token_pack_kernel(const D* __restrict__ logits, int64_t row_stride, int64_t R, int V, float c, int top, TokenOut ans) {
    const Pack<G> p(R, V);
    const D* row = logits + p.r * row_stride;
    const float x = p.i < V ? gf_to_f<D>(row[p.i]) : -INFINITY;
    const float m = pack_max<G>(x), ref = m == -INFINITY ? 0.f : m;
    const float y = (x - ref) * (c * kLog2e), e = exp2_fast(y);
    const float s = pack_sum<G>(e), t = pack_sum<G>(e * fmaxf(y, -3e38f)) * kLn2;
    float ls = 0.f;
    if (p.i == 0 && p.row_on) answer_row<D>(ans, p.r, row, V, c, m, s, t, ls);
    if (top) {
        ls = __shfl(ls, (threadIdx.x & 63) / G * G);
        const unsigned o = ord32(x);
        int rank = 0;
        for (int j = 0; j < V; ++j) {
            const unsigned oj = __shfl(o, (threadIdx.x & 63) / G * G + j);
            rank += oj > o || (oj == o && j < p.i);
        }
        if (p.on && rank < top) answer_top(ans, p.r * top + rank, make_key(x, p.i), c, m, ls);
    }
}

template <typename D, int G>
__global__ __launch_bounds__(kThr) void token_pack_bwd_kernel(const D* __restrict__ logits, int64_t row_stride, const int64_t* __restrict__ tokens, float c,
                                                              int64_t ignore_index, const float* __restrict__ stats, const int64_t* __restrict__ top_tokens,
                                                              int top, const float* __restrict__ dlogp, const float* __restrict__ dentropy,
                                                              const float* __restrict__ dtop, D* __restrict__ dlogits, int64_t R, int V) {
    const Pack<G> p(R, V);
    const float x = p.i < V ? gf_to_f<D>(logits[p.r * row_stride + p.i]) : 0.f;
    const float m = stats[p.r * 3], ls = stats[p.r * 3 + 1], H = stats[p.r * 3 + 2];
    const int64_t tok = tokens[p.r];
    const bool empty = m == -INFINITY && ls == 0.f;
    float w = 0.f;                                              // my output's own weight
    if (dtop)
        for (int k = 0; k < top; ++k) w += top_tokens[p.r * top + k] == p.i ? dtop[p.r * top + k] : 0.f;
    if (dlogp && tok != ignore_index) {
        const float g = dlogp[p.r];
        if (tok < 0 || tok >= V) w = g != 0.f ? NAN : w;        // its log probability is NaN
        else if (tok == p.i) w += g;
    }
    if (empty) w = 0.f;
    const float A = pack_sum<G>(p.i < V ? w : 0.f), gH = (dentropy && !empty) ? dentropy[p.r] : 0.f;
    const float lp = (x - m) * c - ls, q = exp2_fast(lp * kLog2e);
    const float d = ((A == 0.f && gH == 0.f) || q == 0.f) ? 0.f : -c * q * fmaf(gH, lp + H, A);
    if (p.on) dlogits[p.r * V + p.i] = gf_from_f<D>(w != 0.f ? d + c * w : d);
}

template <typename D, int G>
__global__ __launch_bounds__(kThr) void distill_pack_kernel(const D* __restrict__ logits, int64_t row_stride, int64_t R, int V, float c,
                                                            const int64_t* __restrict__ named, int K, Parts out) {
    const Pack<G> p(R, V);
    float x = p.i < V ? gf_to_f<D>(logits[p.r * row_stride + p.i]) : -INFINITY;
    if (named)
        for (int k = 0; k < K; ++k)
            if (named[p.r * K + k] == p.i) x = -INFINITY;
    const float m = pack_max<G>(x), ref = m == -INFINITY ? 0.f : m;
    const float s = pack_sum<G>(exp2_fast((x - ref) * (c * kLog2e)));
    if (p.i == 0 && p.row_on) {
        out.m[p.r] = m;
        out.s[p.r] = s;
    }
}

template <typename D, int G>
__global__ __launch_bounds__(kThr) void distill_pack_bwd_kernel(const D* __restrict__ logits, int64_t row_stride, const int64_t* __restrict__ indices,
                                                                const float* __restrict__ probs, const float* __restrict__ stats, float c,
                                                                const float* __restrict__ dloss, D* __restrict__ dlogits, int64_t R, int V, int K) {
    const Pack<G> p(R, V);
    const float x = p.i < V ? gf_to_f<D>(logits[p.r * row_stride + p.i]) : 0.f;
    const float m = stats[p.r * 3], ls = stats[p.r * 3 + 1], g = c * dloss[p.r], w = g * stats[p.r * 3 + 2];
    const bool none = g == 0.f || w == 0.f || (m == -INFINITY && ls == -INFINITY);
    float d = none ? 0.f : w * exp2_fast(((x - m) * c - ls) * kLog2e);
    for (int k = 0; k < K; ++k)
        if (indices[p.r * K + k] == p.i) d = g == 0.f ? 0.f : g * probs[p.r * K + k];
    if (p.on) dlogits[p.r * V + p.i] = gf_from_f<D>(d);
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// groups (16-byte vectors) per thread of a tile: up to kMaxNV once that gives the chip enough workgroups
template <typename D> int pick_nv(int64_t R, int64_t V) {
    const int64_t groups = row_groups<D>(V);
    for (int nv = kMaxNV; nv > 1; nv >>= 1) {
        const int64_t tiles = (groups + (int64_t)nv * kThr - 1) / ((int64_t)nv * kThr);
        if (R * tiles >= 1024 && groups > (int64_t)(nv / 2) * kThr) return nv;
    }
    return groups > 64 * kThr ? 2 : 1;                          // few rows: small tiles, yet not so many that joining them counts
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

// f(lanes per row) for V <= 64; grid of packed rows
template <typename F> int by_pack(int V, F&& f) {
    if (V <= 8) return f(std::integral_constant<int, 8>());
    if (V <= 16) return f(std::integral_constant<int, 16>());
    if (V <= 32) return f(std::integral_constant<int, 32>());
    return f(std::integral_constant<int, 64>());
}
dim3 pack_grid(int64_t R, int G) { return dim3((unsigned)((R + 4 * (64 / G) - 1) / (4 * (64 / G)))); }

template <typename D, bool TOP, bool ENT, bool MASK, bool ONE>
int run_tiles(const void* logits, int64_t row_stride, int64_t R, int V, int nv, int tiles, float c, int top, const int64_t* indices, int K,
              const Parts& parts, const TokenOut& ans, hipStream_t st) {
    const dim3 grid((unsigned)(R * tiles));
    const D* x = static_cast<const D*>(logits);
    if (nv == 4) tile_kernel<D, 4, TOP, ENT, MASK, ONE><<<grid, kThr, 0, st>>>(x, row_stride, V, tiles, c, top, indices, K, parts, ans);
    else if (nv == 2) tile_kernel<D, 2, TOP, ENT, MASK, ONE><<<grid, kThr, 0, st>>>(x, row_stride, V, tiles, c, top, indices, K, parts, ans);
    else tile_kernel<D, 1, TOP, ENT, MASK, ONE><<<grid, kThr, 0, st>>>(x, row_stride, V, tiles, c, top, indices, K, parts, ans);
    GF_LAUNCH_CHECK("tile_kernel");
    return GF_OK;
}

int check_rows(const char* who, int64_t R, int64_t V, int64_t row_stride, int dtype, float temperature) {
    GF_REQUIRE_ARG(gf_dtype_ok(dtype), "%s: dtype %d", who, dtype);
    GF_REQUIRE_SHAPE(R > 0 && V > 0 && row_stride >= 0, "%s: bad shape R=%lld V=%lld row stride %lld", who, (long long)R, (long long)V, (long long)row_stride);
    // (1 / temperature and the exponents' scale stay finite and normal)
    GF_REQUIRE_ARG(temperature >= 1e-30f && temperature <= 1e30f, "%s: temperature %g (1e-30 .. 1e30)", who, (double)temperature);
    GF_REQUIRE_SHAPE(V < (1ll << 31) - (1 << 16), "%s: rows of V=%lld outputs", who, (long long)V);
    return GF_OK;
}

// rows per launch: one workgroup of 256 threads per (row, tile of at least 1024 elements), and a launch's threads are counted in 32 bits
int64_t rows_per_launch(int64_t V) {
    const int64_t n = (1ll << 23) / (V / 1024 + 2);
    return n < 1 ? 1 : n;
}
template <typename F> int in_batches(int64_t R, int64_t V, F&& f) {   // f(first row, rows)
    const int64_t step = rows_per_launch(V);
    for (int64_t r = 0; r < R; r += step) {
        const int rc = f(r, R - r < step ? R - r : step);
        if (rc != GF_OK) return rc;
    }
    return GF_OK;
}
const char* row_at(const void* p, int64_t r, int64_t stride, int dtype) { return static_cast<const char*>(p) + r * stride * (int64_t)gf_dtype_bytes(dtype); }
char* row_at(void* p, int64_t r, int64_t stride, int dtype) { return static_cast<char*>(p) + r * stride * (int64_t)gf_dtype_bytes(dtype); }
template <typename T> T* at(T* p, int64_t i) { return p ? p + i : nullptr; }

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
    const TokenOut a{tokens, ignore, logp, entropy, top_logp, top_tokens, stats};
    if (V <= kPackMax)
        return by_pack(V, [&](auto g) -> int {
            constexpr int G = decltype(g)::value;
            token_pack_kernel<D, G><<<pack_grid(R, G), kThr, 0, st>>>(static_cast<const D*>(logits), row_stride, R, V, c, top, a);
            GF_LAUNCH_CHECK("token_pack_kernel");
            return GF_OK;
        });
    const int nv = pick_nv<D>(R, V), tiles = (int)tiles_of<D>(V, nv);
    const Parts p = make_parts(ws, R, tiles, top);
    if (tiles == 1)
        return top ? run_tiles<D, true, true, false, true>(logits, row_stride, R, V, nv, 1, c, top, nullptr, 0, p, a, st)
                   : run_tiles<D, false, true, false, true>(logits, row_stride, R, V, nv, 1, c, 0, nullptr, 0, p, a, st);
    const int rc = top ? run_tiles<D, true, true, false, false>(logits, row_stride, R, V, nv, tiles, c, top, nullptr, 0, p, a, st)
                       : run_tiles<D, false, true, false, false>(logits, row_stride, R, V, nv, tiles, c, 0, nullptr, 0, p, a, st);
    if (rc != GF_OK) return rc;
    token_finish_kernel<D><<<dim3((unsigned)R), dim3(top ? kThr : 64), 0, st>>>(static_cast<const D*>(logits), row_stride, c, p, tiles, V, top, a);
    GF_LAUNCH_CHECK("token_finish_kernel");
    return GF_OK;
}

template <typename D>
int token_backward_t(const void* logits, int64_t row_stride, const int64_t* tokens, float c, int64_t ignore, const float* stats, const int64_t* top_tokens,
                     int top, const float* dlogp, const float* dentropy, const float* dtop, void* dlogits, int64_t R, int V, hipStream_t st) {
    if (V <= kPackMax)
        return by_pack(V, [&](auto g) -> int {
            constexpr int G = decltype(g)::value;
            token_pack_bwd_kernel<D, G><<<pack_grid(R, G), kThr, 0, st>>>(static_cast<const D*>(logits), row_stride, tokens, c, ignore, stats, top_tokens, top,
                                                                          dlogp, dentropy, dtop, static_cast<D*>(dlogits), R, V);
            GF_LAUNCH_CHECK("token_pack_bwd_kernel");
            return GF_OK;
        });
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
    const bool pack = V <= kPackMax;
    const int nv = pick_nv<D>(R, V), tiles = pack ? 1 : (int)tiles_of<D>(V, nv);
    const Parts p = make_parts(ws, R, tiles, 0);
    const TokenOut none{};
    const int rc = pack ? by_pack(V, [&](auto g) -> int {
                              constexpr int G = decltype(g)::value;
                              distill_pack_kernel<D, G><<<pack_grid(R, G), kThr, 0, st>>>(static_cast<const D*>(logits), row_stride, R, V, c,
                                                                                          tail ? indices : nullptr, K, p);
                              GF_LAUNCH_CHECK("distill_pack_kernel");
                              return GF_OK;
                          })
                   : tail ? run_tiles<D, false, false, true, false>(logits, row_stride, R, V, nv, tiles, c, 0, indices, K, p, none, st)
                        : run_tiles<D, false, false, false, false>(logits, row_stride, R, V, nv, tiles, c, 0, nullptr, 0, p, none, st);
    if (rc != GF_OK) return rc;
    distill_finish_kernel<D><<<dim3((unsigned)((R + 3) / 4)), kThr, 0, st>>>(static_cast<const D*>(logits), row_stride, indices, values, c, tail, p, tiles,
                                                                             R, V, K, loss, stats, probs);
    GF_LAUNCH_CHECK("distill_finish_kernel");
    return GF_OK;
}

template <typename D>
int distill_backward_t(const void* logits, int64_t row_stride, const int64_t* indices, const float* probs, const float* stats, float c,
                       const float* dloss, void* dlogits, int64_t R, int V, int K, hipStream_t st) {
    if (V <= kPackMax)
        return by_pack(V, [&](auto g) -> int {
            constexpr int G = decltype(g)::value;
            distill_pack_bwd_kernel<D, G><<<pack_grid(R, G), kThr, 0, st>>>(static_cast<const D*>(logits), row_stride, indices, probs, stats, c, dloss,
                                                                            static_cast<D*>(dlogits), R, V, K);
            GF_LAUNCH_CHECK("distill_pack_bwd_kernel");
            return GF_OK;
        });
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

// scratch of the largest batch (the last, shorter one may be cut into smaller tiles: never into more than this bound)
static size_t batch_bytes(int64_t R, int64_t V, int top, int dtype) {
    const int64_t step = rows_per_launch(V), full = R < step ? R : step, last = R % step;
    size_t b = parts_bytes(full, tiles_for(full, V, dtype), top);
    if (R > step && last) {
        const size_t c = parts_bytes(last, tiles_for(last, V, dtype), top);
        b = b > c ? b : c;
    }
    return b;
}

extern "C" size_t gf_token_logp_workspace_bytes(int64_t R, int32_t V, int32_t top, int32_t dtype) {
    if (R <= 0 || V <= 0 || top < 0 || !gf_dtype_ok(dtype)) return 0;
    return batch_bytes(R, V, top, dtype);
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
        return in_batches(R, V, [&](int64_t r, int64_t n) {
            return token_forward_t<decltype(d)>(row_at(logits, r, row_stride, dtype), row_stride, tokens + r, 1.f / temperature, ignore_index, logp + r,
                                                at(entropy, r), at(top_logp, r * top), at(top_tokens, r * top), top, at(stats, r * 3), workspace, n, V,
                                                gf_stream(stream));
        });
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
        return in_batches(R, V, [&](int64_t r, int64_t n) {
            return token_backward_t<decltype(d)>(row_at(logits, r, row_stride, dtype), row_stride, tokens + r, 1.f / temperature, ignore_index, stats + r * 3,
                                                 at(top_tokens, r * top), top, at(dlogp, r), at(dentropy, r), at(dtop, r * top),
                                                 row_at(dlogits, r, V, dtype), n, V, gf_stream(stream));
        });
    });
}

extern "C" size_t gf_distill_top_workspace_bytes(int64_t R, int32_t V, int32_t K, int32_t dtype) {
    if (R <= 0 || V <= 0 || K <= 0 || !gf_dtype_ok(dtype)) return 0;
    return batch_bytes(R, V, 0, dtype);
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
        return in_batches(R, V, [&](int64_t r, int64_t n) {
            return distill_forward_t<decltype(d)>(row_at(logits, r, row_stride, dtype), row_stride, indices + r * K, values + r * K, 1.f / temperature, tail,
                                                  loss + r, stats + r * 3, probs + r * K, workspace, n, V, K, gf_stream(stream));
        });
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
        return in_batches(R, V, [&](int64_t r, int64_t n) {
            return distill_backward_t<decltype(d)>(row_at(logits, r, row_stride, dtype), row_stride, indices + r * K, probs + r * K, stats + r * 3,
                                                   1.f / temperature, dloss + r, row_at(dlogits, r, V, dtype), n, V, K, gf_stream(stream));
        });
    });
}
