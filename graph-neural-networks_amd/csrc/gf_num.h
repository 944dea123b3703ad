// gf_num.h -- element types of the sequence and output operators (fp32, bf16, fp16): vector loads to fp32, stores with one rounding
// (to nearest even; half a step at most), and small wave helpers.  Sums and states are fp32 everywhere.
#pragma once
#include "gf_common.h"

struct gf_bf16 { uint16_t v; };
struct gf_f16 { _Float16 v; };

template <typename D> __device__ __forceinline__ float gf_to_f(D x);
template <> __device__ __forceinline__ float gf_to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float gf_to_f<gf_bf16>(gf_bf16 x) { return __uint_as_float((unsigned)x.v << 16); }
template <> __device__ __forceinline__ float gf_to_f<gf_f16>(gf_f16 x) { return (float)x.v; }

template <typename D> __device__ __forceinline__ D gf_from_f(float x);
template <> __device__ __forceinline__ float gf_from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ gf_bf16 gf_from_f<gf_bf16>(float x) {
    const __bf16 h = static_cast<__bf16>(x);
    gf_bf16 r;
    __builtin_memcpy(&r, &h, 2);
    return r;
}
template <> __device__ __forceinline__ gf_f16 gf_from_f<gf_f16>(float x) { return gf_f16{(_Float16)x}; }

template <typename D, int V> struct alignas(sizeof(D) * V) gf_vec { D e[V]; };

template <typename D, int V> __device__ __forceinline__ void gf_store(D* __restrict__ p, const float (&v)[V]) {
    gf_vec<D, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.e[i] = gf_from_f<D>(v[i]);
    *reinterpret_cast<gf_vec<D, V>*>(p) = r;
}

static inline size_t gf_dtype_bytes(int dtype) { return dtype == GF_F32 ? 4 : 2; }
static inline bool gf_dtype_ok(int dtype) { return dtype == GF_F32 || dtype == GF_BF16 || dtype == GF_F16; }

// the same at any element's address
template <typename D, int V> struct __attribute__((packed, aligned(sizeof(D)))) gf_vec_any { D e[V]; };
template <typename D, int V> __device__ __forceinline__ void gf_load_any(const D* __restrict__ p, float (&out)[V]) {
    const gf_vec_any<D, V> r = *reinterpret_cast<const gf_vec_any<D, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = gf_to_f<D>(r.e[i]);
}
template <typename D, int V> __device__ __forceinline__ void gf_store_any(D* __restrict__ p, const float (&v)[V]) {
    gf_vec_any<D, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.e[i] = gf_from_f<D>(v[i]);
    *reinterpret_cast<gf_vec_any<D, V>*>(p) = r;
}
