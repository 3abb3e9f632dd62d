// Element types of the state space mixer's operators (short_conv.hip, ssm_scan.hip, add_norm.hip): activations are fp32, bf16 or fp16 in
// memory and fp32 in registers; every rounding to 16 bits happens once, at the store.  CDNA4 only: wave = 64 lanes.
#pragma once
#include <type_traits>
#include "w2s_common.h"

typedef _Float16 half_t;
typedef __bf16 bf16_t;

template <typename T, int N> struct mix_vec { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T> struct mix_vec<T, 1> { typedef T type; };

// N elements as floats; p is aligned to N * sizeof(T) (at most 16 bytes a load)
template <typename T, int N> __device__ __forceinline__ void mix_load(const T* p, float* v) {
  constexpr int E = 16 / (int)sizeof(T);
  if constexpr (N > E) {
    mix_load<T, E>(p, v);
    mix_load<T, N - E>(p + E, v + E);
  } else if constexpr (N == 1) {
    v[0] = (float)*p;
  } else {
    typedef typename mix_vec<T, N>::type V;
    const V r = *reinterpret_cast<const V*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)r[i];
  }
}

template <typename T, int N> __device__ __forceinline__ void mix_store(T* p, const float* v) {
  constexpr int E = 16 / (int)sizeof(T);
  if constexpr (N > E) {
    mix_store<T, E>(p, v);
    mix_store<T, N - E>(p + E, v + E);
  } else if constexpr (N == 1) {
    *p = (T)v[0];
  } else {
    typedef typename mix_vec<T, N>::type V;
    V r;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = (T)v[i];
    *reinterpret_cast<V*>(p) = r;
  }
}

// 1 / (1 + e^-x); e^-x may overflow to inf (-> 0) and a NaN stays one
__device__ __forceinline__ float mix_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x)); }

// softplus(x) = max(x, 0) + log1p(e^-|x|).  With e = e^-|x| <= 1 and s = e / (2 + e) <= 1/3: log1p(e) = 2 atanh(s) = 2 (s + s^3/3 + s^5/5 + ...),
// cut after s^15 / 15 (the next term is below 2^-30 of the sum): relative accuracy for tiny time steps too, where log(1 + e) has none
__device__ __forceinline__ float mix_softplus(float x) {
  const float e = __builtin_amdgcn_exp2f(-1.4426950408889634f * __builtin_fabsf(x));
  const float s = e * __builtin_amdgcn_rcpf(2.0f + e);
  const float q = s * s;
  float p = 1.0f / 15.0f;
  p = __builtin_fmaf(p, q, 1.0f / 13.0f);
  p = __builtin_fmaf(p, q, 1.0f / 11.0f);
  p = __builtin_fmaf(p, q, 1.0f / 9.0f);
  p = __builtin_fmaf(p, q, 1.0f / 7.0f);
  p = __builtin_fmaf(p, q, 1.0f / 5.0f);
  p = __builtin_fmaf(p, q, 1.0f / 3.0f);
  p = __builtin_fmaf(p, q, 1.0f);
  const float t = 2.0f * s * p;
  return x > 0.0f ? x + t : (x == x ? t : x);
}

// sum over the lanes of an aligned group of G lanes (a power of two <= 64); every lane gets it, in one fixed order
template <int G> __device__ __forceinline__ float mix_group_sum(float v) {
#pragma unroll
  for (int m = 1; m < G; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}
template <int G> __device__ __forceinline__ float mix_group_max(float v) {
#pragma unroll
  for (int m = 1; m < G; m <<= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}

__device__ __forceinline__ int mix_length(const int32_t* lengths, int b, int L) {
  if (!lengths) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : (n > L ? L : n);
}

static inline bool mix_aligned(const void* p, int64_t s0, int64_t s1, int vec, int esize) {   // base and both strides allow vec-element accesses
  return ((uintptr_t)p % (size_t)(vec * esize)) == 0 && s0 % vec == 0 && s1 % vec == 0;
}
