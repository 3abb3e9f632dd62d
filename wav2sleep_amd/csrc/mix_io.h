// Element types of the state space mixer's operators (short_conv.hip, ssm_scan.hip, add_norm.hip): activations are fp32, bf16 or fp16 in
// memory and fp32 in registers; every rounding to 16 bits happens once, at the store.  CDNA4 only: wave = 64 lanes.
#pragma once
#include <type_traits>
#include "w2s_common.h"

typedef _Float16 half_t;
typedef __bf16 bf16_t;

template <typename T, int N> struct mix_vec { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T> struct mix_vec<T, 1> { typedef T type; };

// N elements as floats.  mix_load / mix_store: p is aligned to N * sizeof(T) (LDS, the library's own scratch memory).  mix_gload / mix_gstore: global memory at
// any element -- gfx950 takes wide global accesses at any address, so rows of odd width, slices of wider rows and offset pointers are read as wide as others.
template <typename T, int N, size_t ALIGN> __device__ __forceinline__ void mix_load_at(const T* p, float* v) {
  constexpr int E = 16 / (int)sizeof(T);
  if constexpr (N > E) {
    mix_load_at<T, E, ALIGN>(p, v);
    mix_load_at<T, N - E, ALIGN>(p + E, v + E);
  } else if constexpr (N == 1) {
    v[0] = (float)*p;
  } else {
    typedef typename mix_vec<T, N>::type V;
    typedef V U __attribute__((aligned(ALIGN ? ALIGN : N * sizeof(T))));
    const V r = *reinterpret_cast<const U*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)r[i];
  }
}
template <typename T, int N, size_t ALIGN> __device__ __forceinline__ void mix_store_at(T* p, const float* v) {
  constexpr int E = 16 / (int)sizeof(T);
  if constexpr (N > E) {
    mix_store_at<T, E, ALIGN>(p, v);
    mix_store_at<T, N - E, ALIGN>(p + E, v + E);
  } else if constexpr (N == 1) {
    *p = (T)v[0];
  } else {
    typedef typename mix_vec<T, N>::type V;
    typedef V U __attribute__((aligned(ALIGN ? ALIGN : N * sizeof(T))));
    V r;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = (T)v[i];
    *reinterpret_cast<U*>(p) = r;
  }
}
template <typename T, int N> __device__ __forceinline__ void mix_load(const T* p, float* v) { mix_load_at<T, N, 0>(p, v); }
template <typename T, int N> __device__ __forceinline__ void mix_store(T* p, const float* v) { mix_store_at<T, N, 0>(p, v); }
template <typename T, int N> __device__ __forceinline__ void mix_gload(const T* p, float* v) { mix_load_at<T, N, sizeof(T)>(p, v); }
template <typename T, int N> __device__ __forceinline__ void mix_gstore(T* p, const float* v) { mix_store_at<T, N, sizeof(T)>(p, v); }

// 1 / (1 + e^-x); e^-x may overflow to inf (-> 0) and a NaN stays one
__device__ __forceinline__ float mix_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x)); }

// softplus(x) = max(x, 0) + log1p(e) with e = e^-|x| <= 1, and its slope sigmoid(x) = (x > 0 ? 1 : e) / (1 + e).  log1p(e): w = 1 + e rounds e's low bits
// away; c = e - (w - 1) is what was lost, exactly, and log(1 + e) = log(w) + c / w up to c^2.  For w in [1, 2] c / w and c differ by at most |c| e, half a
// step of e, so the sum has full relative accuracy for tiny time steps too, where log(1 + e) alone has none.
__device__ __forceinline__ float mix_softplus(float x, float& slope) {
  const float e = __builtin_amdgcn_exp2f(-1.4426950408889634f * __builtin_fabsf(x));
  const float w = 1.0f + e, c = e - (w - 1.0f), r = __builtin_amdgcn_rcpf(w);
  slope = x > 0.0f ? r : e * r;
  return fmaxf(x, 0.0f) + __builtin_fmaf(__builtin_amdgcn_logf(w), 0.6931471805599453f, c);   // (a NaN comes through c)
}
__device__ __forceinline__ float mix_softplus(float x) {
  float slope;
  return mix_softplus(x, slope);
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

// sum over `nparts` rows of part[row][C] at column col of the workgroup's 16 (1024 threads = 64 strided row sums x 16 columns, then a tree: a fixed order);
// valid in the 16 threads of row 0
__device__ __forceinline__ float mix_part_sum(const float* part, int nparts, int64_t C, int64_t col, float (*red)[17]) {
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  float v = 0.0f;
  if (col < C) {
#pragma unroll 4
    for (int p = r; p < nparts; p += 64) v += part[(int64_t)p * C + col];
  }
  red[r][c] = v;
#pragma unroll
  for (int h = 32; h; h >>= 1) {
    __syncthreads();
    if (r < h) red[r][c] = v += red[r + h][c];
  }
  return v;
}
