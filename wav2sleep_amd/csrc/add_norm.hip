// Root-mean-square norm with the residual's addition: r = x + res, y = r rstd w, rstd = 1 / sqrt(mean(r^2) + eps), y in 16 / 32 bits or in e4m3
// with one scale a row.  Three or four elements moved per element and five flops: bound by HBM, so a row is read once and lives in registers
// (G lanes x NV vectors) between the sum of squares and the product; only rows beyond 256 lanes x 8 vectors (4 in the
// backward) are read twice, the second time from L2, by the looped kernel.  Any width, stride and alignment takes the same accesses.  The sum is fp32 and y comes from it before r is rounded.
#include "mix_io.h"

namespace {

// VEC columns from c on of a row of C; behind the row's end zeros / nothing
template <typename T, int VEC> __device__ __forceinline__ void load_cols(const T* row, int c, int C, float* v) {
  if (c + VEC <= C) {
    mix_gload<T, VEC>(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = c + i < C ? (float)row[c + i] : 0.0f;
  }
}
template <typename T, int VEC> __device__ __forceinline__ void store_cols(T* row, int c, int C, const float* v) {
  if (c + VEC <= C) {
    mix_gstore<T, VEC>(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (c + i < C) row[c + i] = (T)v[i];
  }
}

constexpr float kFp8Max = 448.0f;   // largest finite e4m3 value

// sum / maximum over the G lanes of a row: inside a wave by lane exchanges, over a workgroup's four waves through LDS
template <int G, bool MAX> __device__ __forceinline__ float row_reduce(float v, float* red) {
  if constexpr (G <= 64) {
    return MAX ? mix_group_max<G>(v) : mix_group_sum<G>(v);
  } else {
    v = MAX ? mix_group_max<64>(v) : mix_group_sum<64>(v);
    constexpr int W = G / 64;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < W; ++i) v = MAX ? fmaxf(v, red[i]) : v + red[i];
    return v;
  }
}

__device__ __forceinline__ uint8_t fp8_code(float v) { return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xff); }

template <int N> __device__ __forceinline__ void store_fp8(uint8_t* row, int c, int C, const float* v) {   // v within +-448 or NaN
  static_assert(N == 4 || N == 8, "words of four codes");
  if (c + N <= C) {
    typedef uint32_t U __attribute__((ext_vector_type(N / 4)));
    typedef U UU __attribute__((aligned(1)));
    U w;
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const int q = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
      w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], q, true);
    }
    *reinterpret_cast<UU*>(row + c) = w;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i < C) row[c + i] = fp8_code(v[i]);
  }
}

// y / scale into [-448, 448]; a NaN stays one (fmin / fmax would drop it)
__device__ __forceinline__ float to_fp8_range(float y, float scale) {
  const float q = y / scale;
  return q != q ? q : fminf(fmaxf(q, -kFp8Max), kFp8Max);
}

__device__ __forceinline__ float fp8_scale(float top) {   // (never 0: 0 / 0 would make the zeros of such a row NaN)
  return top > 0.0f ? fmaxf(top / kFp8Max, __builtin_bit_cast(float, 1u)) : (top == top ? 1.0f : top);
}

template <typename T, typename RT, bool FP8, int VEC, int G, int NV> __global__ __launch_bounds__(256) void add_norm_fwd_kernel(w2s_add_norm_args a) {
  __shared__ float red[4];
  constexpr int RPB = 256 / G;
  const int lane = threadIdx.x % G, C = a.C;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / G;
  if (G <= 64 && row >= a.rows) return;
  const T* x = (const T*)a.x + row * a.ldx;
  const RT* res = a.res ? (const RT*)a.res + row * a.ldres : nullptr;
  float v[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * G + lane) * VEC;
    load_cols<T, VEC>(x, c, C, v[j]);
  }
  if (res) {
    float q[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * VEC;
      load_cols<RT, VEC>(res, c, C, q[j]);
    }
    RT* r = (RT*)a.r + row * C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * VEC;
      if (c < C) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] += q[j][i];
        store_cols<RT, VEC>(r, c, C, v[j]);
      }
    }
  }
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) s = __builtin_fmaf(v[j][i], v[j][i], s);
  const float rstd = 1.0f / __builtin_sqrtf(row_reduce<G, false>(s, red) / (float)C + a.eps);
  if (a.rstd && lane == 0) a.rstd[row] = rstd;
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * G + lane) * VEC;
    if (c < C) {
      float w[VEC];
      load_cols<float, VEC>(a.w, c, C, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[j][i] *= rstd * w[i];
        if (FP8) top = v[j][i] != v[j][i] || top != top ? __builtin_nanf("") : fmaxf(top, __builtin_fabsf(v[j][i]));
      }
      if (!FP8) store_cols<T, VEC>((T*)a.y + row * C, c, C, v[j]);
    }
  }
  if (FP8) {
    const float bad = top != top ? 1.0f : 0.0f;
    top = row_reduce<G, true>(bad != 0.0f ? 0.0f : top, red);
    if (row_reduce<G, true>(bad, red) != 0.0f) top = __builtin_nanf("");
    const float scale = fp8_scale(top);
    if (lane == 0) a.scale[row] = scale;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * VEC;
      if (c < C) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] = to_fp8_range(v[j][i], scale);
        store_fp8<VEC>((uint8_t*)a.y + row * C, c, C, v[j]);
      }
    }
  }
}

// rows too wide for registers: a workgroup per row, one element a lane, the row's sum formed again in every pass
template <typename T, typename RT, bool FP8> __global__ __launch_bounds__(256) void add_norm_fwd_loop_kernel(w2s_add_norm_args a) {
  __shared__ float red[4];
  const int C = a.C;
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.ldx;
  const RT* res = a.res ? (const RT*)a.res + row * a.ldres : nullptr;
  auto sum_at = [&](int c) { return res ? (float)x[c] + (float)res[c] : (float)x[c]; };
  float s = 0.0f;
  for (int c = threadIdx.x; c < C; c += 256) {
    const float v = sum_at(c);
    s = __builtin_fmaf(v, v, s);
    if (res) ((RT*)a.r)[row * C + c] = (RT)v;
  }
  const float rstd = 1.0f / __builtin_sqrtf(row_reduce<256, false>(s, red) / (float)C + a.eps);
  if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
  if (!FP8) {
    for (int c = threadIdx.x; c < C; c += 256) ((T*)a.y)[row * C + c] = (T)(sum_at(c) * (rstd * a.w[c]));
    return;
  }
  float top = 0.0f, bad = 0.0f;
  for (int c = threadIdx.x; c < C; c += 256) {
    const float v = sum_at(c) * (rstd * a.w[c]);
    if (v != v) bad = 1.0f;
    else top = fmaxf(top, __builtin_fabsf(v));
  }
  top = row_reduce<256, true>(top, red);
  if (row_reduce<256, true>(bad, red) != 0.0f) top = __builtin_nanf("");
  const float scale = fp8_scale(top);
  if (threadIdx.x == 0) a.scale[row] = scale;
  for (int c = threadIdx.x; c < C; c += 256) {
    ((uint8_t*)a.y)[row * C + c] = fp8_code(to_fp8_range(sum_at(c) * (rstd * a.w[c]), scale));
  }
}

// Backward, n = r rstd: gr_total = rstd (gy w - n mean(gy w n)) + gr goes to both addends; gw = sum over rows of gy n.  A workgroup takes rows
// blockIdx, blockIdx + gridDim, ... and keeps its share of gw in registers; the shares are joined in a fixed order.
template <typename T, typename RT, int VEC, int G, int NV> __global__ __launch_bounds__(256) void add_norm_bwd_kernel(w2s_add_norm_args a) {
  __shared__ float red[4];
  __shared__ float acc[G < 256 ? 256 * VEC : 1];
  constexpr int RPB = 256 / G;
  const int lane = threadIdx.x % G, C = a.C;
  float gw[NV][VEC], w[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * G + lane) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) gw[j][i] = w[j][i] = 0.0f;
    load_cols<float, VEC>(a.w, c, C, w[j]);
  }
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + threadIdx.x / G;
    const bool on = row < a.rows;   // (a whole group of lanes; with G = 256 always)
    float n[NV][VEC], g[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) n[j][i] = g[j][i] = 0.0f;
      if (on && c < C) {
        if (a.x) load_cols<T, VEC>((const T*)a.x + row * a.ldx, c, C, n[j]);
        if (a.res) {
          float q[VEC];
          load_cols<RT, VEC>((const RT*)a.res + row * a.ldres, c, C, q);
#pragma unroll
          for (int i = 0; i < VEC; ++i) n[j][i] += q[i];
        }
        if (a.gy) load_cols<T, VEC>((const T*)a.gy + row * a.ldgy, c, C, g[j]);
      }
    }
    const float rstd = on ? a.rstd[row] : 0.0f;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        n[j][i] *= rstd;
        gw[j][i] = __builtin_fmaf(g[j][i], n[j][i], gw[j][i]);
        g[j][i] *= w[j][i];
        s = __builtin_fmaf(g[j][i], n[j][i], s);
      }
    const float m = row_reduce<G, false>(s, red) / (float)C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * VEC;
      if (on && c < C) {
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = 0.0f;
        if (a.gr) load_cols<RT, VEC>((const RT*)a.gr + row * a.ldgr, c, C, o);
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] += rstd * __builtin_fmaf(-n[j][i], m, g[j][i]);
        if (a.gx) store_cols<T, VEC>((T*)a.gx + row * C, c, C, o);
        if (a.gres) store_cols<RT, VEC>((RT*)a.gres + row * C, c, C, o);
      }
    }
  }
  if (!a.gw) return;
  float* part = a.part + (int64_t)blockIdx.x * C;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if constexpr (G == 256) {
      const int c = (j * G + lane) * VEC;
      store_cols<float, VEC>(part, c, C, gw[j]);
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i * 256 + threadIdx.x] = gw[j][i];
      __syncthreads();
      for (int q = threadIdx.x; q < G * VEC; q += 256) {
        const int l = q / VEC, i = q % VEC, c = (j * G + l) * VEC + i;
        if (c < C) {
          float t = 0.0f;
          for (int p = 0; p < RPB; ++p) t += acc[i * 256 + p * G + l];
          part[c] = t;
        }
      }
    }
  }
}

template <typename T, typename RT> __global__ __launch_bounds__(256) void add_norm_bwd_loop_kernel(w2s_add_norm_args a) {
  __shared__ float red[4];
  const int C = a.C;
  float* part = a.gw ? a.part + (int64_t)blockIdx.x * C : nullptr;
  if (part)
    for (int c = threadIdx.x; c < C; c += 256) part[c] = 0.0f;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = a.x ? (const T*)a.x + row * a.ldx : nullptr;
    const RT* res = a.res ? (const RT*)a.res + row * a.ldres : nullptr;
    const T* gy = a.gy ? (const T*)a.gy + row * a.ldgy : nullptr;
    const RT* gr = a.gr ? (const RT*)a.gr + row * a.ldgr : nullptr;
    const float rstd = a.rstd[row];
    auto n_at = [&](int c) { return ((x ? (float)x[c] : 0.0f) + (res ? (float)res[c] : 0.0f)) * rstd; };
    auto g_at = [&](int c) { return gy ? (float)gy[c] : 0.0f; };
    float s = 0.0f;
    for (int c = threadIdx.x; c < C; c += 256) s = __builtin_fmaf(g_at(c) * a.w[c], n_at(c), s);
    const float m = row_reduce<256, false>(s, red) / (float)C;
    for (int c = threadIdx.x; c < C; c += 256) {   // (a column of `part` belongs to one thread)
      const float n = n_at(c), g = g_at(c);
      if (part) part[c] = __builtin_fmaf(g, n, part[c]);
      const float o = (gr ? (float)gr[c] : 0.0f) + rstd * __builtin_fmaf(-n, m, g * a.w[c]);
      if (a.gx) ((T*)a.gx)[row * C + c] = (T)o;
      if (a.gres) ((RT*)a.gres)[row * C + c] = (RT)o;
    }
  }
}

__global__ __launch_bounds__(1024) void add_norm_reduce_kernel(const float* part, int nparts, int C, float* gw) {
  __shared__ float red[64][17];
  const int col = blockIdx.x * 16 + (threadIdx.x & 15);
  const float v = mix_part_sum(part, nparts, C, col, red);
  if (threadIdx.x < 16 && col < C) gw[col] = v;
}

int esize(int dtype) { return dtype == W2S_F32 ? 4 : 2; }

bool valid(const w2s_add_norm_args* a) {
  return a && a->w && a->rows >= 0 && a->rows <= 0x7fffffff && a->C >= 1 && a->C <= (1 << 30) && a->dtype >= 0 && a->dtype <= 2 &&
         (a->rdtype == a->dtype || a->rdtype == W2S_F32);
}

constexpr int64_t kMaxBlocks = 0xffffffffLL / 256;   // a launch has fewer than 2^32 threads

// rows r0 .. r0 + n - 1 of a forward call
w2s_add_norm_args rows_from(const w2s_add_norm_args* a, int64_t r0, int64_t n) {
  w2s_add_norm_args s = *a;
  const int e = esize(a->dtype), er = esize(a->rdtype);
  s.x = (const char*)a->x + r0 * a->ldx * e;
  s.y = (char*)a->y + r0 * a->C * (a->fp8 ? 1 : e);
  if (a->res) {
    s.res = (const char*)a->res + r0 * a->ldres * er;
    s.r = (char*)a->r + r0 * a->C * er;
  }
  if (a->scale) s.scale = a->scale + r0;
  if (a->rstd) s.rstd = a->rstd + r0;
  s.rows = n;
  return s;
}

// workgroups of the backward: enough for 8 waves a SIMD quad on every CU, at most one per row group
int bwd_blocks(const w2s_add_norm_args* a) {
  const int64_t n = a->rows < 1 ? 1 : a->rows;
  return (int)(n < 1024 ? n : 1024);
}

template <typename T, typename RT, int VEC, int G, int NV> int go(const w2s_add_norm_args* a, bool bwd, hipStream_t st) {
  constexpr int RPB = 256 / G;
  if (bwd) {
    if constexpr (NV <= 4) add_norm_bwd_kernel<T, RT, VEC, G, NV><<<bwd_blocks(a), 256, 0, st>>>(*a);
    return W2S_OK;
  }
  for (int64_t r0 = 0; r0 < a->rows; r0 += kMaxBlocks * RPB) {
    const int64_t n = a->rows - r0 < kMaxBlocks * RPB ? a->rows - r0 : kMaxBlocks * RPB;
    const w2s_add_norm_args s = rows_from(a, r0, n);
    const unsigned blocks = (unsigned)((n + RPB - 1) / RPB);
    if (a->fp8) add_norm_fwd_kernel<T, RT, true, VEC, G, NV><<<blocks, 256, 0, st>>>(s);
    else add_norm_fwd_kernel<T, RT, false, VEC, G, NV><<<blocks, 256, 0, st>>>(s);
  }
  return W2S_OK;
}

template <typename T, typename RT> int by_width(const w2s_add_norm_args* a, bool bwd, hipStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const int units = (a->C + V - 1) / V;   // lanes' accesses of 16 bytes (of T) a row
  if (units <= 16) return go<T, RT, V, 16, 1>(a, bwd, st);
  if (units <= 32) return go<T, RT, V, 32, 1>(a, bwd, st);
  if (units <= 64) return go<T, RT, V, 64, 1>(a, bwd, st);
  if (units <= 128) return go<T, RT, V, 64, 2>(a, bwd, st);
  if (units <= 256) return go<T, RT, V, 256, 1>(a, bwd, st);
  if (units <= 512) return go<T, RT, V, 256, 2>(a, bwd, st);
  if (units <= 1024) return go<T, RT, V, 256, 4>(a, bwd, st);
  if (units <= 2048 && !bwd) return go<T, RT, V, 256, 8>(a, bwd, st);   // (the backward keeps four such rows: it would spill)
  if (!bwd && a->rows > kMaxBlocks) return W2S_EINVAL;   // (more than 2^37 elements)
  if (bwd) add_norm_bwd_loop_kernel<T, RT><<<bwd_blocks(a), 256, 0, st>>>(*a);
  else if (a->fp8) add_norm_fwd_loop_kernel<T, RT, true><<<(unsigned)a->rows, 256, 0, st>>>(*a);
  else add_norm_fwd_loop_kernel<T, RT, false><<<(unsigned)a->rows, 256, 0, st>>>(*a);
  return W2S_OK;
}

int dispatch(const w2s_add_norm_args* a, bool bwd, hipStream_t st) {
  const bool wide_r = a->rdtype != a->dtype;
  int rc = W2S_EINVAL;
  switch (a->dtype) {
    case W2S_F32: rc = by_width<float, float>(a, bwd, st); break;
    case W2S_BF16: rc = wide_r ? by_width<bf16_t, float>(a, bwd, st) : by_width<bf16_t, bf16_t>(a, bwd, st); break;
    case W2S_F16: rc = wide_r ? by_width<half_t, float>(a, bwd, st) : by_width<half_t, half_t>(a, bwd, st); break;
  }
  if (rc != W2S_OK) return rc;
  if (bwd && a->gw) add_norm_reduce_kernel<<<(a->C + 15) / 16, 1024, 0, st>>>(a->part, bwd_blocks(a), a->C, a->gw);
  W2S_CHECK_LAUNCH();
  return W2S_OK;
}

}  // namespace

extern "C" int w2s_add_norm_fwd(const w2s_add_norm_args* a, void* stream) {
  if (!valid(a)) return W2S_EINVAL;
  if (a->rows == 0) return W2S_OK;
  if (!a->x || !a->y || (!a->res) != (!a->r) || (a->fp8 && !a->scale)) return W2S_EINVAL;
  return dispatch(a, false, (hipStream_t)stream);
}

extern "C" int64_t w2s_add_norm_part(const w2s_add_norm_args* a) {
  if (!valid(a)) return W2S_EINVAL;
  return (int64_t)bwd_blocks(a) * a->C;
}

extern "C" int w2s_add_norm_bwd(const w2s_add_norm_args* a, void* stream) {
  if (!valid(a) || a->fp8 || (a->gw && !a->part)) return W2S_EINVAL;
  if (a->rows > 0 && ((!a->x && !a->res) || !a->rstd)) return W2S_EINVAL;
  return dispatch(a, true, (hipStream_t)stream);   // no rows: the sums are still written (zeros)
}
