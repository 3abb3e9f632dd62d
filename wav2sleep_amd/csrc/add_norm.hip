// Root-mean-square norm with the residual's addition: r = x + res, y = r rstd w, rstd = 1 / sqrt(mean(r^2) + eps), y in 16 / 32 bits or in e4m3
// with one scale a row.  Three or four elements moved per element and five flops: bound by HBM, so a row is read once and lives in registers
// (G lanes x NV units of 16 bytes) between the sum of squares and the product.  Only rows beyond 4096 units (the backward: 2048), i.e. 32768 (16384) 16-bit or
// 16384 (8192) fp32 columns, are read again for every pass, from L2, by the looped kernels, one element a lane: 67 M elements forward 350 us against 112 in bf16,
// 365 against 203 in fp32, in 8 bits 497 against 122; backward, which also adds its share of gw in global memory row by row, 2.4 ms against 0.11 in bf16 (16385
// columns, 16384) and 1.2 ms against 0.16 in fp32 (8193, 8192).
// Sums and statistics are fp32 and y comes from the sum before r is rounded.
// Measured (bf16, 67 M elements, bytes over time): forward 5.7 TB/s at 4096 columns, 5.5 at 8192; backward 4.9 at 2048, 5.9 at 8192.
#include "mix_io.h"

namespace {

// A row's columns in units of VEC.  Unit u nominally has the columns c = u VEC - shift, ...; with `shift` (the row's first element, counted from address 0, modulo
// VEC) units lie on multiples of their size in memory, which a row of odd width would otherwise take all of its accesses off.  Units that reach over an end
// of the row move inside and share columns with their neighbours: both compute and write the same values, and only one counts in the row's sum.
template <int VEC> struct Unit {
  int c, at;   // nominal first column (behind the row: at >= C), first column in memory
  bool on;
  __device__ __forceinline__ Unit(int u, int shift, int C) : c(u * VEC - shift), on(c < C) {
    const int last = C > VEC ? C - VEC : 0;
    at = c < 0 ? 0 : c < last ? c : last;
  }
  __device__ __forceinline__ bool counts(int i) const { return (unsigned)(at - c + i) < (unsigned)VEC; }
};
// (in the memory's type: a conversion here would wait for the load)
template <typename T, int VEC> struct Cols {
  typedef T V __attribute__((ext_vector_type(VEC)));
  typedef V U __attribute__((aligned(sizeof(T))));
  V v;
  __device__ __forceinline__ void load(const T* row, const Unit<VEC>& u, int C) {
    v = (T)0.0f;
    if (!u.on) return;
    if (C >= VEC) {
      v = *reinterpret_cast<const U*>(row + u.at);
    } else {
#pragma unroll
      for (int i = 0; i < VEC - 1; ++i)
        if (i < C) v[i] = row[i];
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return (float)v[i]; }
};
template <typename T, int VEC> __device__ __forceinline__ void store_cols(T* row, const Unit<VEC>& u, int C, const float* v) {
  if (!u.on) return;
  if (C >= VEC) {
    mix_gstore<T, VEC>(row + u.at, v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC - 1; ++i)
      if (i < C) row[i] = (T)v[i];
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

template <int N> __device__ __forceinline__ void store_fp8(uint8_t* row, const Unit<N>& u, int C, const float* v) {   // v within +-448 or NaN
  static_assert(N == 4 || N == 8, "words of four codes");
  if (!u.on) return;
  if (C >= N) {
    typedef uint32_t W __attribute__((ext_vector_type(N / 4)));
    typedef W UW __attribute__((aligned(1)));
    W w;
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const int q = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
      w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], q, true);
    }
    *reinterpret_cast<UW*>(row + u.at) = w;
  } else {
#pragma unroll
    for (int i = 0; i < N - 1; ++i)
      if (i < C) row[i] = fp8_code(v[i]);
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

template <typename T, typename RT, bool FP8, int VEC, int G, int NV> __global__ __launch_bounds__(G < 256 ? 256 : G) void add_norm_fwd_kernel(w2s_add_norm_args a, int align) {
  __shared__ float red[G < 256 ? 4 : G / 64];
  constexpr int RPB = G < 256 ? 256 / G : 1;
  const int lane = threadIdx.x % G, C = a.C;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / G;
  if (G <= 64 && row >= a.rows) return;
  const T* x = (const T*)a.x + row * a.ldx;
  const RT* res = a.res ? (const RT*)a.res + row * a.ldres : nullptr;
  const int shift = (int)((uint64_t)x / sizeof(T)) & align;
  auto unit = [&](int j) { return Unit<VEC>(j * G + lane, shift, C); };
  float v[NV][VEC];
  Cols<T, VEC> xs[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) xs[j].load(x, unit(j), C);
  if (!res) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = xs[j][i];
  } else {
    Cols<RT, VEC> q[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) q[j].load(res, unit(j), C);
    RT* r = (RT*)a.r + row * C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = xs[j][i] + q[j][i];
      store_cols<RT, VEC>(r, unit(j), C, v[j]);
    }
  }
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const Unit<VEC> u = unit(j);
#pragma unroll
    for (int i = 0; i < VEC; ++i) s = u.counts(i) ? __builtin_fmaf(v[j][i], v[j][i], s) : s;
  }
  const float rstd = 1.0f / __builtin_sqrtf(row_reduce<G, false>(s, red) / (float)C + a.eps);
  if (a.rstd && lane == 0) a.rstd[row] = rstd;
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const Unit<VEC> u = unit(j);
    Cols<float, VEC> w;
    w.load(a.w, u, C);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[j][i] *= rstd * w[i];
      if (FP8 && u.on) top = v[j][i] != v[j][i] || top != top ? __builtin_nanf("") : fmaxf(top, __builtin_fabsf(v[j][i]));
    }
    if (!FP8) store_cols<T, VEC>((T*)a.y + row * C, u, C, v[j]);
  }
  if (FP8) {
    const float bad = top != top ? 1.0f : 0.0f;
    top = row_reduce<G, true>(bad != 0.0f ? 0.0f : top, red);
    if (row_reduce<G, true>(bad, red) != 0.0f) top = __builtin_nanf("");
    const float scale = fp8_scale(top);
    if (lane == 0) a.scale[row] = scale;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = to_fp8_range(v[j][i], scale);
      store_fp8<VEC>((uint8_t*)a.y + row * C, unit(j), C, v[j]);
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
template <typename T, typename RT, int VEC, int G, int NV> __global__ __launch_bounds__(G < 256 ? 256 : G) void add_norm_bwd_kernel(w2s_add_norm_args a, int align) {
  __shared__ float red[G < 256 ? 4 : G / 64];
  __shared__ float acc[G < 256 ? 256 * VEC : 1];
  constexpr int RPB = G < 256 ? 256 / G : 1;
  const int lane = threadIdx.x % G, C = a.C;
  // (the same for all rows of a workgroup, which lie a multiple of VEC apart, so that a thread's columns stay its own)
  const int shift = (int)(a.x ? (uint64_t)a.x / sizeof(T) + blockIdx.x * a.ldx : (uint64_t)a.res / sizeof(RT) + blockIdx.x * a.ldres) & align;
  auto unit = [&](int j) {   // formed again at every use: held for a loop over rows, it and its addresses take registers that the rows need
    int l = lane;
    asm volatile("" : "+v"(l));
    return Unit<VEC>(j * G + l, shift, C);
  };
  float gw[NV][VEC];
  Cols<float, VEC> w[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    w[j].load(a.w, unit(j), C);
#pragma unroll
    for (int i = 0; i < VEC; ++i) gw[j][i] = 0.0f;
  }
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = r0 + threadIdx.x / G;
    const bool on = row < a.rows;   // (a whole group of lanes; from G = 256 on always)
    float n[NV][VEC], g[NV][VEC];
    Cols<T, VEC> x[NV], gy[NV];
    Cols<RT, VEC> res[NV], gr[NV];
    // (gx may be gr's memory: every load of a row, also of a column that two units share, is in front of the row's sum and so of the stores)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Unit<VEC> u = unit(j);
      x[j].v = gy[j].v = (T)0.0f;
      res[j].v = gr[j].v = (RT)0.0f;
      if (on) {
        if (a.x) x[j].load((const T*)a.x + row * a.ldx, u, C);
        if (a.res) res[j].load((const RT*)a.res + row * a.ldres, u, C);
        if (a.gy) gy[j].load((const T*)a.gy + row * a.ldgy, u, C);
        if (a.gr) gr[j].load((const RT*)a.gr + row * a.ldgr, u, C);
      }
    }
    const float rstd = on ? a.rstd[row] : 0.0f;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Unit<VEC> u = unit(j);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        n[j][i] = (x[j][i] + res[j][i]) * rstd;
        gw[j][i] = __builtin_fmaf(gy[j][i], n[j][i], gw[j][i]);
        g[j][i] = gy[j][i] * w[j][i];
        s = u.counts(i) ? __builtin_fmaf(g[j][i], n[j][i], s) : s;
      }
    }
    const float m = row_reduce<G, false>(s, red) / (float)C;
    if (!on) continue;   // (no barrier follows: a workgroup of such groups has waves of their own)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Unit<VEC> u = unit(j);
      float o[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = gr[j][i] + rstd * __builtin_fmaf(-n[j][i], m, g[j][i]);
      if (a.gx) store_cols<T, VEC>((T*)a.gx + row * C, u, C, o);
      if (a.gres) store_cols<RT, VEC>((RT*)a.gres + row * C, u, C, o);
    }
  }
  if (!a.gw) return;
  float* part = a.part + (int64_t)blockIdx.x * C;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if constexpr (G >= 256) {
      store_cols<float, VEC>(part, unit(j), C, gw[j]);
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i * 256 + threadIdx.x] = gw[j][i];
      __syncthreads();
      for (int q = threadIdx.x; q < G * VEC; q += 256) {
        const int l = q / VEC, i = q % VEC;
        const Unit<VEC> u(j * G + l, shift, C);
        if (u.on && u.at + i < C) {
          float t = 0.0f;
          for (int p = 0; p < RPB; ++p) t += acc[i * 256 + p * G + l];
          part[u.at + i] = t;
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

// Rows that start off a multiple of 16 bytes have their units moved there (VEC - 1 as a mask; 0: left where they are): 16001 columns of bf16 forward 108 us
// against 131, backward 121 against 169.  Not where the one unit more would take a row to more lanes than it fills, and not where groups of lanes share a
// workgroup of the backward: they have rows that start differently, and their sum for gw wants one layout.
struct Rule { int units, align; };
Rule rule_of(const w2s_add_norm_args* a, bool bwd) {
  const int V = 16 / esize(a->dtype), plain = (a->C + V - 1) / V, moved = (a->C + 2 * V - 2) / V;
  const int64_t at = a->x ? (int64_t)((uintptr_t)a->x / esize(a->dtype)) : (int64_t)((uintptr_t)a->res / esize(a->rdtype)), ld = a->x ? a->ldx : a->ldres;
  bool more = (at % V || ld % V) && a->C >= V;
  for (int n = 16; n <= 4096 && more; n *= 2) more = !(plain <= n && moved > n);
  if (bwd && plain <= 128) more = false;
  return {more ? moved : plain, more ? V - 1 : 0};
}

// workgroups of the backward: as many as run at once (more leave more shares of gw to join: 2048 for 1024 measured 4 us slower), at most one a row (a narrow row's
// workgroup has up to 16 side by side, so of a few hundred of those most are idle and leave zeros as their shares); a multiple of VEC where a workgroup takes
// one row behind the other
int bwd_blocks(const w2s_add_norm_args* a) {
  const int64_t n = a->rows < 1 ? 1 : a->rows, units = rule_of(a, true).units, top = units <= 512 ? 1024 : 256;
  return (int)(n < top ? n : top);
}

template <typename T, typename RT, int VEC, int G, int NV> int back(const w2s_add_norm_args* a, hipStream_t st) {
  add_norm_bwd_kernel<T, RT, VEC, G, NV><<<bwd_blocks(a), G < 256 ? 256 : G, 0, st>>>(*a, rule_of(a, true).align);
  return W2S_OK;
}

template <typename T, typename RT, int VEC, int G, int NV> int fwd(const w2s_add_norm_args* a, hipStream_t st) {
  constexpr int BLOCK = G < 256 ? 256 : G, RPB = BLOCK / G;
  constexpr int64_t most = 0xffffffffLL / BLOCK * RPB;   // rows a launch, which has fewer than 2^32 threads
  for (int64_t r0 = 0; r0 < a->rows; r0 += most) {
    const int64_t n = a->rows - r0 < most ? a->rows - r0 : most;
    const w2s_add_norm_args s = rows_from(a, r0, n);
    const int align = rule_of(a, false).align;
    const unsigned blocks = (unsigned)((n + RPB - 1) / RPB);
    if (a->fp8) add_norm_fwd_kernel<T, RT, true, VEC, G, NV><<<blocks, BLOCK, 0, st>>>(s, align);
    else add_norm_fwd_kernel<T, RT, false, VEC, G, NV><<<blocks, BLOCK, 0, st>>>(s, align);
  }
  return W2S_OK;
}
template <typename T, typename RT, int VEC, int G, int NV> int go(const w2s_add_norm_args* a, bool bwd, hipStream_t st) {
  return bwd ? back<T, RT, VEC, G, NV>(a, st) : fwd<T, RT, VEC, G, NV>(a, st);
}

// Lanes and units a lane.  Up to 64 lanes a row needs no barrier; from there on as few units a lane as the workgroup allows in the backward, whose registers hold
// four tensors of a row beside the sums of gw: 8192 bf16 columns 108 us with 1024 lanes x 1, 203 with 256 x 4; 4096 columns 122 with 256 x 2, 153 with 512 x 1.
// Forward 8192 columns take 97 us either way and in 8 bits 95 with 256 x 4, 118 with 1024 x 1; 8192 fp32 columns 97 with 1024 x 2, 106 with 256 x 8.
template <typename T, typename RT> int by_width(const w2s_add_norm_args* a, bool bwd, hipStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const int units = rule_of(a, bwd).units;
  if (units <= 16) return go<T, RT, V, 16, 1>(a, bwd, st);
  if (units <= 32) return go<T, RT, V, 32, 1>(a, bwd, st);
  if (units <= 64) return go<T, RT, V, 64, 1>(a, bwd, st);
  if (units <= 128) return go<T, RT, V, 64, 2>(a, bwd, st);
  if (units <= 256) return go<T, RT, V, 256, 1>(a, bwd, st);
  if (units <= 512) return go<T, RT, V, 256, 2>(a, bwd, st);
  if (units <= 1024) return bwd ? back<T, RT, V, 1024, 1>(a, st) : fwd<T, RT, V, 256, 4>(a, st);
  if (units <= 2048) return go<T, RT, V, 1024, 2>(a, bwd, st);
  if (units <= 4096 && !bwd) return fwd<T, RT, V, 1024, 4>(a, st);
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
