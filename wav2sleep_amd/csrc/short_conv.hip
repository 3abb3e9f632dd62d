// Short causal depthwise convolution of a state space mixer: y[t] = act(bias + sum_k w[k] x[t-(K-1)+k]) per channel, K <= 8, channels-last.
// It does 2 K flops per element moved, so it is bound by HBM: every element is read once (plus the K-1 halo rows a run of positions shares
// with the run before it, which hit L2) and written once.  A thread owns 16 bytes of channels and a run of positions whose window slides
// through registers; all its loads are issued before the first multiply.
#include "mix_io.h"

namespace {

constexpr int kRun = 8;   // positions per thread: 8 + K - 1 loads of 16 bytes in flight per lane

struct Shape { int ncg, cx, ty, ncgb, nchb, L, D, runs; };   // runs: how many runs of positions a thread of the backward takes, ty runs apart

// rows r of [state; x] as floats; r counts from the first state row, n = length
template <typename T, int VEC, int K>
__device__ __forceinline__ void full_row(const T* x, int64_t sl, const T* state, int D, int r, int n, float* v) {
  if (r >= K - 1) {
    if (r - (K - 1) < n) { mix_load<T, VEC>(x + (int64_t)(r - (K - 1)) * sl, v); return; }
  } else if (r >= 0 && state) {
    mix_load<T, VEC>(state + (int64_t)r * D, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = 0.0f;
}

template <int VEC, int K> __device__ __forceinline__ void load_weights(const float* w, const float* bias, int d, float (*wk)[VEC], float* bk) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
#pragma unroll
    for (int k = 0; k < K; ++k) wk[k][i] = w[(int64_t)(d + i) * K + k];
    bk[i] = bias ? bias[d + i] : 0.0f;
  }
}

template <typename T, int VEC, int K> __global__ __launch_bounds__(256) void short_conv_fwd_kernel(w2s_short_conv_args a, Shape s) {
  int blk = blockIdx.x;
  const int cgb = blk % s.ncgb;
  blk /= s.ncgb;
  const int chb = blk % s.nchb, b = blk / s.nchb;
  const int cg = cgb * s.cx + (int)threadIdx.x % s.cx, ch = chb * s.ty + (int)threadIdx.x / s.cx;
  const int t0 = ch * kRun;
  if (cg >= s.ncg || (t0 >= s.L && ch > 0)) return;
  const int d = cg * VEC, D = s.D, n = mix_length(a.lengths, b, s.L);
  const T* x = (const T*)a.x + b * a.sx_b + d;
  const T* state = a.state ? (const T*)a.state + (int64_t)b * (K - 1) * D + d : nullptr;
  T* y = (T*)a.y + (int64_t)b * s.L * D + d;
  float win[kRun + K - 1][VEC];
  if (t0 >= K - 1 && t0 + kRun <= n) {
#pragma unroll
    for (int i = 0; i < kRun + K - 1; ++i) mix_load<T, VEC>(x + (int64_t)(t0 - (K - 1) + i) * a.sx_l, win[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kRun + K - 1; ++i) full_row<T, VEC, K>(x, a.sx_l, state, D, t0 + i, n, win[i]);
  }
  float wk[K][VEC], bk[VEC];
  load_weights<VEC, K>(a.w, a.bias, d, wk, bk);
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    const int t = t0 + i;
    if (t >= s.L) break;
    float o[VEC];
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
      float z = bk[c];
#pragma unroll
      for (int k = 0; k < K; ++k) z = __builtin_fmaf(wk[k][c], win[i + k][c], z);
      if (a.act) z *= mix_sigmoid(z);
      o[c] = t < n ? z : 0.0f;
    }
    mix_store<T, VEC>(y + (int64_t)t * D, o);
  }
  if (ch == 0 && a.state_out) {   // the last K-1 rows of [state; x[:n]]
    T* so = (T*)a.state_out + (int64_t)b * (K - 1) * D + d;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      float v[VEC];
      full_row<T, VEC, K>(x, a.sx_l, state, D, n + j, n, v);
      mix_store<T, VEC>(so + (int64_t)j * D, v);
    }
  }
}

// Backward: gz[t] = gy[t] act'(z[t]) is formed again from x for the run and the K-1 positions behind it;
// gx[t] = sum_k w[k] gz[t+K-1-k] (+ the gradient of the final state's rows); gw[k] = sum_t gz[t] x[t-(K-1)+k].
// The sums over positions: in registers along the run, across the workgroup's runs through LDS, across workgroups from `part` in a fixed order.
template <typename T, int VEC, int K> __global__ __launch_bounds__(256) void short_conv_bwd_kernel(w2s_short_conv_args a, Shape s) {
  __shared__ float red[256 * VEC];
  int blk = blockIdx.x;
  const int cgb = blk % s.ncgb;
  blk /= s.ncgb;
  const int chb = blk % s.nchb, b = blk / s.nchb;
  const int cx = (int)threadIdx.x % s.cx, ty = (int)threadIdx.x / s.cx;
  const int cg = cgb * s.cx + cx, D = s.D;
  const int d = cg < s.ncg ? cg * VEC : 0, n = mix_length(a.lengths, b, s.L);
  float gwk[K + 1][VEC];
#pragma unroll
  for (int k = 0; k <= K; ++k)
#pragma unroll
    for (int c = 0; c < VEC; ++c) gwk[k][c] = 0.0f;
  for (int run = 0; run < s.runs; ++run) {
    const int ch = (chb * s.runs + run) * s.ty + ty, t0 = ch * kRun;
    if (cg >= s.ncg || (t0 >= s.L && ch > 0)) break;
    const T* x = (const T*)a.x + b * a.sx_b + d;
    const T* g = a.gy ? (const T*)a.gy + b * a.sg_b + d : nullptr;
    const T* state = a.state ? (const T*)a.state + (int64_t)b * (K - 1) * D + d : nullptr;
    const T* gs = a.gstate ? (const T*)a.gstate + (int64_t)b * (K - 1) * D + d : nullptr;
    constexpr int R = kRun + K - 1;   // positions whose gz this thread needs
    float win[R + K - 1][VEC], gz[R][VEC], wk[K][VEC], bk[VEC];
    if (g && t0 >= K - 1 && t0 + R <= n) {
#pragma unroll
      for (int i = 0; i < R + K - 1; ++i) mix_load<T, VEC>(x + (int64_t)(t0 - (K - 1) + i) * a.sx_l, win[i]);
#pragma unroll
      for (int i = 0; i < R; ++i) mix_load<T, VEC>(g + (int64_t)(t0 + i) * a.sg_l, gz[i]);
    } else {
#pragma unroll
      for (int i = 0; i < R + K - 1; ++i) full_row<T, VEC, K>(x, a.sx_l, state, D, t0 + i, n, win[i]);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (g && t0 + i < n) {
          mix_load<T, VEC>(g + (int64_t)(t0 + i) * a.sg_l, gz[i]);
        } else {
#pragma unroll
          for (int c = 0; c < VEC; ++c) gz[i][c] = 0.0f;
        }
      }
    }
    load_weights<VEC, K>(a.w, a.bias, d, wk, bk);
    if (a.act) {
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (t0 + i < n) {   // (behind the end gz is 0 and z may be anything)
#pragma unroll
          for (int c = 0; c < VEC; ++c) {
            float z = bk[c];
#pragma unroll
            for (int k = 0; k < K; ++k) z = __builtin_fmaf(wk[k][c], win[i + k][c], z);
            const float sg = mix_sigmoid(z);
            gz[i][c] *= sg * (1.0f + z * (1.0f - sg));
          }
        }
    }
    T* gx = (T*)a.gx + (int64_t)b * s.L * D + d;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int t = t0 + i;
      if (t >= s.L) break;
      float o[VEC];
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) v = __builtin_fmaf(wk[k][c], gz[i + K - 1 - k][c], v);
        o[c] = v;
      }
      const int j = t + K - 1 - n;   // row of the final state that x[t] is
      if (gs && t < n && j >= 0) {
        float v[VEC];
        mix_load<T, VEC>(gs + (int64_t)j * D, v);
#pragma unroll
        for (int c = 0; c < VEC; ++c) o[c] += v[c];
      }
      if (t >= n) {
#pragma unroll
        for (int c = 0; c < VEC; ++c) o[c] = 0.0f;
      }
      mix_store<T, VEC>(gx + (int64_t)t * D, o);
    }
    if (ch == 0 && a.gstate_in) {
      T* gi = (T*)a.gstate_in + (int64_t)b * (K - 1) * D + d;
#pragma unroll
      for (int r = 0; r < K - 1; ++r) {   // state row r meets position t through tap k = r - t
        float o[VEC];
#pragma unroll
        for (int c = 0; c < VEC; ++c) o[c] = 0.0f;
#pragma unroll
        for (int t = 0; t <= r; ++t)
#pragma unroll
          for (int c = 0; c < VEC; ++c) o[c] = __builtin_fmaf(wk[r - t][c], gz[t][c], o[c]);
        if (gs && r >= n) {   // a sequence shorter than K-1: the old rows are in the new state
          float v[VEC];
          mix_load<T, VEC>(gs + (int64_t)(r - n) * D, v);
#pragma unroll
          for (int c = 0; c < VEC; ++c) o[c] += v[c];
        }
        mix_store<T, VEC>(gi + (int64_t)r * D, o);
      }
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i)   // gz is 0 behind the end
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
#pragma unroll
        for (int k = 0; k < K; ++k) gwk[k][c] = __builtin_fmaf(gz[i][c], win[i + k][c], gwk[k][c]);
        gwk[K][c] += gz[i][c];
      }
  }
  if (!a.part) return;
  float* part = a.part + ((int64_t)b * s.nchb + chb) * (K + 1) * D;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < VEC; ++c) red[c * 256 + threadIdx.x] = gwk[k][c];
    __syncthreads();
    for (int i = threadIdx.x; i < s.cx * VEC; i += 256) {
      const int lane = i / VEC, c = i % VEC, dd = (cgb * s.cx + lane) * VEC + c;
      if (cgb * s.cx + lane < s.ncg) {
        float v = 0.0f;
        for (int q = 0; q < s.ty; ++q) v += red[c * 256 + q * s.cx + lane];
        part[(int64_t)k * D + dd] = v;
      }
    }
  }
}

// gw[d][k] / gbias[d] = sum over workgroups of part[p][k][d]
__global__ __launch_bounds__(1024) void short_conv_reduce_kernel(const float* part, int nparts, int K, int D, float* gw, float* gbias) {
  __shared__ float red[64][17];
  const int64_t C = (int64_t)(K + 1) * D, col = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
  const float v = mix_part_sum(part, nparts, C, col, red);
  if (threadIdx.x < 16 && col < C) {
    const int k = (int)(col / D), d = (int)(col % D);
    if (k < K) {
      if (gw) gw[(int64_t)d * K + k] = v;
    } else if (gbias) {
      gbias[d] = v;
    }
  }
}

template <typename T, int VEC, int K> __global__ __launch_bounds__(256) void short_conv_step_kernel(w2s_short_conv_args a, int ncg) {
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (item >= (int64_t)a.B * ncg) return;
  const int b = (int)(item / ncg), d = (int)(item % ncg) * VEC, D = a.D;
  float win[K][VEC], wk[K][VEC], bk[VEC];
  mix_load<T, VEC>((const T*)a.x + b * a.sx_b + d, win[K - 1]);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) mix_load<T, VEC>((const T*)a.state + ((int64_t)b * (K - 1) + k) * D + d, win[k]);
  load_weights<VEC, K>(a.w, a.bias, d, wk, bk);
  float o[VEC];
#pragma unroll
  for (int c = 0; c < VEC; ++c) {
    float z = bk[c];
#pragma unroll
    for (int k = 0; k < K; ++k) z = __builtin_fmaf(wk[k][c], win[k][c], z);
    o[c] = a.act ? z * mix_sigmoid(z) : z;
  }
  mix_store<T, VEC>((T*)a.y + (int64_t)b * D + d, o);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) mix_store<T, VEC>((T*)a.state_out + ((int64_t)b * (K - 1) + k) * D + d, win[k + 1]);   // all loads are done: in place is fine
}

Shape shape_of(const w2s_short_conv_args* a, int vec, bool backward) {
  Shape s;
  s.L = a->L;
  s.D = a->D;
  s.ncg = a->D / vec;
  s.cx = 1;
  while (s.cx < 64 && s.cx < s.ncg) s.cx *= 2;
  s.ty = 256 / s.cx;
  s.ncgb = (s.ncg + s.cx - 1) / s.cx;
  const int nch = a->L > 0 ? (a->L + kRun - 1) / kRun : 1;   // (an empty sequence still hands its state on)
  s.nchb = (nch + s.ty - 1) / s.ty;
  s.runs = 1;
  // the sums that a workgroup of the backward leaves are K + 1 floats a channel: with more workgroups than fill the chip (8 a CU) it takes several runs
  while (backward && (int64_t)a->B * s.nchb * s.ncgb > 2048 && s.nchb > 1 && s.runs < 16) {
    s.runs *= 2;
    s.nchb = (s.nchb + 1) / 2;
  }
  return s;
}

int esize(int dtype) { return dtype == W2S_F32 ? 4 : 2; }

bool valid(const w2s_short_conv_args* a) {
  return a && a->w && a->B >= 0 && a->L >= 0 && a->D >= 1 && a->K >= 1 && a->K <= 8 && a->dtype >= 0 && a->dtype <= 2 && (a->act == 0 || a->act == 1);
}

// elements a lane: 16 bytes where every pointer, row and width allows them, one element otherwise.  The backward keeps two windows in
// registers: four elements of either size there (eight would need more registers than a lane has)
int vector_of(const w2s_short_conv_args* a, bool backward) {
  const int e = esize(a->dtype), v = backward ? 4 : 16 / e;
  if (a->D % v) return 1;
  const void* ps[] = {a->x, a->state, a->y, a->state_out, a->gy, a->gstate, a->gx, a->gstate_in};
  for (const void* p : ps)
    if ((uintptr_t)p % (size_t)(v * e)) return 1;
  if (a->sx_b % v || a->sx_l % v || a->sg_b % v || a->sg_l % v) return 1;
  return v;
}

enum { kFwd, kBwd, kStep };

template <typename T, int VEC, int K, bool BWD> int launch(const w2s_short_conv_args* a, int what, hipStream_t st) {
  if constexpr (BWD) {
    const Shape s = shape_of(a, VEC, true);
    const int64_t blocks = (int64_t)a->B * s.nchb * s.ncgb;
    if (blocks > 0x7fffffff) return W2S_EINVAL;
    short_conv_bwd_kernel<T, VEC, K><<<(unsigned)blocks, 256, 0, st>>>(*a, s);
    if (a->part) {
      const int64_t C = (int64_t)(K + 1) * a->D;
      short_conv_reduce_kernel<<<(unsigned)((C + 15) / 16), 1024, 0, st>>>(a->part, a->B * s.nchb, K, a->D, a->gw, a->gbias);
    }
  } else if (what == kStep) {
    const int ncg = a->D / VEC;
    const int64_t blocks = ((int64_t)a->B * ncg + 255) / 256;
    if (blocks > 0x7fffffff) return W2S_EINVAL;
    short_conv_step_kernel<T, VEC, K><<<(unsigned)blocks, 256, 0, st>>>(*a, ncg);
  } else {
    const Shape s = shape_of(a, VEC, false);
    const int64_t blocks = (int64_t)a->B * s.nchb * s.ncgb;
    if (blocks > 0x7fffffff) return W2S_EINVAL;
    short_conv_fwd_kernel<T, VEC, K><<<(unsigned)blocks, 256, 0, st>>>(*a, s);
  }
  W2S_CHECK_LAUNCH();
  return W2S_OK;
}

template <typename T, int VEC, bool BWD> int by_taps(const w2s_short_conv_args* a, int what, hipStream_t st) {
  switch (a->K) {
    case 1: return launch<T, VEC, 1, BWD>(a, what, st);
    case 2: return launch<T, VEC, 2, BWD>(a, what, st);
    case 3: return launch<T, VEC, 3, BWD>(a, what, st);
    case 4: return launch<T, VEC, 4, BWD>(a, what, st);
    case 5: return launch<T, VEC, 5, BWD>(a, what, st);
    case 6: return launch<T, VEC, 6, BWD>(a, what, st);
    case 7: return launch<T, VEC, 7, BWD>(a, what, st);
    case 8: return launch<T, VEC, 8, BWD>(a, what, st);
  }
  return W2S_EINVAL;
}

int dispatch(const w2s_short_conv_args* a, int what, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  const bool bwd = what == kBwd, wide = vector_of(a, bwd) > 1;
  switch (a->dtype) {
    case W2S_F32:
      if (bwd) return wide ? by_taps<float, 4, true>(a, what, st) : by_taps<float, 1, true>(a, what, st);
      return wide ? by_taps<float, 4, false>(a, what, st) : by_taps<float, 1, false>(a, what, st);
    case W2S_BF16:
      if (bwd) return wide ? by_taps<bf16_t, 4, true>(a, what, st) : by_taps<bf16_t, 1, true>(a, what, st);
      return wide ? by_taps<bf16_t, 8, false>(a, what, st) : by_taps<bf16_t, 1, false>(a, what, st);
    case W2S_F16:
      if (bwd) return wide ? by_taps<half_t, 4, true>(a, what, st) : by_taps<half_t, 1, true>(a, what, st);
      return wide ? by_taps<half_t, 8, false>(a, what, st) : by_taps<half_t, 1, false>(a, what, st);
  }
  return W2S_EINVAL;
}

}  // namespace

extern "C" int w2s_short_conv_fwd(const w2s_short_conv_args* a, void* stream) {
  if (!valid(a) || (a->L > 0 && a->B > 0 && (!a->x || !a->y))) return W2S_EINVAL;
  if (a->B == 0 || (a->L == 0 && !a->state_out)) return W2S_OK;
  return dispatch(a, kFwd, stream);
}

extern "C" int64_t w2s_short_conv_part(const w2s_short_conv_args* a) {
  if (!valid(a)) return W2S_EINVAL;
  const Shape s = shape_of(a, vector_of(a, true), true);
  return (int64_t)a->B * s.nchb * (a->K + 1) * a->D;
}

extern "C" int w2s_short_conv_bwd(const w2s_short_conv_args* a, void* stream) {
  if (!valid(a) || (a->L > 0 && a->B > 0 && (!a->x || !a->gx)) || ((a->gw || a->gbias) && !a->part && a->B > 0)) return W2S_EINVAL;
  if (a->B == 0) return (a->gw || a->gbias) ? W2S_EINVAL : W2S_OK;   // nothing would write the sums
  return dispatch(a, kBwd, stream);
}

extern "C" int w2s_short_conv_step(const w2s_short_conv_args* a, void* stream) {
  if (!valid(a)) return W2S_EINVAL;
  if (a->B == 0) return W2S_OK;
  if (!a->x || !a->y || (a->K > 1 && (!a->state || !a->state_out))) return W2S_EINVAL;
  return dispatch(a, kStep, stream);
}
