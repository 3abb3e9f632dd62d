// Short causal depthwise convolution of a state space mixer: y[t] = act(bias + sum_k w[k] x[t-(K-1)+k]) per channel, K <= 8, channels-last.
// It does 2 K flops per element moved, so it is bound by HBM: every element is read once (plus the K-1 halo rows a run of positions shares
// with the run before it, which hit L2) and written once.  A thread owns four channels and runs of
// positions whose window slides through registers; a run's loads are issued before its first multiply.
// Measured, K = 4: 16 x 960 x 256 fp32 (31.6 MB) 8 us = 4.0 TB/s; 8 x 2047 x 1536 bf16 forward 21 us (100 MB, 4.8 TB/s), backward 35 + 4 us (150 MB, 3.9 TB/s).
#include "mix_io.h"

namespace {

constexpr int kRun = 4;   // positions of a run: 4 (8 measured 25 % slower backward -- its two windows take the registers of half the waves)

struct Shape { int ncg, cx, ty, ncgb, nchb, L, D, runs; };   // runs: how many runs of positions a thread takes, one behind the other

// rows r of [state; x] as floats; r counts from the first state row, n = length
template <typename T, int VEC, int K>
__device__ __forceinline__ void full_row(const T* x, int64_t sl, const T* state, int D, int r, int n, float* v) {
  if (r >= K - 1) {
    if (r - (K - 1) < n) { mix_gload<T, VEC>(x + (int64_t)(r - (K - 1)) * sl, v); return; }
  } else if (r >= 0 && state) {
    mix_gload<T, VEC>(state + (int64_t)r * D, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = 0.0f;
}

// A workgroup's weights through LDS: K consecutive floats a channel in memory are one 128-byte line a lane, which as a vector load costs a wave 64 cache
// lines an instruction; staged [tap][channel] they are read once, coalesced, by the workgroup.  (The step has one position to spend them on: load_weights.)
template <int VEC, int K> struct Weights {
  float w[K][64 * VEC + 4], b[64 * VEC + 4];
  __device__ __forceinline__ void stage(const float* gw, const float* gb, int c0, int nc) {   // channels c0 .. c0 + nc - 1 of the tensor's D
    for (int i = threadIdx.x; i < nc * K; i += 256) w[i % K][i / K] = gw[(int64_t)c0 * K + i];
    for (int i = threadIdx.x; i < nc; i += 256) b[i] = gb ? gb[c0 + i] : 0.0f;
    __syncthreads();
  }
  __device__ __forceinline__ void get(int c, bool whole, float (*wk)[VEC], float* bk) const {   // c: the thread's first channel, from c0; whole: a multiple of VEC
    if (whole) {
#pragma unroll
      for (int k = 0; k < K; ++k) mix_load<float, VEC>(&w[k][c], wk[k]);
      mix_load<float, VEC>(&b[c], bk);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k) wk[k][i] = w[k][c + i];
        bk[i] = b[c + i];
      }
    }
  }
};

// first channel of group cg: the last group of a width that is no multiple of VEC moves back and shares channels with the one before it (both compute and
// write the same values)
template <int VEC> __device__ __forceinline__ int channel_of(int cg, int D) { return cg * VEC + VEC <= D ? cg * VEC : D - VEC; }

template <int VEC, int K> __device__ __forceinline__ void load_weights(const float* w, const float* bias, int d, float (*wk)[VEC], float* bk) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
#pragma unroll
    for (int k = 0; k < K; ++k) wk[k][i] = w[(int64_t)(d + i) * K + k];
    bk[i] = bias ? bias[d + i] : 0.0f;
  }
}

// rows r0 .. r0 + M - 1 of [state; x]
template <typename T, int VEC, int K, int M> __device__ __forceinline__ void rows_of(const T* x, int64_t sl, const T* state, int D, int r0, int n, float (*v)[VEC]) {
  if (r0 >= K - 1 && r0 - (K - 1) + M <= n) {
    const T* p = x + (int64_t)(r0 - (K - 1)) * sl;
#pragma unroll
    for (int i = 0; i < M; ++i) mix_gload<T, VEC>(p + i * sl, v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < M; ++i) full_row<T, VEC, K>(x, sl, state, D, r0 + i, n, v[i]);
  }
}

template <typename T, int VEC, int K> __global__ __launch_bounds__(256) void short_conv_fwd_kernel(w2s_short_conv_args a, Shape s) {
  __shared__ Weights<VEC, K> ws;
  int blk = blockIdx.x;
  const int cgb = blk % s.ncgb;
  blk /= s.ncgb;
  const int chb = blk % s.nchb, b = blk / s.nchb, D = s.D, cx = (int)threadIdx.x % s.cx;
  const int c0 = channel_of<VEC>(cgb * s.cx, D), nc = D - c0 < s.cx * VEC ? D - c0 : s.cx * VEC;
  ws.stage(a.w, a.bias, c0, nc);
  const int cg = cgb * s.cx + cx, ch = (chb * s.ty + (int)threadIdx.x / s.cx) * s.runs;   // first run of the thread's
  const int n = mix_length(a.lengths, b, s.L);
  if (cg >= s.ncg || (ch * kRun >= s.L && ch > 0)) return;
  const int d = channel_of<VEC>(cg, D);
  const T* x = (const T*)a.x + b * a.sx_b + d;
  const T* state = a.state ? (const T*)a.state + (int64_t)b * (K - 1) * D + d : nullptr;
  T* y = (T*)a.y + (int64_t)b * s.L * D + d;
  float wk[K][VEC], bk[VEC], win[kRun + K - 1][VEC];
  ws.get(d - c0, D % VEC == 0, wk, bk);
  rows_of<T, VEC, K, K - 1>(x, a.sx_l, state, D, ch * kRun, n, win);
  for (int run = 0; run < s.runs && (ch + run) * kRun < s.L; ++run) {
    const int t0 = (ch + run) * kRun;
    rows_of<T, VEC, K, kRun>(x, a.sx_l, state, D, t0 + K - 1, n, win + (K - 1));
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
      mix_gstore<T, VEC>(y + (int64_t)t * D, o);
    }
#pragma unroll
    for (int i = 0; i < K - 1; ++i)
#pragma unroll
      for (int c = 0; c < VEC; ++c) win[i][c] = win[kRun + i][c];
  }
  if (ch == 0 && a.state_out) {   // the last K-1 rows of [state; x[:n]]
    T* so = (T*)a.state_out + (int64_t)b * (K - 1) * D + d;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      float v[VEC];
      full_row<T, VEC, K>(x, a.sx_l, state, D, n + j, n, v);
      mix_gstore<T, VEC>(so + (int64_t)j * D, v);
    }
  }
}

// Backward: gz[t] = gy[t] act'(z[t]) is formed again from x for the run and the K-1 positions behind it;
// gx[t] = sum_k w[k] gz[t+K-1-k] (+ the gradient of the final state's rows); gw[k] = sum_t gz[t] x[t-(K-1)+k].
// A thread takes `runs` runs one behind the other; the K-1 gz and the 2 (K-1) rows that the next one shares stay in registers.
// The sums over positions: in registers along the runs, across the workgroup through LDS, across workgroups from `part`, in a fixed order.
template <typename T, int VEC, int K> __global__ __launch_bounds__(256) void short_conv_bwd_kernel(w2s_short_conv_args a, Shape s) {
  __shared__ union { Weights<VEC, K> ws; float red[256 * VEC]; } sh;
  int blk = blockIdx.x;
  const int cgb = blk % s.ncgb;
  blk /= s.ncgb;
  const int chb = blk % s.nchb, b = blk / s.nchb, D = s.D, cx = (int)threadIdx.x % s.cx, ty = (int)threadIdx.x / s.cx;
  const int c0 = channel_of<VEC>(cgb * s.cx, D), nc = D - c0 < s.cx * VEC ? D - c0 : s.cx * VEC;
  sh.ws.stage(a.w, a.bias, c0, nc);
  const int cg = cgb * s.cx + cx, ch = (chb * s.ty + ty) * s.runs, n = mix_length(a.lengths, b, s.L);
  float gwk[K + 1][VEC];
#pragma unroll
  for (int k = 0; k <= K; ++k)
#pragma unroll
    for (int c = 0; c < VEC; ++c) gwk[k][c] = 0.0f;
  if (cg < s.ncg && (ch * kRun < s.L || ch == 0)) {
    const int d = channel_of<VEC>(cg, D);
    const T* x = (const T*)a.x + b * a.sx_b + d;
    const T* g = a.gy ? (const T*)a.gy + b * a.sg_b + d : nullptr;
    const T* state = a.state ? (const T*)a.state + (int64_t)b * (K - 1) * D + d : nullptr;
    const T* gs = a.gstate ? (const T*)a.gstate + (int64_t)b * (K - 1) * D + d : nullptr;
    T* gx = (T*)a.gx + (int64_t)b * s.L * D + d;
    float win[kRun + 2 * (K - 1)][VEC], gz[kRun + K - 1][VEC], wk[K][VEC], bk[VEC];
    sh.ws.get(d - c0, D % VEC == 0, wk, bk);
    // gz of position t from its window (rows t .. t + K - 1 of [state; x]); 0 behind the end, where z may be anything
    auto slope = [&](float* v, const float (*row)[VEC], int t) {
      if (!a.act || t >= n) return;
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        float z = bk[c];
#pragma unroll
        for (int k = 0; k < K; ++k) z = __builtin_fmaf(wk[k][c], row[k][c], z);
        const float sg = mix_sigmoid(z);
        v[c] *= sg * (1.0f + z * (1.0f - sg));
      }
    };
    auto load_g = [&](float* v, int t) {
      if (g && t < n) {
        mix_gload<T, VEC>(g + (int64_t)t * a.sg_l, v);
      } else {
#pragma unroll
        for (int c = 0; c < VEC; ++c) v[c] = 0.0f;
      }
    };
    rows_of<T, VEC, K, 2 * (K - 1)>(x, a.sx_l, state, D, ch * kRun, n, win);
#pragma unroll
    for (int i = 0; i < K - 1; ++i) {
      load_g(gz[i], ch * kRun + i);
      slope(gz[i], win + i, ch * kRun + i);
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
          mix_gload<T, VEC>(gs + (int64_t)(r - n) * D, v);
#pragma unroll
          for (int c = 0; c < VEC; ++c) o[c] += v[c];
        }
        mix_gstore<T, VEC>(gi + (int64_t)r * D, o);
      }
    }
    for (int run = 0; run < s.runs && (ch + run) * kRun < s.L; ++run) {
      const int t0 = (ch + run) * kRun;
      rows_of<T, VEC, K, kRun>(x, a.sx_l, state, D, t0 + 2 * (K - 1), n, win + 2 * (K - 1));
      if (g && t0 + K - 1 + kRun <= n) {
        const T* p = g + (int64_t)(t0 + K - 1) * a.sg_l;
#pragma unroll
        for (int i = 0; i < kRun; ++i) mix_gload<T, VEC>(p + i * a.sg_l, gz[K - 1 + i]);
      } else {
#pragma unroll
        for (int i = 0; i < kRun; ++i) load_g(gz[K - 1 + i], t0 + K - 1 + i);
      }
#pragma unroll
      for (int i = 0; i < kRun; ++i) slope(gz[K - 1 + i], win + K - 1 + i, t0 + K - 1 + i);
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
          mix_gload<T, VEC>(gs + (int64_t)j * D, v);
#pragma unroll
          for (int c = 0; c < VEC; ++c) o[c] += v[c];
        }
        if (t >= n) {
#pragma unroll
          for (int c = 0; c < VEC; ++c) o[c] = 0.0f;
        }
        mix_gstore<T, VEC>(gx + (int64_t)t * D, o);
      }
#pragma unroll
      for (int i = 0; i < kRun; ++i)   // gz is 0 behind the end
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
#pragma unroll
          for (int k = 0; k < K; ++k) gwk[k][c] = __builtin_fmaf(gz[i][c], win[i + k][c], gwk[k][c]);
          gwk[K][c] += gz[i][c];
        }
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
#pragma unroll
        for (int i = 0; i < 2 * (K - 1); ++i) win[i][c] = win[kRun + i][c];
#pragma unroll
        for (int i = 0; i < K - 1; ++i) gz[i][c] = gz[kRun + i][c];
      }
    }
  }
  if (!a.part) return;
  float* part = a.part + ((int64_t)b * s.nchb + chb) * (K + 1) * D;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < VEC; ++c) sh.red[c * 256 + threadIdx.x] = gwk[k][c];
    __syncthreads();
    for (int i = threadIdx.x; i < s.cx * VEC; i += 256) {
      const int lane = i / VEC, c = i % VEC, dd = channel_of<VEC>(cgb * s.cx + lane, D) + c;
      if (cgb * s.cx + lane < s.ncg) {
        float v = 0.0f;
        for (int q = 0; q < s.ty; ++q) v += sh.red[c * 256 + q * s.cx + lane];
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
  mix_gload<T, VEC>((const T*)a.x + b * a.sx_b + d, win[K - 1]);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) mix_gload<T, VEC>((const T*)a.state + ((int64_t)b * (K - 1) + k) * D + d, win[k]);
  load_weights<VEC, K>(a.w, a.bias, d, wk, bk);
  float o[VEC];
#pragma unroll
  for (int c = 0; c < VEC; ++c) {
    float z = bk[c];
#pragma unroll
    for (int k = 0; k < K; ++k) z = __builtin_fmaf(wk[k][c], win[k][c], z);
    o[c] = a.act ? z * mix_sigmoid(z) : z;
  }
  mix_gstore<T, VEC>((T*)a.y + (int64_t)b * D + d, o);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) mix_gstore<T, VEC>((T*)a.state_out + ((int64_t)b * (K - 1) + k) * D + d, win[k + 1]);   // all loads are done: in place is fine
}

Shape shape_of(const w2s_short_conv_args* a, int vec, bool backward) {
  Shape s;
  s.L = a->L;
  s.D = a->D;
  s.ncg = (a->D + vec - 1) / vec;
  s.cx = 1;
  while (s.cx < 64 && s.cx < s.ncg) s.cx *= 2;
  s.ty = 256 / s.cx;
  s.ncgb = (s.ncg + s.cx - 1) / s.cx;
  const int nch = a->L > 0 ? (a->L + kRun - 1) / kRun : 1;   // (an empty sequence still hands its state on)
  // Runs a thread: the more, the fewer rows are read twice and the fewer sums a workgroup of the backward leaves (K + 1 floats a channel) -- as long as
  // eight (backward: four) workgroups a CU remain.  8 x 2047 x 1536 bf16 forward: 21 us; with twice as many workgroups 25, with half as many 23.
  s.runs = 1;
  auto blocks = [&](int runs) { return (int64_t)a->B * s.ncgb * ((nch + s.ty * runs - 1) / (s.ty * runs)); };
  while (s.runs < 16 && blocks(s.runs) > (backward ? 1024 : 2048)) s.runs *= 2;
  s.nchb = (nch + s.ty * s.runs - 1) / (s.ty * s.runs);
  return s;
}

constexpr int64_t kMaxBlocks = 0xffffffffLL / 256;   // a launch has fewer than 2^32 threads

bool valid(const w2s_short_conv_args* a) {
  return a && a->w && a->B >= 0 && a->L >= 0 && a->L <= (1 << 30) && a->D >= 1 && a->D <= (1 << 30) && a->K >= 1 && a->K <= 8 && a->dtype >= 0 && a->dtype <= 2 && (a->act == 0 || a->act == 1);
}

// elements a thread: four wherever there are four (8 x 2047 x 1535 bf16 forward 23.5 us against 31.7 one by one, 1536: 21 against 25).  Eight 16-bit elements, a
// full 16-byte access, measured 19 % slower forward: twice the window in registers, half the waves; in the backward they do not fit.  The step may write
// where it reads, so its threads share no channels: one each for other widths.
int vector_of(const w2s_short_conv_args* a, bool step) { return (step ? a->D % 4 == 0 : a->D >= 4) ? 4 : 1; }

enum { kFwd, kBwd, kStep };

template <typename T, int VEC, int K, bool BWD> int launch(const w2s_short_conv_args* a, int what, hipStream_t st) {
  if constexpr (BWD) {
    const Shape s = shape_of(a, VEC, true);
    const int64_t blocks = (int64_t)a->B * s.nchb * s.ncgb;
    if (blocks > kMaxBlocks) return W2S_EINVAL;
    short_conv_bwd_kernel<T, VEC, K><<<(unsigned)blocks, 256, 0, st>>>(*a, s);
    if (a->part) {
      const int64_t C = (int64_t)(K + 1) * a->D;
      short_conv_reduce_kernel<<<(unsigned)((C + 15) / 16), 1024, 0, st>>>(a->part, a->B * s.nchb, K, a->D, a->gw, a->gbias);
    }
  } else if (what == kStep) {
    const int ncg = a->D / VEC;
    const int64_t blocks = ((int64_t)a->B * ncg + 255) / 256;
    if (blocks > kMaxBlocks) return W2S_EINVAL;
    short_conv_step_kernel<T, VEC, K><<<(unsigned)blocks, 256, 0, st>>>(*a, ncg);
  } else {
    const Shape s = shape_of(a, VEC, false);
    const int64_t blocks = (int64_t)a->B * s.nchb * s.ncgb;
    if (blocks > kMaxBlocks) return W2S_EINVAL;
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
  const bool bwd = what == kBwd, wide = vector_of(a, what == kStep) > 1;
  switch (a->dtype) {
    case W2S_F32:
      if (bwd) return wide ? by_taps<float, 4, true>(a, what, st) : by_taps<float, 1, true>(a, what, st);
      return wide ? by_taps<float, 4, false>(a, what, st) : by_taps<float, 1, false>(a, what, st);
    case W2S_BF16:
      if (bwd) return wide ? by_taps<bf16_t, 4, true>(a, what, st) : by_taps<bf16_t, 1, true>(a, what, st);
      return wide ? by_taps<bf16_t, 4, false>(a, what, st) : by_taps<bf16_t, 1, false>(a, what, st);
    case W2S_F16:
      if (bwd) return wide ? by_taps<half_t, 4, true>(a, what, st) : by_taps<half_t, 1, true>(a, what, st);
      return wide ? by_taps<half_t, 4, false>(a, what, st) : by_taps<half_t, 1, false>(a, what, st);
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
  const Shape s = shape_of(a, vector_of(a, false), true);
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
