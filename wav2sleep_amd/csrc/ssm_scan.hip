// Selective state space scan: delta = softplus(dt + bias), h_t[n] = exp(delta A[n]) h_{t-1}[n] + delta u B_t[n], y_t = (sum_n C_t[n] h_t[n] + D u) silu(z),
// its backward and its form for one position.  A lane owns a channel and walks the sequence with the channel's states in registers.
#include "mix_io.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct Tiles { int ntile, dg; };   // 64-channel tiles of a group, channels of a group

__device__ __forceinline__ void tile_of(const w2s_ssm_args& a, const Tiles& s, int& b, int& g, int& tile, int& d, bool& on) {
  int blk = blockIdx.x;
  tile = blk % s.ntile;
  blk /= s.ntile;
  g = blk % a.G;
  b = blk / a.G;
  const int c = tile * 64 + (int)threadIdx.x;
  on = c < s.dg;
  d = g * s.dg + (on ? c : s.dg - 1);
}

template <typename T, int NP> __global__ __launch_bounds__(64) void ssm_fwd_kernel(w2s_ssm_args a, Tiles s) {
  int b, g, tile, d;
  bool on;
  tile_of(a, s, b, g, tile, d, on);
  const int n = mix_length(a.lengths, b, a.L), N = a.N;
  float A[NP], h[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    A[j] = j < N ? a.A[(int64_t)d * N + j] * kLog2e : 0.0f;
    h[j] = j < N && a.h0 ? a.h0[((int64_t)b * a.D + d) * N + j] : 0.0f;
  }
  const float bias = a.dt_bias ? a.dt_bias[d] : 0.0f, Dp = a.Dp ? a.Dp[d] : 0.0f;
  for (int t = 0; t < n; ++t) {
    const float u = (float)((const T*)a.u)[b * a.su_b + t * a.su_l + d];
    float delta = (float)((const T*)a.dt)[b * a.sdt_b + t * a.sdt_l + d] + bias;
    if (a.softplus) delta = mix_softplus(delta);
    const T* Bt = (const T*)a.Bm + b * a.sB_b + t * a.sB_l + g * a.sB_g;
    const T* Ct = (const T*)a.Cm + b * a.sC_b + t * a.sC_l + g * a.sC_g;
    const float du = delta * u;
    float y = 0.0f;
#pragma unroll
    for (int j = 0; j < NP; ++j)
      if (j < N) {
        h[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(delta * A[j]), h[j], du * (float)Bt[j]);
        y = __builtin_fmaf((float)Ct[j], h[j], y);
      }
    y = __builtin_fmaf(Dp, u, y);
    if (a.z) {
      const float z = (float)((const T*)a.z)[b * a.sz_b + t * a.sz_l + d];
      y *= z * mix_sigmoid(z);
    }
    if (on) ((T*)a.y)[((int64_t)b * a.L + t) * a.D + d] = (T)y;
  }
  if (!on) return;
  for (int t = n; t < a.L; ++t) ((T*)a.y)[((int64_t)b * a.L + t) * a.D + d] = (T)0.0f;
  if (a.h_out)
#pragma unroll
    for (int j = 0; j < NP; ++j)
      if (j < N) a.h_out[((int64_t)b * a.D + d) * N + j] = h[j];
}

// backward: the states of the whole sequence are formed again into `hs` [B][L][N][D], then the sequence is walked from its end
template <typename T, int NP> __global__ __launch_bounds__(64) void ssm_bwd_kernel(w2s_ssm_args a, Tiles s, float* hs, float* part_bc, float* part_a) {
  int b, g, tile, d;
  bool on;
  tile_of(a, s, b, g, tile, d, on);
  const int n = mix_length(a.lengths, b, a.L), N = a.N;
  float A[NP], h[NP], e[NP], gA[NP], gD = 0.0f, gbias = 0.0f;
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    A[j] = j < N ? a.A[(int64_t)d * N + j] * kLog2e : 0.0f;
    h[j] = j < N && a.h0 ? a.h0[((int64_t)b * a.D + d) * N + j] : 0.0f;
    e[j] = j < N && a.gh ? a.gh[((int64_t)b * a.D + d) * N + j] : 0.0f;
    gA[j] = 0.0f;
  }
  const float bias = a.dt_bias ? a.dt_bias[d] : 0.0f, Dp = a.Dp ? a.Dp[d] : 0.0f;
  for (int t = 0; t < n; ++t) {
    const float u = (float)((const T*)a.u)[b * a.su_b + t * a.su_l + d];
    float delta = (float)((const T*)a.dt)[b * a.sdt_b + t * a.sdt_l + d] + bias;
    if (a.softplus) delta = mix_softplus(delta);
    const T* Bt = (const T*)a.Bm + b * a.sB_b + t * a.sB_l + g * a.sB_g;
#pragma unroll
    for (int j = 0; j < NP; ++j)
      if (j < N) {
        h[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(delta * A[j]), h[j], delta * u * (float)Bt[j]);
        if (on) hs[(((int64_t)b * a.L + t) * N + j) * a.D + d] = h[j];
      }
  }
  for (int t = n - 1; t >= 0; --t) {
    const int64_t at = ((int64_t)b * a.L + t) * a.D + d;
    const float u = (float)((const T*)a.u)[b * a.su_b + t * a.su_l + d];
    const float raw = (float)((const T*)a.dt)[b * a.sdt_b + t * a.sdt_l + d] + bias;
    const float delta = a.softplus ? mix_softplus(raw) : raw;
    const T* Bt = (const T*)a.Bm + b * a.sB_b + t * a.sB_l + g * a.sB_g;
    const T* Ct = (const T*)a.Cm + b * a.sC_b + t * a.sC_l + g * a.sC_g;
    const float gy = a.gy ? (float)((const T*)a.gy)[b * a.sg_b + t * a.sg_l + d] : 0.0f;
    float gp = gy, z = 0.0f, sz = 0.0f;
    if (a.z) {
      z = (float)((const T*)a.z)[b * a.sz_b + t * a.sz_l + d];
      sz = mix_sigmoid(z);
      gp *= z * sz;
    }
    float y = Dp * u, sB = 0.0f, gdelta = 0.0f;
#pragma unroll
    for (int j = 0; j < NP; ++j)
      if (j < N) {
        const float Bj = (float)Bt[j], Cj = (float)Ct[j];
        const float ht = hs[(((int64_t)b * a.L + t) * N + j) * a.D + d];
        const float hp = t > 0 ? hs[(((int64_t)b * a.L + t - 1) * N + j) * a.D + d] : (a.h0 ? a.h0[((int64_t)b * a.D + d) * N + j] : 0.0f);
        const float G = __builtin_fmaf(Cj, gp, e[j]);
        e[j] = __builtin_amdgcn_exp2f(delta * A[j]) * G;
        const float eh = e[j] * hp;
        gA[j] = __builtin_fmaf(eh, delta, gA[j]);
        gdelta = __builtin_fmaf(eh, A[j], gdelta);
        sB = __builtin_fmaf(G, Bj, sB);
        y = __builtin_fmaf(Cj, ht, y);
        const float pb = mix_group_sum<64>(on ? G * delta * u : 0.0f), pc = mix_group_sum<64>(on ? gp * ht : 0.0f);
        if (threadIdx.x == 0) {
          float* p = part_bc + ((((int64_t)tile * a.B + b) * a.L + t) * a.G + g) * 2 * N;
          p[j] = pb;
          p[N + j] = pc;
        }
      }
    gdelta = __builtin_fmaf(u, sB, gdelta / kLog2e);
    const float graw = a.softplus ? gdelta * mix_sigmoid(raw) : gdelta;
    gD = __builtin_fmaf(gp, u, gD);
    gbias += graw;
    if (on) {
      ((T*)a.gu)[at] = (T)__builtin_fmaf(delta, sB, Dp * gp);
      ((T*)a.gdt)[at] = (T)graw;
      if (a.z) ((T*)a.gz)[at] = (T)(gy * y * sz * (1.0f + z * (1.0f - sz)));
    }
  }
  if (!on) return;
  for (int t = n; t < a.L; ++t) {
    const int64_t at = ((int64_t)b * a.L + t) * a.D + d;
    ((T*)a.gu)[at] = (T)0.0f;
    ((T*)a.gdt)[at] = (T)0.0f;
    if (a.z) ((T*)a.gz)[at] = (T)0.0f;
  }
  float* pa = part_a + ((int64_t)b * a.D + d) * (N + 2);
#pragma unroll
  for (int j = 0; j < NP; ++j)
    if (j < N) {
      pa[j] = gA[j];
      if (a.gh0) a.gh0[((int64_t)b * a.D + d) * N + j] = e[j];
    }
  pa[N] = gD;
  pa[N + 1] = gbias;
}

// gB / gC [B][L][G][N] = sum over the group's channel tiles, in order; 0 behind the end
template <typename T> __global__ __launch_bounds__(256) void ssm_reduce_bc_kernel(w2s_ssm_args a, int ntile, const float* part) {
  const int64_t per = (int64_t)a.B * a.L * a.G * 2 * a.N, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= per) return;
  const int n = (int)(i % (2 * a.N));
  const int64_t row = i / (2 * a.N);   // (b, t, g)
  const int64_t bt = row / a.G;
  float v = 0.0f;
  if (bt % a.L < mix_length(a.lengths, (int)(bt / a.L), a.L))
    for (int k = 0; k < ntile; ++k) v += part[k * per + i];
  (n < a.N ? (T*)a.gB : (T*)a.gC)[row * a.N + (n < a.N ? n : n - a.N)] = (T)v;
}

__global__ __launch_bounds__(256) void ssm_reduce_a_kernel(w2s_ssm_args a, int nparts, const float* part) {
  const int64_t per = (int64_t)a.D * (a.N + 2), i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= per) return;
  float v = 0.0f;
  for (int p = 0; p < nparts; ++p) v += part[p * per + i];
  const int n = (int)(i % (a.N + 2));
  const int64_t d = i / (a.N + 2);
  if (n < a.N) a.gA[d * a.N + n] = v;
  else if (n == a.N) { if (a.gD) a.gD[d] = v; }
  else if (a.gbias) a.gbias[d] = v;
}

// One position.  Four lanes share a channel: with VEC = 4 they read its states as consecutive 16-byte pieces.
template <typename T, int VEC> __global__ __launch_bounds__(256) void ssm_step_kernel(w2s_ssm_args a) {
  const int64_t item = (int64_t)blockIdx.x * 64 + (threadIdx.x >> 2);
  const int q = threadIdx.x & 3, N = a.N;
  if (item >= (int64_t)a.B * a.D) return;   // (the four lanes of a channel leave together)
  const int b = (int)(item / a.D), d = (int)(item % a.D), g = d / (a.D / a.G);
  const float u = (float)((const T*)a.u)[b * a.su_b + d];
  float delta = (float)((const T*)a.dt)[b * a.sdt_b + d] + (a.dt_bias ? a.dt_bias[d] : 0.0f);
  if (a.softplus) delta = mix_softplus(delta);
  const float du = delta * u, dl = delta * kLog2e;
  const T* Bt = (const T*)a.Bm + b * a.sB_b + g * a.sB_g;
  const T* Ct = (const T*)a.Cm + b * a.sC_b + g * a.sC_g;
  float y = 0.0f;
  for (int j = q * VEC; j < N; j += 4 * VEC) {
    float h[VEC], A[VEC], Bv[VEC], Cv[VEC];
    if (a.h0) {
      mix_load<float, VEC>(a.h0 + item * N + j, h);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = 0.0f;
    }
    mix_load<float, VEC>(a.A + (int64_t)d * N + j, A);
    mix_load<T, VEC>(Bt + j, Bv);
    mix_load<T, VEC>(Ct + j, Cv);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      h[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(dl * A[i]), h[i], du * Bv[i]);
      y = __builtin_fmaf(Cv[i], h[i], y);
    }
    mix_store<float, VEC>(a.h_out + item * N + j, h);
  }
  y = mix_group_sum<4>(y);
  if (q != 0) return;
  if (a.Dp) y = __builtin_fmaf(a.Dp[d], u, y);
  if (a.z) {
    const float z = (float)((const T*)a.z)[b * a.sz_b + d];
    y *= z * mix_sigmoid(z);
  }
  ((T*)a.y)[item] = (T)y;
}

int esize(int dtype) { return dtype == W2S_F32 ? 4 : 2; }

bool valid(const w2s_ssm_args* a) {
  return a && a->A && a->B >= 0 && a->L >= 0 && a->D >= 1 && a->N >= 1 && a->N <= 64 && a->G >= 1 && a->D % a->G == 0 && a->dtype >= 0 && a->dtype <= 2;
}

Tiles tiles_of(const w2s_ssm_args* a) { return {(a->D / a->G + 63) / 64, a->D / a->G}; }

template <typename T> int scan_fwd(const w2s_ssm_args* a, hipStream_t st) {
  const Tiles s = tiles_of(a);
  const int64_t blocks = (int64_t)a->B * a->G * s.ntile;
  if (blocks > 0x7fffffff) return W2S_EINVAL;
  if (a->N <= 16) ssm_fwd_kernel<T, 16><<<(unsigned)blocks, 64, 0, st>>>(*a, s);
  else ssm_fwd_kernel<T, 64><<<(unsigned)blocks, 64, 0, st>>>(*a, s);
  W2S_CHECK_LAUNCH();
  return W2S_OK;
}

int64_t floats_hs(const w2s_ssm_args* a) { return (int64_t)a->B * a->L * a->D * a->N; }
int64_t floats_bc(const w2s_ssm_args* a) { return (int64_t)tiles_of(a).ntile * a->B * a->L * a->G * 2 * a->N; }
int64_t floats_a(const w2s_ssm_args* a) { return (int64_t)a->B * a->D * (a->N + 2); }

template <typename T> int scan_bwd(const w2s_ssm_args* a, hipStream_t st) {
  const Tiles s = tiles_of(a);
  const int64_t blocks = (int64_t)a->B * a->G * s.ntile;
  if (blocks > 0x7fffffff) return W2S_EINVAL;
  float* hs = (float*)a->ws;
  float* pbc = hs + floats_hs(a);
  float* pa = pbc + floats_bc(a);
  if (blocks) {
    if (a->N <= 16) ssm_bwd_kernel<T, 16><<<(unsigned)blocks, 64, 0, st>>>(*a, s, hs, pbc, pa);
    else ssm_bwd_kernel<T, 64><<<(unsigned)blocks, 64, 0, st>>>(*a, s, hs, pbc, pa);
  }
  const int64_t nbc = (int64_t)a->B * a->L * a->G * 2 * a->N, na = (int64_t)a->D * (a->N + 2);
  if ((nbc + 255) / 256 > 0x7fffffff) return W2S_EINVAL;
  if (nbc) ssm_reduce_bc_kernel<T><<<(unsigned)((nbc + 255) / 256), 256, 0, st>>>(*a, s.ntile, pbc);
  ssm_reduce_a_kernel<<<(unsigned)((na + 255) / 256), 256, 0, st>>>(*a, a->B, pa);
  W2S_CHECK_LAUNCH();
  return W2S_OK;
}

template <typename T> int step(const w2s_ssm_args* a, hipStream_t st) {
  const int64_t blocks = ((int64_t)a->B * a->D + 63) / 64;
  if (blocks > 0x7fffffff) return W2S_EINVAL;
  const int bytes = 4 * (int)sizeof(T);   // four states of B and C
  const bool wide = a->N % 4 == 0 && mix_aligned(a->h0, 0, 0, 4, 4) && mix_aligned(a->h_out, 0, 0, 4, 4) && mix_aligned(a->A, 0, 0, 4, 4) &&
                    mix_aligned(a->Bm, a->sB_b, a->sB_g, 4, bytes / 4) && mix_aligned(a->Cm, a->sC_b, a->sC_g, 4, bytes / 4);
  if (wide) ssm_step_kernel<T, 4><<<(unsigned)blocks, 256, 0, st>>>(*a);
  else ssm_step_kernel<T, 1><<<(unsigned)blocks, 256, 0, st>>>(*a);
  W2S_CHECK_LAUNCH();
  return W2S_OK;
}

}  // namespace

extern "C" int64_t w2s_ssm_ckpt(const w2s_ssm_args* a) { return valid(a) ? 0 : W2S_EINVAL; }

extern "C" int64_t w2s_ssm_ws(const w2s_ssm_args* a, int backward) {
  if (!valid(a)) return W2S_EINVAL;
  return backward ? 4 * (floats_hs(a) + floats_bc(a) + floats_a(a)) : 0;
}

extern "C" int w2s_ssm_scan_fwd(const w2s_ssm_args* a, void* stream) {
  if (!valid(a)) return W2S_EINVAL;
  if (a->B == 0 || (a->L == 0 && !a->h_out)) return W2S_OK;
  if (a->L > 0 && (!a->u || !a->dt || !a->Bm || !a->Cm || !a->y)) return W2S_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  return a->dtype == W2S_F32 ? scan_fwd<float>(a, st) : a->dtype == W2S_BF16 ? scan_fwd<bf16_t>(a, st) : scan_fwd<half_t>(a, st);
}

extern "C" int w2s_ssm_scan_bwd(const w2s_ssm_args* a, void* stream) {
  if (!valid(a) || !a->gA) return W2S_EINVAL;
  if (a->B > 0 && (!a->ws || (a->L > 0 && (!a->u || !a->dt || !a->Bm || !a->Cm || !a->gu || !a->gdt || !a->gB || !a->gC || (a->z && !a->gz)))))
    return W2S_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  return a->dtype == W2S_F32 ? scan_bwd<float>(a, st) : a->dtype == W2S_BF16 ? scan_bwd<bf16_t>(a, st) : scan_bwd<half_t>(a, st);
}

extern "C" int w2s_ssm_step(const w2s_ssm_args* a, void* stream) {
  if (!valid(a)) return W2S_EINVAL;
  if (a->B == 0) return W2S_OK;
  if (!a->u || !a->dt || !a->Bm || !a->Cm || !a->y || !a->h_out) return W2S_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  return a->dtype == W2S_F32 ? step<float>(a, st) : a->dtype == W2S_BF16 ? step<bf16_t>(a, st) : step<half_t>(a, st);
}
