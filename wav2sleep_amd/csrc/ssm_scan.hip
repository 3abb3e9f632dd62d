// Selective state space scan: delta = softplus(dt + bias), h_t[n] = exp(delta A[n]) h_{t-1}[n] + delta u B_t[n], y_t = (sum_n C_t[n] h_t[n] + D u) silu(z),
// its backward and its form for one position.
//
// The recurrence is sequential in t, and B x D channels do not fill 256 CUs (16 nights x 256 channels = 64 waves of one channel a lane).  So a
// workgroup of 8 waves takes a tile of 8 TT positions of 16 CPL channels and the waves walk their TT positions side by side, which linearity allows:
//   1. every wave walks its positions from a zero state and keeps the decays a_t = exp(delta_t A) in registers (the exponentials, on the quarter-rate
//      unit, are the largest single cost and are computed once);
//   2. the waves' end states and products of decays (exp(A sum delta): one more exponential, no product chain) meet in LDS, and each wave folds those
//      in front of it onto the tile's initial state;
//   3. every wave walks its positions again from the right state -- two fused steps per state, no exponential -- and emits y.
// Four lanes (a quad) share a channel, NPL = N / 4 states each (N padded to 8, 16, 32, 64): sums over states are two DPP adds, the softplus and the
// gate are computed once per quad (the lane of position t mod 4) and broadcast by DPP.  B and C of a tile are staged in LDS in fp32, once per workgroup.
// A tile's global loads are issued one tile ahead.  Where even that leaves CUs idle (few sequences, few channels) the sequence is cut into
// segments: a first launch walks them for their end states alone, the second folds the ones in front of its own segment first.
// Bound: vector issue (about 10 slots per state and position forward, 22 backward, against 4 - 16 bytes per channel and position).
#include "mix_io.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kWaves = 8;

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float quad_bcast(float v, int k) {   // lane k of the quad; k is a constant after unrolling
  switch (k) {
    case 0: return dpp<0x00>(v);
    case 1: return dpp<0x55>(v);
    case 2: return dpp<0xaa>(v);
    default: return dpp<0xff>(v);
  }
}
// the same value as one the compiler knows nothing of.  On a lane offset it keeps the address in its short form, a scalar base and a 32-bit offset, where
// a loop would otherwise carry one 64-bit address a lane for every access.  Between the walks over a tile it keeps what a walk can cheaply form again (broadcasts, LDS reads,
// states) from being carried to the next one in registers, of which the decays take a quarter
__device__ __forceinline__ void forget(float& v) { asm("" : "+v"(v)); }
template <int M, int N> __device__ __forceinline__ void forget(float (&v)[M][N]) {
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) forget(v[i][k]);
}
__device__ __forceinline__ int forgotten(int v) {
  asm("" : "+v"(v));
  return v;
}
__device__ __forceinline__ float quad_sum(float v) {
  v += dpp<0xb1>(v);   // lanes 1 0 3 2
  v += dpp<0x4e>(v);   // lanes 2 3 0 1
  return v;
}
// a + (a of the lane 32 away) in the lower half of the wave, the same of b in the upper half
__device__ __forceinline__ float fold32(float a, float b) {
  auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
  const unsigned x = r[0], y = r[1];
  return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}
// ... of the row of 16 lanes beside: a in rows 0 and 2, b in rows 1 and 3
__device__ __forceinline__ float fold16(float a, float b) {
  auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
  const unsigned x = r[0], y = r[1];
  return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}
__device__ __forceinline__ float sum_quads_of_row(float v) {   // over the four quads of a row of 16 lanes
  v += dpp<0x128>(v);   // row_ror:8
  v += dpp<0x124>(v);   // row_ror:4
  return v;
}

// tile shapes by states per lane: TT positions a wave x CPL channels a quad x NPL states a lane
template <int NPL> struct FwdShape { static constexpr int CPL = 1, TT = NPL <= 4 ? 16 : 64 / NPL; };                  // 64 decays a lane
template <int NPL> struct BwdShape { static constexpr int CPL = NPL <= 2 ? 2 : 1, TT = NPL <= 8 ? 8 : 4; };

struct Plan {
  int dg, ncb, ntile, nseg, tps, nck, vbc, vch;   // channels a group, channel blocks a group, tiles, segments, tiles a segment, checkpoints a sequence; B/C by fours, channels by twos
  float *segh, *segs;                             // [B][nseg][D][NP] end states, [B][nseg][D] sums of delta (nseg > 1)
  float *part_bc, *part_a;                        // backward: [channel block][B][L][G][2 NP], [B nseg][D][N + 2]
};

// Workgroups go to the 8 XCDs in turn; neighbouring channel blocks share cache lines, so each XCD (its own L2) gets a run of consecutive ones.
__device__ __forceinline__ unsigned xcd_order(unsigned blk, unsigned n) {
  const unsigned x = blk & 7, q = n >> 3, r = n & 7;
  return x * q + (x < r ? x : r) + (blk >> 3);
}

struct Where { int b, g, cb, seg; };
__device__ __forceinline__ Where where_of(const w2s_ssm_args& a, const Plan& p) {
  unsigned i = xcd_order(blockIdx.x, gridDim.x);
  Where w;
  w.cb = i % p.ncb;
  i /= p.ncb;
  w.g = i % a.G;
  i /= a.G;
  w.seg = i % p.nseg;
  w.b = i / p.nseg;
  return w;
}

// CPL adjacent channels of one position at a wave-uniform address + 32-bit lane offsets (scalar base, vector offset: no 64-bit arithmetic a lane).
// VCH: the channels come in whole aligned pairs, one access and one offset; else one each, a channel that does not exist reading the group's last
template <typename T, int CPL, bool VCH> __device__ __forceinline__ void load_ch(const T* base, const unsigned (&off)[CPL], float* v) {
  if constexpr (VCH) {
    mix_load<T, CPL>(base + (unsigned)forgotten(off[0]), v);
  } else {
#pragma unroll
    for (int c = 0; c < CPL; ++c) v[c] = (float)base[(unsigned)forgotten(off[c])];
  }
}
template <typename T, int CPL, bool VCH> __device__ __forceinline__ void store_ch(T* base, const unsigned (&off)[CPL], int n, const float* v) {   // n: how many exist
  if constexpr (VCH) {
    if (n > 0) mix_store<T, CPL>(base + (unsigned)forgotten(off[0]), v);
  } else {
#pragma unroll
    for (int c = 0; c < CPL; ++c)
      if (c < n) base[(unsigned)forgotten(off[c])] = (T)v[c];
  }
}
template <int CPL> __device__ __forceinline__ void offsets(unsigned (&off)[CPL], int64_t stride, int q, int ch, int last) {
#pragma unroll
  for (int c = 0; c < CPL; ++c) off[c] = (unsigned)(q * stride) + ch + (c < last ? c : last);
}

// B and C of a tile on their way from global memory to LDS: unit = four states of one position of one of the two
template <typename T, int NP, int TILE> struct StageBC {
  static constexpr int UNITS = TILE * NP / 4 * 2, PER = (UNITS + kWaves * 64 - 1) / (kWaves * 64);
  float v[PER][4];
  __device__ __forceinline__ void load(const w2s_ssm_args& a, const Plan& p, const T* Bg, const T* Cg, int t0, bool with_c) {   // Bg, Cg: the group's first state
    const T* b0 = Bg + (int64_t)t0 * a.sB_l;
    const T* c0 = Cg + (int64_t)t0 * a.sC_l;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = k * kWaves * 64 + (int)threadIdx.x;
      const int half = UNITS / 2, isc = i >= half, r = isc ? i - half : i, row = r / (NP / 4), n = r % (NP / 4) * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = 0.0f;
      if (i < UNITS && (with_c || !isc) && t0 + row < a.L && n < a.N) {
        const T* src = isc ? c0 + (unsigned)forgotten(row * (int)a.sC_l + n) : b0 + (unsigned)forgotten(row * (int)a.sB_l + n);
        if (p.vbc) {
          mix_load<T, 4>(src, v[k]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < a.N) v[k][e] = (float)src[e];
        }
      }
    }
  }
  __device__ __forceinline__ void store(float* lds, int t0, int n) const {   // positions behind the end hold zeros, whatever was there
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = k * kWaves * 64 + (int)threadIdx.x, half = UNITS / 2, r = i >= half ? i - half : i;
      const bool live = t0 + r / (NP / 4) < n;
      if (i < UNITS) *reinterpret_cast<float4*>(lds + i * 4) = live ? make_float4(v[k][0], v[k][1], v[k][2], v[k][3]) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
};

// ------------------------------------------------------------------------------------------------------------------ forward
// STATE: only the segment's end state (from zero) and its sum of delta
template <typename T, int NPL, bool STATE, bool VCH> __global__ __launch_bounds__(kWaves * 64) void ssm_fwd_kernel(w2s_ssm_args a, Plan p) {
  constexpr int CPL = FwdShape<NPL>::CPL, TT = FwdShape<NPL>::TT, TILE = kWaves * TT, NI = TT / 4, NP = 4 * NPL, CW = 16 * CPL;
  constexpr int CK = kWaves * BwdShape<NPL>::TT;   // positions between the states that the backward starts from
  __shared__ float bc[2][TILE * NP * 2];
  __shared__ float ex[kWaves][2][CPL][64 * NPL];
  const Where at = where_of(a, p);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), q = lane & 3;
  const int ch = at.cb * CW + (lane >> 2) * CPL, nch = p.dg - ch;   // channel within the group, how many from there on exist
  const int chc = nch > 0 ? ch : (VCH ? p.dg - CPL : p.dg - 1), last = nch > 0 ? nch - 1 : (VCH ? CPL - 1 : 0), d = at.g * p.dg + chc;
  const int n = mix_length(a.lengths, at.b, a.L), N = a.N, L = a.L;
  float A[CPL][NPL], h[CPL][NPL], hc[CPL][NPL], bias[CPL], Dp[CPL];
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int dc = d + (c < last ? c : last);
    bias[c] = a.dt_bias ? a.dt_bias[dc] : 0.0f;
    Dp[c] = a.Dp ? a.Dp[dc] : 0.0f;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const int s = q * NPL + j;
      A[c][j] = s < N ? a.A[(int64_t)dc * N + s] * kLog2e : 0.0f;
      hc[c][j] = !STATE && s < N && a.h0 ? a.h0[((int64_t)at.b * a.D + dc) * N + s] : 0.0f;
    }
    if (!STATE)
      for (int k = 0; k < at.seg; ++k) {   // the segments in front
        const int64_t r = ((int64_t)at.b * p.nseg + k) * a.D + dc;
        const float S = p.segs[r];
#pragma unroll
        for (int j = 0; j < NPL; ++j) hc[c][j] = __builtin_fmaf(__builtin_amdgcn_exp2f(A[c][j] * S), hc[c][j], p.segh[r * NP + q * NPL + j]);
      }
  }
  const int dg0 = at.g * p.dg;   // uniform: the group's first channel
  const T* pu = (const T*)a.u + at.b * a.su_b + dg0;
  const T* pd = (const T*)a.dt + at.b * a.sdt_b + dg0;
  const T* pz = a.z ? (const T*)a.z + at.b * a.sz_b + dg0 : nullptr;
  const T* pB = (const T*)a.Bm + at.b * a.sB_b + at.g * a.sB_g;
  const T* pC = (const T*)a.Cm + at.b * a.sC_b + at.g * a.sC_g;
  T* py = (T*)a.y + (int64_t)at.b * L * a.D + dg0;
  unsigned ou[CPL], od[CPL], oz[CPL], oy[CPL];
  offsets<CPL>(ou, a.su_l, q, chc, last);
  offsets<CPL>(od, a.sdt_l, q, chc, last);
  offsets<CPL>(oz, a.sz_l, q, chc, last);
  offsets<CPL>(oy, a.D, q, chc, last);
  float ru[NI][CPL], rd[NI][CPL], rz[NI][CPL], Ssum[CPL];
#pragma unroll
  for (int c = 0; c < CPL; ++c) Ssum[c] = 0.0f;
  StageBC<T, NP, TILE> st;
  auto fetch = [&](int t0) {
    const int tb = t0 + w * TT;
    const bool whole = tb + TT <= L;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (whole || tb + 4 * i + q < L) {
        load_ch<T, CPL, VCH>(pu + (int64_t)(tb + 4 * i) * a.su_l, ou, ru[i]);
        load_ch<T, CPL, VCH>(pd + (int64_t)(tb + 4 * i) * a.sdt_l, od, rd[i]);
        if (!STATE && pz) load_ch<T, CPL, VCH>(pz + (int64_t)(tb + 4 * i) * a.sz_l, oz, rz[i]);
      }
    st.load(a, p, pB, pC, t0, !STATE);
  };
  auto put = [&](int t0, const float (&v)[NI][CPL]) {
    const int tb = t0 + w * TT;
    const bool whole = tb + TT <= L;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (whole || tb + 4 * i + q < L) store_ch<T, CPL, VCH>(py + (int64_t)(tb + 4 * i) * a.D, oy, nch, v[i]);
  };
  const int k0 = at.seg * p.tps, k1 = k0 + p.tps < p.ntile ? k0 + p.tps : p.ntile;
  if (k0 < k1 && k0 * TILE < n) fetch(k0 * TILE);
  for (int k = k0; k < k1; ++k) {
    const int t0 = k * TILE;
    if (t0 >= n) {   // (the whole workgroup) behind the end
      if (!STATE) {
        const float zero[NI][CPL] = {};
        put(t0, zero);
      }
      continue;
    }
    float u[NI][CPL], dl[NI][CPL], du[NI][CPL], z[NI][CPL], S[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) S[c] = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const bool live = t0 + w * TT + 4 * i + q < n;
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        const float raw = rd[i][c] + bias[c];
        u[i][c] = live ? ru[i][c] : 0.0f;
        dl[i][c] = live ? (a.softplus ? mix_softplus(raw) : raw) : 0.0f;
        du[i][c] = dl[i][c] * u[i][c];
        z[i][c] = rz[i][c];
        S[c] += dl[i][c];
      }
    }
    float* lds = bc[k & 1];
    st.store(lds, t0, n);
    __syncthreads();
    if (k + 1 < k1 && t0 + TILE < n) fetch(t0 + TILE);
    const float* Bs = lds + w * TT * NP + q * NPL;
    const float* Cs = Bs + TILE * NP;
    float dec[TT][CPL][NPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c)
#pragma unroll
      for (int j = 0; j < NPL; ++j) h[c][j] = 0.0f;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      float Bv[NPL];
      mix_load<float, NPL>(Bs + t * NP, Bv);
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        const float dt = quad_bcast(dl[t / 4][c], t & 3), x = quad_bcast(du[t / 4][c], t & 3);
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
          dec[t][c][j] = __builtin_amdgcn_exp2f(dt * A[c][j]);
          h[c][j] = __builtin_fmaf(dec[t][c][j], h[c][j], x * Bv[j]);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      S[c] = quad_sum(S[c]);
      Ssum[c] += S[c];
      float P[NPL];
#pragma unroll
      for (int j = 0; j < NPL; ++j) P[j] = __builtin_amdgcn_exp2f(A[c][j] * S[c]);
      mix_store<float, NPL>(&ex[w][0][c][lane * NPL], h[c]);
      mix_store<float, NPL>(&ex[w][1][c][lane * NPL], P);
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {   // h: this wave's initial state, hc: the next tile's
      if (v == w) {
#pragma unroll
        for (int c = 0; c < CPL; ++c)
#pragma unroll
          for (int j = 0; j < NPL; ++j) h[c][j] = hc[c][j];
      }
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        float e[NPL], P[NPL];
        mix_load<float, NPL>(&ex[v][0][c][lane * NPL], e);
        mix_load<float, NPL>(&ex[v][1][c][lane * NPL], P);
#pragma unroll
        for (int j = 0; j < NPL; ++j) hc[c][j] = __builtin_fmaf(P[j], hc[c][j], e[j]);
      }
    }
    if constexpr (!STATE) {
      if (a.ckpt && (w * TT) % CK == 0 && t0 + w * TT < n) {
        const int64_t r = ((int64_t)at.b * p.nck + (t0 + w * TT) / CK) * a.D + d;
#pragma unroll
        for (int c = 0; c < CPL; ++c)
          if (c < nch) mix_store<float, NPL>(a.ckpt + (r + c) * NP + q * NPL, h[c]);
      }
      float y[NI][CPL];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        float Bv[NPL], Cv[NPL];
        mix_load<float, NPL>(Bs + t * NP, Bv);
        mix_load<float, NPL>(Cs + t * NP, Cv);
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          const float x = quad_bcast(du[t / 4][c], t & 3);
          float s = 0.0f;
#pragma unroll
          for (int j = 0; j < NPL; ++j) {
            h[c][j] = __builtin_fmaf(dec[t][c][j], h[c][j], x * Bv[j]);
            s = __builtin_fmaf(Cv[j], h[c][j], s);
          }
          s = quad_sum(s);
          y[t / 4][c] = (t & 3) == 0 || q == (t & 3) ? s : y[t / 4][c];
        }
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int t = t0 + w * TT + 4 * i + q;
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          y[i][c] = __builtin_fmaf(Dp[c], u[i][c], y[i][c]);
          if (pz) y[i][c] *= z[i][c] * mix_sigmoid(z[i][c]);
          if (t >= n) y[i][c] = 0.0f;
        }
      }
      put(t0, y);
    }
  }
  if constexpr (STATE) {
    __syncthreads();
    float* red = &ex[0][0][0][0];   // [wave][channel]
    if (q == 0)
#pragma unroll
      for (int c = 0; c < CPL; ++c) red[w * CW + (lane >> 2) * CPL + c] = Ssum[c];
    __syncthreads();
    if (w == 0) {
      const int64_t r = ((int64_t)at.b * p.nseg + at.seg) * a.D + d;
#pragma unroll
      for (int c = 0; c < CPL; ++c)
        if (c < nch) {
          float S = 0.0f;
          for (int v = 0; v < kWaves; ++v) S += red[v * CW + (lane >> 2) * CPL + c];
          if (q == 0) p.segs[r + c] = S;
          mix_store<float, NPL>(p.segh + (r + c) * NP + q * NPL, hc[c]);
        }
    }
  } else if (a.h_out && at.seg == p.nseg - 1 && w == 0) {
#pragma unroll
    for (int c = 0; c < CPL; ++c)
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if (c < nch && q * NPL + j < N) a.h_out[((int64_t)at.b * a.D + d + c) * N + q * NPL + j] = hc[c][j];
  }
}

// ------------------------------------------------------------------------------------------------------------------ backward
// With e_t = a_t G_t, G_t = C_t gy'_t + e_{t+1} (gy' = gy silu(z)): du = delta sum_n G B + D gy', ddelta = sum_n e h_{t-1} A + u sum_n G B, dA = sum_t e h_{t-1} delta,
// dB = sum_channels G delta u, dC = sum_channels gy' h.  Tiles from the sequence's end; inside a tile the waves first walk both ways from zero (forward
// for h, backward for e), meet in LDS, and walk both ways again from the right ends, the states of the second walk staying in registers.  dB and dC are
// summed over the 32 (16) channels of a workgroup by lane exchanges and over workgroups from `part_bc`; everything in a fixed order.
// STATE: only e at the segment's start (from zero) and the sum of delta.
template <typename T, int NPL, bool STATE, bool VCH> __global__ __launch_bounds__(kWaves * 64) void ssm_bwd_kernel(w2s_ssm_args a, Plan p) {
  constexpr int CPL = BwdShape<NPL>::CPL, TT = BwdShape<NPL>::TT, TILE = kWaves * TT, NI = TT / 4, NP = 4 * NPL, CW = 16 * CPL, NX = STATE ? 2 : 3;
  __shared__ float bc[2][TILE * NP * 2];
  __shared__ float ex[kWaves][NX][CPL][64 * NPL];
  const Where at = where_of(a, p);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), q = lane & 3;
  const int ch = at.cb * CW + (lane >> 2) * CPL, nch = p.dg - ch;
  const int chc = nch > 0 ? ch : (VCH ? p.dg - CPL : p.dg - 1), last = nch > 0 ? nch - 1 : (VCH ? CPL - 1 : 0), d = at.g * p.dg + chc;
  const int n = mix_length(a.lengths, at.b, a.L), N = a.N, L = a.L;
  float A[CPL][NPL], ec[CPL][NPL], gA[CPL][NPL], bias[CPL], Dp[CPL], gD[CPL], gb[CPL], Ssum[CPL];
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int dc = d + (c < last ? c : last);
    bias[c] = a.dt_bias ? a.dt_bias[dc] : 0.0f;
    Dp[c] = a.Dp ? a.Dp[dc] : 0.0f;
    gD[c] = gb[c] = Ssum[c] = 0.0f;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const int s = q * NPL + j;
      A[c][j] = s < N ? a.A[(int64_t)dc * N + s] * kLog2e : 0.0f;
      ec[c][j] = !STATE && c < nch && s < N && a.gh ? a.gh[((int64_t)at.b * a.D + dc) * N + s] : 0.0f;   // (a channel that is not there adds nothing to dB)
      gA[c][j] = 0.0f;
    }
    if (!STATE && c < nch)
      for (int k = p.nseg - 1; k > at.seg; --k) {   // the segments behind
        const int64_t r = ((int64_t)at.b * p.nseg + k) * a.D + dc;
        const float S = p.segs[r];
#pragma unroll
        for (int j = 0; j < NPL; ++j) ec[c][j] = __builtin_fmaf(__builtin_amdgcn_exp2f(A[c][j] * S), ec[c][j], p.segh[r * NP + q * NPL + j]);
      }
  }
  const int dg0 = at.g * p.dg;   // uniform: the group's first channel
  const T* pu = (const T*)a.u + at.b * a.su_b + dg0;
  const T* pd = (const T*)a.dt + at.b * a.sdt_b + dg0;
  const T* pz = a.z ? (const T*)a.z + at.b * a.sz_b + dg0 : nullptr;
  const T* pg = a.gy ? (const T*)a.gy + at.b * a.sg_b + dg0 : nullptr;
  const T* pB = (const T*)a.Bm + at.b * a.sB_b + at.g * a.sB_g;
  const T* pC = (const T*)a.Cm + at.b * a.sC_b + at.g * a.sC_g;
  const int64_t o0 = (int64_t)at.b * L * a.D + dg0;
  unsigned ou[CPL], od[CPL], oz[CPL], og[CPL], oo[CPL];
  offsets<CPL>(ou, a.su_l, q, chc, last);
  offsets<CPL>(od, a.sdt_l, q, chc, last);
  offsets<CPL>(oz, a.sz_l, q, chc, last);
  offsets<CPL>(og, a.sg_l, q, chc, last);
  offsets<CPL>(oo, a.D, q, chc, last);
  float ru[NI][CPL], rd[NI][CPL], rz[NI][CPL], rg[NI][CPL];
  StageBC<T, NP, TILE> st;
  auto fetch = [&](int t0) {
    const int tb = t0 + w * TT;
    const bool whole = tb + TT <= L;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (whole || tb + 4 * i + q < L) {
        if (!STATE) load_ch<T, CPL, VCH>(pu + (int64_t)(tb + 4 * i) * a.su_l, ou, ru[i]);
        load_ch<T, CPL, VCH>(pd + (int64_t)(tb + 4 * i) * a.sdt_l, od, rd[i]);
        if (pz) load_ch<T, CPL, VCH>(pz + (int64_t)(tb + 4 * i) * a.sz_l, oz, rz[i]);
        if (pg) load_ch<T, CPL, VCH>(pg + (int64_t)(tb + 4 * i) * a.sg_l, og, rg[i]);
      }
    st.load(a, p, pB, pC, t0, true);
  };
  auto put = [&](void* to, int t0, const float (&v)[NI][CPL]) {
    const int tb = t0 + w * TT;
    const bool whole = tb + TT <= L;
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (whole || tb + 4 * i + q < L) store_ch<T, CPL, VCH>((T*)to + o0 + (int64_t)(tb + 4 * i) * a.D, oo, nch, v[i]);
  };
  const int k0 = at.seg * p.tps, k1 = k0 + p.tps < p.ntile ? k0 + p.tps : p.ntile;
  int kl = k1;   // tiles from kl on lie behind the end
  while (kl > k0 && (kl - 1) * TILE >= n) --kl;
  if (!STATE)
    for (int k = kl; k < k1; ++k) {
      const float zero[NI][CPL] = {};
      put(a.gu, k * TILE, zero);
      put(a.gdt, k * TILE, zero);
      if (pz) put(a.gz, k * TILE, zero);
    }
  if (kl > k0) fetch((kl - 1) * TILE);
  for (int k = kl - 1; k >= k0; --k) {
    const int t0 = k * TILE;
    float u[NI][CPL], dl[NI][CPL], du[NI][CPL], raw[NI][CPL], gp[NI][CPL], gy[NI][CPL], z[NI][CPL], S[CPL], hi[CPL][NPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) S[c] = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int t = t0 + w * TT + 4 * i + q;
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        const bool live = t < n && c < nch;
        raw[i][c] = rd[i][c] + bias[c];
        u[i][c] = !STATE && live ? ru[i][c] : 0.0f;
        dl[i][c] = live ? (a.softplus ? mix_softplus(raw[i][c]) : raw[i][c]) : 0.0f;
        du[i][c] = dl[i][c] * u[i][c];
        gy[i][c] = pg && live ? rg[i][c] : 0.0f;
        z[i][c] = rz[i][c];
        gp[i][c] = pz ? (live ? gy[i][c] * z[i][c] * mix_sigmoid(z[i][c]) : 0.0f) : gy[i][c];
        S[c] += dl[i][c];
      }
    }
    float* lds = bc[k & 1];
    st.store(lds, t0, n);
    __syncthreads();
    if (STATE && k > k0) fetch(t0 - TILE);
    if constexpr (!STATE) {
#pragma unroll
      for (int c = 0; c < CPL; ++c) mix_load<float, NPL>(a.ckpt + (((int64_t)at.b * p.nck + k) * a.D + dg0) * NP + (unsigned)forgotten((chc + (c < last ? c : last)) * NP + q * NPL), hi[c]);
    }
    const float* Bs = lds + forgotten(w * TT * NP + q * NPL);
    const float* Cs = Bs + TILE * NP;
    // (with 16 states a lane the decays do not fit beside the walk's own values: they are computed again wherever they are used)
    constexpr bool KEEP = STATE || NPL < 16;
    float dec[TT][CPL][NPL], e[CPL][NPL], h[CPL][NPL];
    auto decay = [&](int t, int c, int j, float dt) { return KEEP ? dec[t][c][j] : __builtin_amdgcn_exp2f(dt * A[c][j]); };
#pragma unroll
    for (int c = 0; c < CPL; ++c)
#pragma unroll
      for (int j = 0; j < NPL; ++j) h[c][j] = e[c][j] = 0.0f;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      float Bv[NPL];
      if (!STATE) mix_load<float, NPL>(Bs + t * NP, Bv);
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        const float dt = quad_bcast(dl[t / 4][c], t & 3), x = quad_bcast(du[t / 4][c], t & 3);
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
          const float f = __builtin_amdgcn_exp2f(dt * A[c][j]);
          if (KEEP) dec[t][c][j] = f;
          if (!STATE) h[c][j] = __builtin_fmaf(f, h[c][j], x * Bv[j]);
        }
      }
      if (!KEEP) __builtin_amdgcn_sched_barrier(0);   // (registers, not overlap, are short)
    }
    if (!KEEP) {
      forget(A);
      forget(dl);
    }
#pragma unroll
    for (int t = TT - 1; t >= 0; --t) {
      float Cv[NPL];
      mix_load<float, NPL>(Cs + t * NP, Cv);
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        const float g = quad_bcast(gp[t / 4][c], t & 3), dt = quad_bcast(dl[t / 4][c], t & 3);
#pragma unroll
        for (int j = 0; j < NPL; ++j) e[c][j] = decay(t, c, j, dt) * __builtin_fmaf(Cv[j], g, e[c][j]);
      }
      if (!KEEP) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      S[c] = quad_sum(S[c]);
      Ssum[c] += S[c];
      float P[NPL];
#pragma unroll
      for (int j = 0; j < NPL; ++j) P[j] = __builtin_amdgcn_exp2f(A[c][j] * S[c]);
      mix_store<float, NPL>(&ex[w][0][c][lane * NPL], P);
      mix_store<float, NPL>(&ex[w][1][c][lane * NPL], e[c]);
      if constexpr (!STATE) mix_store<float, NPL>(&ex[w][NX - 1][c][lane * NPL], h[c]);
    }
    __syncthreads();
#pragma unroll(NPL < 16 ? 2 : 1)
    for (int v = kWaves - 1; v >= 0; --v) {   // e: what arrives behind this wave's positions, ec: behind the next tile's
      if (v == w) {
#pragma unroll
        for (int c = 0; c < CPL; ++c)
#pragma unroll
          for (int j = 0; j < NPL; ++j) e[c][j] = ec[c][j];
      }
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        float x[NPL], P[NPL];
        mix_load<float, NPL>(&ex[v][0][c][lane * NPL], P);
        mix_load<float, NPL>(&ex[v][1][c][lane * NPL], x);
#pragma unroll
        for (int j = 0; j < NPL; ++j) ec[c][j] = __builtin_fmaf(P[j], ec[c][j], x[j]);
      }
    }
    if constexpr (!STATE) {
#pragma unroll(NPL < 16 ? 2 : 1)
      for (int v = 0; v < w; ++v)
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          float x[NPL], P[NPL];
          mix_load<float, NPL>(&ex[v][0][c][lane * NPL], P);
          mix_load<float, NPL>(&ex[v][NX - 1][c][lane * NPL], x);
#pragma unroll
          for (int j = 0; j < NPL; ++j) hi[c][j] = __builtin_fmaf(P[j], hi[c][j], x[j]);
        }
      // The second walk in parts of HALF positions from the last part to the first, so that only a part's states are in registers; h first reaches a
      // part's start without keeping any.
      constexpr int HALF = NPL == 4 ? TT : NPL == 2 ? TT / 2 : NPL == 8 ? 2 : 1, PARTS = TT / HALF, JB = NPL < 4 ? NPL : 4;
      float oB[NI][CPL], oG[NI][CPL], oY[NI][CPL];
      forget(gp);
      if (!KEEP) forget(A);
      auto forward = [&](const float (*x)[NPL], int t, float (*to)[NPL]) {
        float Bv[NPL];
        mix_load<float, NPL>(Bs + t * NP, Bv);
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          const float v = quad_bcast(du[t / 4][c], t & 3), dt = quad_bcast(dl[t / 4][c], t & 3);
#pragma unroll
          for (int j = 0; j < NPL; ++j) to[c][j] = __builtin_fmaf(decay(t, c, j, dt), x[c][j], v * Bv[j]);
        }
        if (!KEEP) __builtin_amdgcn_sched_barrier(0);
      };
#pragma unroll
      for (int part = PARTS - 1; part >= 0; --part) {
        __builtin_amdgcn_sched_barrier(0);
        if (part == 0 && k > k0) fetch(t0 - TILE);   // (here, not at the tile's start: some of the decays' registers are free by now)
        forget(du);
        forget(dl);
        forget(hi);
        Bs = lds + forgotten(w * TT * NP + q * NPL);
#pragma unroll
        for (int t = 0; t < part * HALF; ++t) forward(t ? h : hi, t, h);
        float hs[HALF][CPL][NPL];
#pragma unroll
        for (int t = 0; t < HALF; ++t) forward(t ? hs[t ? t - 1 : 0] : (part ? h : hi), part * HALF + t, hs[t]);
        forget(du);
        forget(dl);
        Bs = lds + forgotten(w * TT * NP + q * NPL);
        Cs = Bs + TILE * NP;
#pragma unroll
        for (int t = part * HALF + HALF - 1; t >= part * HALF; --t) {
          const int th = t - part * HALF;
          const int tt = t0 + w * TT + t;
          float* out = p.part_bc + ((((int64_t)at.cb * a.B + at.b) * L + tt) * a.G + at.g) * 2 * NP;   // (written where tt < n only)
          float sB[CPL], sG[CPL], sY[CPL];
#pragma unroll
          for (int j0 = 0; j0 < NPL; j0 += JB) {
            float Bv[JB], Cv[JB], pb[JB], pc[JB];
            mix_load<float, JB>(Bs + t * NP + j0, Bv);
            mix_load<float, JB>(Cs + t * NP + j0, Cv);
#pragma unroll
            for (int c = 0; c < CPL; ++c) {
              const float g = quad_bcast(gp[t / 4][c], t & 3), x = quad_bcast(du[t / 4][c], t & 3), dt = quad_bcast(dl[t / 4][c], t & 3);
              if (j0 == 0) sB[c] = sG[c] = sY[c] = 0.0f;
#pragma unroll
              for (int jj = 0; jj < JB; ++jj) {
                const int j = j0 + jj;
                const float ht = hs[th][c][j];
                const float G = __builtin_fmaf(Cv[jj], g, e[c][j]);
                e[c][j] = decay(t, c, j, dt) * G;
                const float eh = e[c][j] * (th ? hs[th ? th - 1 : 0][c][j] : part ? h[c][j] : hi[c][j]);
                gA[c][j] = __builtin_fmaf(eh, dt, gA[c][j]);
                sG[c] = __builtin_fmaf(eh, A[c][j], sG[c]);
                sB[c] = __builtin_fmaf(G, Bv[jj], sB[c]);
                sY[c] = __builtin_fmaf(Cv[jj], ht, sY[c]);
                pb[jj] = c ? __builtin_fmaf(G, x, pb[jj]) : G * x;
                pc[jj] = c ? __builtin_fmaf(g, ht, pc[jj]) : g * ht;
              }
            }
            // sums over the 16 quads; the states of dB and of dC end up spread over the rows of 16 lanes
            if constexpr (JB == 4) {
              const float sb = sum_quads_of_row(fold16(fold32(pb[0], pb[1]), fold32(pb[2], pb[3])));
              const float sc = sum_quads_of_row(fold16(fold32(pc[0], pc[1]), fold32(pc[2], pc[3])));
              const int s = q * NPL + j0 + ((lane >> 4) & 1) * 2 + (lane >> 5);
              if ((lane & 8) == 0 && tt < n) out[(unsigned)forgotten((lane & 4 ? NP : 0) + s)] = lane & 4 ? sc : sb;
            } else {
              const float sv = sum_quads_of_row(fold16(fold32(pb[0], pb[1]), fold32(pc[0], pc[1])));
              if ((lane & 12) == 0 && tt < n) out[(unsigned)forgotten(((lane >> 4) & 1) * NP + q * NPL + (lane >> 5))] = sv;
            }
          }
          const bool mine = q == (t & 3) || (t & 3) == 3;   // (the highest of a lane's four comes first; the others then choose)
#pragma unroll
          for (int c = 0; c < CPL; ++c) {
            const float vB = quad_sum(sB[c]), vG = quad_sum(sG[c]), vY = pz ? quad_sum(sY[c]) : 0.0f;
            oB[t / 4][c] = mine ? vB : oB[t / 4][c];
            oG[t / 4][c] = mine ? vG : oG[t / 4][c];
            oY[t / 4][c] = mine ? vY : oY[t / 4][c];
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const bool live = t0 + w * TT + 4 * i + q < n;
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          float gd = __builtin_fmaf(kLn2, oG[i][c], u[i][c] * oB[i][c]);
          if (a.softplus) gd *= mix_sigmoid(raw[i][c]);
          oG[i][c] = live ? gd : 0.0f;
          oB[i][c] = live ? __builtin_fmaf(dl[i][c], oB[i][c], Dp[c] * gp[i][c]) : 0.0f;
          gD[c] = __builtin_fmaf(gp[i][c], u[i][c], gD[c]);
          gb[c] += oG[i][c];
          if (pz) {
            const float s = mix_sigmoid(z[i][c]), yp = __builtin_fmaf(Dp[c], u[i][c], oY[i][c]);
            oY[i][c] = live ? gy[i][c] * yp * s * (1.0f + z[i][c] * (1.0f - s)) : 0.0f;
          }
        }
      }
      put(a.gu, t0, oB);
      put(a.gdt, t0, oG);
      if (pz) put(a.gz, t0, oY);
    }
  }
  __syncthreads();
  float* red = &ex[0][0][0][0];
  if constexpr (STATE) {
    if (q == 0)
#pragma unroll
      for (int c = 0; c < CPL; ++c) red[w * CW + (lane >> 2) * CPL + c] = Ssum[c];
    __syncthreads();
    if (w == 0) {
      const int64_t r = ((int64_t)at.b * p.nseg + at.seg) * a.D + d;
#pragma unroll
      for (int c = 0; c < CPL; ++c)
        if (c < nch) {
          float S = 0.0f;
          for (int v = 0; v < kWaves; ++v) S += red[v * CW + (lane >> 2) * CPL + c];
          if (q == 0) p.segs[r + c] = S;
          mix_store<float, NPL>(p.segh + (r + c) * NP + q * NPL, ec[c]);
        }
    }
  } else {
    // dA, dD, d(bias) of the workgroup: over the waves in order
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      gD[c] = quad_sum(gD[c]);
      gb[c] = quad_sum(gb[c]);
      mix_store<float, NPL>(&ex[w][0][c][lane * NPL], gA[c]);
      if (q < 2) ex[w][1][c][(lane >> 2) * 2 + q] = q ? gb[c] : gD[c];
    }
    __syncthreads();
    if (w == 0) {
      const int64_t r = ((int64_t)at.b * p.nseg + at.seg) * a.D + d;
#pragma unroll
      for (int c = 0; c < CPL; ++c)
        if (c < nch) {
          float s[NPL] = {}, x = 0.0f;
          for (int v = 0; v < kWaves; ++v) {
            float y[NPL];
            mix_load<float, NPL>(&ex[v][0][c][lane * NPL], y);
#pragma unroll
            for (int j = 0; j < NPL; ++j) s[j] += y[j];
            if (q < 2) x += ex[v][1][c][(lane >> 2) * 2 + q];
          }
          float* o = p.part_a + (r + c) * (N + 2);
#pragma unroll
          for (int j = 0; j < NPL; ++j)
            if (q * NPL + j < N) o[q * NPL + j] = s[j];
          if (q < 2) o[N + q] = x;
          if (a.gh0 && at.seg == 0)
#pragma unroll
            for (int j = 0; j < NPL; ++j)
              if (q * NPL + j < N) a.gh0[((int64_t)at.b * a.D + d + c) * N + q * NPL + j] = ec[c][j];
        }
    }
  }
}

// gB / gC [B][L][G][N]: the group's channel blocks in order; 0 behind the end.  A thread takes four states.
template <typename T> __global__ __launch_bounds__(256) void ssm_reduce_bc_kernel(w2s_ssm_args a, int ncb, int NP, const float* part) {
  const int64_t rows = (int64_t)a.B * a.L * a.G, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = 2 * NP / 4;
  const int64_t row = i / per;   // (b, t, g)
  if (row >= rows) return;
  const int s = (int)(i % per) * 4;
  const int64_t bt = row / a.G;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (bt % a.L < mix_length(a.lengths, (int)(bt / a.L), a.L))
    for (int k = 0; k < ncb; ++k) {
      const float4 x = *reinterpret_cast<const float4*>(part + (k * rows + row) * 2 * NP + s);
      v.x += x.x;
      v.y += x.y;
      v.z += x.z;
      v.w += x.w;
    }
  T* out = (T*)(s < NP ? a.gB : a.gC) + row * a.N;
  const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (s % NP + e < a.N) out[s % NP + e] = (T)o[e];
}

// gA [D][N], gD, gbias [D]: 64 columns x 16 strided sums over the parts a workgroup, then those 16 in order
__global__ __launch_bounds__(1024) void ssm_reduce_a_kernel(w2s_ssm_args a, int nparts, const float* part) {
  __shared__ float red[16][64];
  const int64_t per = (int64_t)a.D * (a.N + 2), i = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const int row = threadIdx.x >> 6;
  float v = 0.0f;
  if (i < per)
    for (int k = row; k < nparts; k += 16) v += part[k * per + i];
  red[row][threadIdx.x & 63] = v;
  __syncthreads();
  if (row || i >= per) return;
  for (int k = 1; k < 16; ++k) v += red[k][threadIdx.x];
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

// rows within a tile are addressed by 32-bit offsets from the tile's 64-bit base: a position's stride stays below 2^22 elements (128 rows of 4 bytes: 2 GiB)
bool near(int64_t s) { return s >= 0 && s < (1 << 22); }

bool valid(const w2s_ssm_args* a) {
  return a && near(a->su_l) && near(a->sdt_l) && near(a->sz_l) && near(a->sB_l) && near(a->sC_l) && near(a->sg_l) && a->D < (1 << 22) && a->A && a->B >= 0 && a->L >= 0 && a->D >= 1 && a->N >= 1 && a->N <= 64 && a->G >= 1 && a->D % a->G == 0 && a->dtype >= 0 && a->dtype <= 2;
}

int npl_of(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }
template <int NPL> constexpr int fwd_tile() { return kWaves * FwdShape<NPL>::TT; }
template <int NPL> constexpr int bwd_tile() { return kWaves * BwdShape<NPL>::TT; }

// Segments a sequence is cut into.  Cutting costs a second walk for the end states, so it pays only where the workgroups of whole sequences leave
// most of the 256 CUs idle.
int segments(int64_t blocks, int ntile) {
  if (blocks <= 0 || blocks > 128 || ntile < 4) return 1;
  int64_t n = 512 / blocks;
  if (n > ntile / 2) n = ntile / 2;
  if (n > 64) n = 64;
  return n < 2 ? 1 : (int)n;
}

template <int NPL> Plan plan_of(const w2s_ssm_args* a, bool backward) {
  Plan p{};
  const int cw = 16 * (backward ? BwdShape<NPL>::CPL : FwdShape<NPL>::CPL), tile = backward ? bwd_tile<NPL>() : fwd_tile<NPL>();
  p.dg = a->D / a->G;
  p.ncb = (p.dg + cw - 1) / cw;
  p.ntile = (int)(((int64_t)a->L + tile - 1) / tile);
  p.nseg = segments((int64_t)a->B * a->G * p.ncb, p.ntile);
  p.tps = (p.ntile + p.nseg - 1) / p.nseg;
  if (p.tps > 0) p.nseg = (p.ntile + p.tps - 1) / p.tps;
  if (p.nseg < 1) p.nseg = 1;
  p.nck = (int)(((int64_t)a->L + bwd_tile<NPL>() - 1) / bwd_tile<NPL>());
  const int e = esize(a->dtype);
  p.vbc = a->N % 4 == 0 && mix_aligned(a->Bm, a->sB_b, a->sB_l, 4, e) && a->sB_g % 4 == 0 && mix_aligned(a->Cm, a->sC_b, a->sC_l, 4, e) && a->sC_g % 4 == 0;
  p.vch = p.dg % 2 == 0 && mix_aligned(a->u, a->su_b, a->su_l, 2, e) && mix_aligned(a->dt, a->sdt_b, a->sdt_l, 2, e) && mix_aligned(a->z, a->sz_b, a->sz_l, 2, e) &&
          mix_aligned(a->gy, a->sg_b, a->sg_l, 2, e) && mix_aligned(a->y, 0, 0, 2, e) && mix_aligned(a->gu, 0, 0, 2, e) && mix_aligned(a->gdt, 0, 0, 2, e) &&
          mix_aligned(a->gz, 0, 0, 2, e);
  return p;
}

int64_t seg_floats(const w2s_ssm_args* a, const Plan& p, int np) { return p.nseg > 1 ? (int64_t)a->B * p.nseg * a->D * (np + 1) : 0; }
int64_t bc_floats(const w2s_ssm_args* a, const Plan& p, int np) { return (int64_t)p.ncb * a->B * a->L * a->G * 2 * np; }
int64_t a_floats(const w2s_ssm_args* a, const Plan& p) { return ((int64_t)a->B * p.nseg * a->D * (a->N + 2) + 3) / 4 * 4; }   // (what follows stays 16-byte aligned)

template <int NPL> int64_t ws_floats(const w2s_ssm_args* a, bool backward) {
  const Plan p = plan_of<NPL>(a, backward);
  return seg_floats(a, p, 4 * NPL) + (backward ? bc_floats(a, p, 4 * NPL) + a_floats(a, p) : 0);
}

template <int NPL> int64_t ckpt_floats(const w2s_ssm_args* a) { return (int64_t)a->B * plan_of<NPL>(a, false).nck * a->D * 4 * NPL; }

template <typename T, int NPL> int scan_fwd(const w2s_ssm_args* a, hipStream_t st) {
  Plan p = plan_of<NPL>(a, false);
  const int64_t blocks = (int64_t)a->B * a->G * p.ncb * p.nseg;
  if (blocks > 0x7fffffff) return W2S_EINVAL;
  if (p.nseg > 1) {
    if (!a->ws) return W2S_EINVAL;
    p.segh = (float*)a->ws;
    p.segs = p.segh + (int64_t)a->B * p.nseg * a->D * 4 * NPL;
    ssm_fwd_kernel<T, NPL, true, false><<<(unsigned)blocks, kWaves * 64, 0, st>>>(*a, p);
  }
  ssm_fwd_kernel<T, NPL, false, false><<<(unsigned)blocks, kWaves * 64, 0, st>>>(*a, p);
  W2S_CHECK_LAUNCH();
  return W2S_OK;
}

template <typename T, int NPL> int scan_bwd(const w2s_ssm_args* a, hipStream_t st) {
  Plan p = plan_of<NPL>(a, true);
  const int64_t blocks = (int64_t)a->B * a->G * p.ncb * p.nseg;
  const int64_t rows = (int64_t)a->B * a->L * a->G, nbc = (rows * (2 * NPL) + 255) / 256, na = ((int64_t)a->D * (a->N + 2) + 63) / 64;
  if (blocks > 0x7fffffff || nbc > 0x7fffffff || na > 0x7fffffff) return W2S_EINVAL;
  p.part_bc = (float*)a->ws;
  p.part_a = p.part_bc + bc_floats(a, p, 4 * NPL);
  p.segh = p.part_a + a_floats(a, p);
  p.segs = p.segh + (int64_t)a->B * p.nseg * a->D * 4 * NPL;
  if (blocks) {
    if (BwdShape<NPL>::CPL > 1 && p.vch) {
      constexpr bool V = BwdShape<NPL>::CPL > 1;
      if (p.nseg > 1) ssm_bwd_kernel<T, NPL, true, V><<<(unsigned)blocks, kWaves * 64, 0, st>>>(*a, p);
      ssm_bwd_kernel<T, NPL, false, V><<<(unsigned)blocks, kWaves * 64, 0, st>>>(*a, p);
    } else {
      if (p.nseg > 1) ssm_bwd_kernel<T, NPL, true, false><<<(unsigned)blocks, kWaves * 64, 0, st>>>(*a, p);
      ssm_bwd_kernel<T, NPL, false, false><<<(unsigned)blocks, kWaves * 64, 0, st>>>(*a, p);
    }
  }
  if (nbc) ssm_reduce_bc_kernel<T><<<(unsigned)nbc, 256, 0, st>>>(*a, p.ncb, 4 * NPL, p.part_bc);
  ssm_reduce_a_kernel<<<(unsigned)na, 1024, 0, st>>>(*a, a->B * p.nseg, p.part_a);
  W2S_CHECK_LAUNCH();
  return W2S_OK;
}

template <typename T> int by_states(const w2s_ssm_args* a, bool backward, hipStream_t st) {
  switch (npl_of(a->N)) {
    case 2: return backward ? scan_bwd<T, 2>(a, st) : scan_fwd<T, 2>(a, st);
    case 4: return backward ? scan_bwd<T, 4>(a, st) : scan_fwd<T, 4>(a, st);
    case 8: return backward ? scan_bwd<T, 8>(a, st) : scan_fwd<T, 8>(a, st);
    default: return backward ? scan_bwd<T, 16>(a, st) : scan_fwd<T, 16>(a, st);
  }
}

int scan(const w2s_ssm_args* a, bool backward, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  switch (a->dtype) {
    case W2S_F32: return by_states<float>(a, backward, st);
    case W2S_BF16: return by_states<bf16_t>(a, backward, st);
    default: return by_states<half_t>(a, backward, st);
  }
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

extern "C" int64_t w2s_ssm_ckpt(const w2s_ssm_args* a) {
  if (!valid(a)) return W2S_EINVAL;
  switch (npl_of(a->N)) {
    case 2: return ckpt_floats<2>(a);
    case 4: return ckpt_floats<4>(a);
    case 8: return ckpt_floats<8>(a);
    default: return ckpt_floats<16>(a);
  }
}

extern "C" int64_t w2s_ssm_ws(const w2s_ssm_args* a, int backward) {
  if (!valid(a)) return W2S_EINVAL;
  switch (npl_of(a->N)) {
    case 2: return 4 * ws_floats<2>(a, backward != 0);
    case 4: return 4 * ws_floats<4>(a, backward != 0);
    case 8: return 4 * ws_floats<8>(a, backward != 0);
    default: return 4 * ws_floats<16>(a, backward != 0);
  }
}

extern "C" int w2s_ssm_scan_fwd(const w2s_ssm_args* a, void* stream) {
  if (!valid(a)) return W2S_EINVAL;
  if (a->B == 0 || (a->L == 0 && !a->h_out)) return W2S_OK;
  if (a->L > 0 && (!a->u || !a->dt || !a->Bm || !a->Cm || !a->y)) return W2S_EINVAL;
  return scan(a, false, stream);
}

extern "C" int w2s_ssm_scan_bwd(const w2s_ssm_args* a, void* stream) {
  if (!valid(a) || !a->gA) return W2S_EINVAL;
  if (a->B > 0 && (!a->ws || (a->L > 0 && (!a->u || !a->dt || !a->Bm || !a->Cm || !a->ckpt || !a->gu || !a->gdt || !a->gB || !a->gC || (a->z && !a->gz)))))
    return W2S_EINVAL;
  return scan(a, true, stream);
}

extern "C" int w2s_ssm_step(const w2s_ssm_args* a, void* stream) {
  if (!valid(a)) return W2S_EINVAL;
  if (a->B == 0) return W2S_OK;
  if (!a->u || !a->dt || !a->Bm || !a->Cm || !a->y || !a->h_out) return W2S_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  return a->dtype == W2S_F32 ? step<float>(a, st) : a->dtype == W2S_BF16 ? step<bf16_t>(a, st) : step<half_t>(a, st);
}
