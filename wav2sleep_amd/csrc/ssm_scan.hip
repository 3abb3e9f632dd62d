// Selective state space scan: delta = softplus(dt + bias), h_t[n] = exp(delta A[n]) h_{t-1}[n] + delta u B_t[n], y_t = (sum_n C_t[n] h_t[n] + D u) silu(z),
// its backward and its form for one position.
//
// The recurrence is sequential in t, and B x D channels do not fill 256 CUs (16 nights x 256 channels = 64 waves of one channel a lane).  So a workgroup
// takes 16 channels of one group and a tile of W TT positions (W = 16 or 8 waves, TT = 8 or 4 positions each), and the waves walk their positions side by
// side, which linearity allows:
//   1. every wave walks its positions from a zero state and keeps the decays a_t = exp(delta_t A) in registers (the exponentials run at a quarter of the
//      rate, are the largest single cost and are computed once);
//   2. the waves' end states and products of decays (exp(A sum delta): one more exponential, no product chain) meet in LDS, and each wave folds those
//      in front of it onto the tile's initial state;
//   3. every wave walks its positions again from the right state -- two fused steps per state, no exponential -- and emits y.
// Four lanes (a quad) share a channel, NPL = N / 4 states each (N padded to 8, 16, 32, 64): sums over states are two DPP adds, the softplus and the
// gate are computed once per quad (the lane of position t mod 4) and broadcast by DPP.  B and C of a tile are staged in LDS in fp32, once per workgroup.
// A tile's global loads are issued one tile ahead.  Where even that leaves CUs idle (few sequences, few channels) the sequence is cut into
// segments: a first launch walks them for their end states alone, the second folds the ones in front of its own segment first.
// Bound: the vector units (counters of 16 nights: 67 % busy both ways; 13.4 M and 33.1 M wave instructions), not HBM.  Measured, N = 16, gated: 16 nights
// x 960 x 256 fp32 (65 MB) 38 us forward = 1.7 TB/s, with the backward 149 us (130 MB by the least count, 0.9 TB/s); 4 x 2047 x 1536 bf16 in three groups
// 124 + 330 us; one row of 16384 x 512 bf16 107 us, of which the end states of its segments are about four tenths.  One state a lane and positions one after
// another, without tiles, took 58 us for a night.
#include "mix_io.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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
template <int N> __device__ __forceinline__ void forget(float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) forget(v[i]);
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

// Tile shapes: W waves, TT positions a wave, SIMD waves a SIMD (what the registers have to allow).
// WIDE where there is at most one workgroup a CU and nothing to gain from cutting sequences: the forward then takes sixteen waves, which hide each other's LDS
// and barrier waits, and the backward eight with a long walk each (sixteen: 109 us against 100).  With more workgroups than CUs, eight waves of at most 128
// registers a lane, so that a CU holds two workgroups and the last round of them is short.  fp32, L = 960, D = 256, N = 16, wide / not, forward and with the
// backward: 256 workgroups 38 / 43 and 141 / 165 us, 288 workgroups 72 / 59 and 262 / 228 us, 512 workgroups 74 / 60 and 284 / 252 us.  One workgroup more than
// there are CUs costs half as much again: some CU then has two, which share its vector units, and the others wait for it; up to 512 it costs no more.  (256 and 288
// workgroups of 512 channels 39 and 59 us, with the backward 145 and 232; 240 and 300 of 3000 positions and 8 states in bf16 77 and 122, 295 and 494.)
// From eight states a lane on the registers of a walk leave one shape; at 16 states a lane TT = 4 (forward of N = 64, 16 x 960 x 256: 174 us; TT = 8 spills: 276).
template <int NPL, bool WIDE> struct FwdShape { static constexpr int W = NPL <= 4 && WIDE ? 16 : 8, TT = NPL <= 8 ? 8 : 4, SIMD = NPL <= 4 ? 4 : 2; };
template <int NPL, bool WIDE> struct BwdShape { static constexpr int W = 8, TT = NPL == 16 || (NPL <= 4 && !WIDE) ? 4 : 8, SIMD = NPL <= 4 && !WIDE ? 4 : 2; };

struct Plan {
  int dg, ncb, ntile, nseg, tps, ck, nck, vbc;   // channels a group, channel blocks a group, tiles, segments, tiles a segment, positions from checkpoint to checkpoint (the backward's tile) and how many; B / C: 0 one by one, 1 by fours, 2 and N needs no padding
  float *segh, *segs;                        // [B][nseg][D][NP] end states, [B][nseg][D] sums of delta (nseg > 1)
  float *part_bc, *part_a;                   // backward: [channel block][B][L][G][2 NP], [B nseg][D][N + 2]
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

// One channel's values of a tensor [L][channels], four positions to a quad (lane q has positions 4 i + q of its wave's TT): a wave-uniform running row, moved
// on a tile at a time, and one 32-bit lane offset, so that an access is a scalar base and an offset and costs no 64-bit arithmetic a lane.
template <typename T> struct Column {
  T* row;         // position 0 of this wave's TT in the current tile, the group's first channel
  int sl;         // elements from position to position (below 2^22)
  unsigned off;
  __device__ __forceinline__ void start(const void* base, int64_t sb, int64_t stride, int b, int channel0, int t, int q, int ch) {
    sl = (int)stride;
    row = (T*)base + b * sb + t * stride + channel0;
    off = (unsigned)(q * sl) + ch;
  }
  template <int TILE> __device__ __forceinline__ void move() { row += TILE * sl; }
  __device__ __forceinline__ T get(int i) const { return (row + i * 4 * sl)[(unsigned)forgotten(off)]; }
  __device__ __forceinline__ void put(int i, float v) const { (row + i * 4 * sl)[(unsigned)forgotten(off)] = (T)v; }
};
// (values stay in the memory's type until a tile is worked on: a conversion here would wait for the load that it is to hide)
template <typename T, int NI> __device__ __forceinline__ void get_all(const Column<const T>& c, bool whole, int left, int q, T (&v)[NI]) {   // left: positions up to L
  if (whole) {
#pragma unroll
    for (int i = 0; i < NI; ++i) v[i] = c.get(i);
  } else {
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (4 * i + q < left) v[i] = c.get(i);
  }
}
template <typename T, int NI> __device__ __forceinline__ void put_all(const Column<T>& c, bool whole, int left, int q, bool on, const float (&v)[NI]) {
  if (whole) {
    if (on) {
#pragma unroll
      for (int i = 0; i < NI; ++i) c.put(i, v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (on && 4 * i + q < left) c.put(i, v[i]);
  }
}

// B and C of a tile on their way from global memory to LDS: unit = four states of one position of one of the two; a wave's 64 units of a round lie in one
template <typename T, int NP, int TILE, int W> struct StageBC {
  static constexpr int HALF = TILE * NP / 4, PER = (2 * HALF + W * 64 - 1) / (W * 64);
  static_assert(HALF % 64 == 0, "a wave's units are all of B or all of C");
  const T *rowB, *rowC;   // the tile's first position
  int slB, slC;
  unsigned off[PER];
  typedef typename mix_vec<T, 4>::type V;
  typedef V U __attribute__((aligned(sizeof(T))));   // (at any element: B and C are slices of a projection)
  V v[PER];
  __device__ __forceinline__ void start(const w2s_ssm_args& a, const Where& at, int t, int w, int lane) {
    rowB = (const T*)a.Bm + at.b * a.sB_b + at.g * a.sB_g + t * a.sB_l;
    rowC = (const T*)a.Cm + at.b * a.sC_b + at.g * a.sC_g + t * a.sC_l;
    slB = (int)a.sB_l;
    slC = (int)a.sC_l;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int u0 = (k * W + w) * 64, isc = u0 >= HALF, r = u0 - isc * HALF + lane;
      off[k] = r / (NP / 4) * (isc ? slC : slB) + r % (NP / 4) * 4;
    }
  }
  template <int STEP> __device__ __forceinline__ void move() {
    rowB += STEP * slB;
    rowC += STEP * slC;
  }
  __device__ __forceinline__ void load(const w2s_ssm_args& a, int vbc, int left, bool with_c, int w, int lane) {   // left: positions of the tile up to L
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int u0 = (k * W + w) * 64, isc = u0 >= HALF;
      if (u0 >= 2 * HALF || (isc && !with_c)) continue;
      const T* src = (isc ? rowC : rowB) + (unsigned)forgotten(off[k]);
      if (vbc == 2 && left >= TILE) {
        v[k] = *reinterpret_cast<const U*>(src);
      } else {
        const int r = u0 - isc * HALF + lane, n = r % (NP / 4) * 4;
        v[k] = V{};
        if (r / (NP / 4) < left && n < a.N) {
          if (vbc) {
            v[k] = *reinterpret_cast<const U*>(src);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n + e < a.N) v[k][e] = src[e];
          }
        }
      }
    }
  }
  __device__ __forceinline__ void store(float* lds, int live, int w, int lane) {   // live: positions of the tile up to the end; behind it zeros, whatever was there
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int u0 = (k * W + w) * 64, r = u0 - (u0 >= HALF) * HALF + lane;
      float4 o = make_float4((float)v[k][0], (float)v[k][1], (float)v[k][2], (float)v[k][3]);
      if (live < TILE && r / (NP / 4) >= live) o = make_float4(0.f, 0.f, 0.f, 0.f);
      if (u0 < 2 * HALF) *reinterpret_cast<float4*>(lds + (u0 + lane) * 4) = o;
    }
  }
};

// ------------------------------------------------------------------------------------------------------------------ forward
// GATE: z is there.  STATE: only the segment's end state (from zero) and its sum of delta
template <typename T, int NPL, bool STATE, bool GATE, bool WIDE> __global__ __launch_bounds__((FwdShape<NPL, WIDE>::W * 64), (FwdShape<NPL, WIDE>::SIMD)) void ssm_fwd_kernel(w2s_ssm_args a, Plan p) {
  constexpr int W = FwdShape<NPL, WIDE>::W, TT = FwdShape<NPL, WIDE>::TT, TILE = W * TT, NI = TT / 4, NP = 4 * NPL;
  __shared__ float bc[2][TILE * NP * 2];
  __shared__ float ex[W][2][64 * NPL];
  __shared__ float carry[2][64 * NPL];   // the state in front of a tile, from the last wave of the tile before
  const Where at = where_of(a, p);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), q = lane & 3;
  const bool on = at.cb * 16 + (lane >> 2) < p.dg;   // (a channel that does not exist walks along on the group's last one and writes nothing)
  const int ch = on ? at.cb * 16 + (lane >> 2) : p.dg - 1, dg0 = at.g * p.dg, d = dg0 + ch;
  const int n = mix_length(a.lengths, at.b, a.L), N = a.N, L = a.L;
  const int k0 = at.seg * p.tps, k1 = k0 + p.tps < p.ntile ? k0 + p.tps : p.ntile;
  float A[NPL], hc[NPL];
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const int s = q * NPL + j;
    A[j] = s < N ? a.A[(int64_t)d * N + s] * kLog2e : 0.0f;
    hc[j] = !STATE && w == W - 1 && s < N && a.h0 ? a.h0[((int64_t)at.b * a.D + d) * N + s] : 0.0f;
  }
  if (w == W - 1) {
    if (!STATE)
      for (int k = 0; k < at.seg; ++k) {   // the segments in front
        const int64_t r = ((int64_t)at.b * p.nseg + k) * a.D + d;
        const float S = p.segs[r];
#pragma unroll
        for (int j = 0; j < NPL; ++j) hc[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(A[j] * S), hc[j], p.segh[r * NP + q * NPL + j]);
      }
    mix_store<float, NPL>(&carry[0][lane * NPL], hc);
  }
  const float bias = a.dt_bias ? a.dt_bias[d] : 0.0f, Dp = a.Dp ? a.Dp[d] : 0.0f;
  const int t00 = k0 * TILE + w * TT;
  Column<const T> cu, cd, cz;
  Column<T> cy;
  cu.start(a.u, a.su_b, a.su_l, at.b, dg0, t00, q, ch);
  cd.start(a.dt, a.sdt_b, a.sdt_l, at.b, dg0, t00, q, ch);
  cz.start(a.z, a.sz_b, a.sz_l, at.b, dg0, t00, q, ch);
  cy.start(a.y, (int64_t)L * a.D, a.D, at.b, dg0, t00, q, ch);
  StageBC<T, NP, TILE, W> st;
  st.start(a, at, k0 * TILE, w, lane);
  T ru[NI], rd[NI], rz[NI];
  float Ssum = 0.0f;
  auto fetch = [&](int t0) {   // ... and on to the tile behind it
    const int left = L - t0 - w * TT;
    const bool whole = left >= TT;
    get_all(cu, whole, left, q, ru);
    get_all(cd, whole, left, q, rd);
    if (GATE) get_all(cz, whole, left, q, rz);
    st.load(a, p.vbc, L - t0, !STATE, w, lane);
    cu.template move<TILE>();
    cd.template move<TILE>();
    cz.template move<TILE>();
    st.template move<TILE>();
  };
  if (k0 < k1 && k0 * TILE < n) fetch(k0 * TILE);
  for (int k = k0; k < k1; ++k) {
    const int t0 = k * TILE, par = (k - k0) & 1, tw = t0 + w * TT;
    if (t0 >= n) {   // (the whole workgroup) behind the end
      if (!STATE) {
        const float zero[NI] = {};
        put_all(cy, L - tw >= TT, L - tw, q, on, zero);
        cy.template move<TILE>();
      }
      continue;
    }
    float u[NI], dl[NI], du[NI], z[NI], S = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const float raw = (float)rd[i] + bias;
      u[i] = (float)ru[i];
      dl[i] = a.softplus ? mix_softplus(raw) : raw;
      z[i] = (float)rz[i];
    }
    if (n - tw < TT) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const bool live = 4 * i + q < n - tw;
        u[i] = live ? u[i] : 0.0f;
        dl[i] = live ? dl[i] : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      du[i] = dl[i] * u[i];
      S += dl[i];
    }
    float* lds = bc[par];
    st.store(lds, n - t0, w, lane);
    __syncthreads();
    if (k + 1 < k1 && t0 + TILE < n) fetch(t0 + TILE);
    const float* Bs = lds + w * TT * NP + q * NPL;
    const float* Cs = Bs + TILE * NP;
    float dec[TT][NPL], h[NPL], e[NPL], P[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) e[j] = 0.0f;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      float Bv[NPL];
      mix_load<float, NPL>(Bs + t * NP, Bv);
      const float dt = quad_bcast(dl[t / 4], t & 3), x = quad_bcast(du[t / 4], t & 3);
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        dec[t][j] = __builtin_amdgcn_exp2f(dt * A[j]);
        e[j] = __builtin_fmaf(dec[t][j], e[j], x * Bv[j]);
      }
    }
    S = quad_sum(S);
    Ssum += S;
#pragma unroll
    for (int j = 0; j < NPL; ++j) P[j] = __builtin_amdgcn_exp2f(A[j] * S);
    mix_store<float, NPL>(&ex[w][0][lane * NPL], e);
    mix_store<float, NPL>(&ex[w][1][lane * NPL], P);
    __syncthreads();
    // h: the state in front of this wave's positions; the last wave goes on to the next tile's
    mix_load<float, NPL>(&carry[par][lane * NPL], h);
#pragma unroll(NPL < 8 ? 4 : NPL < 16 ? 2 : 1)
    for (int v = 0; v < w; ++v) {
      float x[NPL], y[NPL];
      mix_load<float, NPL>(&ex[v][0][lane * NPL], x);
      mix_load<float, NPL>(&ex[v][1][lane * NPL], y);
#pragma unroll
      for (int j = 0; j < NPL; ++j) h[j] = __builtin_fmaf(y[j], h[j], x[j]);
    }
    if (w == W - 1) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) hc[j] = __builtin_fmaf(P[j], h[j], e[j]);
      mix_store<float, NPL>(&carry[par ^ 1][lane * NPL], hc);
    }
    if constexpr (!STATE) {
      if (a.ckpt && ((w * TT) & (p.ck - 1)) == 0 && tw < n && on)   // (a power of two, at most a tile)
        mix_store<float, NPL>(a.ckpt + (((int64_t)at.b * p.nck + tw / p.ck) * a.D + dg0) * NP + (unsigned)(ch * NP + q * NPL), h);
      float y[NI];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        float Bv[NPL], Cv[NPL], s = 0.0f;
        mix_load<float, NPL>(Bs + t * NP, Bv);
        mix_load<float, NPL>(Cs + t * NP, Cv);
        const float x = quad_bcast(du[t / 4], t & 3);
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
          h[j] = __builtin_fmaf(dec[t][j], h[j], x * Bv[j]);
          s = __builtin_fmaf(Cv[j], h[j], s);
        }
        s = quad_sum(s);
        y[t / 4] = (t & 3) == 0 || q == (t & 3) ? s : y[t / 4];
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) y[i] = __builtin_fmaf(Dp, u[i], y[i]);
      if (GATE) {
#pragma unroll
        for (int i = 0; i < NI; ++i) y[i] *= z[i] * mix_sigmoid(z[i]);
      }
      if (n - tw < TT) {
#pragma unroll
        for (int i = 0; i < NI; ++i) y[i] = 4 * i + q < n - tw ? y[i] : 0.0f;
      }
      put_all(cy, L - tw >= TT, L - tw, q, on, y);
      cy.template move<TILE>();
    }
  }
  if constexpr (STATE) {
    __syncthreads();
    float* red = &ex[0][0][0];   // [wave][channel]
    if (q == 0) red[w * 16 + (lane >> 2)] = Ssum;
    __syncthreads();
    if (w == W - 1 && on) {
      const int64_t r = ((int64_t)at.b * p.nseg + at.seg) * a.D + d;
      float S = 0.0f;
      for (int v = 0; v < W; ++v) S += red[v * 16 + (lane >> 2)];
      if (q == 0) p.segs[r] = S;
      mix_store<float, NPL>(p.segh + r * NP + q * NPL, hc);
    }
  } else if (a.h_out && at.seg == p.nseg - 1 && w == W - 1 && on) {
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (q * NPL + j < N) a.h_out[((int64_t)at.b * a.D + d) * N + q * NPL + j] = hc[j];
  }
}

// ------------------------------------------------------------------------------------------------------------------ backward
// With e_t = a_t G_t, G_t = C_t gy'_t + e_{t+1} (gy' = gy silu(z)): du = delta sum_n G B + D gy', ddelta = sum_n e h_{t-1} A + u sum_n G B, dA = sum_t e h_{t-1} delta,
// dB = sum_channels G delta u, dC = sum_channels gy' h.  Tiles from the sequence's end; inside a tile the waves first walk both ways from zero (forward
// for h, backward for e), meet in LDS, and walk both ways again from the right ends, the states of the second walk staying in registers.  dB and dC are
// summed over the 16 channels of a workgroup by lane exchanges and over workgroups from `part_bc`; everything in a fixed order.
// STATE: only e at the segment's start (from zero) and the sum of delta.
template <typename T, int NPL, bool STATE, bool GATE, bool WIDE> __global__ __launch_bounds__((BwdShape<NPL, WIDE>::W * 64), (BwdShape<NPL, WIDE>::SIMD)) void ssm_bwd_kernel(w2s_ssm_args a, Plan p) {
  constexpr int W = BwdShape<NPL, WIDE>::W, TT = BwdShape<NPL, WIDE>::TT, TILE = W * TT, NI = TT / 4, NP = 4 * NPL, NX = STATE ? 2 : 3;
  __shared__ float bc[2][TILE * NP * 2];
  __shared__ float ex[W][NX][64 * NPL];
  __shared__ float carry[2][64 * NPL];   // e in front of a tile, from the first wave of the tile behind
  const Where at = where_of(a, p);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), q = lane & 3;
  const bool on = at.cb * 16 + (lane >> 2) < p.dg;   // (a channel that does not exist has a gradient of zero, so that it adds nothing to dB and dC)
  const int ch = on ? at.cb * 16 + (lane >> 2) : p.dg - 1, dg0 = at.g * p.dg, d = dg0 + ch;
  const int n = mix_length(a.lengths, at.b, a.L), N = a.N, L = a.L;
  const int k0 = at.seg * p.tps, k1 = k0 + p.tps < p.ntile ? k0 + p.tps : p.ntile;
  const bool has_gy = a.gy != nullptr;
  float A[NPL], ec[NPL], gA[NPL], gD = 0.0f, gb = 0.0f, Ssum = 0.0f;
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const int s = q * NPL + j;
    A[j] = s < N ? a.A[(int64_t)d * N + s] * kLog2e : 0.0f;
    ec[j] = !STATE && w == 0 && on && s < N && a.gh ? a.gh[((int64_t)at.b * a.D + d) * N + s] : 0.0f;
    gA[j] = 0.0f;
  }
  if (w == 0) {
    if (!STATE && on)
      for (int k = p.nseg - 1; k > at.seg; --k) {   // the segments behind
        const int64_t r = ((int64_t)at.b * p.nseg + k) * a.D + d;
        const float S = p.segs[r];
#pragma unroll
        for (int j = 0; j < NPL; ++j) ec[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(A[j] * S), ec[j], p.segh[r * NP + q * NPL + j]);
      }
    mix_store<float, NPL>(&carry[0][lane * NPL], ec);
  }
  const float bias = a.dt_bias ? a.dt_bias[d] : 0.0f, Dp = a.Dp ? a.Dp[d] : 0.0f;
  int kl = k1;   // tiles from kl on lie behind the end
  while (kl > k0 && (kl - 1) * TILE >= n) --kl;
  const int64_t LD = (int64_t)L * a.D;
  if (!STATE)
    for (int k = kl; k < k1; ++k) {
      const int tw = k * TILE + w * TT;
      const float zero[NI] = {};
      Column<T> c;
      c.start(a.gu, LD, a.D, at.b, dg0, tw, q, ch);
      put_all(c, false, L - tw, q, on, zero);
      c.start(a.gdt, LD, a.D, at.b, dg0, tw, q, ch);
      put_all(c, false, L - tw, q, on, zero);
      c.start(a.gz, LD, a.D, at.b, dg0, tw, q, ch);
      if (GATE) put_all(c, false, L - tw, q, on, zero);
    }
  const int t00 = (kl - 1) * TILE + w * TT;
  Column<const T> cu, cd, cz, cg;
  Column<T> co;   // one row pointer for the three outputs, which are alike: gdt and gz at fixed distances
  cu.start(a.u, a.su_b, a.su_l, at.b, dg0, t00, q, ch);
  cd.start(a.dt, a.sdt_b, a.sdt_l, at.b, dg0, t00, q, ch);
  cz.start(a.z, a.sz_b, a.sz_l, at.b, dg0, t00, q, ch);
  cg.start(a.gy, a.sg_b, a.sg_l, at.b, dg0, t00, q, ch);
  co.start(a.gu, LD, a.D, at.b, dg0, t00, q, ch);
  StageBC<T, NP, TILE, W> st;
  st.start(a, at, (kl - 1) * TILE, w, lane);
  T ru[NI], rd[NI], rz[NI], rg[NI];
  auto fetch = [&](int t0) {   // ... and on to the tile in front of it
    const int left = L - t0 - w * TT;
    const bool whole = left >= TT;
    if (!STATE) get_all(cu, whole, left, q, ru);
    get_all(cd, whole, left, q, rd);
    if (GATE) get_all(cz, whole, left, q, rz);
    if (has_gy) get_all(cg, whole, left, q, rg);
    st.load(a, p.vbc, L - t0, true, w, lane);
    cu.template move<-TILE>();
    cd.template move<-TILE>();
    cz.template move<-TILE>();
    cg.template move<-TILE>();
    st.template move<-TILE>();
  };
  // where a lane leaves its share of dB and dC (the walk's reduction below)
  const unsigned out_off = NPL < 4 ? ((lane >> 4) & 1) * NP + q * NPL + (lane >> 5) : (lane & 4 ? NP : 0) + q * NPL + ((lane >> 4) & 1) * 2 + (lane >> 5);
  const bool out_on = NPL < 4 ? (lane & 12) == 0 : (lane & 8) == 0;
  if (kl > k0) fetch((kl - 1) * TILE);
  for (int k = kl - 1; k >= k0; --k) {
    const int t0 = k * TILE, par = (kl - 1 - k) & 1, tw = t0 + w * TT;
    float u[NI], dl[NI], du[NI], slope[NI], gp[NI], gy[NI], z[NI], sz[NI], S = 0.0f, hi[NPL];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const float r = (float)rd[i] + bias;
      u[i] = STATE ? 0.0f : (float)ru[i];
      slope[i] = 1.0f;
      dl[i] = a.softplus ? mix_softplus(r, slope[i]) : r;
      gy[i] = has_gy ? (float)rg[i] : 0.0f;
      z[i] = (float)rz[i];
    }
    if (n - tw < TT || !on) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const bool live = 4 * i + q < n - tw && on;
        u[i] = live ? u[i] : 0.0f;
        dl[i] = live ? dl[i] : 0.0f;
        gy[i] = live ? gy[i] : 0.0f;
        z[i] = live ? z[i] : 0.0f;
        slope[i] = live ? slope[i] : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      du[i] = dl[i] * u[i];
      sz[i] = GATE ? mix_sigmoid(z[i]) : 0.0f;
      gp[i] = GATE ? gy[i] * z[i] * sz[i] : gy[i];
      S += dl[i];
    }
    float* lds = bc[par];
    st.store(lds, n - t0, w, lane);
    __syncthreads();
    if (STATE && k > k0) fetch(t0 - TILE);
    if constexpr (!STATE) mix_load<float, NPL>(a.ckpt + (((int64_t)at.b * p.nck + k) * a.D + dg0) * NP + (unsigned)forgotten(ch * NP + q * NPL), hi);
    const float* Bs = lds + forgotten(w * TT * NP + q * NPL);
    const float* Cs = Bs + TILE * NP;
    // (with 16 states a lane the decays do not fit beside the walk's own values: they are computed again wherever they are used)
    constexpr bool KEEP = STATE || NPL < 16;
    float dec[TT][NPL], e[NPL], h[NPL], P[NPL], own[NPL];
    auto decay = [&](int t, int j, float dt) { return KEEP ? dec[t][j] : __builtin_amdgcn_exp2f(dt * A[j]); };
#pragma unroll
    for (int j = 0; j < NPL; ++j) h[j] = own[j] = 0.0f;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      float Bv[NPL];
      if (!STATE) mix_load<float, NPL>(Bs + t * NP, Bv);
      const float dt = quad_bcast(dl[t / 4], t & 3), x = quad_bcast(du[t / 4], t & 3);
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        const float f = __builtin_amdgcn_exp2f(dt * A[j]);
        if (KEEP) dec[t][j] = f;
        if (!STATE) h[j] = __builtin_fmaf(f, h[j], x * Bv[j]);
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
      const float g = quad_bcast(gp[t / 4], t & 3), dt = quad_bcast(dl[t / 4], t & 3);
#pragma unroll
      for (int j = 0; j < NPL; ++j) own[j] = decay(t, j, dt) * __builtin_fmaf(Cv[j], g, own[j]);
      if (!KEEP) __builtin_amdgcn_sched_barrier(0);
    }
    S = quad_sum(S);
    Ssum += S;
#pragma unroll
    for (int j = 0; j < NPL; ++j) P[j] = __builtin_amdgcn_exp2f(A[j] * S);
    mix_store<float, NPL>(&ex[w][0][lane * NPL], P);
    mix_store<float, NPL>(&ex[w][1][lane * NPL], own);
    if constexpr (!STATE) mix_store<float, NPL>(&ex[w][NX - 1][lane * NPL], h);
    __syncthreads();
    // e: what arrives behind this wave's positions; the first wave goes on to what arrives behind the next tile
    mix_load<float, NPL>(&carry[par][lane * NPL], e);
#pragma unroll(NPL < 8 ? 4 : NPL < 16 ? 2 : 1)
    for (int v = W - 1; v > w; --v) {
      float x[NPL], y[NPL];
      mix_load<float, NPL>(&ex[v][0][lane * NPL], y);
      mix_load<float, NPL>(&ex[v][1][lane * NPL], x);
#pragma unroll
      for (int j = 0; j < NPL; ++j) e[j] = __builtin_fmaf(y[j], e[j], x[j]);
    }
    if (w == 0) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) ec[j] = __builtin_fmaf(P[j], e[j], own[j]);
      mix_store<float, NPL>(&carry[par ^ 1][lane * NPL], ec);
    }
    if constexpr (!STATE) {
#pragma unroll(NPL < 8 ? 4 : NPL < 16 ? 2 : 1)
      for (int v = 0; v < w; ++v) {
        float x[NPL], y[NPL];
        mix_load<float, NPL>(&ex[v][0][lane * NPL], y);
        mix_load<float, NPL>(&ex[v][NX - 1][lane * NPL], x);
#pragma unroll
        for (int j = 0; j < NPL; ++j) hi[j] = __builtin_fmaf(y[j], hi[j], x[j]);
      }
      // The second walk in parts of HALF positions from the last part to the first, so that only a part's states are in registers; h first reaches a
      // part's start without keeping any.
      constexpr int HALF = NPL <= 4 ? TT : NPL == 8 ? 2 : 1, PARTS = TT / HALF, JB = NPL < 4 ? NPL : 4;
      constexpr bool LATE = NPL <= 4 && TT > 4;   // a lane's shares of dB and dC wait in registers for the walk's end, which then has no branch inside
      float oB[NI], oG[NI], oY[NI], share[TT];
      forget(gp);
      if (!KEEP) forget(A);
      auto forward = [&](const float* x, int t, float* to) {
        float Bv[NPL];
        mix_load<float, NPL>(Bs + t * NP, Bv);
        const float v = quad_bcast(du[t / 4], t & 3), dt = quad_bcast(dl[t / 4], t & 3);
#pragma unroll
        for (int j = 0; j < NPL; ++j) to[j] = __builtin_fmaf(decay(t, j, dt), x[j], v * Bv[j]);
        if (!KEEP) __builtin_amdgcn_sched_barrier(0);
      };
      float* out = p.part_bc + ((((int64_t)at.cb * a.B + at.b) * L + tw) * a.G + at.g) * 2 * NP;   // (written where the position exists only)
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
        float hs[HALF][NPL];
#pragma unroll
        for (int t = 0; t < HALF; ++t) forward(t ? hs[t ? t - 1 : 0] : (part ? h : hi), part * HALF + t, hs[t]);
        forget(du);
        forget(dl);
        Bs = lds + forgotten(w * TT * NP + q * NPL);
        Cs = Bs + TILE * NP;
#pragma unroll
        for (int t = part * HALF + HALF - 1; t >= part * HALF; --t) {
          const int th = t - part * HALF;
          float* row = out + (int64_t)t * a.G * 2 * NP;
          float sB = 0.0f, sG = 0.0f, sY = 0.0f;
          const float g = quad_bcast(gp[t / 4], t & 3), x = quad_bcast(du[t / 4], t & 3), dt = quad_bcast(dl[t / 4], t & 3);
#pragma unroll
          for (int j0 = 0; j0 < NPL; j0 += JB) {
            float Bv[JB], Cv[JB], pb[JB], pc[JB];
            mix_load<float, JB>(Bs + t * NP + j0, Bv);
            mix_load<float, JB>(Cs + t * NP + j0, Cv);
#pragma unroll
            for (int jj = 0; jj < JB; ++jj) {
              const int j = j0 + jj;
              const float ht = hs[th][j];
              const float G = __builtin_fmaf(Cv[jj], g, e[j]);
              e[j] = decay(t, j, dt) * G;
              const float eh = e[j] * (th ? hs[th ? th - 1 : 0][j] : part ? h[j] : hi[j]);
              gA[j] = __builtin_fmaf(eh, dt, gA[j]);
              sG = __builtin_fmaf(eh, A[j], sG);
              sB = __builtin_fmaf(G, Bv[jj], sB);
              sY = __builtin_fmaf(Cv[jj], ht, sY);
              pb[jj] = G * x;
              pc[jj] = g * ht;
            }
            // sums over the 16 quads; the states of dB and of dC end up spread over the rows of 16 lanes
            float v;
            if constexpr (JB == 4) {
              const float sb = sum_quads_of_row(fold16(fold32(pb[0], pb[1]), fold32(pb[2], pb[3])));
              const float sc = sum_quads_of_row(fold16(fold32(pc[0], pc[1]), fold32(pc[2], pc[3])));
              v = lane & 4 ? sc : sb;
            } else {
              v = sum_quads_of_row(fold16(fold32(pb[0], pb[1]), fold32(pc[0], pc[1])));
            }
            if (LATE) share[t] = v;
            else if (out_on && t < n - tw) (row + j0)[(unsigned)forgotten(out_off)] = v;
          }
          const bool mine = q == (t & 3) || (t & 3) == 3;   // (the highest of a lane's four comes first; the others then choose)
          const float vB = quad_sum(sB), vG = quad_sum(sG), vY = GATE ? quad_sum(sY) : 0.0f;
          oB[t / 4] = mine ? vB : oB[t / 4];
          oG[t / 4] = mine ? vG : oG[t / 4];
          oY[t / 4] = mine ? vY : oY[t / 4];
          if (!LATE) __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (LATE && out_on) {
        const int step = a.G * 2 * NP;
        if (n - tw >= TT) {
#pragma unroll
          for (int t = 0; t < TT; ++t) (out + t * step)[(unsigned)forgotten(out_off)] = share[t];
        } else {
#pragma unroll
          for (int t = 0; t < TT; ++t)
            if (t < n - tw) (out + t * step)[(unsigned)forgotten(out_off)] = share[t];
        }
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {   // (behind the end u, delta, its slope, gy and gy' are zero, and so are these)
        const float gd = slope[i] * __builtin_fmaf(kLn2, oG[i], u[i] * oB[i]);
        oB[i] = __builtin_fmaf(dl[i], oB[i], Dp * gp[i]);
        gD = __builtin_fmaf(gp[i], u[i], gD);
        gb += gd;
        oG[i] = gd;
        if (GATE) oY[i] = gy[i] * __builtin_fmaf(Dp, u[i], oY[i]) * sz[i] * (1.0f + z[i] * (1.0f - sz[i]));
      }
      const bool whole = L - tw >= TT;
      put_all(co, whole, L - tw, q, on, oB);
      Column<T> c = co;
      c.row = co.row + ((T*)a.gdt - (T*)a.gu);
      put_all(c, whole, L - tw, q, on, oG);
      c.row = co.row + ((T*)a.gz - (T*)a.gu);
      if (GATE) put_all(c, whole, L - tw, q, on, oY);
      co.template move<-TILE>();
    }
  }
  __syncthreads();
  float* red = &ex[0][0][0];
  if constexpr (STATE) {
    if (q == 0) red[w * 16 + (lane >> 2)] = Ssum;
    __syncthreads();
    if (w == 0 && on) {
      const int64_t r = ((int64_t)at.b * p.nseg + at.seg) * a.D + d;
      float S = 0.0f;
      for (int v = 0; v < W; ++v) S += red[v * 16 + (lane >> 2)];
      if (q == 0) p.segs[r] = S;
      mix_store<float, NPL>(p.segh + r * NP + q * NPL, ec);
    }
  } else {
    // dA, dD, d(bias) of the workgroup: over the waves in order
    gD = quad_sum(gD);
    gb = quad_sum(gb);
    mix_store<float, NPL>(&ex[w][0][lane * NPL], gA);
    if (q < 2) ex[w][1][(lane >> 2) * 2 + q] = q ? gb : gD;
    __syncthreads();
    if (w == 0 && on) {
      const int64_t r = ((int64_t)at.b * p.nseg + at.seg) * a.D + d;
      float s[NPL] = {}, x = 0.0f;
      for (int v = 0; v < W; ++v) {
        float y[NPL];
        mix_load<float, NPL>(&ex[v][0][lane * NPL], y);
#pragma unroll
        for (int j = 0; j < NPL; ++j) s[j] += y[j];
        if (q < 2) x += ex[v][1][(lane >> 2) * 2 + q];
      }
      float* o = p.part_a + r * (N + 2);
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if (q * NPL + j < N) o[q * NPL + j] = s[j];
      if (q < 2) o[N + q] = x;
      if (a.gh0 && at.seg == 0)
#pragma unroll
        for (int j = 0; j < NPL; ++j)
          if (q * NPL + j < N) a.gh0[((int64_t)at.b * a.D + d) * N + q * NPL + j] = ec[j];
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

// gA [D][N], gD, gbias [D] from the workgroups' shares
__global__ __launch_bounds__(1024) void ssm_reduce_a_kernel(w2s_ssm_args a, int nparts, const float* part) {
  __shared__ float red[64][17];
  const int64_t C = (int64_t)a.D * (a.N + 2), i = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
  const float v = mix_part_sum(part, nparts, C, i, red);
  if (threadIdx.x >= 16 || i >= C) return;
  const int n = (int)(i % (a.N + 2));
  const int64_t d = i / (a.N + 2);
  if (n < a.N) a.gA[d * a.N + n] = v;
  else if (n == a.N) { if (a.gD) a.gD[d] = v; }
  else if (a.gbias) a.gbias[d] = v;
}

// One position.  Bound by HBM: 8 N bytes of state a channel, read and written.  Four lanes share a channel; with N a multiple of 4 they read its states as
// consecutive 16-byte pieces (256 x 512 channels, N = 16: 5.7 us against 6.9 one by one; 2048 x 512: 27 us = 5.5 TB/s against 35).
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
      mix_gload<float, VEC>(a.h0 + item * N + j, h);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = 0.0f;
    }
    mix_gload<float, VEC>(a.A + (int64_t)d * N + j, A);
    mix_gload<T, VEC>(Bt + j, Bv);
    mix_gload<T, VEC>(Ct + j, Cv);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      h[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(dl * A[i]), h[i], du * Bv[i]);
      y = __builtin_fmaf(Cv[i], h[i], y);
    }
    mix_gstore<float, VEC>(a.h_out + item * N + j, h);
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

// rows within a tile are addressed by 32-bit offsets from the tile's 64-bit base: a position's stride stays below 2^22 elements (128 rows of 4 bytes: 2 GiB)
bool near(int64_t s) { return s >= 0 && s < (1 << 22); }

bool valid(const w2s_ssm_args* a) {
  return a && near(a->su_l) && near(a->sdt_l) && near(a->sz_l) && near(a->sB_l) && near(a->sC_l) && near(a->sg_l) && near(a->D) && a->A && a->B >= 0 && a->L >= 0 &&
         a->L <= (1 << 30) && a->D >= 1 && a->N >= 1 && a->N <= 64 && a->G >= 1 && a->D % a->G == 0 && a->dtype >= 0 && a->dtype <= 2;
}
bool launches(int64_t blocks, int threads) { return blocks * threads <= 0xffffffffLL; }   // a launch has fewer than 2^32 threads

int npl_of(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }
// Segments a sequence is cut into.  Cutting costs a second walk for the end states (half of a whole one), so it pays only where the workgroups of whole
// sequences leave half of the 256 CUs idle or more: then up to two workgroups a CU, of two tiles at least.  fp32, L = 960, D = 256, N = 16, cut / whole, forward and
// with the backward: 16 workgroups 20 / 36 and 66 / 134 us, 128 workgroups 33 / 37 and 111 / 139 us, 192 workgroups 45 / 37 and 149 / 140 us; one row of
// 16384 x 512 bf16 113 / 515 and 352 / 1967 us.
int segments(int64_t blocks, int ntile) {
  if (blocks <= 0 || blocks > 128 || ntile < 4) return 1;
  int64_t n = 512 / blocks;
  if (n > ntile / 2) n = ntile / 2;
  if (n > 64) n = 64;
  return n < 2 ? 1 : (int)n;
}

bool wide(int NPL, int64_t blocks, int nseg) { return NPL <= 4 && nseg == 1 && blocks <= 256; }

template <int NPL> Plan plan_of(const w2s_ssm_args* a, bool backward, bool* is_wide) {
  Plan p{};
  p.dg = a->D / a->G;
  p.ncb = (p.dg + 15) / 16;
  const int64_t blocks = (int64_t)a->B * a->G * p.ncb;
  auto tiles = [&](int tile) { return (int)(((int64_t)a->L + tile - 1) / tile); };
  constexpr int ft = FwdShape<NPL, false>::W * FwdShape<NPL, false>::TT, ftw = FwdShape<NPL, true>::W * FwdShape<NPL, true>::TT;
  constexpr int bt = BwdShape<NPL, false>::W * BwdShape<NPL, false>::TT, btw = BwdShape<NPL, true>::W * BwdShape<NPL, true>::TT;
  const bool bw = wide(NPL, blocks, segments(blocks, tiles(bt)));
  p.ck = bw ? btw : bt;
  p.nck = tiles(p.ck);
  p.nseg = segments(blocks, tiles(backward ? bt : ft));
  *is_wide = backward ? bw : wide(NPL, blocks, p.nseg);
  p.ntile = backward ? p.nck : tiles(*is_wide ? ftw : ft);
  p.tps = (p.ntile + p.nseg - 1) / p.nseg;
  if (p.tps > 0) p.nseg = (p.ntile + p.tps - 1) / p.tps;
  if (p.nseg < 1) p.nseg = 1;
  p.vbc = a->N == 4 * NPL ? 2 : a->N % 4 == 0 ? 1 : 0;
  return p;
}

int64_t seg_floats(const w2s_ssm_args* a, const Plan& p, int np) { return p.nseg > 1 ? (int64_t)a->B * p.nseg * a->D * (np + 1) : 0; }
int64_t bc_floats(const w2s_ssm_args* a, const Plan& p, int np) { return (int64_t)p.ncb * a->B * a->L * a->G * 2 * np; }
int64_t a_floats(const w2s_ssm_args* a, const Plan& p) { return ((int64_t)a->B * p.nseg * a->D * (a->N + 2) + 3) / 4 * 4; }   // (what follows stays 16-byte aligned)

template <int NPL> int64_t ws_floats(const w2s_ssm_args* a, bool backward) {
  bool w;
  const Plan p = plan_of<NPL>(a, backward, &w);
  return seg_floats(a, p, 4 * NPL) + (backward ? bc_floats(a, p, 4 * NPL) + a_floats(a, p) : 0);
}

template <int NPL> int64_t ckpt_floats(const w2s_ssm_args* a) {
  bool w;
  return (int64_t)a->B * plan_of<NPL>(a, false, &w).nck * a->D * 4 * NPL;
}

template <typename T, int NPL, bool GATE> int scan_fwd(const w2s_ssm_args* a, hipStream_t st) {
  bool w;
  Plan p = plan_of<NPL>(a, false, &w);
  const int64_t blocks = (int64_t)a->B * a->G * p.ncb * p.nseg;
  if (!launches(blocks, 1024)) return W2S_EINVAL;
  if (p.nseg > 1) {
    if (!a->ws) return W2S_EINVAL;
    p.segh = (float*)a->ws;
    p.segs = p.segh + (int64_t)a->B * p.nseg * a->D * 4 * NPL;
    ssm_fwd_kernel<T, NPL, true, false, false><<<(unsigned)blocks, FwdShape<NPL, false>::W * 64, 0, st>>>(*a, p);
  }
  constexpr bool V = NPL <= 4;
  if (w) ssm_fwd_kernel<T, NPL, false, GATE, V><<<(unsigned)blocks, FwdShape<NPL, V>::W * 64, 0, st>>>(*a, p);
  else ssm_fwd_kernel<T, NPL, false, GATE, false><<<(unsigned)blocks, FwdShape<NPL, false>::W * 64, 0, st>>>(*a, p);
  W2S_CHECK_LAUNCH();
  return W2S_OK;
}

template <typename T, int NPL, bool GATE> int scan_bwd(const w2s_ssm_args* a, hipStream_t st) {
  bool w;
  Plan p = plan_of<NPL>(a, true, &w);
  const int64_t blocks = (int64_t)a->B * a->G * p.ncb * p.nseg;
  const int64_t rows = (int64_t)a->B * a->L * a->G, nbc = (rows * (2 * NPL) + 255) / 256, na = ((int64_t)a->D * (a->N + 2) + 15) / 16;
  if (!launches(blocks, 512) || !launches(nbc, 256) || !launches(na, 1024)) return W2S_EINVAL;
  p.part_bc = (float*)a->ws;
  p.part_a = p.part_bc + bc_floats(a, p, 4 * NPL);
  p.segh = p.part_a + a_floats(a, p);
  p.segs = p.segh + (int64_t)a->B * p.nseg * a->D * 4 * NPL;
  if (blocks) {
    constexpr bool V = NPL <= 4;
    if (p.nseg > 1) ssm_bwd_kernel<T, NPL, true, GATE, false><<<(unsigned)blocks, BwdShape<NPL, false>::W * 64, 0, st>>>(*a, p);
    if (w) ssm_bwd_kernel<T, NPL, false, GATE, V><<<(unsigned)blocks, BwdShape<NPL, V>::W * 64, 0, st>>>(*a, p);
    else ssm_bwd_kernel<T, NPL, false, GATE, false><<<(unsigned)blocks, BwdShape<NPL, false>::W * 64, 0, st>>>(*a, p);
  }
  if (nbc) ssm_reduce_bc_kernel<T><<<(unsigned)nbc, 256, 0, st>>>(*a, p.ncb, 4 * NPL, p.part_bc);
  ssm_reduce_a_kernel<<<(unsigned)na, 1024, 0, st>>>(*a, a->B * p.nseg, p.part_a);
  W2S_CHECK_LAUNCH();
  return W2S_OK;
}

template <typename T, int NPL> int by_gate(const w2s_ssm_args* a, bool backward, hipStream_t st) {
  if (a->z) return backward ? scan_bwd<T, NPL, true>(a, st) : scan_fwd<T, NPL, true>(a, st);
  return backward ? scan_bwd<T, NPL, false>(a, st) : scan_fwd<T, NPL, false>(a, st);
}

template <typename T> int by_states(const w2s_ssm_args* a, bool backward, hipStream_t st) {
  switch (npl_of(a->N)) {
    case 2: return by_gate<T, 2>(a, backward, st);
    case 4: return by_gate<T, 4>(a, backward, st);
    case 8: return by_gate<T, 8>(a, backward, st);
    default: return by_gate<T, 16>(a, backward, st);
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
  if (!launches(blocks, 256)) return W2S_EINVAL;
  if (a->N % 4 == 0) ssm_step_kernel<T, 4><<<(unsigned)blocks, 256, 0, st>>>(*a);
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
