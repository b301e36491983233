// Selective scan, forward:
//
//   delta = softplus(dt + dt_bias),  h_t = exp(delta_t A) h_{t-1} + delta_t x_t B_t,
//   y_t = (C_t . h_t + skip x_t) silu(z_t)
//
// S exponentials a (step, row, channel) on the special function units, 16 a clock and SM, against
// 8 to 16 bytes of sequences: for S = 16 those units bound it, not HBM.
#include <algorithm>

#include "selective_scan.cuh"

namespace hb {
namespace scan {
namespace {

// A channel's states lie in Q lanes, four in each, for the whole sequence.  The block stages a tile
// of TT steps: (delta, delta x) per channel and B, C per step, and walks it; the next tile's loads
// are under way meanwhile.  The Q partial sums of C . h are added for Q steps together.
template <typename T, int Q, int THREADS>
struct Fwd {
  static constexpr int CB = THREADS / Q;
  static constexpr int TT = Q <= 2 ? 8 : Q <= 16 ? 16 : 32;
  static constexpr int PER = TT * CB / THREADS;      // staged (step, channel) pairs of a thread
  static constexpr int SP = Q * NS;
  static constexpr int PB = (TT * SP + THREADS - 1) / THREADS;
  static constexpr int YS = CB + 32 / Q;             // row of y sums, shifted so that lanes miss each other's banks
};

template <typename T, int Q, int THREADS>
__global__ void __launch_bounds__(THREADS) scan_fwd(Args<T> a) {
  using F = Fwd<T, Q, THREADS>;
  constexpr int CB = F::CB, TT = F::TT, PER = F::PER, SP = F::SP, PB = F::PB, YS = F::YS;
  __shared__ float2 dd[TT][CB];
  __shared__ __align__(16) float Bs[TT][SP], Cs[TT][SP];
  __shared__ float ys[TT][YS];
  const Place at(a, CB);
  const int tid = threadIdx.x, lane = tid % 32;
  const int q = tid % Q, c = tid / Q, s0 = q * NS;
  const int n = at.n, len = row_length(a.lengths, n, a.T_);
  // staging: pairs e = i * THREADS + tid, step e / CB, channel e % CB
  const int cs = tid % CB, ts = tid / CB;
  const bool has = cs < at.count;
  const int ds = at.d0 + (has ? cs : 0);
  const float bias = has && a.dt_bias ? a.dt_bias[ds] : 0.f, skip = has && a.skip ? a.skip[ds] : 0.f;

  float A[NS], h[NS];
  const bool mine = c < at.count;
  const long long row = ((long long)n * a.D + at.d0 + (mine ? c : 0)) * a.S;
#pragma unroll
  for (int i = 0; i < NS; ++i) A[i] = h[i] = 0.f;
  if (mine) {
    load_states(a.A + (long long)(at.d0 + c) * a.S, s0, a.S, A);
    if (a.state) load_states(a.state + row, s0, a.S, h);
  }
#pragma unroll
  for (int i = 0; i < NS; ++i) A[i] *= LOG2E;

  float xn[PER], dn[PER], zn[PER], bn[PB], cn[PB];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int t = t0 + ts + i * (THREADS / CB);
      const bool ok = has && t < len;
      xn[i] = ok ? ld(a.x.at(t, n) + ds) : 0.f;
      dn[i] = ok ? ld(a.dt.at(t, n) + ds) : 0.f;
      zn[i] = ok && a.z.p ? ld(a.z.at(t, n) + ds) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const int e = i * THREADS + tid, t = t0 + e / SP, s = e % SP;
      const bool ok = e < TT * SP && t < len && s < a.S;
      bn[i] = ok ? ld(a.B.at(t, n) + at.g * a.B_g + s) : 0.f;
      cn[i] = ok ? ld(a.C.at(t, n) + at.g * a.C_g + s) : 0.f;
    }
  };
  fetch(0);
  for (int t0 = 0; t0 < a.T_; t0 += TT) {
    float x[PER], z[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = ts + i * (THREADS / CB);
      const float v = dn[i] + bias;
      const float delta = t0 + k >= len ? 0.f : a.softplus ? softplus(v) : v;  // 0: the state stays
      x[i] = xn[i];
      z[i] = zn[i];
      dd[k][cs] = make_float2(delta, delta * x[i]);
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const int e = i * THREADS + tid;
      if (e < TT * SP) {
        Bs[e / SP][e % SP] = bn[i];
        Cs[e / SP][e % SP] = cn[i];
      }
    }
    __syncthreads();
    if (t0 + TT < a.T_) fetch(t0 + TT);
    constexpr int GR = Q < CKPT ? CKPT : Q;  // steps between two sums over the lanes
#pragma unroll 1
    for (int k0 = 0; k0 < TT; k0 += GR) {
      float y[GR];
#pragma unroll
      for (int k = 0; k < GR; ++k) {
        if (k % CKPT == 0 && a.checkpoints && mine && t0 + k0 + k < a.T_)
          store_states(a.checkpoints + (long long)((t0 + k0 + k) / CKPT) * a.N * a.D * a.S + row, s0, a.S, h);
        const float2 w = dd[k0 + k][c];
        const float4 b = *reinterpret_cast<const float4*>(&Bs[k0 + k][s0]);
        const float4 g = *reinterpret_cast<const float4*>(&Cs[k0 + k][s0]);
        h[0] = fmaf(exp2_fast(w.x * A[0]), h[0], w.y * b.x);
        h[1] = fmaf(exp2_fast(w.x * A[1]), h[1], w.y * b.y);
        h[2] = fmaf(exp2_fast(w.x * A[2]), h[2], w.y * b.z);
        h[3] = fmaf(exp2_fast(w.x * A[3]), h[3], w.y * b.w);
        y[k] = fmaf(h[0], g.x, h[1] * g.y) + fmaf(h[2], g.z, h[3] * g.w);
      }
      bool owner;
      const int first = lane_sums<GR, Q, 1>(y, lane, owner);
      if (owner)
#pragma unroll
        for (int i = 0; i < GR / Q; ++i) ys[k0 + first + i][c] = y[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = ts + i * (THREADS / CB), t = t0 + k;
      if (!has || t >= a.T_) continue;
      float v = fmaf(skip, x[i], ys[k][cs]);
      if (a.z.p) v *= silu(z[i]);
      st(a.y.at(t, n) + ds, t < len ? v : 0.f);
    }
  }
  if (mine && a.final_state) store_states(a.final_state + row, s0, a.S, h);
}

// A single step: the states are read and written once, so HBM (or, for few rows, the launch) bounds it.
// Q lanes of four states per (row, channel).
template <typename T, int Q>
__global__ void __launch_bounds__(256) scan_step(Args<T> a) {
  const long long pair = ((long long)blockIdx.x * 256 + threadIdx.x) / Q;
  const int lane = threadIdx.x % 32, s0 = (threadIdx.x % Q) * NS;
  const bool ok = pair < (long long)a.N * a.D;
  const int n = ok ? (int)(pair / a.D) : 0, d = ok ? (int)(pair % a.D) : 0, g = d / a.per;
  const bool live = row_length(a.lengths, n, 1) > 0;
  float A[NS], h[NS] = {0.f, 0.f, 0.f, 0.f};
  load_states(a.A + (long long)d * a.S, s0, a.S, A);
  const long long row = ((long long)n * a.D + d) * a.S;
  if (a.state) load_states(a.state + row, s0, a.S, h);
  float x = 0.f, y = 0.f;
  if (live) {
    x = ld(a.x.at(0, n) + d);
    const float v = ld(a.dt.at(0, n) + d) + (a.dt_bias ? a.dt_bias[d] : 0.f);
    const float delta = a.softplus ? softplus(v) : v;
    const T *B = a.B.at(0, n) + g * a.B_g, *C = a.C.at(0, n) + g * a.C_g;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if (s0 + i >= a.S) continue;
      h[i] = fmaf(exp2_fast(delta * A[i] * LOG2E), h[i], delta * x * ld(B + s0 + i));
      y = fmaf(h[i], ld(C + s0 + i), y);
    }
  }
  if (ok && a.final_state) store_states(a.final_state + row, s0, a.S, h);
#pragma unroll
  for (int o = Q / 2; o > 0; o /= 2) y += __shfl_xor_sync(0xffffffffu, y, o);
  if (ok && lane % Q == 0) {
    y = live ? fmaf(a.skip ? a.skip[d] : 0.f, x, y) : 0.f;
    if (live && a.z.p) y *= silu(ld(a.z.at(0, n) + d));
    st(a.y.at(0, n) + d, y);
  }
}

template <typename T, int Q>
int launch(const haste_b200_selective_scan& a, cudaStream_t s) {
  if (a.T == 1 && !a.checkpoints) {
    const Args<T> k = pack<T>(a, 1);
    scan_step<T, Q><<<ceil_div((long long)a.N * a.D * Q, 256), 256, 0, s>>>(k);
  } else {
    constexpr int THREADS = Q >= 16 ? 256 : 128;
    const Args<T> k = pack<T>(a, THREADS / Q);
    scan_fwd<T, Q, THREADS><<<a.N * a.G * k.ctiles, THREADS, 0, s>>>(k);
  }
  HB_LAUNCH_OK();
  count_launch(1);
  return HASTE_B200_OK;
}

template <typename T>
int by_lanes(const haste_b200_selective_scan& a, cudaStream_t s) {
  switch (lanes(a.S)) {
    case 1: return launch<T, 1>(a, s);
    case 2: return launch<T, 2>(a, s);
    case 4: return launch<T, 4>(a, s);
    case 8: return launch<T, 8>(a, s);
    case 16: return launch<T, 16>(a, s);
    default: return launch<T, 32>(a, s);
  }
}

}  // namespace

int check(const haste_b200_selective_scan& a, bool backward) {
  HB_REQUIRE(storage_dtype(a.dtype), "dtype");
  HB_REQUIRE(a.T >= 0 && a.N >= 0 && a.D >= 0, "T,N,D");
  HB_REQUIRE(a.S >= 1 && a.S <= 128, "S must be 1..128");
  HB_REQUIRE(a.G >= 1 && a.D % a.G == 0, "G must divide D");
  HB_REQUIRE((long long)a.D * (a.S + 2) < (1LL << 31) && (long long)a.N * a.D < (1LL << 31), "N*D too large");
  HB_REQUIRE((long long)a.N * a.D * a.S < (1LL << 37), "N*D*S too large");
  if (a.N == 0 || a.D == 0) return HASTE_B200_OK;
  HB_REQUIRE(a.A, "null pointer");
  if (backward) HB_REQUIRE(a.dA && a.scratch, "null pointer");
  if (a.T == 0) return HASTE_B200_OK;
  HB_REQUIRE(a.x.data && a.dt.data && a.B.data && a.C.data, "null pointer");
  if (backward) {
    HB_REQUIRE(a.checkpoints && a.dy.data && a.dx.data && a.ddt.data && a.dB.data && a.dC.data, "null pointer");
    HB_REQUIRE(!a.z.data == !a.dz.data, "dz goes with z");
  } else {
    HB_REQUIRE(a.y.data, "null pointer");
  }
  return HASTE_B200_OK;
}

}  // namespace scan

int selective_scan_forward(const haste_b200_selective_scan& a, cudaStream_t s) {
  HB_TRY(scan::check(a, false));
  if (a.N == 0 || a.D == 0) return HASTE_B200_OK;
  ProfScope p(PH_REC_FWD, s);
  if (a.dtype == HASTE_B200_F32) return scan::by_lanes<float>(a, s);
  if (a.dtype == HASTE_B200_BF16) return scan::by_lanes<__nv_bfloat16>(a, s);
  return scan::by_lanes<__half>(a, s);
}

long long selective_scan_checkpoints(const haste_b200_selective_scan& a) {
  if (a.T <= 0 || a.N <= 0 || a.D <= 0 || a.S <= 0) return 0;
  return (long long)ceil_div(a.T, scan::CKPT) * a.N * a.D * a.S;
}

}  // namespace hb
