// Selective scan, backward.  With dy already multiplied by silu(z), from the last step to the first:
//
//   lam_t = C_t dy_t + a_{t+1} lam_{t+1}          a_t = exp(delta_t A)
//   dC_t = sum_d dy_t h_t,   dB_t = sum_d lam_t delta_t x_t
//   dx_t = delta_t (lam_t . B_t) + skip dy_t
//   ddelta_t = x_t (lam_t . B_t) + lam_t . (A a_t h_{t-1}),   dA = sum_t lam_t delta_t a_t h_{t-1}
//
// The forward pass left the state in front of every CKPT steps; a thread computes those steps' states
// and decays again, keeps them in registers, and walks back over them.
#include <algorithm>

#include "selective_scan.cuh"

namespace hb {
namespace scan {
namespace {

constexpr int THREADS = 128;

// Threads and channels as in the forward kernel.  The sums over channels (dB, dC) are added over the
// lanes of a warp, over the warps in shared memory, and over the blocks from partial rows
// [ctiles][T][N][G][2][SP] in a fixed order.
template <typename T, int Q>
__global__ void __launch_bounds__(THREADS) scan_bwd(Args<T> a) {
  constexpr int CB = THREADS / Q, TT = CKPT, SP = Q * NS, WARPS = THREADS / 32;
  constexpr int PER = (TT * CB + THREADS - 1) / THREADS;
  constexpr int PB = (TT * SP + THREADS - 1) / THREADS;
  constexpr int STEP = THREADS / CB;     // = Q: staged steps lie Q apart in a thread
  constexpr int LANES = 32 / Q;          // channels of a warp
  __shared__ float4 in[TT][CB];          // delta, delta x, dy
  __shared__ float out[3][TT][CB + 1];   // C . h, lam . B, lam . (A a h)
  __shared__ __align__(16) float Bs[TT][SP], Cs[TT][SP];
  __shared__ float red[WARPS][TT][2 * SP];
  const Place at(a, CB);
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int q = tid % Q, c = tid / Q, s0 = q * NS;
  const int n = at.n, len = row_length(a.lengths, n, a.T_);
  const int ct = blockIdx.x % a.ctiles;
  const int cs = tid % CB, ts = tid / CB;
  const bool has = cs < at.count;
  const int ds = at.d0 + (has ? cs : 0);
  const float bias = has && a.dt_bias ? a.dt_bias[ds] : 0.f, skip = has && a.skip ? a.skip[ds] : 0.f;
  const bool mine = c < at.count;
  const long long row = ((long long)n * a.D + at.d0 + (mine ? c : 0)) * a.S;
  float A[NS], carry[NS], dA[NS];  // carry: a_{t+1} lam_{t+1}
#pragma unroll
  for (int i = 0; i < NS; ++i) A[i] = carry[i] = dA[i] = 0.f;
  if (mine) {
    load_states(a.A + (long long)(at.d0 + c) * a.S, s0, a.S, A);
    if (a.dfinal) load_states(a.dfinal + row, s0, a.S, carry);
  }
  float dskip = 0.f, dbias = 0.f;
  for (int t0 = a.T_ > 0 ? (a.T_ - 1) / TT * TT : -TT; t0 >= 0; t0 -= TT) {
    float x[PER], raw[PER], z[PER], dy[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = ts + i * STEP, t = t0 + k;
      const bool ok = has && k < TT && t < len;
      x[i] = ok ? ld(a.x.at(t, n) + ds) : 0.f;
      raw[i] = ok ? ld(a.dt.at(t, n) + ds) + bias : 0.f;
      z[i] = ok && a.z.p ? ld(a.z.at(t, n) + ds) : 0.f;
      dy[i] = ok ? ld(a.dy.at(t, n) + ds) : 0.f;
      const float delta = !ok ? 0.f : a.softplus ? softplus(raw[i]) : raw[i];
      const float g = a.z.p ? dy[i] * silu(z[i]) : dy[i];
      if (k < TT) in[k][cs] = make_float4(delta, delta * x[i], g, 0.f);
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const int e = i * THREADS + tid, k = e / SP, s = e % SP, t = t0 + k;
      if (e >= TT * SP) break;
      const bool ok = t < len && s < a.S;
      Bs[k][s] = ok ? ld(a.B.at(t, n) + at.g * a.B_g + s) : 0.f;
      Cs[k][s] = ok ? ld(a.C.at(t, n) + at.g * a.C_g + s) : 0.f;
    }
    float h0[NS] = {0.f, 0.f, 0.f, 0.f};
    if (mine) load_states(a.checkpoints + (long long)(t0 / CKPT) * a.N * a.D * a.S + row, s0, a.S, h0);
    __syncthreads();
    float decay[TT][NS], h[TT][NS], v[TT];
#pragma unroll
    for (int k = 0; k < TT; ++k) {
      const float4 w = in[k][c];
      const float4 b4 = *reinterpret_cast<const float4*>(&Bs[k][s0]);
      const float4 c4 = *reinterpret_cast<const float4*>(&Cs[k][s0]);
      const float b[NS] = {b4.x, b4.y, b4.z, b4.w}, g[NS] = {c4.x, c4.y, c4.z, c4.w};
      v[k] = 0.f;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        decay[k][i] = exp2_fast(w.x * A[i] * LOG2E);
        h[k][i] = fmaf(decay[k][i], k ? h[k ? k - 1 : 0][i] : h0[i], w.y * b[i]);
        v[k] = fmaf(g[i], h[k][i], v[k]);
      }
    }
    bool owner;
    if (a.z.p) {
      const int first = lane_sums<TT, Q, 1>(v, lane, owner);
      if (owner)
#pragma unroll
        for (int i = 0; i < (TT > Q ? TT / Q : 1); ++i) out[0][first + i][c] = v[i];
    }
    float lb[TT], da[TT];
#pragma unroll
    for (int k = TT - 1; k >= 0; --k) {
      const float4 w = in[k][c];
      const float4 b4 = *reinterpret_cast<const float4*>(&Bs[k][s0]);
      const float4 c4 = *reinterpret_cast<const float4*>(&Cs[k][s0]);
      const float b[NS] = {b4.x, b4.y, b4.z, b4.w}, g[NS] = {c4.x, c4.y, c4.z, c4.w};
      float bc[2 * NS];
      lb[k] = da[k] = 0.f;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const float lam = fmaf(g[i], w.z, carry[i]);
        bc[i] = lam * w.y;
        bc[NS + i] = w.z * h[k][i];
        lb[k] = fmaf(lam, b[i], lb[k]);
        carry[i] = decay[k][i] * lam;
        const float u = carry[i] * (k ? h[k ? k - 1 : 0][i] : h0[i]);  // lam a h_{t-1}
        da[k] = fmaf(u, A[i], da[k]);
        dA[i] = fmaf(u, w.x, dA[i]);
      }
      const int first = lane_sums<2 * NS, LANES, Q>(bc, lane, owner);
      if (owner)
#pragma unroll
        for (int i = 0; i < (2 * NS > LANES ? 2 * NS / LANES : 1); ++i) {
          const int e = first + i;  // 0..3 dB, 4..7 dC of the thread's states
          red[warp][k][(e / NS) * SP + s0 + e % NS] = bc[i];
        }
    }
    {
      const int first = lane_sums<TT, Q, 1>(lb, lane, owner);
      lane_sums<TT, Q, 1>(da, lane, owner);
      if (owner)
#pragma unroll
        for (int i = 0; i < (TT > Q ? TT / Q : 1); ++i) {
          out[1][first + i][c] = lb[i];
          out[2][first + i][c] = da[i];
        }
    }
    __syncthreads();
    for (int e = tid; e < TT * 2 * SP; e += THREADS) {
      const int k = e / (2 * SP), j = e % (2 * SP);
      if (t0 + k >= a.T_) break;
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) s += red[w][k][j];
      a.part[((((long long)ct * a.T_ + t0 + k) * a.N + n) * a.G + at.g) * (2 * SP) + j] = s;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = ts + i * STEP, t = t0 + k;
      if (!has || k >= TT || t >= a.T_) continue;
      const float4 w = in[k][cs];
      const float l = out[1][k][cs];
      const float ddelta = fmaf(l, x[i], out[2][k][cs]);
      const float ddt = t >= len ? 0.f : a.softplus ? ddelta * sigmoid(raw[i]) : ddelta;
      st(a.dx.at(t, n) + ds, fmaf(w.x, l, skip * w.z));
      st(a.ddt.at(t, n) + ds, ddt);
      if (a.z.p) {
        const float y = fmaf(skip, x[i], out[0][k][cs]);
        st(a.dz.at(t, n) + ds, dy[i] * y * silu_slope(z[i], sigmoid(z[i])));
      }
      dskip = fmaf(w.z, x[i], dskip);
      dbias += ddt;
    }
    __syncthreads();
  }
  if (mine && a.dstate) store_states(a.dstate + row, s0, a.S, carry);
  // row n of the partial sums: dA [D][S], dskip [D], ddt_bias [D]
  float* sums = a.part + (long long)a.ctiles * a.T_ * a.N * a.G * (2 * SP) + (long long)n * a.D * (a.S + 2);
#pragma unroll
  for (int i = 0; i < NS; ++i)
    if (mine && s0 + i < a.S) sums[(long long)(at.d0 + c) * a.S + s0 + i] = dA[i];
  // the Q threads that staged a channel
  __syncthreads();
  float* shared = &red[0][0][0];  // 2 * THREADS floats: fewer than WARPS * TT * 2 * SP
  shared[tid] = dskip;
  shared[THREADS + tid] = dbias;
  __syncthreads();
  if (ts == 0 && has) {
    for (int j = 1; j < STEP; ++j) {
      dskip += shared[j * CB + cs];
      dbias += shared[THREADS + j * CB + cs];
    }
    sums[(long long)a.D * a.S + ds] = dskip;
    sums[(long long)a.D * (a.S + 1) + ds] = dbias;
  }
}

// dB and dC from the blocks' partial rows.
template <typename T>
__global__ void __launch_bounds__(256) scan_bwd_finish(Args<T> a, int SP, long long rows) {
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long r = e / (2 * a.S);
  if (r >= rows) return;
  const int j = (int)(e % (2 * a.S)), which = j / a.S, s = j % a.S;
  const float* p = a.part + r * (2 * SP) + which * SP + s;
  float v = 0.f;
  for (int ct = 0; ct < a.ctiles; ++ct) v += p[(long long)ct * rows * (2 * SP)];
  const int g = (int)(r % a.G), n = (int)(r / a.G % a.N);
  const long long t = r / a.G / a.N;
  if (which == 0) st(a.dB.at(t, n) + g * a.dB_g + s, v);
  else st(a.dC.at(t, n) + g * a.dC_g + s, v);
}

long long bc_floats(const haste_b200_selective_scan& a) {
  const int Q = lanes(a.S), ctiles = ceil_div(a.D / a.G, THREADS / Q);
  return (long long)ctiles * a.T * a.N * a.G * 2 * Q * NS;
}

template <typename T, int Q>
int launch(const haste_b200_selective_scan& a, cudaStream_t s) {
    const Args<T> k = pack<T>(a, THREADS / Q);
  scan_bwd<T, Q><<<a.N * a.G * k.ctiles, THREADS, 0, s>>>(k);
  HB_LAUNCH_OK();
  const long long rows = (long long)a.T * a.N * a.G;
  if (rows) {
    HB_REQUIRE(rows * 2 * a.S / 256 < (1LL << 31) - 1, "T*N too large");
    scan_bwd_finish<T><<<ceil_div(rows * 2 * a.S, 256), 256, 0, s>>>(k, Q * NS, rows);
    HB_LAUNCH_OK();
  }
  count_launch(rows ? 2 : 1);
  SumJobs jobs;
  jobs.add(a.dA, 0, 1, a.D * a.S, HASTE_B200_F32);
  jobs.add(a.dskip, (long long)a.D * a.S, 1, a.D, HASTE_B200_F32);
  jobs.add(a.ddt_bias, (long long)a.D * (a.S + 1), 1, a.D, HASTE_B200_F32);
  return sum_parts(a.scratch + bc_floats(a), a.N, (long long)a.D * (a.S + 2), jobs, s);
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
}  // namespace scan

int selective_scan_backward(const haste_b200_selective_scan& a, cudaStream_t s) {
  HB_TRY(scan::check(a, true));
  if (a.N == 0 || a.D == 0) return HASTE_B200_OK;
  ProfScope p(PH_REC_BWD, s);
  if (a.dtype == HASTE_B200_F32) return scan::by_lanes<float>(a, s);
  if (a.dtype == HASTE_B200_BF16) return scan::by_lanes<__nv_bfloat16>(a, s);
  return scan::by_lanes<__half>(a, s);
}

long long selective_scan_scratch(const haste_b200_selective_scan& a, bool backward) {
  if (!backward || a.T < 0 || a.N <= 0 || a.D <= 0 || a.S < 1 || a.S > 128 || a.G < 1) return 0;
  return scan::bc_floats(a) + (long long)a.N * a.D * (a.S + 2);
}

}  // namespace hb
