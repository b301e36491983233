// Selective scan, forward:
//
//   delta = softplus(dt + dt_bias),  h_t = exp(delta_t A) h_{t-1} + delta_t x_t B_t,
//   y_t = (C_t . h_t + skip x_t) silu(z_t)
//
// S exponentials a (step, row, channel) on the special function units, 16 a clock and SM, against
// 8 to 16 bytes of sequences: for S = 16 those units bound it, not HBM.
#pragma once

#include <algorithm>

#include "selective_scan.cuh"

namespace hb {
namespace scan {
namespace {

// A channel's states lie in Q lanes, four in each, for the whole piece; a thread walks CH channels side by
// side, because shared memory hands a warp 128 bytes a clock, copies of one value included, and reading
// B and C for every channel alone took more of it than the exponentials take of their units.
// The block stages a tile of TT steps: (delta, delta x) per channel and B, C per step, and walks it; the
// next tile's loads are under way meanwhile.  The Q partial sums of C . h meet in shared memory, where
// the thread that writes y adds them.
//
// Few channels leave most of the GPU idle, so their sequences are cut into pieces, walked twice: first
// (Ends) each piece but the last computes what it adds to a state that is zero in front of it, and its
// sum of delta; then each piece starts from the state that those of the pieces before it give.
template <typename T, int Q, int CH, int V, bool Gate, bool Ends>
__global__ void __launch_bounds__(THREADS, CH == 2 ? 4 : 5) scan_fwd(Args<T> a) {
  constexpr int TT = fwd_steps(Q);
  using F = Tile<Q, CH, TT>;
  constexpr int CB = F::CB, CT = F::CT, SP = F::SP, YC = F::YC, BR = F::BR, PB = F::PB;
  constexpr int SL = F::PER / V, ROWS = THREADS * V / CT;  // slots of V channels, steps between them
  __shared__ __align__(16) float2 dd[TT][CT];              // delta, delta x
  __shared__ __align__(16) float Bs[TT][SP], Cs[Ends ? 1 : TT][SP];
  __shared__ __align__(16) float ys[Ends ? 1 : TT][Q][YC];
  const Place at(a, CT);
  const int tid = threadIdx.x;
  const int q = tid % Q, c = tid / Q, s0 = q * NS;
  const int n = at.n, len = row_length(a.lengths, n, a.T_);
  const int cs = tid * V % CT, ts = tid * V / CT;
  const bool has = cs < at.count && ts < TT;  // (with 32 lanes a channel some threads stage nothing)
  const int ds = at.d0 + (has ? cs : 0);
  float bias[V], skip[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    bias[v] = has && a.dt_bias ? a.dt_bias[ds + v] : 0.f;
    skip[v] = has && a.skip ? a.skip[ds + v] : 0.f;
  }

  const long long pairs = (long long)a.N * a.D, rown = (long long)n * a.D + at.d0;
  float2 A[CH][2] = {}, h[CH][2] = {};
  float total[CH] = {};
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int ch = j * CB + c;
    if (ch >= at.count) continue;
    const long long row = (rown + ch) * a.S;
    load_states(a.A + (long long)(at.d0 + ch) * a.S, s0, a.S, A[j]);
#pragma unroll
    for (int i = 0; i < 2; ++i) A[j][i] = __fmul2_rn(A[j][i], both(LOG2E));
    if (Ends) continue;
    if (a.state) load_states(a.state + row, s0, a.S, h[j]);
#pragma unroll 4
    for (int p = 0; p < at.piece; ++p) {
      float2 e[2];
      load_states(a.ends + p * pairs * a.S + row, s0, a.S, e);
      const float2 sum = both(a.sums[p * pairs + rown + ch]);
#pragma unroll
      for (int i = 0; i < 2; ++i) h[j][i] = __ffma2_rn(decay(sum, A[j][i]), h[j][i], e[i]);
    }
  }

  Raw<T, V> xn[SL], dn[SL], zn[SL];
  Raw<T, 1> bn[PB], cn[PB];
  const T *px = a.x.at(at.first + ts, n) + ds, *pd = a.dt.at(at.first + ts, n) + ds,
          *pz = Gate ? a.z.at(at.first + ts, n) + ds : nullptr;
  const int bt = tid / SP, bs = tid % SP;
  const T *pb = a.B.at(at.first + bt, n) + at.g * a.B_g + bs, *pc = a.C.at(at.first + bt, n) + at.g * a.C_g + bs;
  int left = has ? len - at.first - ts : 0, bleft = bs < a.S ? len - at.first - bt : 0;  // steps that exist from here on
  auto fetch = [&]() {
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const bool ok = i * ROWS < left;
      xn[i] = load_if<T, V>(ok, px + (long long)(i * ROWS) * a.x.t);
      dn[i] = load_if<T, V>(ok, pd + (long long)(i * ROWS) * a.dt.t);
      if (Gate && !Ends) zn[i] = load_if<T, V>(ok, pz + (long long)(i * ROWS) * a.z.t);
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const bool ok = i * BR < bleft && (TT % BR == 0 || i * BR + bt < TT);
      bn[i] = load_if<T, 1>(ok, pb + (long long)(i * BR) * a.B.t);
      if (!Ends) cn[i] = load_if<T, 1>(ok, pc + (long long)(i * BR) * a.C.t);
    }
    px += (long long)TT * a.x.t;
    pd += (long long)TT * a.dt.t;
    if (Gate) pz += (long long)TT * a.z.t;
    pb += (long long)TT * a.B.t;
    pc += (long long)TT * a.C.t;
    left -= TT;
    bleft -= TT;
  };
  fetch();
  T* py = Ends ? nullptr : a.y.at(at.first + ts, n) + ds;
  for (int t0 = at.first; t0 < at.last; t0 += TT) {
    Raw<T, V> x[SL], z[SL];
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int k = ts + i * ROWS;
      x[i] = xn[i];
      z[i] = zn[i];
      float xv[V], delta[V];
      unpack<T, V>(x[i], xv);
      unpack<T, V>(dn[i], delta);
#pragma unroll
      for (int v = 0; v < V; ++v) delta[v] += bias[v];
      if (a.softplus) softplus<V, false>(delta, delta);
      if (t0 + k >= len)
#pragma unroll
        for (int v = 0; v < V; ++v) delta[v] = 0.f;  // the state stays
      if (ts < TT)
#pragma unroll
        for (int v = 0; v < V; ++v) dd[k][cs + v] = make_float2(delta[v], delta[v] * xv[v]);
    }
#pragma unroll
    for (int i = 0; i < PB; ++i)
      if (TT % BR == 0 || i * BR + bt < TT) {
        Bs[i * BR + bt][bs] = one(bn[i]);
        if (!Ends) Cs[i * BR + bt][bs] = one(cn[i]);
      }
    __syncthreads();
    if (t0 + TT < at.last) fetch();
#pragma unroll 1
    for (int k0 = 0; k0 < TT; k0 += CKPT) {
      if (!Ends && a.checkpoints && t0 + k0 < at.last)
#pragma unroll
        for (int j = 0; j < CH; ++j)
          if (j * CB + c < at.count)
            store_states(a.checkpoints + (t0 + k0) / CKPT * (pairs * a.S) + (rown + j * CB + c) * a.S, s0, a.S, h[j]);
      // Four steps at a time: first what does not hang on the state, so that the exponentials are on their
      // way when the chain needs them.
#pragma unroll
      for (int k1 = k0; k1 < k0 + CKPT; k1 += 4) {
        float2 e[4][CH][2], u[4][CH][2];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float2 b[2];
          load_pairs(&Bs[k1 + k][s0], b);
#pragma unroll
          for (int j = 0; j < CH; ++j) {
            const float2 w = dd[k1 + k][j * CB + c];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              e[k][j][i] = decay(both(w.x), A[j][i]);
              u[k][j][i] = __fmul2_rn(both(w.y), b[i]);
            }
            if (Ends) total[j] += w.x;
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float2 g[2];
          if (!Ends) load_pairs(&Cs[k1 + k][s0], g);
#pragma unroll
          for (int j = 0; j < CH; ++j) {
#pragma unroll
            for (int i = 0; i < 2; ++i) h[j][i] = __ffma2_rn(e[k][j][i], h[j][i], u[k][j][i]);
            if (!Ends) {
              const float2 s = __ffma2_rn(h[j][1], g[1], __fmul2_rn(h[j][0], g[0]));
              ys[k1 + k][q][j * CB + c] = s.x + s.y;
            }
          }
        }
      }
    }
    __syncthreads();
    if constexpr (!Ends) {
#pragma unroll
      for (int i = 0; i < SL; ++i) {
        const int k = ts + i * ROWS, t = t0 + k;
        if (!has || t >= at.last) continue;
        float y[V], xv[V];
        sum_parts_of<Q, V, YC>(&ys[k][0][cs], y);
        unpack<T, V>(x[i], xv);
#pragma unroll
        for (int v = 0; v < V; ++v) y[v] = fmaf(skip[v], xv[v], y[v]);
        if (Gate) {
          float zv[V];
          unpack<T, V>(z[i], zv);
#pragma unroll
          for (int v = 0; v < V; ++v) y[v] *= silu(zv[v]);
        }
        if (t >= len)
#pragma unroll
          for (int v = 0; v < V; ++v) y[v] = 0.f;
        store<T, V>(py + (long long)(i * ROWS) * a.y.t, y);
      }
      py += (long long)TT * a.y.t;
    }
  }
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int ch = j * CB + c;
    if (ch >= at.count) continue;
    if (Ends) {
      store_states(a.ends + at.piece * pairs * a.S + (rown + ch) * a.S, s0, a.S, h[j]);
      if (q == 0) a.sums[at.piece * pairs + rown + ch] = total[j];
    } else if (a.final_state && at.piece == a.chunks - 1) {
      store_states(a.final_state + (rown + ch) * a.S, s0, a.S, h[j]);
    }
  }
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
  float2 A[2], h[2] = {};
  load_states(a.A + (long long)d * a.S, s0, a.S, A);
  const long long row = ((long long)n * a.D + d) * a.S;
  if (a.state) load_states(a.state + row, s0, a.S, h);
  float x = 0.f, y = 0.f;
  if (live) {
    x = ld(a.x.at(0, n) + d);
    const float v = ld(a.dt.at(0, n) + d) + (a.dt_bias ? a.dt_bias[d] : 0.f);
    const float delta = a.softplus ? softplus(v) : v, u = delta * x;
    const T *B = a.B.at(0, n) + g * a.B_g, *C = a.C.at(0, n) + g * a.C_g;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int s = s0 + 2 * i;
      const float2 b = make_float2(s < a.S ? ld(B + s) : 0.f, s + 1 < a.S ? ld(B + s + 1) : 0.f);
      const float2 w = make_float2(s < a.S ? ld(C + s) : 0.f, s + 1 < a.S ? ld(C + s + 1) : 0.f);
      h[i] = __ffma2_rn(decay(make_float2(delta, delta), __fmul2_rn(A[i], make_float2(LOG2E, LOG2E))), h[i],
                        __fmul2_rn(make_float2(u, u), b));
      y = fmaf(h[i].x, w.x, fmaf(h[i].y, w.y, y));
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


template <typename T, int Q, int CH, int V>
void launch_scan(const Args<T>& k, int blocks, cudaStream_t s) {
  // (the last piece's end is nobody's start)
  if (k.chunks > 1) scan_fwd<T, Q, CH, V, false, true><<<blocks * (k.chunks - 1), THREADS, 0, s>>>(k);
  if (k.z.p) scan_fwd<T, Q, CH, V, true, false><<<blocks * k.chunks, THREADS, 0, s>>>(k);
  else scan_fwd<T, Q, CH, V, false, false><<<blocks * k.chunks, THREADS, 0, s>>>(k);
}

template <typename T, int Q>
int launch(const haste_b200_selective_scan& a, cudaStream_t s) {
  if (a.T == 1 && !a.checkpoints) {
    scan_step<T, Q><<<ceil_div((long long)a.N * a.D * Q, 256), 256, 0, s>>>(pack<T>(a, 1));
  } else {
    constexpr int TT = fwd_steps(Q), V1 = Tile<Q, 1, TT>::V, V2 = Tile<Q, 2, TT>::V;
    constexpr int CB = THREADS / Q;
    const long long rows = (long long)a.N * a.G;
    // two channels a thread while their blocks fill the GPU
    const bool two = rows * ceil_div(a.D / a.G, 2 * CB) >= 4LL * sm_count() && wide(a, V2, false);
    Args<T> k = pack<T>(a, two ? 2 * CB : CB);
    const long long blocks = rows * k.ctiles;
    k.chunks = two || !a.scratch ? 1 : forward_pieces(a);
    if (k.chunks > 1) {
      k.chunk = ceil_div(ceil_div(a.T, k.chunks), TT) * TT;
      k.ends = a.scratch;
      k.sums = a.scratch + (long long)k.chunks * a.N * a.D * a.S;
      k.chunks = ceil_div(a.T, k.chunk);
    }
    HB_REQUIRE(blocks * k.chunks < (1LL << 31), "N*D too large");
    if (two) launch_scan<T, Q, 2, V2>(k, (int)blocks, s);
    else if (V1 > 1 && wide(a, V1, false)) launch_scan<T, Q, 1, V1>(k, (int)blocks, s);
    else launch_scan<T, Q, 1, 1>(k, (int)blocks, s);
    if (k.chunks > 1) count_launch(1);
  }
  HB_LAUNCH_OK();
  count_launch(1);
  return HASTE_B200_OK;
}

}  // namespace

template <typename T>
int forward(const haste_b200_selective_scan& a, cudaStream_t s) {
  switch (lanes(a.S)) {
    case 1: return launch<T, 1>(a, s);
    case 2: return launch<T, 2>(a, s);
    case 4: return launch<T, 4>(a, s);
    case 8: return launch<T, 8>(a, s);
    case 16: return launch<T, 16>(a, s);
    default: return launch<T, 32>(a, s);
  }
}

}  // namespace scan
}  // namespace hb
