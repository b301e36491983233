// Selective scan, backward.  With dy already multiplied by silu(z), from the last step to the first:
//
//   lam_t = C_t dy_t + a_{t+1} lam_{t+1}          a_t = exp(delta_t A)
//   dC_t = sum_d dy_t h_t,   dB_t = sum_d lam_t delta_t x_t
//   dx_t = delta_t (lam_t . B_t) + skip dy_t
//   ddelta_t = x_t (lam_t . B_t) + lam_t . (A a_t h_{t-1}),   dA = sum_t lam_t delta_t a_t h_{t-1}
//
// The forward pass left the state in front of every CKPT steps; a thread computes those steps' states
// and decays again, H at a time, keeps them in registers, and walks back over them.  bf16 T=1000 N=64 D=1024
// S=16: 1400 us.  A step of eight channels takes 102 instructions (28 of them pairs of products and sums) and
// about 35 turns of shared memory against 15 clocks of exponentials; with 168 registers twelve warps are
// resident, which issue every second clock.  Tried, us: one channel a thread 1735; H = 2 with sixteen
// warps 1596; B and C as 16-bit values in shared memory 1504; pairs stored twice there 1680.
#pragma once

#include <algorithm>

#include "selective_scan.cuh"

namespace hb {
namespace scan {
namespace {

// Lanes, channels and shared memory as in the forward kernel.  dB and dC are sums over channels: a thread
// adds its CH channels, then they are added over the lanes of a warp, over the warps in shared memory,
// and over the blocks from partial rows [ctiles][T][rows][G][2][SP], all in a fixed order.
template <int Q, int CH>
struct Shared {
  using F = Tile<Q, CH, CKPT>;
  // B and C, once for each order in which a thread's four states may come: see add_channels
  static constexpr int NP = Q <= 8 ? 4 : 32 / Q;
  float B[NP][CKPT][F::SP], C[NP][CKPT][F::SP];
  float2 dd[CKPT][F::CT];                     // delta, delta x
  float dy[CKPT][F::CT];
  float red[THREADS / 32][CKPT][2 * F::SP];
  float part[3][CKPT][Q][F::YC];              // each lane's part of lam . B, lam . (A a h), C . h
  // What a thread keeps from tile to tile, each word its own: registers are what limits this kernel.
  float4 dA[CH][THREADS];
  float4 start[CH][THREADS];                  // the state in front of the next tile
  float4 sums[2][THREADS];                    // of dskip and ddt_bias
};

template <typename T, int Q, int CH, int V, bool Gate>
__global__ void __launch_bounds__(THREADS, CH == 1 ? 4 : 3) scan_bwd(Args<T> a) {
  using M = Shared<Q, CH>;
  using F = Tile<Q, CH, CKPT>;
  constexpr int TT = CKPT, CB = F::CB, CT = F::CT, SP = F::SP, YC = F::YC, BR = F::BR, PB = F::PB, WARPS = THREADS / 32;
  constexpr int SL = F::PER / V, ROWS = THREADS * V / CT;
  static_assert(ROWS >= 1 && SL * ROWS >= TT, "the threads stage every channel of every step");
  constexpr int LANES = 32 / Q;  // channels of a warp
  constexpr int H = 4;  // steps whose states and decays a thread holds; of 8, all would not fit the registers
  extern __shared__ __align__(16) char memory[];
  M& m = *reinterpret_cast<M*>(memory);
  const Place at(a, CT);
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int q = tid % Q, c = tid / Q, s0 = q * NS;
  // Order of this thread's states: register i is state s0 + (i ^ order).  Lanes that exchange sums of
  // different states then have the values to keep and to give in the same registers.
  const int order = (LANES >= 2 && (lane & LANES / 2 * Q) ? 2 : 0) + (LANES >= 4 && (lane & LANES / 4 * Q) ? 1 : 0);
  const int copy = LANES >= 4 ? order : order / 2;
  const int n = at.n, len = row_length(a.lengths, n, a.T_);
  const int cs = tid * V % CT, ts = tid * V / CT;
  const bool has = cs < at.count && ts < TT;
  const int d = at.d0 + (has ? cs : 0);
  const long long pairs = (long long)a.N * a.D, rown = (long long)n * a.D + at.d0;
  // (parameters are read again for every tile, from the L1 cache)
  auto parameter = [&](const float* p, float (&out)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) out[v] = has && p ? __ldg(p + d + v) : 0.f;
  };
  m.sums[0][tid] = m.sums[1][tid] = make_float4(0.f, 0.f, 0.f, 0.f);
  float2 A2[CH][2] = {}, carry[CH][2] = {};  // A2: A log2(e); carry: a_{t+1} lam_{t+1}, from dfinal through the pieces behind
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int ch = j * CB + c;
    m.dA[j][tid] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (ch >= at.count) continue;
    const long long row = (rown + ch) * a.S;
    load_states(a.A + (long long)(at.d0 + ch) * a.S, s0, a.S, A2[j]);
    reorder(A2[j], order);
#pragma unroll
    for (int i = 0; i < 2; ++i) A2[j][i] = __fmul2_rn(A2[j][i], both(LOG2E));
    if (a.dfinal) load_states(a.dfinal + row, s0, a.S, carry[j]);
    reorder(carry[j], order);
#pragma unroll 4
    for (int p = a.chunks - 1; p > at.piece; --p) {
      float2 e[2];
      load_states(a.ends + p * pairs * a.S + row, s0, a.S, e);
      reorder(e, order);
      const float sum = a.sums[p * pairs + rown + ch];
#pragma unroll
      for (int i = 0; i < 2; ++i) carry[j][i] = behind(sum, A2[j][i], carry[j][i], e[i]);
    }
  }

  // Behind the row's end the carry stays and all gradients are zero: whole tiles of that are written at once.
  const int tiles = (max(at.first, min(at.last, len)) - at.first + TT - 1) / TT;
  for (int t = at.first + tiles * TT + ts; t < at.last; t += min(ROWS, TT)) {
    if (!has) break;
    const float none[V] = {};
    store<T, V>(a.dx.at(t, n) + d, none);
    store<T, V>(a.ddt.at(t, n) + d, none);
    if (Gate) store<T, V>(a.dz.at(t, n) + d, none);
  }
  for (int t = at.first + tiles * TT; t < at.last; ++t)
    for (int e = tid; e < 2 * SP; e += THREADS)
      a.part[((((long long)at.ct * a.T_ + t) * a.rows + n - a.n0) * a.G + at.g) * (2 * SP) + e] = 0.f;
  Raw<T, V> xn[SL], dn[SL], zn[SL], gn[SL];
  Raw<T, 1> bn[PB], cn[PB];
  const int bt = tid / SP, bs = tid % SP;
  auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int t = t0 + ts + i * ROWS;
      const bool ok = has && t < len;
      xn[i] = load_if<T, V>(ok, a.x.at(t, n) + d);
      dn[i] = load_if<T, V>(ok, a.dt.at(t, n) + d);
      gn[i] = load_if<T, V>(ok, a.dy.at(t, n) + d);
      if (Gate) zn[i] = load_if<T, V>(ok, a.z.at(t, n) + d);
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const int k = i * BR + bt, t = t0 + k;
      const bool ok = bs < a.S && t < len && (TT % BR == 0 || k < TT);
      bn[i] = load_if<T, 1>(ok, a.B.at(t, n) + at.g * a.B_g + bs);
      cn[i] = load_if<T, 1>(ok, a.C.at(t, n) + at.g * a.C_g + bs);
    }
  };
  // Sums over the channels of the warp.  Lanes that differ in the bit behind order's first exchange two states
  // for two, those in the second one for one, without a select; then the one half goes on with dB, the other with dC.
  auto add_channels = [&](float* to, const float2 (&dB)[2], const float2 (&dC)[2]) {
    float v[8] = {dB[0].x, dB[0].y, dB[1].x, dB[1].y, dC[0].x, dC[0].y, dC[1].x, dC[1].y};
    constexpr unsigned all = 0xffffffffu;
    if (LANES >= 2) {
      v[0] += __shfl_xor_sync(all, v[2], LANES / 2 * Q);
      v[1] += __shfl_xor_sync(all, v[3], LANES / 2 * Q);
      v[4] += __shfl_xor_sync(all, v[6], LANES / 2 * Q);
      v[5] += __shfl_xor_sync(all, v[7], LANES / 2 * Q);
    }
    if (LANES >= 4) {
      v[0] += __shfl_xor_sync(all, v[1], LANES / 4 * Q);
      v[4] += __shfl_xor_sync(all, v[5], LANES / 4 * Q);
    }
    if constexpr (LANES >= 8) {
      const bool up = lane & LANES / 8 * Q;
      const float give = up ? v[0] : v[4];
      v[0] = (up ? v[4] : v[0]) + __shfl_xor_sync(all, give, LANES / 8 * Q);
#pragma unroll
      for (int o = LANES / 16; o > 0; o /= 2) v[0] += __shfl_xor_sync(all, v[0], o * Q);
      if (LANES == 8 || (lane & (LANES / 8 - 1) * Q) == 0) to[(up ? SP : 0) + order] = v[0];
    } else {
#pragma unroll
      for (int i = 0; i < (LANES == 1 ? 4 : LANES == 2 ? 2 : 1); ++i) {
        to[i ^ order] = v[i];
        to[SP + (i ^ order)] = v[4 + i];
      }
    }
  };
  // the states in front of a tile, on their way to shared memory
  const bool fours = a.S % NS == 0 && (reinterpret_cast<uintptr_t>(a.checkpoints) & 15) == 0;
  auto before = [&](int t0) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const float* p = a.checkpoints + t0 / CKPT * (pairs * a.S) + (rown + j * CB + c) * a.S + s0;
      const bool mine = j * CB + c < at.count;
      float* to = &m.start[j][tid].x;
      if (fours) copy_async<16>(to, mine && s0 < a.S ? p : a.checkpoints, mine && s0 < a.S);
      else
#pragma unroll
        for (int i = 0; i < NS; ++i) copy_async<4>(to + i, mine && s0 + i < a.S ? p + i : a.checkpoints, mine && s0 + i < a.S);
    }
  };
  if (tiles > 0) {
    fetch(at.first + (tiles - 1) * TT);
    before(at.first + (tiles - 1) * TT);
  }
#pragma unroll 1
  for (int tile = tiles - 1; tile >= 0; --tile) {
    const int t0 = at.first + tile * TT;
    Raw<T, V> x[SL], z[SL], dy[SL];
    float slope[SL][V], bias[V];
    copies_done();
    float2 h0[CH][2];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      load_pairs(&m.start[j][tid].x, h0[j]);
      reorder(h0[j], order);
    }
    parameter(a.dt_bias, bias);
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int k = ts + i * ROWS;
      x[i] = xn[i];
      z[i] = zn[i];
      dy[i] = gn[i];
      float xv[V], delta[V], g[V];
      unpack<T, V>(x[i], xv);
      unpack<T, V>(dn[i], delta);
      unpack<T, V>(dy[i], g);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        delta[v] += bias[v];
        slope[i][v] = 1.f;
      }
      if (a.softplus) softplus<V, true>(delta, slope[i]);
      if (Gate) {
        float zv[V];
        unpack<T, V>(z[i], zv);
#pragma unroll
        for (int v = 0; v < V; ++v) g[v] *= silu(zv[v]);
      }
      if (t0 + k >= len)
#pragma unroll
        for (int v = 0; v < V; ++v) delta[v] = slope[i][v] = 0.f;
      if (ts < TT) {
#pragma unroll
        for (int v = 0; v < V; ++v) m.dd[k][cs + v] = make_float2(delta[v], delta[v] * xv[v]);
        store<float, V>(&m.dy[k][cs], g);
      }
    }
#pragma unroll
    for (int i = 0; i < PB; ++i)
      if (TT % BR == 0 || i * BR + bt < TT) {
        const float b = one(bn[i]), g = one(cn[i]);
#pragma unroll
        for (int p = 0; p < M::NP; ++p) {
          const int to = bs ^ (M::NP == 2 ? 2 * p : p);
          m.B[p][i * BR + bt][to] = b;
          m.C[p][i * BR + bt][to] = g;
        }
      }
    __syncthreads();
    if (tile > 0) {
      fetch(t0 - TT);
      before(t0 - TT);
    }
    float2 sum[CH][2] = {};  // dA of these steps: short sums keep their bits
#pragma unroll 1
    for (int k0 = TT - H; k0 >= 0; k0 -= H) {
      // the H steps at hand in shared memory, from this thread's first word on
      const float *pB = &m.B[copy][k0][s0], *pC = &m.C[copy][k0][s0], *pdy = &m.dy[k0][c];
      const float2* pdd = &m.dd[k0][c];
      float* pp = &m.part[0][k0][q][c];
      float* pred = &m.red[warp][k0][s0];
      constexpr int PK = Q * YC, PW = TT * Q * YC;  // from step to step of the parts, and from one kind to the next
      float2 hs[CH][2], decays[CH][H][2], h[CH][H][2];
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        hs[j][0] = h0[j][0];
        hs[j][1] = h0[j][1];
      }
      // up to the H steps at hand, then over them
#pragma unroll 1
      for (int k = 0; k < k0; k += H)
#pragma unroll
        for (int l = 0; l < H; ++l) {
          float2 b[2];
          load_pairs(&m.B[copy][k + l][s0], b);
#pragma unroll
          for (int j = 0; j < CH; ++j) {
            const float2 w = m.dd[k + l][j * CB + c];
#pragma unroll
            for (int i = 0; i < 2; ++i) hs[j][i] = __ffma2_rn(decay(both(w.x), A2[j][i]), hs[j][i], __fmul2_rn(both(w.y), b[i]));
          }
        }
#pragma unroll
      for (int k = 0; k < H; ++k) {
        float2 b[2];
        load_pairs(pB + k * SP, b);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          const float2 w = pdd[k * CT + j * CB];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            decays[j][k][i] = decay(both(w.x), A2[j][i]);
            h[j][k][i] = __fmul2_rn(both(w.y), b[i]);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < H; ++k) {
        float2 g[2];
        if (Gate) load_pairs(pC + k * SP, g);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            h[j][k][i] = __ffma2_rn(decays[j][k][i], k ? h[j][k ? k - 1 : 0][i] : hs[j][i], h[j][k][i]);
          if (Gate) {
            const float2 s = __ffma2_rn(h[j][k][1], g[1], __fmul2_rn(h[j][k][0], g[0]));
            pp[2 * PW + k * PK + j * CB] = s.x + s.y;
          }
        }
      }
      float2 lastB[2], lastC[2];
#pragma unroll
      for (int k = H - 1; k >= 0; --k) {
        float2 b[2], g[2], dB[2], dC[2];
        load_pairs(pB + k * SP, b);
        load_pairs(pC + k * SP, g);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          const float2 w = pdd[k * CT + j * CB], dyk = both(pdy[k * CT + j * CB]);
          float2 lb, da;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 lam = __ffma2_rn(g[i], dyk, carry[j][i]);
            dB[i] = j ? __ffma2_rn(lam, both(w.y), dB[i]) : __fmul2_rn(lam, both(w.y));
            dC[i] = j ? __ffma2_rn(dyk, h[j][k][i], dC[i]) : __fmul2_rn(dyk, h[j][k][i]);
            lb = i ? __ffma2_rn(lam, b[i], lb) : __fmul2_rn(lam, b[i]);
            carry[j][i] = __fmul2_rn(decays[j][k][i], lam);
            const float2 u = __fmul2_rn(carry[j][i], k ? h[j][k ? k - 1 : 0][i] : hs[j][i]);  // lam a h_{t-1}
            da = i ? __ffma2_rn(u, A2[j][i], da) : __fmul2_rn(u, A2[j][i]);
            sum[j][i] = __ffma2_rn(u, both(w.x), sum[j][i]);
          }
          pp[k * PK + j * CB] = lb.x + lb.y;
          pp[PW + k * PK + j * CB] = da.x + da.y;
        }
        // the step before's, whose shuffles then run beside this one's arithmetic
        if (k < H - 1) add_channels(pred + (k + 1) * 2 * SP, lastB, lastC);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          lastB[i] = dB[i];
          lastC[i] = dC[i];
        }
      }
      add_channels(pred, lastB, lastC);
    }
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      float2 v[2];
      load_pairs(&m.dA[j][tid].x, v);
      v[0] = __fadd2_rn(v[0], sum[j][0]);
      v[1] = __fadd2_rn(v[1], sum[j][1]);
      m.dA[j][tid] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    }
    __syncthreads();
#pragma unroll 1
    for (int e = tid; e < TT * 2 * SP; e += THREADS) {
      const int k = e / (2 * SP), i = e % (2 * SP);
      if (t0 + k >= at.last) break;
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) s += m.red[w][k][i];
      if (t0 + k >= len) s = 0.f;  // (the state that stays may be no number)
      a.part[((((long long)at.ct * a.T_ + t0 + k) * a.rows + n - a.n0) * a.G + at.g) * (2 * SP) + i] = s;
    }
    float skip[V], ds[V], db[V];
    parameter(a.skip, skip);
    load<float, V>(&m.sums[0][tid].x, ds);
    load<float, V>(&m.sums[1][tid].x, db);
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int k = ts + i * ROWS;
      if (!has || t0 + k >= at.last) continue;
      if (t0 + k >= len) {
        const float none[V] = {};
        store<T, V>(a.dx.at(t0 + k, n) + d, none);
        store<T, V>(a.ddt.at(t0 + k, n) + d, none);
        if (Gate) store<T, V>(a.dz.at(t0 + k, n) + d, none);
        continue;
      }
      float g[V], xv[V], lb[V], da[V], dx[V], ddt[V];
      load<float, V>(&m.dy[k][cs], g);
      unpack<T, V>(x[i], xv);
      sum_parts_of<Q, V, YC>(&m.part[0][k][0][cs], lb);
      sum_parts_of<Q, V, YC>(&m.part[1][k][0][cs], da);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        dx[v] = fmaf(m.dd[k][cs + v].x, lb[v], skip[v] * g[v]);
        ddt[v] = fmaf(lb[v], xv[v], da[v] * LN2) * slope[i][v];
        ds[v] = fmaf(g[v], xv[v], ds[v]);
        db[v] += ddt[v];
      }
      store<T, V>(a.dx.at(t0 + k, n) + d, dx);
      store<T, V>(a.ddt.at(t0 + k, n) + d, ddt);
      if (Gate) {
        float zv[V], dyv[V], y[V];
        unpack<T, V>(z[i], zv);
        unpack<T, V>(dy[i], dyv);
        sum_parts_of<Q, V, YC>(&m.part[2][k][0][cs], y);
#pragma unroll
        for (int v = 0; v < V; ++v) y[v] = dyv[v] * fmaf(skip[v], xv[v], y[v]) * silu_slope(zv[v], sigmoid(zv[v]));
        store<T, V>(a.dz.at(t0 + k, n) + d, y);
      }
    }
    store<float, V>(&m.sums[0][tid].x, ds);
    store<float, V>(&m.sums[1][tid].x, db);
  }
  // row (piece, n) of the partial sums: dA [D][S], dskip [D], ddt_bias [D]
  float* sums = a.part + (long long)a.ctiles * a.T_ * a.most * a.G * (2 * SP) +
                ((long long)at.piece * a.N + n) * a.D * (a.S + 2);
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int ch = j * CB + c;
    if (ch >= at.count) continue;
    const float4 w = m.dA[j][tid];
    float2 e4[2] = {make_float2(w.x, w.y), make_float2(w.z, w.w)};
    reorder(e4, order);
    const float e[NS] = {e4[0].x, e4[0].y, e4[1].x, e4[1].y};
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (s0 + i < a.S) sums[(long long)(at.d0 + ch) * a.S + s0 + i] = e[i];
    reorder(carry[j], order);
    if (at.piece == 0 && a.dstate) store_states(a.dstate + (rown + ch) * a.S, s0, a.S, carry[j]);
  }
  // the threads that staged a channel
  __syncthreads();
  if (ts == 0 && has)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float dskip = 0.f, dbias = 0.f;
      for (int j = 0; j < ROWS && j < TT; ++j) {
        const int other = (j * CT + cs) / V;
        dskip += (&m.sums[0][other].x)[v];
        dbias += (&m.sums[1][other].x)[v];
      }
      sums[(long long)a.D * a.S + d + v] = dskip;
      sums[(long long)a.D * (a.S + 1) + d + v] = dbias;
    }
}

// What a piece hands to the one in front of it if nothing comes from behind: the recursion of lam alone.
template <typename T, int Q, int V, bool Gate>
__global__ void __launch_bounds__(THREADS) scan_bwd_ends(Args<T> a) {
  constexpr int TT = fwd_steps(Q);
  using F = Tile<Q, 1, TT>;
  constexpr int CB = F::CB, SP = F::SP, BR = F::BR, PB = F::PB;
  constexpr int SL = F::PER / V, ROWS = THREADS * V / CB;
  static_assert(ROWS >= 1 && SL * ROWS >= TT, "the threads stage every channel of every step");
  __shared__ __align__(16) float2 in[TT][CB];  // delta, dy
  __shared__ __align__(16) float Cs[TT][SP];
  Place at(a, CB);
  at.piece += 1;  // the first piece hands to nobody
  at.first += a.chunk;
  at.last = min(a.T_, at.first + a.chunk);
  const int tid = threadIdx.x, q = tid % Q, c = tid / Q, s0 = q * NS;
  const int n = at.n, len = row_length(a.lengths, n, a.T_);
  const int cs = tid * V % CB, ts = tid * V / CB;
  const bool has = cs < at.count && ts < TT, mine = c < at.count;
  const int ds = at.d0 + (has ? cs : 0);
  float bias[V];
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = has && a.dt_bias ? a.dt_bias[ds + v] : 0.f;
  float2 A[2] = {}, carry[2] = {};
  float total = 0.f;
  if (mine) load_states(a.A + (long long)(at.d0 + c) * a.S, s0, a.S, A);
#pragma unroll
  for (int i = 0; i < 2; ++i) A[i] = __fmul2_rn(A[i], both(LOG2E));
  const int tiles = (max(at.first, min(at.last, len)) - at.first + TT - 1) / TT;
  Raw<T, V> dn[SL], gn[SL], zn[SL];
  Raw<T, 1> cn[PB];
  const int bt = tid / SP, bs = tid % SP;
  auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int t = t0 + ts + i * ROWS;
      const bool ok = has && t < len;
      dn[i] = load_if<T, V>(ok, a.dt.at(t, n) + ds);
      gn[i] = load_if<T, V>(ok, a.dy.at(t, n) + ds);
      if (Gate) zn[i] = load_if<T, V>(ok, a.z.at(t, n) + ds);
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      const int k = i * BR + bt;
      cn[i] = load_if<T, 1>(k < TT && t0 + k < len && bs < a.S, a.C.at(t0 + k, n) + at.g * a.C_g + bs);
    }
  };
  if (tiles > 0) fetch(at.first + (tiles - 1) * TT);
#pragma unroll 1
  for (int tile = tiles - 1; tile >= 0; --tile) {
    const int t0 = at.first + tile * TT;
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const int k = ts + i * ROWS;
      float delta[V], g[V];
      unpack<T, V>(dn[i], delta);
      unpack<T, V>(gn[i], g);
#pragma unroll
      for (int v = 0; v < V; ++v) delta[v] += bias[v];
      if (a.softplus) softplus<V, false>(delta, delta);
      if (Gate) {
        float zv[V];
        unpack<T, V>(zn[i], zv);
#pragma unroll
        for (int v = 0; v < V; ++v) g[v] *= silu(zv[v]);
      }
      if (t0 + k >= len)
#pragma unroll
        for (int v = 0; v < V; ++v) delta[v] = 0.f;
      if (ts < TT)
#pragma unroll
        for (int v = 0; v < V; ++v) in[k][cs + v] = make_float2(delta[v], g[v]);
    }
#pragma unroll
    for (int i = 0; i < PB; ++i)
      if (TT % BR == 0 || i * BR + bt < TT) Cs[i * BR + bt][bs] = one(cn[i]);
    __syncthreads();
    if (tile > 0) fetch(t0 - TT);
#pragma unroll 8
    for (int k = TT - 1; k >= 0; --k) {
      const float2 w = in[k][c];
      float2 g[2];
      load_pairs(&Cs[k][s0], g);
#pragma unroll
      for (int i = 0; i < 2; ++i) carry[i] = __fmul2_rn(decay(both(w.x), A[i]), __ffma2_rn(g[i], both(w.y), carry[i]));
      total += w.x;
    }
    __syncthreads();
  }
  if (!mine) return;
  const long long pairs = (long long)a.N * a.D, pair = (long long)n * a.D + at.d0 + c;
  store_states(a.ends + at.piece * pairs * a.S + pair * a.S, s0, a.S, carry);
  if (q == 0) a.sums[at.piece * pairs + pair] = total;
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
#pragma unroll 8
  for (int ct = 0; ct < a.ctiles; ++ct) v += p[(long long)ct * rows * (2 * SP)];
  const int g = (int)(r % a.G), n = a.n0 + (int)(r / a.G % a.rows);
  const int t = (int)(r / a.G / a.rows);
  if (which == 0) st(a.dB.at(t, n) + g * a.dB_g + s, v);
  else st(a.dC.at(t, n) + g * a.dC_g + s, v);
}

template <typename T, int Q, int CH, int V, bool Gate>
int launch_scan(const Args<T>& k, cudaStream_t s) {
  constexpr int bytes = sizeof(Shared<Q, CH>);
  if (bytes > 48 * 1024)
    HB_CUDA_OK(cudaFuncSetAttribute(scan_bwd<T, Q, CH, V, Gate>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  scan_bwd<T, Q, CH, V, Gate><<<k.rows * k.G * k.ctiles * k.chunks, THREADS, bytes, s>>>(k);
  HB_LAUNCH_OK();
  return HASTE_B200_OK;
}
template <typename T, int Q, int CH, int V>
int by_gate(const Args<T>& k, cudaStream_t s) {
  return k.z.p ? launch_scan<T, Q, CH, V, true>(k, s) : launch_scan<T, Q, CH, V, false>(k, s);
}

template <typename T, int Q>
int launch_rows(const haste_b200_selective_scan& a, const Args<T>& k, const BwdShape& sh, cudaStream_t s) {
  if (sh.chunks > 1) {
    Args<T> e = k;
    e.ctiles = ceil_div(k.per, THREADS / Q);
    const int blocks = k.rows * a.G * e.ctiles * (sh.chunks - 1);
    constexpr int V = Tile<Q, 1, fwd_steps(Q)>::V;
    if (V > 1 && wide(a, V, true)) {
      if (k.z.p) scan_bwd_ends<T, Q, V, true><<<blocks, THREADS, 0, s>>>(e);
      else scan_bwd_ends<T, Q, V, false><<<blocks, THREADS, 0, s>>>(e);
    } else {
      if (k.z.p) scan_bwd_ends<T, Q, 1, true><<<blocks, THREADS, 0, s>>>(e);
      else scan_bwd_ends<T, Q, 1, false><<<blocks, THREADS, 0, s>>>(e);
    }
    HB_LAUNCH_OK();
    count_launch(1);
  }
  constexpr int V1 = Tile<Q, 1, CKPT>::V, V2 = Tile<Q, 2, CKPT>::V;
  if (sh.CH == 1) {
    if (wide(a, V1, true)) HB_TRY((by_gate<T, Q, 1, V1>(k, s)));
    else HB_TRY((by_gate<T, Q, 1, 1>(k, s)));
  } else if constexpr (Q > 1) {
    if (wide(a, V2, true)) HB_TRY((by_gate<T, Q, 2, V2>(k, s)));
    else HB_TRY((by_gate<T, Q, 2, 1>(k, s)));
  }
  const long long rows = (long long)a.T * k.rows * a.G;
  if (rows) {
    HB_REQUIRE(rows * 2 * a.S / 256 < (1LL << 31) - 1, "T*N too large");
    scan_bwd_finish<T><<<ceil_div(rows * 2 * a.S, 256), 256, 0, s>>>(k, Q * NS, rows);
    HB_LAUNCH_OK();
  }
  count_launch(rows ? 2 : 1);
  return HASTE_B200_OK;
}

template <typename T, int Q>
int launch(const haste_b200_selective_scan& a, cudaStream_t s) {
  const BwdShape sh(a);
  HB_REQUIRE(sh.blocks * sh.chunks < (1LL << 31), "N*D too large");
  Args<T> k = pack<T>(a, THREADS / Q * sh.CH);
  k.chunks = sh.chunks;
  k.chunk = sh.chunk;
  k.most = sh.rows;
  if (sh.chunks > 1) {
    k.ends = a.scratch + sh.bc_floats(a) + sh.sum_floats(a);
    k.sums = k.ends + (long long)sh.chunks * a.N * a.D * a.S;
  }
  for (k.n0 = 0; k.n0 < a.N; k.n0 += sh.rows) {
    k.rows = std::min(sh.rows, a.N - k.n0);
    HB_TRY((launch_rows<T, Q>(a, k, sh, s)));
  }
  SumJobs jobs;
  jobs.add(a.dA, 0, 1, a.D * a.S, HASTE_B200_F32);
  jobs.add(a.dskip, (long long)a.D * a.S, 1, a.D, HASTE_B200_F32);
  jobs.add(a.ddt_bias, (long long)a.D * (a.S + 1), 1, a.D, HASTE_B200_F32);
  return sum_parts(a.scratch + sh.bc_floats(a), sh.chunks * a.N, (long long)a.D * (a.S + 2), jobs, s);
}

}  // namespace

template <typename T>
int backward(const haste_b200_selective_scan& a, cudaStream_t s) {
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
