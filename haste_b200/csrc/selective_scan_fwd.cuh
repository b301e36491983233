// Selective scan, forward:
//
//   delta = softplus(dt + dt_bias),  h_t = exp(delta_t A) h_{t-1} + delta_t x_t B_t,
//   y_t = (C_t . h_t + skip x_t) silu(z_t)
//
// S exponentials a (step, row, channel) on the special function units, 16 a clock and SM (measured), against
// 8 to 16 bytes of sequences: for S = 16 those units bound it, not HBM.  bf16 T=1000 N=64 D=1024 S=16: 377 us
// (413 with checkpoints); the units' floor, with softplus and SiLU, is 290 us, and they are busy 65 % of the
// time, shared memory 63 %, the issue slots 56 % at 33 instructions per step of eight channels.
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
  static_assert(ROWS >= 1 && SL * ROWS >= TT, "the threads stage every channel of every step");
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
      const float sum = a.sums[p * pairs + rown + ch];
#pragma unroll
      for (int i = 0; i < 2; ++i) h[j][i] = behind(sum, A[j][i], h[j][i], e[i]);
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
  // (behind the row's end the state stays and y is zero)
  const int stop = len <= at.first ? at.first : min(at.last, at.first + (len - at.first + TT - 1) / TT * TT);
  for (int t0 = at.first; t0 < stop; t0 += TT) {
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
    if (t0 + TT < stop) fetch();
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
  if constexpr (!Ends) {
    for (int t0 = stop; t0 < at.last; t0 += TT) {
      const float none[V] = {};
#pragma unroll
      for (int i = 0; i < SL; ++i)
        if (has && t0 + ts + i * ROWS < at.last) store<T, V>(py + (long long)(i * ROWS) * a.y.t, none);
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
// Q lanes of four states per channel; a thread takes R rows, whose loads go out together.
template <typename T, int Q, int R, bool Fours>
__global__ void __launch_bounds__(256) scan_step(Args<T> a, int dblocks) {
  const int at = blockIdx.x % dblocks * 256 + threadIdx.x, d = at / Q, s0 = at % Q * NS;
  const int n0 = blockIdx.x / dblocks * R;
  const bool ok = d < a.D;
  const int dd = ok ? d : 0, g = dd / a.per;
  float2 A[2], h[R][2] = {};
  Raw<T, 1> x[R], dt[R], z[R];
  Raw<T, Fours ? 4 : 1> B[R][Fours ? 1 : 4], C[R][Fours ? 1 : 4];
  load_states(a.A + (long long)dd * a.S, s0, a.S, A);
  const float bias = a.dt_bias ? a.dt_bias[dd] : 0.f, skip = a.skip ? a.skip[dd] : 0.f;
  bool live[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int n = n0 + r;
    live[r] = ok && n < a.N && row_length(a.lengths, n, 1) > 0;
    if (ok && n < a.N && a.state) load_states(a.state + ((long long)n * a.D + d) * a.S, s0, a.S, h[r]);
    x[r] = load_if<T, 1>(live[r], a.x.at(0, n) + dd);
    dt[r] = load_if<T, 1>(live[r], a.dt.at(0, n) + dd);
    z[r] = load_if<T, 1>(live[r] && a.z.p, a.z.at(0, n) + dd);
    const T *pb = a.B.at(0, n) + g * a.B_g + s0, *pc = a.C.at(0, n) + g * a.C_g + s0;
    if constexpr (Fours) {
      B[r][0] = load_if<T, 4>(live[r] && s0 < a.S, pb);
      C[r][0] = load_if<T, 4>(live[r] && s0 < a.S, pc);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        B[r][i] = load_if<T, 1>(live[r] && s0 + i < a.S, pb + i);
        C[r][i] = load_if<T, 1>(live[r] && s0 + i < a.S, pc + i);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) A[i] = __fmul2_rn(A[i], both(LOG2E));
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int n = n0 + r;
    float b[4], c[4];
    if constexpr (Fours) {
      unpack<T, 4>(B[r][0], b);
      unpack<T, 4>(C[r][0], c);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        b[i] = one(B[r][i]);
        c[i] = one(C[r][i]);
      }
    }
    const float xv = one(x[r]), v = one(dt[r]) + bias;
    const float delta = !live[r] ? 0.f : a.softplus ? softplus(v) : v, u = delta * xv;
    float2 y = both(0.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (live[r]) h[r][i] = __ffma2_rn(decay(both(delta), A[i]), h[r][i], __fmul2_rn(both(u), make_float2(b[2 * i], b[2 * i + 1])));
      y = __ffma2_rn(h[r][i], make_float2(c[2 * i], c[2 * i + 1]), y);
    }
    if (ok && n < a.N && a.final_state) store_states(a.final_state + ((long long)n * a.D + d) * a.S, s0, a.S, h[r]);
    float sum = y.x + y.y;
#pragma unroll
    for (int o = Q / 2; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (ok && n < a.N && at % Q == 0) {
      sum = fmaf(skip, xv, sum);
      if (a.z.p) sum *= silu(one(z[r]));
      st(a.y.at(0, n) + d, live[r] ? sum : 0.f);
    }
  }
}

template <typename T, int Q, int CH, int V>
void launch_scan(const Args<T>& k, int blocks, cudaStream_t s) {
  // (the last piece's end is nobody's start; two channels a thread take whole sequences)
  if constexpr (CH == 1)
    if (k.chunks > 1) scan_fwd<T, Q, CH, V, false, true><<<blocks * (k.chunks - 1), THREADS, 0, s>>>(k);
  if (k.z.p) scan_fwd<T, Q, CH, V, true, false><<<blocks * k.chunks, THREADS, 0, s>>>(k);
  else scan_fwd<T, Q, CH, V, false, false><<<blocks * k.chunks, THREADS, 0, s>>>(k);
}

template <typename T, int Q>
int launch(const haste_b200_selective_scan& a, cudaStream_t s) {
  if (a.T == 1 && !a.checkpoints) {
    const Args<T> k = pack<T>(a, 1);
    const int dblocks = ceil_div((long long)a.D * Q, 256), e = sizeof(T);
    // four rows a thread once there are more threads than the GPU holds (bf16 N=128 D=2048 S=16: 16.4 us
    // with one, 12.3 with four)
    const bool many = (long long)a.N * a.D * Q > 2048LL * sm_count();
    const bool fours = a.S % 4 == 0 && aligned(a.B, e, 4 * e) && aligned(a.C, e, 4 * e) && a.B_g % 4 == 0 && a.C_g % 4 == 0;
    const long long blocks = (long long)dblocks * (many ? ceil_div(a.N, 4) : a.N);
    HB_REQUIRE(blocks < (1LL << 31), "N*D too large");
    if (many && fours) scan_step<T, Q, 4, true><<<(int)blocks, 256, 0, s>>>(k, dblocks);
    else if (many) scan_step<T, Q, 4, false><<<(int)blocks, 256, 0, s>>>(k, dblocks);
    else if (fours) scan_step<T, Q, 1, true><<<(int)blocks, 256, 0, s>>>(k, dblocks);
    else scan_step<T, Q, 1, false><<<(int)blocks, 256, 0, s>>>(k, dblocks);
  } else {
    constexpr int TT = fwd_steps(Q), V1 = Tile<Q, 1, TT>::V, V2 = Tile<Q, 2, TT>::V;
    constexpr int CB = THREADS / Q;
    const long long rows = (long long)a.N * a.G;
    // two channels a thread while their blocks fill the GPU
    const bool two = rows * ceil_div(a.D / a.G, 2 * CB) >= 4LL * sm_count() && wide(a, V2, false);
    Args<T> k = pack<T>(a, two ? 2 * CB : CB);
    const long long blocks = rows * k.ctiles;
    // (every piece reads the initial state, so a final state in its place takes whole sequences)
    k.chunks = two || !a.scratch || (a.state && a.final_state == a.state) ? 1 : forward_pieces(a);
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
