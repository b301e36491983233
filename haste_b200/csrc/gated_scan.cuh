// Gated linear recurrence, one state a channel:
//
//   r = sigmoid(gate),  with decay: log a = decay r, w = sqrt(1 - a^2);  without: a = r, w = 1 - a
//   h_t = a_t h_{t-1} + w_t x_t sigmoid(input_gate_t),  y_t = h_t
//
// and its gradients.  With lam_t = dy_t + a_{t+1} lam_{t+1}, u_t = x_t sigmoid(input_gate_t):
//
//   dx = lam w sigmoid(i),  di = lam w u (1 - sigmoid(i)),
//   without decay: dgate = lam (h_{t-1} - u) r (1 - r),
//   with: dlog_a = lam (a h_{t-1} - u a^2 / w),  ddecay = sum dlog_a r,  dgate = dlog_a decay r (1 - r).
//
// Each sequence is read once and each output written once: HBM bounds it, at 3 to 9 words a (step, row, channel).
#pragma once

#include <algorithm>

#include "state_space.cuh"

namespace hb {

long long gated_scan_scratch(const haste_b200_gated_scan& a, bool backward);

namespace gated {

using namespace ss;

constexpr int THREADS = 256, SEG = THREADS / 32;  // a warp walks one of the tile's segments
constexpr int FWD_L = 8, BWD_L = 4;               // steps of a segment
constexpr int FWD_TT = SEG * FWD_L, BWD_TT = SEG * BWD_L;
constexpr int CKPT = BWD_TT;                      // steps between the states left for the backward pass

template <typename T>
struct Args {
  int T_, N, D, ctiles;
  int pieces, piece;  // of the sequence, that blocks work on side by side; steps of one
  Seq<const T> x, gate, inner, dy;
  Seq<T> y, dx, dgate, dinner;
  const float *decay, *state, *dfinal;
  float *final_state, *checkpoints, *dstate;
  float2* ends;  // [pieces][N][D]: a piece's product of decays, and what it adds to the state (backward: to a lam)
  float* part;   // [pieces][N][D]: sums of ddecay
  const long long* lengths;
};

// Where a block works: lane `c` has channels d .. d + V - 1 of row n; steps first .. last - 1.
template <int V>
struct Place {
  int n, d, piece, first, last, len;
  bool ok;
  template <typename A>
  __device__ __forceinline__ explicit Place(const A& a) {
    const int r = blockIdx.x / a.ctiles;
    d = (blockIdx.x % a.ctiles * 32 + threadIdx.x % 32) * V;
    ok = d < a.D;
    n = r % a.N;
    piece = r / a.N;
    first = piece * a.piece;
    last = min(a.T_, first + a.piece);
    len = row_length(a.lengths, n, a.T_);
  }
};

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rsqrt_fast(float v) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float LOG2E = 1.4426950408889634f;

// sigmoid(v), sigmoid(-v) and their product, each to its own last bits.
struct Gate {
  float r, rest, slope;
  __device__ __forceinline__ explicit Gate(float v) {
    const float e = exp2_fast(fabsf(v) * -LOG2E), big = reciprocal(1.f + e), small = e * big;
    const bool up = v > 0.f;
    r = up ? big : small;
    rest = up ? small : big;
    slope = small * big;
  }
};

// What a step does to the state.  A decay lies next to one, where the special function unit's results are low by
// 2.4e-8 on average; a state that keeps 1 / (1 - a) steps would add that up.  So 1 - a is computed to its own last
// bits (the exponential's series, where a is above 0.7), and a, its difference from one, is rounded once, to either side.
template <bool Decay>
struct Step {
  float a, w, over;  // over: 1 / w, 0 where w is
  __device__ __forceinline__ Step(const Gate& g, float decay) {
    if constexpr (Decay) {
      const float l = decay * g.r;
      float p = 1.f / 5040;
      p = fmaf(p, l, 1.f / 720);
      p = fmaf(p, l, 1.f / 120);
      p = fmaf(p, l, 1.f / 24);
      p = fmaf(p, l, 1.f / 6);
      p = fmaf(p, l, 0.5f);
      p = fmaf(p, l, 1.f);
      const bool slow = l > -0.35f;
      const float far = exp2_fast(l * LOG2E), m = slow ? -l * p : 1.f - far;
      a = slow ? 1.f - m : far;
      const float v = fmaf(m, a, m);  // 1 - a^2
      over = v >= 1.1754944e-38f ? rsqrt_fast(v) : v * 0.f;  // (a NaN stays)
      w = v * over;
    } else {
      a = g.r > 0.5f ? 1.f - g.rest : g.r;
      w = g.rest;
      over = 0.f;
    }
  }
};

// A channel's decay: values above zero count as zero, so that no state grows.
template <bool Decay>
__device__ __forceinline__ float decay_of(const float* decay, int d, bool ok) {
  if (!Decay || !ok) return 0.f;
  const float v = decay[d];
  return v > 0.f ? 0.f : v;
}

// ------------------------------------------------------------------ forward
// A block takes 32 words of neighbouring channels (two channels of 16 bits, one of 32) and tiles of 64 steps, eight to a
// warp.  A warp folds its steps into (product of decays, what they add to a state of zero), the warps' pairs meet in
// shared memory, each warp folds those in front of its own into the tile's starting state, and walks its steps again
// from registers.  One barrier a tile: pairs and the state behind the tile have two buffers.  The next tile's words are
// under way from when the present ones have been used.
//
// Few channels leave most of the GPU idle, so their sequences are cut into pieces and read twice (the second time from
// L2): first (Ends) each piece but the last leaves its pair, then each piece starts from those in front of it.
template <typename T, int V, bool Decay, bool In, bool Ends>
__global__ void __launch_bounds__(THREADS, 2) gated_fwd(Args<T> a) {
  constexpr int L = FWD_L, TT = FWD_TT;
  __shared__ float2 pairs[2][SEG][V][32];
  __shared__ float behind[2][V][32];
  const Place<V> at(a);
  const int lane = threadIdx.x % 32, seg = threadIdx.x / 32;
  const int d = at.ok ? at.d : 0;
  const long long rows = (long long)a.N * a.D, row = (long long)at.n * a.D + d;
  float decay[V], start[V], total[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    decay[v] = decay_of<Decay>(a.decay, d + v, at.ok);
    start[v] = !Ends && at.ok && a.state ? a.state[row + v] : 0.f;
    total[v] = 1.f;
  }
  if (!Ends)
#pragma unroll 4
    for (int p = 0; p < at.piece; ++p)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 e = a.ends[p * rows + row + v];
        start[v] = fmaf(e.x, start[v], e.y);
      }

  const int stop = min(at.last, at.len);  // tiles from here on are behind the row's end
  Raw<T, V> xn[L], gn[L], in[L];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const int t = t0 + seg * L + j;
      const bool ok = at.ok && t < stop;
      xn[j] = load_if<T, V>(ok, a.x.at(t, at.n) + d);
      gn[j] = load_if<T, V>(ok, a.gate.at(t, at.n) + d);
      if (In) in[j] = load_if<T, V>(ok, a.inner.at(t, at.n) + d);
    }
  };
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = start[v];
  fetch(at.first);
  int k = 0;
  for (int t0 = at.first; t0 < stop; t0 += TT, ++k) {
    float s[L][V], b[L][V];
#pragma unroll
    for (int j = 0; j < L; ++j) {
      float x[V], g[V], i[V];
      unpack<T, V>(xn[j], x);
      unpack<T, V>(gn[j], g);
      if (In) unpack<T, V>(in[j], i);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Step<Decay> step(Gate(g[v]), decay[v]);
        s[j][v] = step.a;
        b[j][v] = step.w * (In ? x[v] * sigmoid(i[v]) : x[v]);
      }
    }
    if (t0 + TT > stop)
#pragma unroll
      for (int j = 0; j < L; ++j)
        if (t0 + seg * L + j >= stop)
#pragma unroll
          for (int v = 0; v < V; ++v) s[j][v] = 1.f, b[j][v] = 0.f;
    if (t0 + TT < stop) fetch(t0 + TT);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float p = s[0][v], e = b[0][v];
#pragma unroll
      for (int j = 1; j < L; ++j) {
        e = fmaf(s[j][v], e, b[j][v]);
        p *= s[j][v];
      }
      pairs[k & 1][seg][v][lane] = make_float2(p, e);
    }
    __syncthreads();
    if constexpr (Ends) {
      if (seg == 0)
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int q = 0; q < SEG; ++q) {
            const float2 e = pairs[k & 1][q][v][lane];
            h[v] = fmaf(e.x, h[v], e.y);
            total[v] *= e.x;
          }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        h[v] = k ? behind[(k - 1) & 1][v][lane] : start[v];
        for (int q = 0; q < seg; ++q) {
          const float2 e = pairs[k & 1][q][v][lane];
          h[v] = fmaf(e.x, h[v], e.y);
        }
      }
      const int ts = t0 + seg * L;
      if (a.checkpoints && seg * L % CKPT == 0 && at.ok && ts < at.last)
#pragma unroll
        for (int v = 0; v < V; ++v) a.checkpoints[ts / CKPT * rows + row + v] = h[v];
#pragma unroll
      for (int j = 0; j < L; ++j) {
        float y[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h[v] = fmaf(s[j][v], h[v], b[j][v]);
          y[v] = ts + j < stop ? h[v] : 0.f;
        }
        if (at.ok && ts + j < at.last) store<T, V>(a.y.at(ts + j, at.n) + d, y);
      }
      if (seg == SEG - 1)
#pragma unroll
        for (int v = 0; v < V; ++v) behind[k & 1][v][lane] = h[v];
    }
  }
  if (!at.ok) return;
  if constexpr (Ends) {
    if (seg == 0)
#pragma unroll
      for (int v = 0; v < V; ++v) a.ends[at.piece * rows + row + v] = make_float2(total[v], h[v]);
  } else {
    const float none[V] = {};
    for (int t = at.first + k * TT + seg; t < at.last; t += SEG) store<T, V>(a.y.at(t, at.n) + d, none);
    if (a.final_state && at.piece == a.pieces - 1 && seg == SEG - 1)
#pragma unroll
      for (int v = 0; v < V; ++v) a.final_state[row + v] = h[v];
  }
}

// A single step: HBM or, for few rows, the launch bounds it.
template <typename T, int V, bool Decay>
__global__ void __launch_bounds__(256) gated_step(Args<T> a) {
  const int words = a.D / V;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int n = (int)(i / words), d = (int)(i - (long long)n * words) * V;
  if (n >= a.N) return;
  const bool live = row_length(a.lengths, n, 1) > 0;
  const Raw<T, V> xr = load_if<T, V>(live, a.x.at(0, n) + d), gr = load_if<T, V>(live, a.gate.at(0, n) + d),
                  ir = load_if<T, V>(live && a.inner.p, a.inner.at(0, n) + d);
  const long long row = (long long)n * a.D + d;
  float h[V], x[V], g[V], in[V], y[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = a.state ? a.state[row + v] : 0.f;
  unpack<T, V>(xr, x);
  unpack<T, V>(gr, g);
  unpack<T, V>(ir, in);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const Step<Decay> step(Gate(g[v]), decay_of<Decay>(a.decay, d + v, true));
    if (live) h[v] = fmaf(step.a, h[v], step.w * (a.inner.p ? x[v] * sigmoid(in[v]) : x[v]));
    y[v] = live ? h[v] : 0.f;
    if (a.final_state) a.final_state[row + v] = h[v];
  }
  store<T, V>(a.y.at(0, n) + d, y);
}

// ------------------------------------------------------------------ backward
// The same blocks and barriers, from the last tile to the first, with four steps to a warp.  A tile's states come from
// the one that the forward pass left in front of it; a segment is a pair for the states, and for the adjoint
// mu = a lam, which runs the other way, the same product and a third number.
// Ends: pieces but the first leave (product, mu that they give to one of zero behind them).
template <typename T, int V, bool Decay, bool In, bool Ends>
__global__ void __launch_bounds__(THREADS, 2) gated_bwd(Args<T> a) {
  constexpr int L = BWD_L, TT = BWD_TT;
  __shared__ float2 pairs[2][SEG][V][32];
  __shared__ float backs[2][SEG][V][32];
  __shared__ float before[2][V][32];
  const Place<V> at(a);
  const int lane = threadIdx.x % 32, seg = threadIdx.x / 32;
  const int d = at.ok ? at.d : 0;
  const long long rows = (long long)a.N * a.D, row = (long long)at.n * a.D + d;
  float decay[V], start[V], total[V], mu[V], sum[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    decay[v] = decay_of<Decay>(a.decay, d + v, at.ok);
    start[v] = !Ends && at.ok && a.dfinal ? a.dfinal[row + v] : 0.f;
    total[v] = 1.f;
    sum[v] = 0.f;
  }
  if (!Ends)
#pragma unroll 4
    for (int p = a.pieces - 1; p > at.piece; --p)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 e = a.ends[p * rows + row + v];
        start[v] = fmaf(e.x, start[v], e.y);
      }
#pragma unroll
  for (int v = 0; v < V; ++v) mu[v] = start[v];

  const int stop = min(at.last, at.len);
  const int tiles = stop > at.first ? (stop - at.first + TT - 1) / TT : 0;
  Raw<T, V> xn[L], gn[L], in[L], yn[L];
  float hn[V];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const int t = t0 + seg * L + j;
      const bool ok = at.ok && t < stop;
      if (!Ends) xn[j] = load_if<T, V>(ok, a.x.at(t, at.n) + d);
      gn[j] = load_if<T, V>(ok, a.gate.at(t, at.n) + d);
      if (In && !Ends) in[j] = load_if<T, V>(ok, a.inner.at(t, at.n) + d);
      yn[j] = load_if<T, V>(ok, a.dy.at(t, at.n) + d);
    }
    if (!Ends)
#pragma unroll
      for (int v = 0; v < V; ++v) hn[v] = at.ok ? a.checkpoints[t0 / CKPT * rows + row + v] : 0.f;
  };
  if (tiles) fetch(at.first + (tiles - 1) * TT);
  if constexpr (!Ends) {
    const float none[V] = {};
    if (at.ok)
      for (int t = at.first + tiles * TT + seg; t < at.last; t += SEG) {
        store<T, V>(a.dx.at(t, at.n) + d, none);
        store<T, V>(a.dgate.at(t, at.n) + d, none);
        if (In) store<T, V>(a.dinner.at(t, at.n) + d, none);
      }
  }
  for (int k = 0; k < tiles; ++k) {
    const int t0 = at.first + (tiles - 1 - k) * TT, ts = t0 + seg * L;
    const bool whole = t0 + TT <= stop;
    float x[L][V], s[L][V], dy[L][V], i[L][V], islope[L][V], w[L][V], over[L][V], r[L][V], slope[L][V], h[V];
#pragma unroll
    for (int j = 0; j < L; ++j) {
      float g[V];
      unpack<T, V>(gn[j], g);
      unpack<T, V>(yn[j], dy[j]);
      if (!Ends) unpack<T, V>(xn[j], x[j]);
      if (In && !Ends) unpack<T, V>(in[j], i[j]);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gate gate(g[v]);
        const Step<Decay> step(gate, decay[v]);
        s[j][v] = step.a;
        w[j][v] = step.w;
        over[j][v] = step.over;
        r[j][v] = gate.r;
        slope[j][v] = gate.slope;
        if (In && !Ends) {
          const Gate inner(i[j][v]);
          i[j][v] = inner.r;
          islope[j][v] = inner.slope;
        } else {
          i[j][v] = 1.f;
          islope[j][v] = 0.f;
        }
      }
    }
    if (!whole)
#pragma unroll
      for (int j = 0; j < L; ++j)
        if (ts + j >= stop)
#pragma unroll
          for (int v = 0; v < V; ++v) s[j][v] = 1.f, w[j][v] = 0.f;  // (x and dy are zeros)
    if (!Ends)
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = hn[v];
    if (k + 1 < tiles) fetch(t0 - TT);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float p = 1.f, e = 0.f, m = 0.f;
#pragma unroll
      for (int j = 0; j < L; ++j) {
        if (!Ends) e = fmaf(s[j][v], e, w[j][v] * (x[j][v] * i[j][v]));
        p *= s[j][v];
        m = s[L - 1 - j][v] * (dy[L - 1 - j][v] + m);
      }
      pairs[k & 1][seg][v][lane] = make_float2(p, e);
      backs[k & 1][seg][v][lane] = m;
    }
    __syncthreads();
    if constexpr (Ends) {
      if (seg == 0)
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int q = SEG - 1; q >= 0; --q) {
            const float p = pairs[k & 1][q][v][lane].x;
            mu[v] = fmaf(p, mu[v], backs[k & 1][q][v][lane]);
            total[v] *= p;
          }
    } else {
      float hs[L][V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        for (int q = 0; q < seg; ++q) {
          const float2 e = pairs[k & 1][q][v][lane];
          h[v] = fmaf(e.x, h[v], e.y);
        }
        mu[v] = k ? before[(k - 1) & 1][v][lane] : start[v];
        for (int q = SEG - 1; q > seg; --q) mu[v] = fmaf(pairs[k & 1][q][v][lane].x, mu[v], backs[k & 1][q][v][lane]);
#pragma unroll
        for (int j = 0; j < L; ++j) {
          hs[j][v] = h[v];
          h[v] = fmaf(s[j][v], h[v], w[j][v] * (x[j][v] * i[j][v]));
        }
      }
#pragma unroll
      for (int j = L - 1; j >= 0; --j) {
        float dx[V], dg[V], di[V];
        const bool live = ts + j < stop;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float lam = dy[j][v] + mu[v], u = x[j][v] * i[j][v], lw = lam * w[j][v];
          if (Decay) {
            const float dl = lam * (s[j][v] * (hs[j][v] - u * (s[j][v] * over[j][v])));
            dg[v] = dl * (decay[v] * slope[j][v]);
            sum[v] = live ? fmaf(dl, r[j][v], sum[v]) : sum[v];
          } else {
            dg[v] = lam * (hs[j][v] - u) * slope[j][v];
          }
          dx[v] = lw * i[j][v];
          di[v] = lw * x[j][v] * islope[j][v];
          mu[v] = s[j][v] * lam;
          if (!live) dx[v] = dg[v] = di[v] = 0.f;
        }
        if (at.ok && ts + j < at.last) {
          store<T, V>(a.dx.at(ts + j, at.n) + d, dx);
          store<T, V>(a.dgate.at(ts + j, at.n) + d, dg);
          if (In) store<T, V>(a.dinner.at(ts + j, at.n) + d, di);
        }
      }
      if (seg == 0)
#pragma unroll
        for (int v = 0; v < V; ++v) before[k & 1][v][lane] = mu[v];
    }
  }
  if constexpr (Ends) {
    if (seg == 0 && at.ok)
#pragma unroll
      for (int v = 0; v < V; ++v) a.ends[at.piece * rows + row + v] = make_float2(total[v], mu[v]);
  } else {
    if (a.dstate && at.piece == 0 && seg == 0 && at.ok)
#pragma unroll
      for (int v = 0; v < V; ++v) a.dstate[row + v] = mu[v];
    if constexpr (Decay) {
      __syncthreads();  // the last tile's numbers have been read
#pragma unroll
      for (int v = 0; v < V; ++v) backs[0][seg][v][lane] = sum[v];
      __syncthreads();
      if (seg == 0 && at.ok)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float s = backs[0][0][v][lane];
#pragma unroll
          for (int q = 1; q < SEG; ++q) s += backs[0][q][v][lane];
          a.part[at.piece * rows + row + v] = a.decay[d + v] > 0.f ? 0.f : s;
        }
    }
  }
}

// ------------------------------------------------------------------ host side
// Pieces of the sequence: none while the channels make two blocks an SM, else as many as make four, of two tiles at least.
inline int pieces_of(const haste_b200_gated_scan& a, int V, int tile) {
  const long long blocks = (long long)a.N * ceil_div(a.D, 32 * V);
  if (blocks >= 2LL * sm_count()) return 1;
  const long long most = a.T / (2 * tile), want = (4LL * sm_count() + blocks - 1) / blocks;
  return (int)std::max(1LL, std::min(most, want));
}
// (Scratch is asked for before the pointers are there: whole words are one channel a lane or two, so the most of both.)
inline int most_pieces(const haste_b200_gated_scan& a, int tile) {
  return std::max(pieces_of(a, 1, tile), pieces_of(a, 2, tile));
}

template <typename T>
Args<T> pack(const haste_b200_gated_scan& a, int V) {
  Args<T> k;
  k.T_ = a.T; k.N = a.N; k.D = a.D;
  k.ctiles = ceil_div(a.D, 32 * V);
  k.pieces = 1;
  k.piece = std::max(a.T, 1);
  k.x = Seq<const T>(a.x); k.gate = Seq<const T>(a.gate); k.inner = Seq<const T>(a.input_gate); k.dy = Seq<const T>(a.dy);
  k.y = Seq<T>(a.y); k.dx = Seq<T>(a.dx); k.dgate = Seq<T>(a.dgate); k.dinner = Seq<T>(a.dinput_gate);
  k.decay = a.decay; k.state = a.state; k.dfinal = a.dfinal_state;
  k.final_state = a.final_state; k.checkpoints = a.checkpoints; k.dstate = a.dstate;
  k.ends = nullptr; k.part = nullptr;
  k.lengths = a.lengths;
  return k;
}
template <typename T>
bool words(const haste_b200_gated_scan& a) {
  if (sizeof(T) == 4 || a.D % 2) return false;
  for (const haste_b200_sequence* q : {&a.x, &a.gate, &a.input_gate, &a.y, &a.dy, &a.dx, &a.dgate, &a.dinput_gate})
    if (!aligned(*q, sizeof(T), 4)) return false;
  return true;
}

template <typename T, int V, bool Decay, bool In>
int run_forward(const haste_b200_gated_scan& a, cudaStream_t s) {
  Args<T> k = pack<T>(a, V);
  // (every piece reads the initial state, so a final state in its place takes whole sequences)
  const bool cut = a.scratch && !(a.state && a.final_state == a.state);
  const int pieces = cut ? pieces_of(a, V, FWD_TT) : 1;
  if (pieces > 1) {
    k.piece = ceil_div(ceil_div(a.T, pieces), FWD_TT) * FWD_TT;
    k.pieces = ceil_div(a.T, k.piece);
    k.ends = reinterpret_cast<float2*>(a.scratch);
  }
  const long long blocks = (long long)k.ctiles * a.N;
  HB_REQUIRE(blocks * k.pieces < (1LL << 31), "N*D too large");
  if (k.pieces > 1) {
    gated_fwd<T, V, Decay, In, true><<<(int)(blocks * (k.pieces - 1)), THREADS, 0, s>>>(k);
    HB_LAUNCH_OK();
    count_launch(1);
  }
  gated_fwd<T, V, Decay, In, false><<<(int)(blocks * k.pieces), THREADS, 0, s>>>(k);
  HB_LAUNCH_OK();
  count_launch(1);
  return HASTE_B200_OK;
}
template <typename T, int V, bool Decay, bool In>
int run_backward(const haste_b200_gated_scan& a, cudaStream_t s) {
  Args<T> k = pack<T>(a, V);
  const int pieces = pieces_of(a, V, BWD_TT);
  if (pieces > 1) {
    k.piece = ceil_div(ceil_div(a.T, pieces), BWD_TT) * BWD_TT;
    k.pieces = ceil_div(a.T, k.piece);
  }
  k.ends = reinterpret_cast<float2*>(a.scratch);
  const long long rows = (long long)a.N * a.D;
  if (Decay) k.part = a.scratch + (k.pieces > 1 ? 2LL * k.pieces * rows : 0);
  const long long blocks = (long long)k.ctiles * a.N;
  HB_REQUIRE(blocks * k.pieces < (1LL << 31), "N*D too large");
  if (k.pieces > 1) {
    // (the first piece's pair is nobody's start, but blocks are numbered from it)
    gated_bwd<T, V, Decay, false, true><<<(int)(blocks * k.pieces), THREADS, 0, s>>>(k);
    HB_LAUNCH_OK();
    count_launch(1);
  }
  gated_bwd<T, V, Decay, In, false><<<(int)(blocks * k.pieces), THREADS, 0, s>>>(k);
  HB_LAUNCH_OK();
  count_launch(1);
  if (Decay) {
    SumJobs jobs;
    jobs.add(a.ddecay, 0, 1, a.D, HASTE_B200_F32);
    HB_TRY(sum_parts(k.part, a.N * k.pieces, a.D, jobs, s));
  }
  return HASTE_B200_OK;
}

template <typename T, int V>
int run_step(const haste_b200_gated_scan& a, cudaStream_t s) {
  const Args<T> k = pack<T>(a, V);
  const long long blocks = ((long long)a.N * (a.D / V) + 255) / 256;
  HB_REQUIRE(blocks < (1LL << 31), "N*D too large");
  if (a.decay) gated_step<T, V, true><<<(int)blocks, 256, 0, s>>>(k);
  else gated_step<T, V, false><<<(int)blocks, 256, 0, s>>>(k);
  HB_LAUNCH_OK();
  count_launch(1);
  return HASTE_B200_OK;
}

template <typename T, int V>
int run_gates(const haste_b200_gated_scan& a, bool backward, cudaStream_t s) {
  if (!backward && a.T == 1 && !a.checkpoints) return run_step<T, V>(a, s);
  const bool in = a.input_gate.data != nullptr;
  if (backward) {
    if (a.decay) return in ? run_backward<T, V, true, true>(a, s) : run_backward<T, V, true, false>(a, s);
    return in ? run_backward<T, V, false, true>(a, s) : run_backward<T, V, false, false>(a, s);
  }
  if (a.decay) return in ? run_forward<T, V, true, true>(a, s) : run_forward<T, V, true, false>(a, s);
  return in ? run_forward<T, V, false, true>(a, s) : run_forward<T, V, false, false>(a, s);
}

// One definition per storage type, each in a file of its own.
template <typename T>
int run(const haste_b200_gated_scan& a, bool backward, cudaStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (words<T>(a)) return run_gates<T, 2>(a, backward, s);
  return run_gates<T, 1>(a, backward, s);
}

}  // namespace gated
}  // namespace hb
