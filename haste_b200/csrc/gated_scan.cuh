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
#include <cmath>

#include "state_space.cuh"

namespace hb {

long long gated_scan_scratch(const haste_b200_gated_scan& a, bool backward);

namespace gated {

using namespace ss;

constexpr int THREADS = 128, SEG = THREADS / 32;  // a warp walks one of the tile's segments
constexpr int FWD_L = 4, BWD_L = 4;               // steps of a segment
constexpr int FWD_BLOCKS = 7, BWD_BLOCKS = 4;     // of an SM, as registers allow
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

// Two neighbouring channels go through each instruction (V of one: the second is idle).
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
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
__device__ __forceinline__ float sqrt_fast(float v) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float at_most(float v, float most) {  // (a NaN stays)
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(most));
  return r;
}
// A decay is an exponential and never zero: where it, or a product of them, rounds to zero, float's smallest number stands
// for it.  So an infinite state stays infinite however the sequence is cut, where zero times it would be a NaN, and a finite one
// is off by 2^-149 of itself at most, as its product's rounding is.
__device__ __forceinline__ float not_zero(float v) {  // (a NaN stays)
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(0x1p-149f));
  return r;
}
__device__ __forceinline__ float2 not_zero(float2 v) { return make_float2(not_zero(v.x), not_zero(v.y)); }
template <int V, typename F>
__device__ __forceinline__ float2 each(float2 v, const F& f) {
  return make_float2(f(v.x), V == 2 ? f(v.y) : 0.f);
}
template <typename T, int V>
__device__ __forceinline__ float2 pair_of(const Raw<T, V>& r) {
  float v[V];
  unpack<T, V>(r, v);
  return make_float2(v[0], v[V - 1]);
}
template <typename T, int V>
__device__ __forceinline__ void store_pair(T* p, float2 v) {
  const float w[2] = {v.x, v.y};
  store<T, V>(p, reinterpret_cast<const float(&)[V]>(w));
}
template <int V>
__device__ __forceinline__ float2 load_floats(const float* p) {
  return make_float2(p[0], V == 2 ? p[V - 1] : 0.f);
}
template <int V>
__device__ __forceinline__ void store_floats(float* p, float2 v) {
  p[0] = v.x;
  if (V == 2) p[V - 1] = v.y;
}
constexpr float LOG2E = 1.4426950408889634f;

// (Where a factor is a number, the two channels take an instruction each: the number is part of it, where an instruction for
// two wants it in registers.)

// r = sigmoid(v) and 1 - r, each to its own last bits; exponentials above 2^125 are held there, so that 1 - r, which is
// their product with r, stays one.
template <int V>
__device__ __forceinline__ void sigmoids(float2 v, float2& r, float2& rest) {
  const float2 e = each<V>(v, [](float x) { return at_most(exp2_fast(x * -LOG2E), 0x1p125f); });
  r = each<V>(e, [](float x) { return reciprocal(x + 1.f); });
  rest = __fmul2_rn(e, r);
}
template <int V>
__device__ __forceinline__ float2 sigmoids(float2 v) {
  return each<V>(v, [](float x) { return sigmoid(x); });
}
// 2^l - 1 for l from -0.505 to 0: the exponential's series.
__device__ __forceinline__ constexpr float series(int k) {  // ln(2)^(7 - k) / (7 - k)!
  constexpr float c[] = {1.5252733804059840e-05f, 1.5403530393381608e-04f, 1.3333558146428441e-03f, 9.6181291076284772e-03f,
                         5.5504108664821576e-02f, 2.4022650695910069e-01f, 6.9314718055994529e-01f};
  return c[k];
}
__device__ __forceinline__ float exp2_less_one(float l) {
  float p = series(0);
#pragma unroll
  for (int k = 1; k < 7; ++k) p = fmaf(p, l, series(k));
  return p * l;
}
// a = 2^l for l <= 0, and a - 1.  A decay lies next to one, where the special function unit's results are low by
// 2.4e-8 on average; a state that keeps 1 / (1 - a) steps would add that up.  So a - 1 is computed to its own last bits
// (where a is above 0.7; `far`: some of the block's channels may go below), and a rounded once, to either side.
// Packed: the series' numbers lie in registers, of which the forward pass has enough.
template <int V, bool Packed>
__device__ __forceinline__ void decays(float2 l, bool far, float2& a, float2& n) {
  if constexpr (Packed) {
    float2 p = both(series(0));
#pragma unroll
    for (int k = 1; k < 7; ++k) p = __ffma2_rn(p, l, both(series(k)));
    n = __fmul2_rn(p, l);
  } else {
    n = each<V>(l, [](float x) { return exp2_less_one(x); });
  }
  a = make_float2(n.x + 1.f, n.y + 1.f);
  if (far) {
    const float2 e = each<V>(l, [](float x) { return not_zero(exp2_fast(x)); });
    const bool x = l.x < -0.505f, y = l.y < -0.505f;
    a = make_float2(x ? e.x : a.x, y ? e.y : a.y);
    n = make_float2(x ? e.x - 1.f : n.x, y ? e.y - 1.f : n.y);
  }
}
// Without decay: a = r, rounded once to either side where it is near one.
__device__ __forceinline__ float2 kept(float2 r, float2 rest) {
  return make_float2(r.x > 0.5f ? 1.f - rest.x : r.x, r.y > 0.5f ? 1.f - rest.y : r.y);
}

// A channel's decay in units of log(2): values above zero count as zero, so that no state grows.
template <bool Decay, int V>
__device__ __forceinline__ float2 decay_of(const float* decay, int d) {
  if (!Decay) return both(0.f);
  return each<V>(load_floats<V>(decay + d), [](float v) { return at_most(v, 0.f) * LOG2E; });
}
__device__ __forceinline__ bool goes_far(float2 decay) { return __any_sync(0xffffffffu, decay.x < -0.5f || decay.y < -0.5f); }

// A thread's place in a sequence, which it walks tile by tile: one addition each, where an address anew is two products.
template <typename T>
struct Walk {
  T* p;
  long long by;
  int t;
  __device__ __forceinline__ Walk(const Seq<T>& q, int first, int n, int d, int steps) : p(q.at(first, n) + d), by((long long)steps * q.t), t(q.t) {}
  __device__ __forceinline__ void next() { p += by; }
  __device__ __forceinline__ T* at(int j) const { return p + (long long)j * t; }
};
// A load that needs no predicate.
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p) {
  Raw<T, V> r;
  constexpr int B = sizeof(T) * V;
  if constexpr (B == 2) {
    unsigned short w;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(w) : "l"(p));
    r.w[0] = w;
  } else if constexpr (B == 4) {
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(r.w[0]) : "l"(p));
  } else {
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
  }
  return r;
}
// The steps of a segment, `left` of which exist where not all of the tile's do.
template <int L, int V, typename T, typename U>
__device__ __forceinline__ void fetch_steps(Raw<T, V> (&r)[L], Walk<U>& q, int left, bool whole) {
  if (whole) {
#pragma unroll
    for (int j = 0; j < L; ++j) r[j] = load_raw<T, V>(q.at(j));
  } else {
#pragma unroll
    for (int j = 0; j < L; ++j) r[j] = load_if<T, V>(j < left, q.at(j));
  }
  q.next();
}

// Waits for the launch in front (which this one may have overtaken so far), and lets the next one come.
__device__ __forceinline__ void after_launch_in_front() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_launch_come() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// What comes into a piece from those in front of it (backward: behind it): `count` pairs (product, addend), `step` apart, the
// nearest last, folded by the block's warps a quarter each, many loads at a time.
template <int V>
__device__ __forceinline__ float2 fold_pieces(const float2* first, int count, long long step, float2 start, float4 (&shared)[SEG][32]) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, each = (count + SEG - 1) / SEG;
  float2 p = both(1.f), e = both(0.f);
#pragma unroll 8
  for (int i = warp * each; i < min(count, (warp + 1) * each); ++i) {
    const float2 *q = first + i * step, x = q[0], y = V == 2 ? q[V - 1] : both(0.f);
    e = __ffma2_rn(make_float2(x.x, y.x), e, make_float2(x.y, y.y));
    p = not_zero(__fmul2_rn(p, make_float2(x.x, y.x)));
  }
  shared[warp][lane] = make_float4(p.x, p.y, e.x, e.y);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SEG; ++w) {
    const float4 q = shared[w][lane];
    start = __ffma2_rn(make_float2(q.x, q.y), start, make_float2(q.z, q.w));
  }
  return start;
}

// ------------------------------------------------------------------ forward
// A block takes 64 neighbouring channels, two a lane (32, one a lane, where rows do not start on whole pairs), and tiles of
// four steps to each of its four warps.  A warp folds its steps into (product of decays, what they add to a state of
// zero), the warps' pairs meet in shared memory, each warp folds those in front of its own into the tile's starting state,
// and walks its steps again from registers.  One barrier a tile: pairs and the state behind the tile have two buffers.
// The next tile's words are under way from when the present ones have been used.
// bf16 1000 x 64 x 1024 with both gates: 129 us, 4.1 TB/s (fp32 161, 6.5 TB/s, at the copy bandwidth); with the sigmoids, series and root left out 99 us, which is what
// the accesses and barriers take.  Eight steps a warp and blocks of 256 threads 135 us (fewer instructions, but 3.5 blocks
// an SM to share out); words copied to shared memory tiles ahead 142; one reciprocal for both gates 129.
//
// Few channels leave most of the GPU idle, so their sequences are cut into pieces and read twice (the second time from
// L2): first (Ends) each piece but the last leaves its pair, then each piece starts from those in front of it.
template <typename T, int V, bool Decay, bool In, bool Ends>
__global__ void __launch_bounds__(THREADS, FWD_BLOCKS) gated_fwd(Args<T> a) {
  constexpr int L = FWD_L, TT = FWD_TT;
  __shared__ float4 pairs[2][SEG][32];
  __shared__ float2 behind[2][32];
  const Place<V> at(a);
  const int lane = threadIdx.x % 32, seg = threadIdx.x / 32;
  const int d = at.ok ? at.d : a.D - V;  // (lanes without channels repeat the last ones)
  const long long rows = (long long)a.N * a.D, row = (long long)at.n * a.D + d;
  const float2 decay = decay_of<Decay, V>(a.decay, d);
  const bool far = goes_far(decay);
  float2 start = !Ends && a.state ? load_floats<V>(a.state + row) : both(0.f), total = both(1.f);
  const int stop = min(at.last, at.len);  // tiles from here on are behind the row's end
  const int ts0 = at.first + seg * L;
  Walk<const T> px(a.x, ts0, at.n, d, TT), pg(a.gate, ts0, at.n, d, TT), pi(In ? a.inner : a.x, ts0, at.n, d, TT);
  Walk<T> py(a.y, Ends ? 0 : ts0, at.n, d, TT);
  Raw<T, V> xn[L], gn[L], in[L];
  auto fetch = [&](int t0) {
    const bool whole = t0 + TT <= stop;
    const int left = stop - t0 - seg * L;
    fetch_steps<L>(xn, px, left, whole);
    fetch_steps<L>(gn, pg, left, whole);
    if (In) fetch_steps<L>(in, pi, left, whole);
  };
  if (at.first < stop) fetch(at.first);
  if (Ends) {
    let_next_launch_come();
  } else if (a.pieces > 1) {
    after_launch_in_front();
    // (the first tile's pairs go into the other buffer)
    start = fold_pieces<V>(a.ends + row, at.piece, rows, start, pairs[1]);
  }
  float2 h = start;
  int k = 0;
  for (int t0 = at.first; t0 < stop; t0 += TT, ++k) {
    const int ts = t0 + seg * L;
    float2 s[L], b[L], p, e;
#pragma unroll
    for (int j = 0; j < L; ++j) {
      float2 w, r, rest;
      if constexpr (Decay) r = sigmoids<V>(pair_of<T, V>(gn[j]));
      else sigmoids<V>(pair_of<T, V>(gn[j]), r, rest);
      if constexpr (Decay) {
        float2 n;
        decays<V, true>(__fmul2_rn(decay, r), far, s[j], n);
        w = each<V>(__ffma2_rn(n, s[j], n), [](float x) { return sqrt_fast(-x); });  // 1 - a^2 = -n (1 + a)
      } else {
        w = rest;
        s[j] = kept(r, w);
      }
      b[j] = __fmul2_rn(w, pair_of<T, V>(xn[j]));
      if (In) b[j] = __fmul2_rn(b[j], sigmoids<V>(pair_of<T, V>(in[j])));
    }
    if (t0 + TT > stop)
#pragma unroll
      for (int j = 0; j < L; ++j)
        if (ts + j >= stop) s[j] = both(1.f), b[j] = both(0.f);
    if (t0 + TT < stop) fetch(t0 + TT);
    p = s[0];
    e = b[0];
#pragma unroll
    for (int j = 1; j < L; ++j) {
      e = __ffma2_rn(s[j], e, b[j]);
      p = __fmul2_rn(p, s[j]);
    }
    p = not_zero(p);
    pairs[k & 1][seg][lane] = make_float4(p.x, p.y, e.x, e.y);
    __syncthreads();
    if constexpr (Ends) {
      if (seg == 0)
#pragma unroll
        for (int q = 0; q < SEG; ++q) {
          const float4 w = pairs[k & 1][q][lane];
          h = __ffma2_rn(make_float2(w.x, w.y), h, make_float2(w.z, w.w));
          total = not_zero(__fmul2_rn(total, make_float2(w.x, w.y)));
        }
    } else {
      h = k ? behind[(k - 1) & 1][lane] : start;
      for (int q = 0; q < seg; ++q) {
        const float4 w = pairs[k & 1][q][lane];
        h = __ffma2_rn(make_float2(w.x, w.y), h, make_float2(w.z, w.w));
      }
      if (a.checkpoints && seg * L % CKPT == 0 && at.ok && ts < at.last) store_floats<V>(a.checkpoints + ts / CKPT * rows + row, h);
      if (t0 + TT <= stop) {
#pragma unroll
        for (int j = 0; j < L; ++j) {
          h = __ffma2_rn(s[j], h, b[j]);
          if (at.ok) store_pair<T, V>(py.at(j), h);
        }
      } else {
#pragma unroll
        for (int j = 0; j < L; ++j) {
          h = __ffma2_rn(s[j], h, b[j]);
          if (at.ok && ts + j < at.last) store_pair<T, V>(py.at(j), ts + j < stop ? h : both(0.f));
        }
      }
      py.next();
      if (seg == SEG - 1) behind[k & 1][lane] = h;
    }
  }
  if (!at.ok) return;
  if constexpr (Ends) {
    if (seg == 0) {
      float2* e = a.ends + at.piece * rows + row;
      e[0] = make_float2(total.x, h.x);
      if (V == 2) e[V - 1] = make_float2(total.y, h.y);
    }
  } else {
    for (int t = at.first + k * TT + seg; t < at.last; t += SEG) store_pair<T, V>(a.y.at(t, at.n) + d, both(0.f));
    if (a.final_state && at.piece == a.pieces - 1 && seg == SEG - 1) store_floats<V>(a.final_state + row, h);
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
  float2 h = a.state ? load_floats<V>(a.state + row) : both(0.f), w, s;
  const float2 decay = decay_of<Decay, V>(a.decay, d);
  if constexpr (Decay) {
    float2 m;
    decays<V, false>(__fmul2_rn(decay, sigmoids<V>(pair_of<T, V>(gr))), true, s, m);
    w = each<V>(__ffma2_rn(m, s, m), [](float x) { return sqrt_fast(-x); });
  } else {
    float2 r;
    sigmoids<V>(pair_of<T, V>(gr), r, w);
    s = kept(r, w);
  }
  float2 b = __fmul2_rn(w, pair_of<T, V>(xr));
  if (a.inner.p) b = __fmul2_rn(b, sigmoids<V>(pair_of<T, V>(ir)));
  if (live) h = __ffma2_rn(s, h, b);
  if (a.final_state) store_floats<V>(a.final_state + row, h);
  store_pair<T, V>(a.y.at(0, n) + d, live ? h : both(0.f));
}

// ------------------------------------------------------------------ backward
// The same blocks and barriers, from the last tile to the first, with four steps to a warp.  A tile's states come from
// the one that the forward pass left in front of it; a segment is a pair for the states, and for the adjoint
// mu = a lam, which runs the other way, the same product and a third number.
// Ends: pieces but the first leave (product, mu that they give to one of zero behind them).
// bf16 1000 x 64 x 1024 with both gates: 227 us, 4.0 TB/s (by itself, from a cold L2, 234), bound by what 16 warps an SM issue
// next to each other (0.6 of the slots): a step's numbers fill 128 registers a thread; fp32 350 us, 5.2 TB/s.  Five blocks an SM spill (629 us), blocks of 256 threads 242.
template <typename T, int V, bool Decay, bool In, bool Ends>
__global__ void __launch_bounds__(THREADS, BWD_BLOCKS) gated_bwd(Args<T> a) {
  constexpr int L = BWD_L, TT = BWD_TT;
  __shared__ float4 pairs[2][SEG][32];
  __shared__ float2 backs[2][SEG][32];
  __shared__ float2 before[2][32];
  const Place<V> at(a);
  const int lane = threadIdx.x % 32, seg = threadIdx.x / 32;
  const int d = at.ok ? at.d : a.D - V;
  const long long rows = (long long)a.N * a.D, row = (long long)at.n * a.D + d;
  const float2 decay = decay_of<Decay, V>(a.decay, d);
  const bool far = goes_far(decay);
  const float2 natural = __fmul2_rn(decay, both(0.6931471805599453f));  // decay as it was given
  // (a channel whose decay is zero adds nothing to its state: w, whose slope has no value there, counts as constant)
  const float2 moves = make_float2(decay.x != 0.f ? 1.f : 0.f, decay.y != 0.f ? 1.f : 0.f);
  float2 start = !Ends && a.dfinal ? load_floats<V>(a.dfinal + row) : both(0.f), total = both(1.f), sum = both(0.f);

  const int stop = min(at.last, at.len);
  const int tiles = stop > at.first ? (stop - at.first + TT - 1) / TT : 0;
  const int ts0 = at.first + max(tiles - 1, 0) * TT + seg * L;
  Walk<const T> pg(a.gate, ts0, at.n, d, -TT), py(a.dy, ts0, at.n, d, -TT), px(a.x, ts0, at.n, d, -TT),
      pi(In ? a.inner : a.x, ts0, at.n, d, -TT);
  Walk<T> qx(a.dx, Ends ? 0 : ts0, at.n, d, -TT), qg(a.dgate, Ends ? 0 : ts0, at.n, d, -TT),
      qi(In ? a.dinner : a.dx, Ends ? 0 : ts0, at.n, d, -TT);
  const float* ph = a.checkpoints + (ts0 - seg * L) / CKPT * rows + row;
  Raw<T, V> xn[L], gn[L], in[L], yn[L];
  float2 hn = both(0.f);
  auto fetch = [&](int t0) {
    const bool whole = t0 + TT <= stop;
    const int left = stop - t0 - seg * L;
    fetch_steps<L>(gn, pg, left, whole);
    fetch_steps<L>(yn, py, left, whole);
    if (Ends) return;
    fetch_steps<L>(xn, px, left, whole);
    if (In) fetch_steps<L>(in, pi, left, whole);
    hn = load_floats<V>(ph);
    ph -= rows;
  };
  if (tiles) fetch(at.first + (tiles - 1) * TT);
  if (Ends) {
    let_next_launch_come();
  } else if (a.pieces > 1) {
    after_launch_in_front();
    start = fold_pieces<V>(a.ends + (a.pieces - 1) * rows + row, a.pieces - 1 - at.piece, -rows, start, pairs[1]);
  }
  float2 mu = start;
  if constexpr (!Ends) {
    if (at.ok)
      for (int t = at.first + tiles * TT + seg; t < at.last; t += SEG) {
        store_pair<T, V>(a.dx.at(t, at.n) + d, both(0.f));
        store_pair<T, V>(a.dgate.at(t, at.n) + d, both(0.f));
        if (In) store_pair<T, V>(a.dinner.at(t, at.n) + d, both(0.f));
      }
  }
  for (int k = 0; k < tiles; ++k) {
    const int t0 = at.first + (tiles - 1 - k) * TT, ts = t0 + seg * L;
    const bool whole = t0 + TT <= stop;
    // b: what a step adds to the state; wi: w sigmoid(i); c: -u a / w (without decay -u); r, rest: the gate's sigmoid and
    // (with decay) decay (1 - r); irest: 1 - sigmoid(i)
    float2 s[L], b[L], wi[L], c[L], r[L], rest[L], irest[L], dy[L], h;
#pragma unroll
    for (int j = 0; j < L; ++j) {
      float2 w, i;
      dy[j] = pair_of<T, V>(yn[j]);
      sigmoids<V>(pair_of<T, V>(gn[j]), r[j], rest[j]);
      if constexpr (Decay) {
        float2 n;
        decays<V, false>(__fmul2_rn(decay, r[j]), far, s[j], n);
        if (Ends) continue;
        const float2 v = __ffma2_rn(n, s[j], n);  // a^2 - 1
        // (1 / w with 1e-30 added to w^2, so that it stays finite where w is zero)
        const float2 over = each<V>(v, [](float x) { return -rsqrt_fast(1e-30f - x); });
        w = __fmul2_rn(v, over);
        c[j] = __fmul2_rn(__fmul2_rn(s[j], moves), over);
        rest[j] = __fmul2_rn(rest[j], natural);
      } else {
        w = rest[j];
        s[j] = kept(r[j], w);
        if (Ends) continue;
        c[j] = both(-1.f);
      }
      const float2 x = pair_of<T, V>(xn[j]);
      float2 u = x;
      wi[j] = w;
      if (In) {
        sigmoids<V>(pair_of<T, V>(in[j]), i, irest[j]);
        u = __fmul2_rn(x, i);
        wi[j] = __fmul2_rn(w, i);
      }
      b[j] = __fmul2_rn(w, u);
      c[j] = __fmul2_rn(c[j], u);
    }
    if (!whole)
#pragma unroll
      for (int j = 0; j < L; ++j)
        if (ts + j >= stop) s[j] = both(1.f), b[j] = both(0.f);  // (dy is zero)
    if (!Ends) h = hn;
    if (k + 1 < tiles) fetch(t0 - TT);
    float2 p = s[0], e = both(0.f), m = both(0.f);
    if (!Ends) e = b[0];
#pragma unroll
    for (int j = 1; j < L; ++j) {
      if (!Ends) e = __ffma2_rn(s[j], e, b[j]);
      p = __fmul2_rn(p, s[j]);
    }
    p = not_zero(p);
#pragma unroll
    for (int j = L - 1; j >= 0; --j) m = __fmul2_rn(s[j], __fadd2_rn(dy[j], m));
    pairs[k & 1][seg][lane] = make_float4(p.x, p.y, e.x, e.y);
    backs[k & 1][seg][lane] = m;
    __syncthreads();
    if constexpr (Ends) {
      if (seg == 0)
#pragma unroll
        for (int q = SEG - 1; q >= 0; --q) {
          const float4 w = pairs[k & 1][q][lane];
          mu = __ffma2_rn(make_float2(w.x, w.y), mu, backs[k & 1][q][lane]);
          total = not_zero(__fmul2_rn(total, make_float2(w.x, w.y)));
        }
    } else {
      for (int q = 0; q < seg; ++q) {
        const float4 w = pairs[k & 1][q][lane];
        h = __ffma2_rn(make_float2(w.x, w.y), h, make_float2(w.z, w.w));
      }
      mu = k ? before[(k - 1) & 1][lane] : start;
      for (int q = SEG - 1; q > seg; --q) {
        const float4 w = pairs[k & 1][q][lane];
        mu = __ffma2_rn(make_float2(w.x, w.y), mu, backs[k & 1][q][lane]);
      }
#pragma unroll
      for (int j = 0; j < L; ++j) {
        c[j] = __fadd2_rn(c[j], h);  // h_{t-1} - u a / w
        h = __ffma2_rn(s[j], h, b[j]);
      }
      auto gradients = [&](auto every) {  // every: all of the tile's steps are in front of the row's end
#pragma unroll
        for (int j = L - 1; j >= 0; --j) {
          const float2 lam = __fadd2_rn(dy[j], mu);
          mu = __fmul2_rn(lam, s[j]);
          float2 dx = __fmul2_rn(lam, wi[j]), dg, di = both(0.f), by_decay = both(0.f);
          if (Decay) {
            by_decay = __fmul2_rn(__fmul2_rn(mu, c[j]), r[j]);
            dg = __fmul2_rn(by_decay, rest[j]);
          } else {
            dg = __fmul2_rn(__fmul2_rn(mu, c[j]), rest[j]);
          }
          if (In) di = __fmul2_rn(__fmul2_rn(lam, b[j]), irest[j]);
          if (!every.value && ts + j >= stop) dx = dg = di = by_decay = both(0.f);
          if (Decay) sum = __fadd2_rn(sum, by_decay);
          if (at.ok && (every.value || ts + j < at.last)) {
            store_pair<T, V>(qx.at(j), dx);
            store_pair<T, V>(qg.at(j), dg);
            if (In) store_pair<T, V>(qi.at(j), di);
          }
        }
      };
      if (whole) gradients(std::true_type());
      else gradients(std::false_type());
      qx.next();
      qg.next();
      if (In) qi.next();
      if (seg == 0) before[k & 1][lane] = mu;
    }
  }
  if constexpr (Ends) {
    if (seg == 0 && at.ok) {
      float2* e = a.ends + at.piece * rows + row;
      e[0] = make_float2(total.x, mu.x);
      if (V == 2) e[V - 1] = make_float2(total.y, mu.y);
    }
  } else {
    if (a.dstate && at.piece == 0 && seg == 0 && at.ok) store_floats<V>(a.dstate + row, mu);
    if constexpr (Decay) {
      __syncthreads();  // the last tile's numbers have been read
      backs[0][seg][lane] = sum;
      __syncthreads();
      if (seg == 0 && at.ok) {
        float2 s = backs[0][0][lane];
#pragma unroll
        for (int q = 1; q < SEG; ++q) s = __fadd2_rn(s, backs[0][q][lane]);
        const float2 raw = load_floats<V>(a.decay + d);
        store_floats<V>(a.part + at.piece * rows + row, make_float2(raw.x > 0.f ? 0.f : s.x, raw.y > 0.f ? 0.f : s.y));
      }
    }
  }
}

// ------------------------------------------------------------------ host side
// Pieces of the sequence: none while the channels make blocks enough (two an SM; backward, which keeps four on an SM where
// the forward pass keeps seven, one and a half), else as many as make seven an SM (four: bf16 1000 x 8 x 1024 47 us,
// backward 62), of a tile at least and three times the root of the steps at most, beyond which folding them takes longer than
// walking them.  Forward / backward in us with once, twice, three times, 4.5 times the root and without a bound: bf16 4000 x 1 x 256
// 12.8 / 15.5, 11.2 / 12.9, 11.2 / 12.9, 13.7 / 17.8, the same; 16000 x 1 x 64 20.6 / 22.5, 15.9 / 17.7, 15.5 / 17.4, 17.3 / 18.4,
// 31.4 / 30.8; fp32 23.9 / 27.6, 19.4 / 20.8, 19.3 / 20.1, 23.0 / 20.9, 39.4 / 31.5; bf16 64000 x 1 x 64 40.0 / 42.0, 31.8 / 34.0,
// 35.8 / 39.3, 42.1 / 45.6, the same.  us, whole / in pieces, both gates, bf16 1000 x N x 1024: N = 8 forward 70 / 39, backward 86 / 51; 16 78 / 66, 96 / 100; 32 92 / 111, 128 / 172; fp32
// 2000 x 1 x 1024 162 / 17, 221 / 26; bf16 100 x 8 x 1024 14 / 12, 18 / 17.
inline int pieces_of(const haste_b200_gated_scan& a, int V, bool backward) {
  const long long blocks = (long long)a.N * ceil_div(a.D, 32 * V), sms = sm_count();
  const int tile = backward ? BWD_TT : FWD_TT;
  if (blocks * 2 >= sms * (backward ? 3 : 4) || a.T < 4 * tile) return 1;
  const long long most = std::min(a.T / tile, (int)(3 * std::sqrt((double)a.T)));
  return (int)std::min(most, (7 * sms + blocks - 1) / blocks);
}
// (Scratch is asked for before the pointers are there, which decide on one channel a lane or two: the most of both.)
inline int most_pieces(const haste_b200_gated_scan& a, bool backward) {
  return std::max(pieces_of(a, 1, backward), pieces_of(a, 2, backward));
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
bool in_pairs(const haste_b200_gated_scan& a) {
  if (a.D % 2) return false;
  for (const haste_b200_sequence* q : {&a.x, &a.gate, &a.input_gate, &a.y, &a.dy, &a.dx, &a.dgate, &a.dinput_gate})
    if (!aligned(*q, sizeof(T), 2 * sizeof(T))) return false;
  return true;
}

// A launch that may begin while the one in front of it ends; it waits for that itself.
template <typename K, typename A>
int launch_behind(K kernel, long long blocks, const A& args, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  HB_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, args));
  count_launch(1);
  return HASTE_B200_OK;
}

template <typename T, int V, bool Decay, bool In>
int run_forward(const haste_b200_gated_scan& a, cudaStream_t s) {
  Args<T> k = pack<T>(a, V);
  // (every piece reads the initial state, so a final state in its place takes whole sequences)
  const bool cut = a.scratch && !(a.state && a.final_state == a.state);
  const int pieces = cut ? pieces_of(a, V, false) : 1;
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
    return launch_behind(gated_fwd<T, V, Decay, In, false>, blocks * k.pieces, k, s);
  }
  gated_fwd<T, V, Decay, In, false><<<(int)blocks, THREADS, 0, s>>>(k);
  HB_LAUNCH_OK();
  count_launch(1);
  return HASTE_B200_OK;
}
template <typename T, int V, bool Decay, bool In>
int run_backward(const haste_b200_gated_scan& a, cudaStream_t s) {
  Args<T> k = pack<T>(a, V);
  const int pieces = pieces_of(a, V, true);
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
    HB_TRY(launch_behind(gated_bwd<T, V, Decay, In, false>, blocks * k.pieces, k, s));
  } else {
    gated_bwd<T, V, Decay, In, false><<<(int)blocks, THREADS, 0, s>>>(k);
    HB_LAUNCH_OK();
    count_launch(1);
  }
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
  if (in_pairs<T>(a)) return run_gates<T, 2>(a, backward, s);
  return run_gates<T, 1>(a, backward, s);
}

}  // namespace gated
}  // namespace hb
