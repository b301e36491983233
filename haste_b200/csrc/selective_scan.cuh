// Arguments and arithmetic shared by the selective scan's forward and backward kernels.
#pragma once

#include "state_space.cuh"

namespace hb {
namespace scan {

using namespace ss;

constexpr int NS = 4;    // states of one thread
constexpr int CKPT = 8;  // steps between the states that the forward pass leaves for the backward pass

template <typename T>
struct Args {
  int T_, N, D, G, S, per, ctiles;  // per: channels of a group, ctiles: blocks that share them out
  int n0, rows, most;               // the rows of this launch, and the most of any
  int chunks, chunk;                // pieces of the sequence that blocks work on side by side, steps of one
  bool softplus;
  Seq<const T> x, dt, z, B, C, dy;
  Seq<T> y, dx, ddt, dz, dB, dC;
  long long B_g, C_g, dB_g, dC_g;
  const float *A, *skip, *dt_bias, *state, *dfinal;
  float *final_state, *checkpoints, *dstate, *part;
  float *ends, *sums;  // [chunks][N][D][S], [chunks][N][D]: what a piece adds to the state, and its sum of delta
  const long long* lengths;
};

// Where a block works: channels d0 .. d0 + count - 1 of group g in row n, steps first .. last - 1.
struct Place {
  int ct, n, g, d0, count, piece, first, last;
  template <typename A>
  __device__ __forceinline__ Place(const A& a, int CB) {
    int r = blockIdx.x / a.ctiles;
    ct = blockIdx.x % a.ctiles;
    g = r % a.G;
    r /= a.G;
    n = a.n0 + r % a.rows;
    piece = r / a.rows;
    d0 = g * a.per + ct * CB;
    count = min(CB, a.per - ct * CB);
    first = piece * a.chunk;
    last = min(a.T_, first + a.chunk);
  }
};

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// 2^v on the special function unit, whose results are low by 2.4e-8 of their value on average for v in
// [-1/64, 0] and by 5.4e-8 below (measured).  A state that decays slowly adds that bias up over
// 1 / (1 - a) steps, so decay() shifts the argument by half of it, in the same instruction.
__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float EXP2_LOW = 3e-8f;
// exp(delta A) for two states, A in units of log2(e).
__device__ __forceinline__ float2 decay(float2 delta, float2 A) {
  const float2 v = __ffma2_rn(delta, A, make_float2(EXP2_LOW, EXP2_LOW));
  return make_float2(exp2_fast(v.x), exp2_fast(v.y));
}
// exp(sum A) h + e: what stands behind a piece whose steps add up to `sum`.  Decays above one (A or delta of the
// other sign) may have a product beyond float32 where the state that they meet is zero or small: two factors.
__device__ __forceinline__ float behind(float sum, float A, float h, float e) {
  const float v = fmaf(sum, A, EXP2_LOW), first = v > 127.f ? 127.f : v;  // (a NaN stays)
  h *= exp2_fast(first);
  if (h != 0.f) h *= exp2_fast(v - first);
  return h + e;
}
__device__ __forceinline__ float2 behind(float sum, float2 A, float2 h, float2 e) {
  return make_float2(behind(sum, A.x, h.x, e.x), behind(sum, A.y, h.y, e.y));
}

// delta = log(1 + exp(v)) = max(v, 0) + log(1 + e) and its slope, with e = exp(-|v|).  The product
// -|v| log2(e) is taken in two parts, so that e keeps its bits for large |v|; log(1 + e) / e on [0, 1] is a
// polynomial of degree 8, fitted for the least relative error (3e-8).
template <int V, bool Slope>
__device__ __forceinline__ void softplus(float (&v)[V], float (&slope)[V]) {
  constexpr float c[] = {0.00523269070233413f, -0.02950522894050519f, 0.0782259443637453f, -0.13663246046340774f,
                         0.191060074281249f,   -0.2484298258665141f,  0.33319096896971945f, -0.4999949314926837f,
                         0.9999999698819679f};
#pragma unroll
  for (int i = 0; i < V; i += 2) {  // two values to an instruction
    const float2 x = make_float2(v[i], v[i + 1 < V ? i + 1 : i]);
    float2 m = make_float2(fabsf(x.x), fabsf(x.y));
    m.x = m.x > 128.f ? 128.f : m.x;  // (a NaN stays)
    m.y = m.y > 128.f ? 128.f : m.y;
    const float2 hi = __fmul2_rn(m, both(-LOG2E));
    const float2 lo = __ffma2_rn(m, both(-1.925963033500e-8f), __ffma2_rn(m, both(-LOG2E), make_float2(-hi.x, -hi.y)));
    const float2 r = make_float2(exp2_fast(hi.x), exp2_fast(hi.y)), e = __ffma2_rn(r, __fmul2_rn(lo, both(LN2)), r);
    float2 p = both(c[0]);
#pragma unroll
    for (int k = 1; k < 9; ++k) p = __ffma2_rn(p, e, both(c[k]));
    p = __ffma2_rn(p, e, make_float2(fmaxf(x.x, 0.f), fmaxf(x.y, 0.f)));
    v[i] = p.x;
    if (Slope) slope[i] = (x.x >= 0.f ? 1.f : e.x) * reciprocal(1.f + e.x);
    if (i + 1 < V) {
      v[i + 1] = p.y;
      if (Slope) slope[i + 1] = (x.y >= 0.f ? 1.f : e.y) * reciprocal(1.f + e.y);
    }
  }
}
__device__ __forceinline__ float softplus(float v) {
  float x[1] = {v}, none[1];
  softplus<1, false>(x, none);
  return x[0];
}

// A thread's NS neighbouring values of a row of S, zero beyond its end.
__device__ __forceinline__ void load_states(const float* p, int s0, int S, float2 (&v)[NS / 2]) {
  if (S % NS == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    const float4 w = s0 < S ? *reinterpret_cast<const float4*>(p + s0) : make_float4(0.f, 0.f, 0.f, 0.f);
    v[0] = make_float2(w.x, w.y);
    v[1] = make_float2(w.z, w.w);
    return;
  }
#pragma unroll
  for (int i = 0; i < NS / 2; ++i) {
    v[i].x = s0 + 2 * i < S ? p[s0 + 2 * i] : 0.f;
    v[i].y = s0 + 2 * i + 1 < S ? p[s0 + 2 * i + 1] : 0.f;
  }
}
__device__ __forceinline__ void store_states(float* p, int s0, int S, const float2 (&v)[NS / 2]) {
  if (S % NS == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    if (s0 < S) *reinterpret_cast<float4*>(p + s0) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    return;
  }
#pragma unroll
  for (int i = 0; i < NS / 2; ++i) {
    if (s0 + 2 * i < S) p[s0 + 2 * i] = v[i].x;
    if (s0 + 2 * i + 1 < S) p[s0 + 2 * i + 1] = v[i].y;
  }
}
// Four floats of shared memory as two pairs.
__device__ __forceinline__ void load_pairs(const float* p, float2 (&v)[2]) {
  const float4 w = *reinterpret_cast<const float4*>(p);
  v[0] = make_float2(w.x, w.y);
  v[1] = make_float2(w.z, w.w);
}
// B bytes of global to shared memory behind the thread's back, zeros unless `ok`.
template <int B>
__device__ __forceinline__ void copy_async(float* to, const float* from, bool ok) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  const int bytes = ok ? B : 0;
  if constexpr (B == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(at), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// How a block is laid out: Q lanes of NS states a channel, CH channels a thread, tiles of TT staged steps.
constexpr int THREADS = 128;
template <int Q, int CH, int TT>
struct Tile {
  static constexpr int CB = THREADS / Q, CT = CB * CH, SP = Q * NS;
  static constexpr int PER = TT * CT >= THREADS ? TT * CT / THREADS : 1;  // staged (step, channel) pairs of a thread
  static constexpr int V = PER < 4 ? PER : 4;                            // neighbouring channels among them, at most
  // A row of the lanes' partial sums, one per lane of a channel: shifted so that a warp's stores fall into 32 banks.
  static constexpr int YC = CT + (Q == 1 ? 0 : 32 / Q);
  // rows of B or C that the block loads together, and how often
  static constexpr int BR = THREADS / SP, PB = (TT + BR - 1) / BR;
};
constexpr int fwd_steps(int Q) { return Q <= 2 ? 8 : 16; }

// The sums of the Q lanes' parts for V neighbouring channels; p: the first lane's.
template <int Q, int V, int YC>
__device__ __forceinline__ void sum_parts_of(const float* p, float (&s)[V]) {
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    float w[V];
    load<float, V>(p + i * YC, w);
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = i ? s[v] + w[v] : w[v];
  }
}

// A thread's four states in another order: register i gets state i ^ order.
__device__ __forceinline__ void reorder(float2 (&v)[2], int order) {
  if (order & 2) {
    const float2 w = v[0];
    v[0] = v[1];
    v[1] = w;
  }
  if (order & 1) {
    v[0] = make_float2(v[0].y, v[0].x);
    v[1] = make_float2(v[1].y, v[1].x);
  }
}

// Whether a group's width, the strides and the starts allow accesses of V channels.
inline bool wide(const haste_b200_selective_scan& a, int V, bool backward) {
  const int e = (int)dtype_size(a.dtype), b = V * e;
  bool ok = (a.D / a.G) % V == 0 && aligned(a.x, e, b) && aligned(a.dt, e, b) && aligned(a.z, e, b);
  if (!backward) return ok && aligned(a.y, e, b);
  return ok && aligned(a.dy, e, b) && aligned(a.dx, e, b) && aligned(a.ddt, e, b) && aligned(a.dz, e, b);
}

// Lanes per channel: states in fours, a power of two.
inline int lanes(int S) {
  int q = 1;
  while (q * NS < S) q *= 2;
  return q;
}

int check(const haste_b200_selective_scan& a, bool backward);

// One definition per storage type, each in a file of its own.
template <typename T>
int forward(const haste_b200_selective_scan& a, cudaStream_t s);
template <typename T>
int backward(const haste_b200_selective_scan& a, cudaStream_t s);
int forward_pieces(const haste_b200_selective_scan& a);

// How a backward call is cut: channels per thread, and pieces of the sequence.
struct BwdShape {
  int Q, CH, ctiles, chunks, chunk;
  int rows;          // of one launch
  long long blocks;  // of a piece and all rows
  explicit BwdShape(const haste_b200_selective_scan& a) {
    Q = lanes(a.S);
    const int per = a.D / a.G, CB = THREADS / Q;
    const long long lines = (long long)a.N * a.G;
    // two channels a thread while their blocks fill the GPU (bf16 T=1000 N=64 D=1024 S=16: 1735 us with one, 1617 with two)
    // (One lane a channel takes one: two would be 256 channels a block, more than its threads stage one by one, and
    // spill; bf16 T=400 N=64 D=2048 S=4 667 us with two, 470 with one; fp32 300 x 16 x 8192 709 and 428.  A rule on
    // sizes alone: the scratch may be asked for before the pointers, whose alignment decides on wider staging, are there.)
    CH = Q > 1 && lines * ceil_div(per, 2 * CB) >= 3LL * sm_count() ? 2 : 1;
    ctiles = ceil_div(per, CB * CH);
    blocks = lines * ctiles;
    chunks = 1;
    chunk = a.T > 0 ? a.T : 1;
    // As in the forward pass; the walk that pieces add is a quarter of the pass.  fp32 T=333 N=7 D=250 S=24, us:
    // whole 79, pieces for 2, 3, 5, 8 blocks per SM 63, 61, 54, 54.
    if (blocks < 2LL * sm_count()) {
      const long long most = ceil_div(a.T, 64), want = (5LL * sm_count() + blocks - 1) / blocks;
      if (want >= 2 && most >= 2) {
        chunk = ceil_div(ceil_div(a.T, want < most ? want : most), 32) * 32;
        chunks = ceil_div(a.T, chunk);
      }
    }
    // Many states make few channels a block and many partial rows of dB and dC: beyond a GB of them the rows
    // of the batch are taken in turn, as long as each turn fills the GPU.
    const long long a_row = (long long)ctiles * a.T * a.G * 2 * Q * NS, fill = (3LL * sm_count() * a.N + blocks * chunks - 1) / (blocks * chunks);
    long long most = a_row > 0 ? (1LL << 28) / a_row : a.N;
    if (most < fill) most = fill;
    rows = most < 1 ? 1 : most < a.N ? (int)most : a.N;
  }
  // scratch: partial rows of dB and dC, sums of dA, dskip and ddt_bias, the pieces' ends
  long long bc_floats(const haste_b200_selective_scan& a) const { return (long long)ctiles * a.T * rows * a.G * 2 * Q * NS; }
  long long sum_floats(const haste_b200_selective_scan& a) const { return (long long)chunks * a.N * a.D * (a.S + 2); }
  long long floats(const haste_b200_selective_scan& a) const {
    return bc_floats(a) + sum_floats(a) + (chunks > 1 ? (long long)chunks * a.N * a.D * (a.S + 1) : 0);
  }
};

template <typename T>
Args<T> pack(const haste_b200_selective_scan& a, int CB) {
  Args<T> k;
  k.T_ = a.T; k.N = a.N; k.n0 = 0; k.rows = k.most = a.N; k.D = a.D; k.G = a.G; k.S = a.S;
  k.per = a.D / a.G;
  k.ctiles = ceil_div(k.per, CB);
  k.chunks = 1;
  k.chunk = a.T;
  k.softplus = a.softplus != 0;
  k.x = Seq<const T>(a.x); k.dt = Seq<const T>(a.dt); k.z = Seq<const T>(a.z);
  k.B = Seq<const T>(a.B); k.C = Seq<const T>(a.C); k.dy = Seq<const T>(a.dy);
  k.y = Seq<T>(a.y); k.dx = Seq<T>(a.dx); k.ddt = Seq<T>(a.ddt); k.dz = Seq<T>(a.dz);
  k.dB = Seq<T>(a.dB); k.dC = Seq<T>(a.dC);
  k.B_g = a.B_g; k.C_g = a.C_g; k.dB_g = a.dB_g; k.dC_g = a.dC_g;
  k.A = a.A; k.skip = a.skip; k.dt_bias = a.dt_bias; k.state = a.state; k.dfinal = a.dfinal_state;
  k.final_state = a.final_state; k.checkpoints = a.checkpoints; k.dstate = a.dstate; k.part = a.scratch;
  k.ends = k.sums = nullptr;
  k.lengths = a.lengths;
  return k;
}

}  // namespace scan
}  // namespace hb
