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
  bool softplus;
  Seq<const T> x, dt, z, B, C, dy;
  Seq<T> y, dx, ddt, dz, dB, dC;
  long long B_g, C_g, dB_g, dC_g;
  const float *A, *skip, *dt_bias, *state, *dfinal;
  float *final_state, *checkpoints, *dstate, *part;
  const long long* lengths;
};

// Where a block works: channels d0 .. d0 + CB - 1 of group g in row n.
struct Place {
  int n, g, d0, count;  // count: channels that exist
  template <typename A>
  __device__ __forceinline__ Place(const A& a, int CB) {
    const int ct = blockIdx.x % a.ctiles, r = blockIdx.x / a.ctiles;
    g = r % a.G;
    n = r / a.G;
    const int first = ct * CB;
    d0 = g * a.per + first;
    count = min(CB, a.per - first);
  }
};

// 2^v on the special function unit; a = exp(delta A) is exp2(delta (A log2 e)).
__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float LOG2E = 1.4426950408889634f;

// log(1 + exp(v)), from the side where the exponential is small.
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.f) + log1pf(__expf(-fabsf(v))); }

// A thread's NS neighbouring values of a row of S, zero beyond its end.
__device__ __forceinline__ void load_states(const float* p, int s0, int S, float (&v)[NS]) {
  if (S % NS == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    if (s0 < S) {
      const float4 w = *reinterpret_cast<const float4*>(p + s0);
      v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    } else {
      v[0] = v[1] = v[2] = v[3] = 0.f;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < NS; ++i) v[i] = s0 + i < S ? p[s0 + i] : 0.f;
}
__device__ __forceinline__ void store_states(float* p, int s0, int S, const float (&v)[NS]) {
  if (S % NS == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    if (s0 < S) *reinterpret_cast<float4*>(p + s0) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < NS; ++i)
    if (s0 + i < S) p[s0 + i] = v[i];
}

// Sums COUNT values over the LANES lanes that differ in the bits of LANES / 2 * STRIDE .. STRIDE.  While
// there are several values a lane hands half of them over and keeps the other half (COUNT - 1
// shuffles for COUNT = LANES); afterwards v[0 .. max(1, COUNT / LANES) - 1] are the sums of the values
// from the returned index on.  Of lanes that end with the same value, `owner` is set for one.
template <int COUNT, int LANES, int STRIDE>
__device__ __forceinline__ int lane_sums(float (&v)[COUNT], int lane, bool& owner) {
  int base = 0;
  owner = true;
  int count = COUNT;
#pragma unroll
  for (int o = LANES / 2; o > 0; o /= 2) {
    const bool up = lane & (o * STRIDE);
    if (count > 1) {
      const int half = count / 2;
#pragma unroll
      for (int i = 0; i < COUNT / 2; ++i)
        if (i < half) {
          const float give = up ? v[i] : v[i + half], keep = up ? v[i + half] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o * STRIDE);
        }
      base += up ? half : 0;
      count = half;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o * STRIDE);
      owner = owner && !up;
    }
  }
  return base;
}

// Lanes per channel: states in fours, a power of two.
inline int lanes(int S) {
  int q = 1;
  while (q * NS < S) q *= 2;
  return q;
}

int check(const haste_b200_selective_scan& a, bool backward);

template <typename T>
Args<T> pack(const haste_b200_selective_scan& a, int CB) {
  Args<T> k;
  k.T_ = a.T; k.N = a.N; k.D = a.D; k.G = a.G; k.S = a.S;
  k.per = a.D / a.G;
  k.ctiles = ceil_div(k.per, CB);
  k.softplus = a.softplus != 0;
  k.x = Seq<const T>(a.x); k.dt = Seq<const T>(a.dt); k.z = Seq<const T>(a.z);
  k.B = Seq<const T>(a.B); k.C = Seq<const T>(a.C); k.dy = Seq<const T>(a.dy);
  k.y = Seq<T>(a.y); k.dx = Seq<T>(a.dx); k.ddt = Seq<T>(a.ddt); k.dz = Seq<T>(a.dz);
  k.dB = Seq<T>(a.dB); k.dC = Seq<T>(a.dC);
  k.B_g = a.B_g; k.C_g = a.C_g; k.dB_g = a.dB_g; k.dC_g = a.dC_g;
  k.A = a.A; k.skip = a.skip; k.dt_bias = a.dt_bias; k.state = a.state; k.dfinal = a.dfinal_state;
  k.final_state = a.final_state; k.checkpoints = a.checkpoints; k.dstate = a.dstate; k.part = a.scratch;
  k.lengths = a.lengths;
  return k;
}

}  // namespace scan
}  // namespace hb
