// What a projection does to its sums before it stores them: y = act(sum + bias) + residual, and the slopes of its
// activations for the backward pass.
#pragma once

#include "state_space.cuh"

namespace hb {

// Pointers into dense or row-strided matrices [rows, outputs]; null where absent.
struct Epilogue {
  const void* bias;      // float or the operands' type
  const void* residual;  // the output's type
  long long ld_res;
  void* pre;             // sum + bias in the operands' type, kept for the backward pass
  long long ld_pre;
  int bias_f32, act;
};

namespace epi {

using namespace ss;

// Accurate (tanh and gelu): CUDA's own functions, for float32 sequences; otherwise within 2e-7 of the function's own size, and
// the rounding of an exponent, which is nothing to 16 bits, in a third of the instructions.  Infinities come out as the
// formulas have them: p times zero is a NaN.
__device__ __forceinline__ float exp2_(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// (1 - e) / (1 + e), e = exp(-2 |v|); near zero, where that cancels, the series up to v^9.
template <bool Accurate>
__device__ __forceinline__ float tanh_(float v) {
  if constexpr (Accurate) return tanhf(v);
  const float a = fabsf(v), e = exp2_(a * -2.885390081777927f);
  const float far = copysignf((1.f - e) * reciprocal(1.f + e), v), q = v * v;
  float p = 62.f / 2835;
  p = fmaf(p, q, -17.f / 315);
  p = fmaf(p, q, 2.f / 15);
  p = fmaf(p, q, -1.f / 3);
  return a < 0.25f ? fmaf(v * q, p, v) : far;
}
// The normal distribution Phi(v) and exp(-v^2 / 2).  Not accurate: the complementary error function as erfcc of "Numerical
// Recipes" (Press and others) has it, t exp(-z^2 + a polynomial of t), t = 1 / (1 + z / 2), which is off by 1.2e-7 of its
// value at most, small ones included.
template <bool Accurate>
__device__ __forceinline__ float normal(float v, float& bell) {
  constexpr float LOG2E = 1.4426950408889634f;
  bell = exp2_(v * v * -0.7213475204444817f);
  if constexpr (Accurate) return 0.5f * erfcf(v * -0.7071067811865476f);
  const float t = reciprocal(fmaf(fabsf(v), 0.5f * 0.7071067811865476f, 1.f));
  float p = 0.17087277f * LOG2E;
  p = fmaf(p, t, -0.82215223f * LOG2E);
  p = fmaf(p, t, 1.48851587f * LOG2E);
  p = fmaf(p, t, -1.13520398f * LOG2E);
  p = fmaf(p, t, 0.27886807f * LOG2E);
  p = fmaf(p, t, -0.18628806f * LOG2E);
  p = fmaf(p, t, 0.09678418f * LOG2E);
  p = fmaf(p, t, 0.37409196f * LOG2E);
  p = fmaf(p, t, 1.00002368f * LOG2E);
  p = fmaf(p, t, -1.26551223f * LOG2E - 1.f);  // (the half of Phi)
  const float tail = t * exp2_(fmaf(v * v, -0.5f * LOG2E, p));
  return v < 0.f ? tail : 1.f - tail;
}

template <bool Accurate, int Act>
__device__ __forceinline__ float activate(float p) {
  if constexpr (Act == HASTE_B200_RELU) return p < 0.f ? 0.f : p;  // (a NaN stays)
  if constexpr (Act == HASTE_B200_SILU) return silu(p);
  if constexpr (Act == HASTE_B200_GELU) {
    float bell;
    return p * normal<Accurate>(p, bell);
  }
  if constexpr (Act == HASTE_B200_TANH) return tanh_<Accurate>(p);
  if constexpr (Act == HASTE_B200_SIGMOID) return sigmoid(p);
  return p;
}
// Of infinite p its limit, 0 or 1: a sum beyond 16 bits' range is kept as an infinity, at which the formulas of SiLU and GELU
// have infinity times zero; from 1000 on they are at their limits.  (Kept as the type's largest value instead, which the
// product's epilogue has to see to: bf16 64000 x 2048, K = 1024 with sums 263 us, where it takes 245.)
template <bool Accurate, int Act>
__device__ __forceinline__ float slope(float p) {
  if constexpr (Act == HASTE_B200_SILU || Act == HASTE_B200_GELU) asm("max.NaN.f32 %0, %0, %1;\n\tmin.NaN.f32 %0, %0, %2;" : "+f"(p) : "f"(-1000.f), "f"(1000.f));
  if constexpr (Act == HASTE_B200_RELU) return p > 0.f ? 1.f : p != p ? p : 0.f;
  if constexpr (Act == HASTE_B200_SILU) return silu_slope(p, sigmoid(p));
  if constexpr (Act == HASTE_B200_GELU) {
    float bell;
    const float n = normal<Accurate>(p, bell);
    return fmaf(p * 0.3989422804014327f, bell, n);
  }
  if constexpr (Act == HASTE_B200_TANH) {
    const float e = exp2_(fabsf(p) * -2.885390081777927f), r = reciprocal(1.f + e);
    return 4.f * e * r * r;  // 1 - tanh^2
  }
  if constexpr (Act == HASTE_B200_SIGMOID) {
    const float e = exp2_(fabsf(p) * -1.4426950408889634f), r = reciprocal(1.f + e);
    return e * r * r;
  }
  return 1.f;
}
// f with the activation as a compile-time number: chosen once for all elements that f walks (chosen for each, next to
// the others' code, a pass waits for its instructions: bf16 64000 x 2048 slopes 260 us).
template <int A>
struct Act {
  static constexpr int value = A;
};
template <typename F>
__host__ __device__ __forceinline__ void with_activation(int act, const F& f) {
  switch (act) {
    case HASTE_B200_RELU: f(Act<HASTE_B200_RELU>()); break;
    case HASTE_B200_SILU: f(Act<HASTE_B200_SILU>()); break;
    case HASTE_B200_GELU: f(Act<HASTE_B200_GELU>()); break;
    case HASTE_B200_TANH: f(Act<HASTE_B200_TANH>()); break;
    case HASTE_B200_SIGMOID: f(Act<HASTE_B200_SIGMOID>()); break;
    default: f(Act<HASTE_B200_IDENTITY>());
  }
}

template <typename T>
__device__ __forceinline__ float bias_at(const Epilogue& e, int n) {
  return e.bias_f32 ? static_cast<const float*>(e.bias)[n] : ld(static_cast<const T*>(e.bias) + n);
}
// Element (m, n) of y from its sum.
template <typename T, typename TO>
__device__ __forceinline__ void finish(const Epilogue& e, float v, int m, int n, TO* y) {
  if (e.bias) v += bias_at<T>(e, n);
  if (e.pre) st(static_cast<T*>(e.pre) + m * e.ld_pre + n, v);
  with_activation(e.act, [&](auto act) { v = activate<sizeof(T) == 4, decltype(act)::value>(v); });
  if (e.residual) v += ld(static_cast<const TO*>(e.residual) + m * e.ld_res + n);
  st(y, v);
}
// Four neighbouring elements, whose rows take accesses of four (`wide`); bias: theirs.
template <typename T, typename TO>
__device__ __forceinline__ void finish4(const Epilogue& e, float (&v)[4], const float (&bias)[4], int m, int n, TO* y) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] += bias[j];
  if (e.pre) store<T, 4>(static_cast<T*>(e.pre) + m * e.ld_pre + n, v);
  with_activation(e.act, [&](auto act) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = activate<sizeof(T) == 4, decltype(act)::value>(v[j]);
  });
  if (e.residual) {
    float r[4];
    load<TO, 4>(static_cast<const TO*>(e.residual) + m * e.ld_res + n, r);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += r[j];
  }
  store<TO, 4>(y, v);
}

}  // namespace epi
}  // namespace hb
