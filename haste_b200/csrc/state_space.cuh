// What the state space operators (causal_conv1d.cu, selective_scan*.cu, fused_norm*) share.
#pragma once

#include <cstring>
#include <type_traits>

#include "util.cuh"

namespace hb {
namespace ss {

// V neighbouring elements, moved with accesses of up to 16 bytes.
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V>& w, float (&out)[V]) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      uint32_t bits;
      memcpy(&bits, &w.v[2 * i], 4);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // one instruction a value
        out[2 * i] = __uint_as_float(bits << 16);
        out[2 * i + 1] = __uint_as_float(bits & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&bits));
        out[2 * i] = f.x;
        out[2 * i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = ld(&w.v[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&out)[V]) {
  unpack<T, V>(*reinterpret_cast<const Pack<T, V>*>(p), out);
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&in)[V]) {
  Pack<T, V> w;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(in[2 * i], in[2 * i + 1]);
        memcpy(&w.v[2 * i], &h, 4);
      } else {
        const __half2 h = __floats2half2_rn(in[2 * i], in[2 * i + 1]);
        memcpy(&w.v[2 * i], &h, 4);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) st(&w.v[i], in[i]);
  }
  *reinterpret_cast<Pack<T, V>*>(p) = w;
}

// V neighbouring elements as they come from memory, for loads issued long before their use: whole words,
// because taking elements apart would wait for the load where it is issued.
template <typename T, int V>
struct Raw {
  uint32_t w[(sizeof(T) * V + 3) / 4];
};
// Zeros unless `ok`: a predicated load.  (Written as a branch, the merge of the two values waits for it.)
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_if(bool ok, const T* p) {
  constexpr int B = sizeof(T) * V;
  static_assert(B == 2 || B == 4 || B == 8 || B == 16, "one access");
  Raw<T, V> r;
  if constexpr (B == 2)
    asm volatile("{\n.reg .pred p;\nsetp.ne.s32 p, %2, 0;\nmov.u32 %0, 0;\n@p ld.global.u16 %0, [%1];\n}"
                 : "=&r"(r.w[0]) : "l"(p), "r"((int)ok));
  else if constexpr (B == 4)
    asm volatile("{\n.reg .pred p;\nsetp.ne.s32 p, %2, 0;\nmov.u32 %0, 0;\n@p ld.global.u32 %0, [%1];\n}"
                 : "=&r"(r.w[0]) : "l"(p), "r"((int)ok));
  else if constexpr (B == 8)
    asm volatile("{\n.reg .pred p;\nsetp.ne.s32 p, %3, 0;\nmov.u32 %0, 0;\nmov.u32 %1, 0;\n"
                 "@p ld.global.v2.u32 {%0, %1}, [%2];\n}"
                 : "=&r"(r.w[0]), "=&r"(r.w[1]) : "l"(p), "r"((int)ok));
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.s32 p, %5, 0;\nmov.u32 %0, 0;\nmov.u32 %1, 0;\nmov.u32 %2, 0;\nmov.u32 %3, 0;\n"
                 "@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n}"
                 : "=&r"(r.w[0]), "=&r"(r.w[1]), "=&r"(r.w[2]), "=&r"(r.w[3]) : "l"(p), "r"((int)ok));
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& r, float (&out)[V]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t w = r.w[i / 2];
      if constexpr (std::is_same<T, __nv_bfloat16>::value) out[i] = __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16);
      else out[i] = __half2float(__ushort_as_half((unsigned short)(i % 2 ? w >> 16 : w)));
    }
  }
}

template <typename T>
__device__ __forceinline__ float one(const Raw<T, 1>& r) {
  float v[1];
  unpack<T, 1>(r, v);
  return v[0];
}

// A parameter vector is fp32 or has the sequences' type.
template <typename T>
__device__ __forceinline__ float ldp(const void* p, bool f32, long long i) {
  return f32 ? static_cast<const float*>(p)[i] : ld(static_cast<const T*>(p) + i);
}

template <typename T>
struct Seq {
  T* p;
  int t;  // a step's stride: below 2^31 elements (strides_fit), so that an address is one multiplication
  long long n;
  __host__ Seq() {}
  __host__ explicit Seq(const haste_b200_sequence& s) : p(static_cast<T*>(s.data)), t((int)s.t_stride), n(s.n_stride) {}
  __device__ __forceinline__ T* at(int ti, int ni) const { return p + ni * n + (long long)ti * t; }
};
inline bool strides_fit(int T, const haste_b200_sequence& s) {
  return !s.data || T <= 1 || (s.t_stride < (1LL << 31) && s.t_stride > -(1LL << 31));
}

// Whether every row of a sequence starts on a multiple of `bytes`.
inline bool aligned(const haste_b200_sequence& s, int elem, int bytes) {
  return !s.data || (reinterpret_cast<uintptr_t>(s.data) % bytes == 0 && s.t_stride * elem % bytes == 0 &&
                     s.n_stride * elem % bytes == 0);
}
inline bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

__device__ __forceinline__ int row_length(const long long* lengths, int n, int T) {
  if (!lengths) return T;
  const long long l = lengths[n];
  return l < 0 ? 0 : l < T ? (int)l : T;
}

// sigmoid(v) = 1 / (1 + 2^(-v log2 e)), two approximate instructions (2^-22 relative and one unit in the last
// place).  The product -v log2 e is rounded once, which puts the exponential, and for negative v the result, off by
// up to |v| 2^-24 of its value (6e-7 at -10, 3.6e-6 at -60); an overflowing exponential gives zero.
// silu(v) = v s and its slope from s = sigmoid(v).
__device__ __forceinline__ float reciprocal(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float sigmoid(float v) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  return reciprocal(1.0f + e);
}
__device__ __forceinline__ float silu(float v) { return v * sigmoid(v); }
__device__ __forceinline__ float silu_slope(float v, float s) { return fmaf(v * s, 1.0f - s, s); }

inline bool storage_dtype(int d) { return d == HASTE_B200_F32 || d == HASTE_B200_BF16 || d == HASTE_B200_F16; }

// out_k[j * stride_k] = sum over p of part[p * parts + offset_k + j], j < width_k, in a fixed order;
// out_k (fp32 or `dtype`) may be null.  Up to 8 jobs in one launch.
struct SumJob {
  void* out;
  long long offset, stride;
  int width, dtype;
};
struct SumJobs {
  SumJob job[8];
  int n = 0;
  void add(void* out, long long offset, long long stride, int width, int dtype) {
    if (out) job[n++] = SumJob{out, offset, stride, width, dtype};
  }
};
int sum_parts(const float* part, int P, long long stride, const SumJobs& jobs, cudaStream_t s);

}  // namespace ss
}  // namespace hb
