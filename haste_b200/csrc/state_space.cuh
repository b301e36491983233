// What the state space operators (causal_conv1d.cu, selective_scan*.cu, fused_norm.cu) share.
#pragma once

#include "util.cuh"

namespace hb {
namespace ss {

// V neighbouring elements, moved with accesses of up to 16 bytes.
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&out)[V]) {
  const Pack<T, V> w = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = ld(&w.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&in)[V]) {
  Pack<T, V> w;
#pragma unroll
  for (int i = 0; i < V; ++i) st(&w.v[i], in[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = w;
}

// A parameter vector is fp32 or has the sequences' type.
template <typename T>
__device__ __forceinline__ float ldp(const void* p, bool f32, long long i) {
  return f32 ? static_cast<const float*>(p)[i] : ld(static_cast<const T*>(p) + i);
}

template <typename T>
struct Seq {
  T* p;
  long long t, n;
  __host__ Seq() {}
  __host__ explicit Seq(const haste_b200_sequence& s) : p(static_cast<T*>(s.data)), t(s.t_stride), n(s.n_stride) {}
  __device__ __forceinline__ T* at(long long ti, long long ni) const { return p + ti * t + ni * n; }
};

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

// silu(v) = v s and its slope, from s = sigmoid(v).
__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }
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
