// Norm fused with a block's gate and residual, forward and backward:
//
//   u = x silu(gate),  r = residual + scale u,  y = (r - mean) inv weight + bias
//
// A stream (a dozen operations a value), so HBM bounds it.  A block keeps a whole row in registers,
// at most 16 values a thread, so that every tensor is read once and the variance is that of the
// centred values; r is normalised as computed, before it is rounded to storage.  The backward pass
// computes u and r again from the inputs (the same bytes as reading r, and no rounding between).
#include <algorithm>

#include "state_space.cuh"

namespace hb {
namespace {

using namespace ss;

template <typename T, typename R>
struct NormArgs {
  int rows, N, H;
  bool param_f32, layer;
  float eps;
  Seq<const T> x, gate, dy;
  Seq<const R> residual, dr;
  Seq<T> y, dx, dgate;
  Seq<R> r, dresidual;
  const void *scale, *weight, *bias;
  float* stats;
  float* part;
};

// Sums of K values over the block, to every thread.  `sums` holds 2 * 32 * K floats; consecutive calls alternate `turn`.
template <int K>
__device__ __forceinline__ void block_sum(float (&v)[K], float* sums, int turn) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  const int warps = blockDim.x / 32;
  if (warps == 1) return;
  float* s = sums + (turn & 1) * 32 * K;
  if (threadIdx.x % 32 == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) s[(threadIdx.x / 32) * K + k] = v[k];
  __syncthreads();  // the buffer of the call before last is free again after the barrier in between
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = 0.f;
  for (int w = 0; w < warps; ++w)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += s[w * K + k];
}

// Vectors of V neighbouring values, thread by thread across the row; K of them a thread.
template <typename T, typename R, int V, int K>
__global__ void __launch_bounds__(512) norm_fwd(NormArgs<T, R> a) {
  __shared__ float sums[2 * 32];
  float w[K][V], b[K][V], sc[K][V];
  int col[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    col[k] = (k * blockDim.x + threadIdx.x) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const bool ok = col[k] < a.H;
      w[k][i] = ok ? ldp<T>(a.weight, a.param_f32, col[k] + i) : 0.f;
      b[k][i] = ok && a.bias ? ldp<T>(a.bias, a.param_f32, col[k] + i) : 0.f;
      sc[k][i] = ok && a.scale ? ldp<T>(a.scale, a.param_f32, col[k] + i) : 1.f;
    }
  }
  const float over = 1.0f / a.H;
  int turn = 0;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int t = row / a.N, n = row % a.N;
    float r[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) r[k][i] = 0.f;
      if (col[k] < a.H) {
        load<T, V>(a.x.at(t, n) + col[k], r[k]);
        if (a.gate.p) {
          float g[V];
          load<T, V>(a.gate.at(t, n) + col[k], g);
#pragma unroll
          for (int i = 0; i < V; ++i) r[k][i] *= silu(g[i]);
        }
        if (a.residual.p) {
          float q[V];
          load<R, V>(a.residual.at(t, n) + col[k], q);
#pragma unroll
          for (int i = 0; i < V; ++i) r[k][i] = fmaf(sc[k][i], r[k][i], q[i]);
          if (a.r.p) store<R, V>(a.r.at(t, n) + col[k], r[k]);
        }
      }
    }
    float s[1], mean = 0.f;
    if (a.layer) {
      s[0] = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) s[0] += r[k][i];
      block_sum<1>(s, sums, turn++);
      mean = s[0] * over;
    }
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (col[k] < a.H)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          r[k][i] -= mean;
          s[0] = fmaf(r[k][i], r[k][i], s[0]);
        }
    block_sum<1>(s, sums, turn++);
    const float inv = rsqrtf(s[0] * over + a.eps);
    if (a.stats && threadIdx.x == 0) {
      a.stats[2LL * row] = mean;
      a.stats[2LL * row + 1] = inv;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (col[k] < a.H) {
#pragma unroll
        for (int i = 0; i < V; ++i) r[k][i] = fmaf(r[k][i] * inv, w[k][i], b[k][i]);
        store<T, V>(a.y.at(t, n) + col[k], r[k]);
      }
  }
}

// With n = (r - mean) inv and dn = dy weight:
//   dr += inv (dn - n mean(dn n) - mean(dn))   (the last term with the mean only)
//   dresidual = dr,  dscale = sum dr u,  dx = dr scale silu(gate),  dgate = dr scale x silu'(gate)
// The column sums stay over the rows that a block takes in turn: in registers, or with 16 values a
// thread (rows beyond 4096), where those and the parameters do not fit, in shared memory.
template <typename T, typename R, int V, int K>
__global__ void __launch_bounds__(512) norm_bwd(NormArgs<T, R> a) {
  constexpr bool Wide = V * K > 8;
  constexpr int KR = Wide ? 1 : K;  // rows of the register arrays that only the narrow form has
  __shared__ float sums[2 * 32 * 2];
  extern __shared__ float columns[];  // Wide: [3][H], each entry its thread's own
  float w_[KR][V], sc_[KR][V], dw_[KR][V], db_[KR][V], ds_[KR][V];
  int col[K];
#pragma unroll
  for (int k = 0; k < K; ++k) col[k] = (k * blockDim.x + threadIdx.x) * V;
  auto weight = [&](int k, int i) { return Wide ? ldp<T>(a.weight, a.param_f32, col[k] + i) : w_[Wide ? 0 : k][i]; };
  auto scale = [&](int k, int i) {
    return !Wide ? sc_[Wide ? 0 : k][i] : a.scale ? ldp<T>(a.scale, a.param_f32, col[k] + i) : 1.f;
  };
  auto dw = [&](int k, int i) -> float& { return Wide ? columns[col[k] + i] : dw_[Wide ? 0 : k][i]; };
  auto db = [&](int k, int i) -> float& { return Wide ? columns[a.H + col[k] + i] : db_[Wide ? 0 : k][i]; };
  auto ds = [&](int k, int i) -> float& { return Wide ? columns[2 * a.H + col[k] + i] : ds_[Wide ? 0 : k][i]; };
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const bool ok = col[k] < a.H;
      if (!Wide) {
        w_[Wide ? 0 : k][i] = ok ? ldp<T>(a.weight, a.param_f32, col[k] + i) : 0.f;
        sc_[Wide ? 0 : k][i] = ok && a.scale ? ldp<T>(a.scale, a.param_f32, col[k] + i) : 1.f;
      }
      if (!Wide || ok) dw(k, i) = db(k, i) = ds(k, i) = 0.f;
    }
  }
  const float over = 1.0f / a.H;
  int turn = 0;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int t = row / a.N, n = row % a.N;
    const float mean = a.stats[2LL * row], inv = a.stats[2LL * row + 1];
    float x[K][V], g[K][V], q[K][V], d[K][V], s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) x[k][i] = g[k][i] = q[k][i] = d[k][i] = 0.f;
      if (col[k] < a.H) {
        load<T, V>(a.x.at(t, n) + col[k], x[k]);
        load<T, V>(a.dy.at(t, n) + col[k], d[k]);
        if (a.gate.p) load<T, V>(a.gate.at(t, n) + col[k], g[k]);
        if (a.residual.p) load<R, V>(a.residual.at(t, n) + col[k], q[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (col[k] < a.H)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float u = a.gate.p ? x[k][i] * silu(g[k][i]) : x[k][i];
          q[k][i] = ((a.residual.p ? fmaf(scale(k, i), u, q[k][i]) : u) - mean) * inv;  // n
          dw(k, i) = fmaf(d[k][i], q[k][i], dw(k, i));
          db(k, i) += d[k][i];
          d[k][i] *= weight(k, i);  // dn
          s[0] = fmaf(d[k][i], q[k][i], s[0]);
          s[1] += d[k][i];
        }
    block_sum<2>(s, sums, turn++);
    const float p = s[0] * over, m = a.layer ? s[1] * over : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (col[k] < a.H) {
#pragma unroll
        for (int i = 0; i < V; ++i) d[k][i] = inv * (d[k][i] - q[k][i] * p - m);
        if (a.residual.p) {
          if (a.dr.p) {
            load<R, V>(a.dr.at(t, n) + col[k], q[k]);
#pragma unroll
            for (int i = 0; i < V; ++i) d[k][i] += q[k][i];
          }
          if (a.dresidual.p) store<R, V>(a.dresidual.at(t, n) + col[k], d[k]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float sg = a.gate.p ? sigmoid(g[k][i]) : 1.f;
          const float act = a.gate.p ? g[k][i] * sg : 1.f;
          ds(k, i) = fmaf(d[k][i], x[k][i] * act, ds(k, i));
          d[k][i] *= scale(k, i);
          q[k][i] = d[k][i] * x[k][i] * silu_slope(g[k][i], sg);
          d[k][i] *= act;
        }
        if (a.dx.p) store<T, V>(a.dx.at(t, n) + col[k], d[k]);
        if (a.dgate.p) store<T, V>(a.dgate.at(t, n) + col[k], q[k]);
      }
  }
  float* row = a.part + (long long)blockIdx.x * 3 * a.H;
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (col[k] < a.H)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        row[col[k] + i] = dw(k, i);
        row[a.H + col[k] + i] = db(k, i);
        row[2 * a.H + col[k] + i] = ds(k, i);
      }
}

int check(const haste_b200_fused_norm& a, bool backward) {
  HB_REQUIRE(storage_dtype(a.dtype), "dtype");
  HB_REQUIRE(a.residual_dtype == HASTE_B200_F32 || a.residual_dtype == a.dtype, "residual_dtype");
  HB_REQUIRE(a.param_dtype == HASTE_B200_F32 || a.param_dtype == a.dtype, "param_dtype");
  HB_REQUIRE(a.T >= 0 && a.N >= 0, "T,N");
  HB_REQUIRE((long long)a.T * a.N < (1LL << 31) - 65536, "T*N too large");
  HB_REQUIRE(a.H >= 1 && a.H <= 8192, "H must be 1..8192");
  HB_REQUIRE(a.eps >= 0.f, "eps");
  HB_REQUIRE(strides_fit(a.T, a.x) && strides_fit(a.T, a.gate) && strides_fit(a.T, a.residual) && strides_fit(a.T, a.y) && strides_fit(a.T, a.r) && strides_fit(a.T, a.dy) && strides_fit(a.T, a.dr) && strides_fit(a.T, a.dx) && strides_fit(a.T, a.dgate) && strides_fit(a.T, a.dresidual),
             "a step's stride must be below 2^31 elements");
  HB_REQUIRE(!a.scale || a.residual.data || a.T == 0 || a.N == 0, "scale needs a residual");
  HB_REQUIRE(a.weight, "null pointer");
  if (backward) HB_REQUIRE(a.scratch && a.dweight, "null pointer");
  if (a.T == 0 || a.N == 0) return HASTE_B200_OK;
  HB_REQUIRE(a.x.data, "null pointer");
  if (backward) HB_REQUIRE(a.dy.data && a.stats, "null pointer");
  else HB_REQUIRE(a.y.data, "null pointer");
  return HASTE_B200_OK;
}

// Values per access: 16 bytes of the narrower type where width, strides and starts allow.
int width(const haste_b200_fused_norm& a) {
  const int e = (int)dtype_size(a.dtype), f = (int)dtype_size(a.residual_dtype);
  for (int v = 16 / e; v > 1; v /= 2) {
    const int w = std::min(16, v * e), q = std::min(16, v * f);
    if (a.H % v == 0 && aligned(a.x, e, w) && aligned(a.gate, e, w) && aligned(a.y, e, w) && aligned(a.dy, e, w) &&
        aligned(a.dx, e, w) && aligned(a.dgate, e, w) && aligned(a.residual, f, q) && aligned(a.r, f, q) &&
        aligned(a.dr, f, q) && aligned(a.dresidual, f, q))
      return v;
  }
  return 1;
}

int threads(int H, int per) { return ceil_div(ceil_div(H, per), 32) * 32; }

// Blocks of the backward pass, each of which leaves a row of partial sums: enough threads to fill the SMs.
int parts(const haste_b200_fused_norm& a) {
  const int th = threads(a.H, a.H <= 4096 ? 8 : 16), per_sm = std::max(1, std::min(16, 1024 / th));
  return std::max(1, std::min(a.T * a.N, per_sm * sm_count()));
}

template <typename T, typename R, int V, int K>
int launch(const haste_b200_fused_norm& a, bool backward, cudaStream_t s) {
  NormArgs<T, R> k;
  k.rows = a.T * a.N; k.N = a.N; k.H = a.H;
  k.param_f32 = a.param_dtype == HASTE_B200_F32;
  k.layer = a.layer_norm != 0;
  k.eps = a.eps;
  k.x = Seq<const T>(a.x); k.gate = Seq<const T>(a.gate); k.dy = Seq<const T>(a.dy);
  k.residual = Seq<const R>(a.residual); k.dr = Seq<const R>(a.dr);
  k.y = Seq<T>(a.y); k.dx = Seq<T>(a.dx); k.dgate = Seq<T>(a.dgate);
  k.r = Seq<R>(a.r); k.dresidual = Seq<R>(a.dresidual);
  k.scale = a.scale; k.weight = a.weight; k.bias = a.bias;
  k.stats = a.stats;
  k.part = a.scratch;
  const int th = threads(a.H, V * K);
  if (!backward) {
    if (k.rows == 0) return HASTE_B200_OK;
    const int blocks = std::min(k.rows, std::max(1, std::min(32, 2048 / th)) * sm_count());
    norm_fwd<T, R, V, K><<<blocks, th, 0, s>>>(k);
    HB_LAUNCH_OK();
    count_launch(1);
    return HASTE_B200_OK;
  }
  const int blocks = parts(a);
  const size_t smem = V * K > 8 ? 3 * sizeof(float) * a.H : 0;
  if (smem > 48 * 1024)
    HB_CUDA_OK(cudaFuncSetAttribute(norm_bwd<T, R, V, K>, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * 4 * 8192));
  norm_bwd<T, R, V, K><<<blocks, th, smem, s>>>(k);
  HB_LAUNCH_OK();
  count_launch(1);
  SumJobs jobs;
  jobs.add(a.dweight, 0, 1, a.H, a.param_dtype);
  jobs.add(a.dbias, a.H, 1, a.H, a.param_dtype);
  jobs.add(a.dscale, 2LL * a.H, 1, a.H, a.param_dtype);
  return sum_parts(a.scratch, blocks, 3LL * a.H, jobs, s);
}

template <typename T, typename R, int V>
int by_count(const haste_b200_fused_norm& a, bool backward, cudaStream_t s) {
  return a.H <= 4096 ? launch<T, R, V, 8 / V>(a, backward, s) : launch<T, R, V, 16 / V>(a, backward, s);
}

template <typename T, typename R>
int by_width(const haste_b200_fused_norm& a, bool backward, cudaStream_t s) {
  const int v = width(a);
  if constexpr (sizeof(T) == 2)
    if (v == 8) return by_count<T, R, 8>(a, backward, s);
  return v == 4 ? by_count<T, R, 4>(a, backward, s)
       : v == 2 ? by_count<T, R, 2>(a, backward, s)
                : by_count<T, R, 1>(a, backward, s);
}

int run(const haste_b200_fused_norm& a, bool backward, cudaStream_t s) {
  HB_TRY(check(a, backward));
  const bool wide = a.residual_dtype == HASTE_B200_F32;
  if (a.dtype == HASTE_B200_F32) return by_width<float, float>(a, backward, s);
  if (a.dtype == HASTE_B200_BF16)
    return wide ? by_width<__nv_bfloat16, float>(a, backward, s) : by_width<__nv_bfloat16, __nv_bfloat16>(a, backward, s);
  return wide ? by_width<__half, float>(a, backward, s) : by_width<__half, __half>(a, backward, s);
}

}  // namespace

int fused_norm_forward(const haste_b200_fused_norm& a, cudaStream_t s) {
  ProfScope p(PH_OTHER, s);
  return run(a, false, s);
}
int fused_norm_backward(const haste_b200_fused_norm& a, cudaStream_t s) {
  ProfScope p(PH_OTHER, s);
  return run(a, true, s);
}
long long fused_norm_scratch(const haste_b200_fused_norm& a) {
  if (a.T < 0 || a.N < 0 || a.H < 1 || a.H > 8192) return 0;
  return 3LL * parts(a) * a.H;
}

}  // namespace hb
