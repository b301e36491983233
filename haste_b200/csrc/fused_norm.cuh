// Norm fused with a block's gate and residual, forward and backward:
//
//   u = x silu(gate),  r = residual + scale u,  y = (r - mean) inv weight + bias
//
// A stream (a dozen operations a value), so HBM bounds it.  A block keeps a whole row in registers, at most
// 16 values a thread, so that every tensor is read once and the variance is that of the centred values; rows
// of up to 128 values share warps.  r is normalised as computed, before it is rounded to storage.  The
// backward pass computes u and r again from the inputs (the same bytes as reading r, and no rounding between).
// bf16 64000 x 1024 with residual, scale and bias: forward 101 us, 5.2 TB/s (0.80 of the measured copy),
// backward 171 us with its sums, 4.6 TB/s; without the next row under way 146 and 357 us.
#pragma once

#include <algorithm>

#include "state_space.cuh"

namespace hb {
namespace norm {

using namespace ss;

int parts(const haste_b200_fused_norm& a);
template <typename T>
int run(const haste_b200_fused_norm& a, bool backward, cudaStream_t s);

namespace {

template <typename T, typename R, typename P>
struct NormArgs {
  int rows, N, H;
  bool layer;
  float eps;
  Seq<const T> x, gate, dy;
  Seq<const R> residual, dr;
  Seq<T> y, dx, dgate;
  Seq<R> r, dresidual;
  const P *scale, *weight, *bias;
  float* stats;
  float* part;
};

// Sums of K values over the block, to every thread.  `sums` holds two rows of 16 * K floats, which consecutive calls take in turn.
template <int K>
__device__ __forceinline__ void block_sum(float (&v)[K], float* sums, int turn) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  const int warps = blockDim.x / 32;
  if (warps == 1) return;
  float* s = sums + (turn & 1) * 16 * K;
  if (threadIdx.x % 32 == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) s[k * 16 + threadIdx.x / 32] = v[k];
  __syncthreads();  // the buffer of the call before last is free again after the barrier in between
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const float4 first = *reinterpret_cast<const float4*>(s + k * 16);  // (entries beyond the warps stay zero)
    v[k] = (first.x + first.y) + (first.z + first.w);
    for (int w = 4; w < warps; ++w) v[k] += s[k * 16 + w];
  }
}

// Rows of up to 128 values take a part of a warp each (Sub lanes): sums over those lanes, no barrier.
constexpr int SUB_THREADS = 128;
template <int Sub, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* sums, int turn) {
  if constexpr (Sub == 0) {
    block_sum<K>(v, sums, turn);
  } else {
#pragma unroll
    for (int o = Sub / 2; o > 0; o /= 2)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
}

// V values as they come from memory, in accesses of at most 16 bytes.
template <typename T, int V>
struct Line {
  static constexpr int U = V * sizeof(T) > 16 ? 16 / sizeof(T) : V;
  Raw<T, U> part[V / U];
  __device__ __forceinline__ void load(bool ok, const T* p) {
#pragma unroll
    for (int i = 0; i < V / U; ++i) part[i] = load_if<T, U>(ok, p + i * U);
  }
  __device__ __forceinline__ void get(float (&out)[V]) const {
#pragma unroll
    for (int i = 0; i < V / U; ++i) {
      float f[U];
      unpack<T, U>(part[i], f);
#pragma unroll
      for (int k = 0; k < U; ++k) out[i * U + k] = f[k];
    }
  }
};

struct Where {
  int t, n;
  template <typename A>
  __device__ __forceinline__ Where(const A& a, int row) : t(row < a.N ? 0 : row / a.N), n(row - t * a.N) {}
};

// A row's tensors on their way.
template <bool Backward, typename T, typename R, typename P, int V, int K>
struct Row {
  Line<T, V> x[K], gate[K], dy[Backward ? K : 1];
  Line<R, V> q[K];
  float mean, inv;
  __device__ __forceinline__ void fetch(const NormArgs<T, R, P>& a, int row, const int (&col)[K]) {
    const bool ok = row < a.rows;
    const Where at(a, row);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool in = ok && col[k] < a.H;
      x[k].load(in, a.x.at(at.t, at.n) + col[k]);
      gate[k].load(in && a.gate.p, a.gate.at(at.t, at.n) + col[k]);
      if (Backward) dy[k].load(in, a.dy.at(at.t, at.n) + col[k]);
      q[k].load(in && a.residual.p, a.residual.at(at.t, at.n) + col[k]);
    }
    if (Backward) {
      mean = __uint_as_float(load_if<float, 1>(ok, a.stats + 2LL * row).w[0]);
      inv = __uint_as_float(load_if<float, 1>(ok, a.stats + 2LL * row + 1).w[0]);
    }
  }
};

// Vectors of V neighbouring values, thread by thread across the row; K of them a thread.  The next row
// of a block is under way while one is computed; the parameters stay in registers as they are stored.
template <typename T, typename R, typename P, int V, int K, int Sub>
__global__ void __launch_bounds__(Sub ? SUB_THREADS : 512) norm_fwd(NormArgs<T, R, P> a) {
  __shared__ __align__(16) float sums[2 * 16];
  if (threadIdx.x < 32) sums[threadIdx.x] = 0.f;
  __syncthreads();
  int col[K];
  Line<P, V> weight[K], bias[K], scale[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    col[k] = (k * (Sub ? Sub : blockDim.x) + (Sub ? threadIdx.x % Sub : threadIdx.x)) * V;
    const bool in = col[k] < a.H;
    weight[k].load(in, a.weight + col[k]);
    bias[k].load(in && a.bias, a.bias + col[k]);
    scale[k].load(in && a.scale, a.scale + col[k]);
  }
  const float over = 1.0f / a.H;
  int turn = 0;
  Row<false, T, R, P, V, K> now, next;
  constexpr int ROWS = Sub ? SUB_THREADS / Sub : 1;  // rows of the block side by side
  const int mine = Sub ? threadIdx.x / (Sub ? Sub : 1) : 0;
  now.fetch(a, blockIdx.x * ROWS + mine, col);
  for (int first = blockIdx.x * ROWS; first < a.rows; first += gridDim.x * ROWS) {
    const int row = first + mine;
    next.fetch(a, row + gridDim.x * ROWS, col);
    const Where at(a, row);
    const bool ok = !Sub || row < a.rows;
    float r[K][V], f[V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      now.x[k].get(r[k]);
      if (a.gate.p) {
        now.gate[k].get(f);
#pragma unroll
        for (int i = 0; i < V; ++i) r[k][i] *= silu(f[i]);
      }
      if (a.residual.p) {
        if (a.scale) {
          scale[k].get(f);
#pragma unroll
          for (int i = 0; i < V; ++i) r[k][i] *= f[i];
        }
        now.q[k].get(f);
#pragma unroll
        for (int i = 0; i < V; ++i) r[k][i] += f[i];
        if (a.r.p && ok && col[k] < a.H) store<R, V>(a.r.at(at.t, at.n) + col[k], r[k]);
      }
    }
    float s[1], mean = 0.f;
    if (a.layer) {
      s[0] = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) s[0] += r[k][i];
      row_sum<Sub, 1>(s, sums, turn++);
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
    row_sum<Sub, 1>(s, sums, turn++);
    const float inv = rsqrtf(s[0] * over + a.eps);
    if (a.stats && ok && col[0] == 0) *reinterpret_cast<float2*>(a.stats + 2LL * row) = make_float2(mean, inv);
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (ok && col[k] < a.H) {
        weight[k].get(f);
#pragma unroll
        for (int i = 0; i < V; ++i) r[k][i] *= inv * f[i];
        if (a.bias) {
          bias[k].get(f);
#pragma unroll
          for (int i = 0; i < V; ++i) r[k][i] += f[i];
        }
        store<T, V>(a.y.at(at.t, at.n) + col[k], r[k]);
      }
    now = next;
  }
}

// With n = (r - mean) inv and dn = dy weight:
//   dr += inv (dn - n mean(dn n) - mean(dn))   (the last term with the mean only)
//   dresidual = dr,  dscale = sum dr u,  dx = dr scale silu(gate),  dgate = dr scale x silu'(gate)
// The column sums stay over the rows that a block takes in turn: in registers, or with 16 values a
// thread (rows beyond 4096), where those and the next row do not fit, in shared memory.
template <typename T, typename R, typename P, int V, int K, int Sub>
__global__ void __launch_bounds__(Sub ? SUB_THREADS : 512) norm_bwd(NormArgs<T, R, P> a) {
  constexpr bool Wide = V * K > 8;
  constexpr int KR = Wide ? 1 : K;  // rows of the register arrays that only the narrow form has
  __shared__ __align__(16) float sums[2 * 16 * 2];
  if (threadIdx.x < 64) sums[threadIdx.x] = 0.f;
  if (blockDim.x < 64) sums[32 + threadIdx.x] = 0.f;
  __syncthreads();
  extern __shared__ float columns[];  // Wide: [3][H], each entry its thread's own
  float dw_[KR][V], db_[KR][V], ds_[KR][V];
  int col[K];
  Line<P, V> weight[K], scale[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    col[k] = (k * (Sub ? Sub : blockDim.x) + (Sub ? threadIdx.x % Sub : threadIdx.x)) * V;
    weight[k].load(col[k] < a.H, a.weight + col[k]);
    scale[k].load(col[k] < a.H && a.scale, a.scale + col[k]);
  }
  auto dw = [&](int k, int i) -> float& { return Wide ? columns[col[k] + i] : dw_[Wide ? 0 : k][i]; };
  auto db = [&](int k, int i) -> float& { return Wide ? columns[a.H + col[k] + i] : db_[Wide ? 0 : k][i]; };
  auto ds = [&](int k, int i) -> float& { return Wide ? columns[2 * a.H + col[k] + i] : ds_[Wide ? 0 : k][i]; };
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (!Wide || col[k] < a.H) dw(k, i) = db(k, i) = ds(k, i) = 0.f;
  const float over = 1.0f / a.H;
  int turn = 0;
  Row<true, T, R, P, V, K> now, next;
  constexpr int ROWS = Sub ? SUB_THREADS / Sub : 1;  // rows of the block side by side
  const int mine = Sub ? threadIdx.x / (Sub ? Sub : 1) : 0;
  now.fetch(a, blockIdx.x * ROWS + mine, col);
  // By twos: copying `next` would wait for its loads, two turns exchange the registers instead.  (184 -> 171 us at
  // 64000 x 1024 in bf16; in fp32 the registers do not suffice, and the forward pass has enough blocks without.)
#pragma unroll(sizeof(T) == 2 ? 2 : 1)
  for (int first = blockIdx.x * ROWS; first < a.rows; first += gridDim.x * ROWS) {
    const int row = first + mine;
    const Where at(a, row);
    const bool ok = !Sub || row < a.rows;
    Line<R, V> dr[K];
#pragma unroll
    for (int k = 0; k < K; ++k) dr[k].load(ok && a.dr.p && col[k] < a.H, a.dr.at(at.t, at.n) + col[k]);
    if (!Wide) next.fetch(a, row + gridDim.x * ROWS, col);
    const float mean = now.mean, inv = now.inv;
    float q[K][V], d[K][V], s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (col[k] < a.H) {
        float u[V], f[V];
        now.x[k].get(u);
        now.dy[k].get(d[k]);
        now.q[k].get(q[k]);
        if (a.gate.p) {
          now.gate[k].get(f);
#pragma unroll
          for (int i = 0; i < V; ++i) u[i] *= silu(f[i]);
        }
        if (a.scale) {
          scale[k].get(f);
#pragma unroll
          for (int i = 0; i < V; ++i) u[i] *= f[i];
        }
        weight[k].get(f);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          q[k][i] = (u[i] + q[k][i] - mean) * inv;  // n
          dw(k, i) = fmaf(d[k][i], q[k][i], dw(k, i));
          db(k, i) += d[k][i];
          d[k][i] *= f[i];  // dn
          s[0] = fmaf(d[k][i], q[k][i], s[0]);
          s[1] += d[k][i];
        }
      }
    row_sum<Sub, 2>(s, sums, turn++);
    const float p = s[0] * over, m = a.layer ? s[1] * over : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (ok && col[k] < a.H) {
        float x[V], g[V], e[V];
        dr[k].get(e);
#pragma unroll
        for (int i = 0; i < V; ++i) d[k][i] = fmaf(inv, d[k][i] - q[k][i] * p - m, e[i]);
        if (a.dresidual.p) store<R, V>(a.dresidual.at(at.t, at.n) + col[k], d[k]);
        now.x[k].get(x);
        if (a.gate.p) {
          now.gate[k].get(g);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float sg = sigmoid(g[i]);
            e[i] = x[i] * silu_slope(g[i], sg);
            g[i] *= sg;
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) g[i] = 1.f;
        }
        if (a.scale) {
          float f[V];
          scale[k].get(f);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            ds(k, i) = fmaf(d[k][i], x[i] * g[i], ds(k, i));
            d[k][i] *= f[i];
          }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          e[i] *= d[k][i];
          d[k][i] *= g[i];
        }
        if (a.dx.p) store<T, V>(a.dx.at(at.t, at.n) + col[k], d[k]);
        if (a.dgate.p) store<T, V>(a.dgate.at(at.t, at.n) + col[k], e);
      }
    if (Wide) now.fetch(a, row + gridDim.x * ROWS, col);
    else now = next;
  }
  float* row = a.part + (long long)blockIdx.x * 3 * a.H;
  if constexpr (Sub > 0) {  // the block's rows of partial sums, added in order
    __shared__ float all[SUB_THREADS * V * K];
    auto add = [&](float (&v)[KR][V], float* to) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) all[threadIdx.x * V * K + k * V + i] = v[k][i];
      __syncthreads();
      if (threadIdx.x >= Sub) return;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float sum = 0.f;
          for (int r = 0; r < ROWS; ++r) sum += all[(r * Sub + threadIdx.x) * V * K + k * V + i];
          if (col[k] < a.H) to[col[k] + i] = sum;
        }
    };
    add(dw_, row);
    add(db_, row + a.H);
    add(ds_, row + 2 * a.H);
  } else {
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
}

// Values per access: 16 bytes of the narrower type where width, strides and starts allow.
int width(const haste_b200_fused_norm& a) {
  const int e = (int)dtype_size(a.dtype), f = (int)dtype_size(a.residual_dtype), g = (int)dtype_size(a.param_dtype);
  for (int v = 16 / e; v > 1; v /= 2) {
    const int w = std::min(16, v * e), q = std::min(16, v * f), r = std::min(16, v * g);
    if (a.H % v == 0 && aligned(a.weight, r) && aligned(a.bias, r) && aligned(a.scale, r) && aligned(a.x, e, w) && aligned(a.gate, e, w) && aligned(a.y, e, w) && aligned(a.dy, e, w) &&
        aligned(a.dx, e, w) && aligned(a.dgate, e, w) && aligned(a.residual, f, q) && aligned(a.r, f, q) &&
        aligned(a.dr, f, q) && aligned(a.dresidual, f, q))
      return v;
  }
  return 1;
}

int threads(int H, int per) { return ceil_div(ceil_div(H, per), 32) * 32; }

template <typename T, typename R, typename P, int V, int K, int Sub>
int launch(const haste_b200_fused_norm& a, bool backward, cudaStream_t s) {
  NormArgs<T, R, P> k;
  k.rows = a.T * a.N; k.N = a.N; k.H = a.H;
  k.layer = a.layer_norm != 0;
  k.eps = a.eps;
  k.x = Seq<const T>(a.x); k.gate = Seq<const T>(a.gate); k.dy = Seq<const T>(a.dy);
  k.residual = Seq<const R>(a.residual); k.dr = Seq<const R>(a.dr);
  k.y = Seq<T>(a.y); k.dx = Seq<T>(a.dx); k.dgate = Seq<T>(a.dgate);
  k.r = Seq<R>(a.r); k.dresidual = Seq<R>(a.dresidual);
  k.scale = static_cast<const P*>(a.scale); k.weight = static_cast<const P*>(a.weight);
  k.bias = static_cast<const P*>(a.bias);
  k.stats = a.stats;
  k.part = a.scratch;
  bool even = true;  // rows at one distance throughout: no division by N
  for (const haste_b200_sequence* q : {&a.x, &a.gate, &a.residual, &a.y, &a.r, &a.dy, &a.dr, &a.dx, &a.dgate, &a.dresidual})
    even &= !q->data || q->t_stride == a.N * q->n_stride;
  if (even) k.N = std::max(1, k.rows);
  const int th = Sub ? SUB_THREADS : threads(a.H, V * K), rows = Sub ? SUB_THREADS / (Sub ? Sub : 1) : 1;
  if (!backward) {
    if (k.rows == 0) return HASTE_B200_OK;
    const int blocks = std::min(ceil_div(k.rows, rows), std::max(1, std::min(32, 768 / th)) * sm_count());
    norm_fwd<T, R, P, V, K, Sub><<<blocks, th, 0, s>>>(k);
    HB_LAUNCH_OK();
    count_launch(1);
    return HASTE_B200_OK;
  }
  const int blocks = parts(a);
  const size_t smem = V * K > 8 ? 3 * sizeof(float) * a.H : 0;
  if (smem > 48 * 1024)
    HB_CUDA_OK(cudaFuncSetAttribute(norm_bwd<T, R, P, V, K, Sub>, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * 4 * 8192));
  norm_bwd<T, R, P, V, K, Sub><<<blocks, th, smem, s>>>(k);
  HB_LAUNCH_OK();
  count_launch(1);
  SumJobs jobs;
  jobs.add(a.dweight, 0, 1, a.H, a.param_dtype);
  jobs.add(a.dbias, a.H, 1, a.H, a.param_dtype);
  jobs.add(a.dscale, 2LL * a.H, 1, a.H, a.param_dtype);
  return sum_parts(a.scratch, blocks, 3LL * a.H, jobs, s);
}

template <typename T, typename R, typename P, int V>
int by_count(const haste_b200_fused_norm& a, bool backward, cudaStream_t s) {
  // Short rows: 8 or 16 lanes each, against a block for every row (us, bf16, forward and backward with residual
  // and scale: 1001000 x 64 825 -> 257, 641000 x 100 595 -> 324).  The same widths stand in parts().
  if (a.H <= 64) return launch<T, R, P, V, 8 / V, 8>(a, backward, s);
  if (a.H <= 128) return launch<T, R, P, V, 8 / V, 16>(a, backward, s);
  return a.H <= 4096 ? launch<T, R, P, V, 8 / V, 0>(a, backward, s) : launch<T, R, P, V, 16 / V, 0>(a, backward, s);
}

template <typename T, typename R, typename P>
int by_width(const haste_b200_fused_norm& a, bool backward, cudaStream_t s) {
  const int v = width(a);
  if constexpr (sizeof(T) == 2)
    if (v == 8) return by_count<T, R, P, 8>(a, backward, s);
  return v >= 4 ? by_count<T, R, P, 4>(a, backward, s)
       : v == 2 ? by_count<T, R, P, 2>(a, backward, s)
                : by_count<T, R, P, 1>(a, backward, s);
}

}  // namespace

template <typename T>
int run(const haste_b200_fused_norm& a, bool backward, cudaStream_t s) {
  const bool r = a.residual_dtype == HASTE_B200_F32, p = a.param_dtype == HASTE_B200_F32;
  if constexpr (sizeof(T) == 4) return by_width<T, T, T>(a, backward, s);
  else if (r) return p ? by_width<T, float, float>(a, backward, s) : by_width<T, float, T>(a, backward, s);
  else return p ? by_width<T, T, float>(a, backward, s) : by_width<T, T, T>(a, backward, s);
}

}  // namespace norm
}  // namespace hb
