// Projections: y = act(x W^T + bias) + residual, and their gradients
//
//   dp = dy act'(p),  dx = dp W,  dW = dp^T x,  dbias = sum of dp over the rows,  dresidual = dy.
//
// Each is one contraction, bound by the tensor cores where there are many rows (gemm_sm100.cu, with what follows the
// sums in its epilogue) and by the weight's bytes where there are few (linear_few.cuh).  dp is computed and summed up in
// one pass over dy and p = x W^T + bias, which the forward pass leaves in x's type: that rounding moves a slope by
// half a step of p, as the rounding of y moves whatever reads it; where it makes an infinity of p, the slope is its limit
// there.  dp is rounded to x's type too, which the tensor cores multiply: half a step of it, in 16 bits as much again as the
// rounding of dx and dW themselves (bf16 64000 x 1024 x 2048, SiLU, against float64: 2.4e-3, where dp in fp32 leaves 1.7e-3;
// p's rounding is 0.1e-3 of that).  A float32 dy beside fp16 operands meets fp16's range in dp.
#include <algorithm>

#include "epilogue.cuh"
#include "linear_few.cuh"

namespace hb {
namespace lin {
namespace {

using namespace ss;

constexpr int THREADS = 256, ROWS = THREADS / 32;

// A block takes 32 lanes of V columns and every chunks-th row in eights: a warp a row, four rows ahead.
template <typename T, typename TO, int V, int Act>
__global__ void __launch_bounds__(THREADS) slope_kernel(const T* pre, const TO* dy, long long dy_ld, T* dp, int M, int H,
                                                        float* part) {
  constexpr bool act = Act != HASTE_B200_IDENTITY;
  __shared__ float sums[ROWS][32][V + 1];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int n = (blockIdx.x * 32 + lane) * V;
  const bool ok = n < H;
  float sum[V] = {};
  constexpr int AHEAD = 4;
  const long long step = (long long)gridDim.y * ROWS;
  for (long long m0 = blockIdx.y * ROWS + warp; m0 < M; m0 += step * AHEAD) {
    Raw<TO, V> y[AHEAD];
    Raw<T, V> p[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const long long m = m0 + i * step;
      const bool in = ok && m < M;
      y[i] = load_if<TO, V>(in, dy + m * dy_ld + n);
      if (act) p[i] = load_if<T, V>(in, pre + m * H + n);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const long long m = m0 + i * step;
      float v[V], q[V];
      unpack<TO, V>(y[i], v);
      if (act) {
        unpack<T, V>(p[i], q);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= epi::slope<sizeof(T) == 4, Act>(q[j]);
      }
      if (!ok || m >= M) continue;
      if (dp) store<T, V>(dp + m * H + n, v);
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += v[j];
    }
  }
  if (!part) return;
#pragma unroll
  for (int j = 0; j < V; ++j) sums[warp][lane][j] = sum[j];
  __syncthreads();
  if (warp == 0 && ok)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float s = sums[0][lane][j];
#pragma unroll
      for (int w = 1; w < ROWS; ++w) s += sums[w][lane][j];
      part[(long long)blockIdx.y * H + n + j] = s;
    }
}

// Blocks that share out the rows: four an SM together.
int chunks_of(int M, int H, int V) {
  const long long across = ceil_div(H, 32 * V);
  return (int)std::max(1LL, std::min((4LL * sm_count() + across - 1) / across, (long long)ceil_div(M, 4 * ROWS)));
}
int most_chunks(const haste_b200_linear& a) { return std::max(chunks_of(a.M, a.H, 1), std::max(chunks_of(a.M, a.H, 4), chunks_of(a.M, a.H, 8))); }

bool direct(const haste_b200_linear& a) { return a.activation == HASTE_B200_IDENTITY && a.out_dtype == a.dtype; }  // dp is dy

template <typename T, typename TO, int V>
int launch_slope(const haste_b200_linear& a, T* dp, float* part, int* chunks, cudaStream_t s) {
  *chunks = chunks_of(a.M, a.H, V);
  epi::with_activation(a.activation, [&](auto act) {
    slope_kernel<T, TO, V, decltype(act)::value><<<dim3(ceil_div(a.H, 32 * V), *chunks), THREADS, 0, s>>>(
        static_cast<const T*>(a.pre), static_cast<const TO*>(a.dy), a.dy_ld, dp, a.M, a.H, part);
  });
  HB_LAUNCH_OK();
  count_launch(1);
  return HASTE_B200_OK;
}
template <typename T, typename TO>
int slopes(const haste_b200_linear& a, void* dp_, float* part, int* chunks, cudaStream_t s) {
  // (16 bytes of the widest type at a time)
  constexpr int V = sizeof(TO) == 4 ? 4 : 8;
  T* dp = static_cast<T*>(dp_);
  if (a.H % V == 0 && a.dy_ld % V == 0 && aligned(a.dy, 16) && aligned(a.pre, 16)) return launch_slope<T, TO, V>(a, dp, part, chunks, s);
  return launch_slope<T, TO, 1>(a, dp, part, chunks, s);
}

// The three contractions, with operands where they lie.
GemmDesc product(const haste_b200_linear& a, int M, int N, int K, const void* x, long long x_rs, long long x_cs, const void* w,
                 long long w_rs, long long w_cs, void* c, long long ldc, int dtype_c, void* scratch) {
  GemmDesc g{a.dtype, dtype_c, M, N, K, x, x_rs, x_cs, w, w_rs, w_cs, c, ldc, 0};
  g.precise = 1;
  g.projection = true;
  g.scratch = scratch;
  static const Epilogue nothing{};
  if (a.dtype == HASTE_B200_F32) g.epilogue = &nothing;  // (by the projections' own, more exact product)
  return g;
}
GemmDesc forward_product(const haste_b200_linear& a, void* scratch) {
  return product(a, a.M, a.H, a.C, a.x, a.x_ld, 1, a.weight, 1, a.C, a.y, a.y_ld, a.out_dtype, scratch);
}
GemmDesc dx_product(const haste_b200_linear& a, const void* dp, long long ld, void* scratch) {
  return product(a, a.M, a.C, a.H, dp, ld, 1, a.weight, a.C, 1, a.dx, a.dx_ld, a.dtype, scratch);
}
GemmDesc dw_product(const haste_b200_linear& a, const void* dp, long long ld, void* scratch) {
  return product(a, a.H, a.C, a.M, dp, 1, ld, a.x, a.x_ld, 1, a.dweight, a.C, a.dtype, scratch);
}

// Few rows: 32 of 16 bits, 8 of fp32, which has no matrix instruction of its own.
bool few_rows(const haste_b200_linear& a) { return a.M <= (a.dtype == HASTE_B200_F32 ? 8 : 32); }

struct Layout {
  size_t dp, part, gemm, bytes;
  explicit Layout(const haste_b200_linear& a) {
    dp = direct(a) ? 0 : Arena::pad((size_t)a.M * a.H * dtype_size(a.dtype));
    part = a.dbias ? Arena::pad((size_t)most_chunks(a) * a.H * 4) : 0;
    const void* from = direct(a) ? a.dy : nullptr;
    const long long ld = direct(a) ? a.dy_ld : a.H;
    const size_t x = a.dx ? gemm_scratch(dx_product(a, from, ld, nullptr)) : 0, w = a.dweight ? gemm_scratch(dw_product(a, from, ld, nullptr)) : 0;
    gemm = std::max(x, w);
    bytes = dp + part + gemm;
  }
};

int check(const haste_b200_linear& a, bool backward) {
  HB_REQUIRE(storage_dtype(a.dtype), "dtype");
  HB_REQUIRE(a.out_dtype == a.dtype || a.out_dtype == HASTE_B200_F32, "out_dtype");
  HB_REQUIRE(a.param_dtype == a.dtype || a.param_dtype == HASTE_B200_F32, "param_dtype");
  HB_REQUIRE(a.activation >= HASTE_B200_IDENTITY && a.activation <= HASTE_B200_SIGMOID, "activation");
  HB_REQUIRE(a.M >= 0 && a.C >= 1 && a.H >= 1, "M,C,H");
  HB_REQUIRE(a.M <= (1 << 30) && a.C < (1 << 20) && a.H < (1 << 20), "M, C or H too large");
  if (a.M == 0 && !backward) return HASTE_B200_OK;
  HB_REQUIRE(aligned(a.scratch, 256), "scratch must be aligned to 256 bytes");
  if (a.M > 0) {
    HB_REQUIRE(a.x && a.weight, "null pointer");
    HB_REQUIRE(a.x_ld >= a.C, "x_ld");
    if (backward) {
      HB_REQUIRE(a.dy && a.dy_ld >= a.H && (a.activation == HASTE_B200_IDENTITY || a.pre), "null pointer");
      HB_REQUIRE(!a.dx || a.dx_ld >= a.C, "dx_ld");
    } else {
      HB_REQUIRE(a.y && a.y_ld >= a.H && (!a.residual || a.residual_ld >= a.H), "null pointer");
      HB_REQUIRE(a.residual != a.y || a.residual_ld == a.y_ld || a.M == 1, "a residual in y's place has its rows");
    }
  }
  return HASTE_B200_OK;
}

template <typename T, typename TO>
int few_forward(const haste_b200_linear& a, const Epilogue& e, cudaStream_t s) {
  return few::run<T, TO>(few::Args{a.x, a.weight, a.x_ld, a.y, a.y_ld, a.M, a.C, a.H, 1, 0, e}, s);
}

}  // namespace
}  // namespace lin

int linear_forward(const haste_b200_linear& a, cudaStream_t s) {
  HB_TRY(lin::check(a, false));
  if (a.M == 0) return HASTE_B200_OK;
  ProfScope p(PH_PROJ, s);
  const Epilogue e{a.bias, a.residual, a.residual_ld, a.pre, a.H, a.param_dtype == HASTE_B200_F32, a.activation};
  if (lin::few_rows(a)) {
    if (a.dtype == HASTE_B200_F32) return lin::few_forward<float, float>(a, e, s);
    if (a.dtype == HASTE_B200_BF16)
      return a.out_dtype == HASTE_B200_F32 ? lin::few_forward<__nv_bfloat16, float>(a, e, s) : lin::few_forward<__nv_bfloat16, __nv_bfloat16>(a, e, s);
    return a.out_dtype == HASTE_B200_F32 ? lin::few_forward<__half, float>(a, e, s) : lin::few_forward<__half, __half>(a, e, s);
  }
  HB_REQUIRE(a.scratch, "null pointer");
  GemmDesc g = lin::forward_product(a, a.scratch);
  g.epilogue = &e;
  return gemm_sm100(g, s);
}

int linear_backward(const haste_b200_linear& a, cudaStream_t s) {
  HB_TRY(lin::check(a, true));
  if (a.M == 0) {
    if (a.dweight) HB_CUDA_OK(cudaMemsetAsync(a.dweight, 0, (size_t)a.H * a.C * dtype_size(a.dtype), s));
    if (a.dbias) HB_CUDA_OK(cudaMemsetAsync(a.dbias, 0, (size_t)a.H * dtype_size(a.param_dtype), s));
    return HASTE_B200_OK;
  }
  HB_REQUIRE(a.scratch, "null pointer");
  const lin::Layout at(a);
  char* base = static_cast<char*>(a.scratch);
  const bool direct = lin::direct(a);
  void* dp = direct ? nullptr : base;
  float* part = a.dbias ? reinterpret_cast<float*>(base + at.dp) : nullptr;
  void* scratch = base + at.dp + at.part;
  if (dp || part) {
    ProfScope p(PH_OTHER, s);
    int chunks = 0;
    if (a.dtype == HASTE_B200_F32) HB_TRY((lin::slopes<float, float>(a, dp, part, &chunks, s)));
    else if (a.dtype == HASTE_B200_BF16 && a.out_dtype == HASTE_B200_F32) HB_TRY((lin::slopes<__nv_bfloat16, float>(a, dp, part, &chunks, s)));
    else if (a.dtype == HASTE_B200_BF16) HB_TRY((lin::slopes<__nv_bfloat16, __nv_bfloat16>(a, dp, part, &chunks, s)));
    else if (a.out_dtype == HASTE_B200_F32) HB_TRY((lin::slopes<__half, float>(a, dp, part, &chunks, s)));
    else HB_TRY((lin::slopes<__half, __half>(a, dp, part, &chunks, s)));
    if (part) {
      ss::SumJobs jobs;
      jobs.add(a.dbias, 0, 1, a.H, a.param_dtype);
      HB_TRY(ss::sum_parts(part, chunks, a.H, jobs, s));
    }
  }
  const void* from = direct ? a.dy : dp;
  const long long ld = direct ? a.dy_ld : a.H;
  if (a.dx) {
    ProfScope p(PH_DGRAD, s);
    HB_TRY(gemm_sm100(lin::dx_product(a, from, ld, scratch), s));
  }
  if (a.dweight) {
    ProfScope p(PH_WGRAD, s);
    HB_TRY(gemm_sm100(lin::dw_product(a, from, ld, scratch), s));
  }
  return HASTE_B200_OK;
}

long long linear_scratch(const haste_b200_linear& a, bool backward) {
  if (a.M <= 0 || a.C < 1 || a.H < 1 || !ss::storage_dtype(a.dtype)) return 0;
  if (backward) return (long long)lin::Layout(a).bytes;
  return lin::few_rows(a) ? 0 : (long long)gemm_scratch(lin::forward_product(a, nullptr));
}

}  // namespace hb
