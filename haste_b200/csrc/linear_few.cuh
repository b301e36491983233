// Projections of few rows (tokens): y[M,H] = act(x[M,C] W[H,C]^T + bias) + residual, M up to 32.
//
// The weight is read once and nothing else counts: HBM bounds it.  So the weights go from memory straight into the
// registers that the matrix instruction takes them from, many loads ahead; tcgen05, whose operands go through shared
// memory and whose sums through tensor memory, has nothing to win at 2 M operations a byte.
#pragma once

#include "epilogue.cuh"
#include "tcgen05.cuh"

namespace hb {
namespace few {

using namespace ss;

constexpr int WARPS = 8;

struct Args {
  const void *x, *w;
  long long x_ld;
  void* y;
  long long y_ld;
  int M, C, H, splits, per;  // splits: blocks that share C out, `per` values each
  Epilogue e;
};

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight (fp32: four) neighbouring values from `at` on, zeros from `end` on: one load where rows start on 16 bytes.
template <typename T, bool Wide>
__device__ __forceinline__ Raw<T, 16 / (int)sizeof(T)> load16(bool ok, const T* row, int at, int end) {
  constexpr int V = 16 / sizeof(T);
  if constexpr (Wide) return load_if<T, V>(ok && at < end, row + at);
  Raw<T, V> r = {};
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const Raw<T, 1> one = load_if<T, 1>(ok && at + i < end, row + at + i);
    if constexpr (sizeof(T) == 4) r.w[i] = one.w[0];
    else r.w[i / 2] |= (one.w[0] & 0xffffu) << (i % 2 * 16);
  }
  return r;
}

// A block takes RT times 16 rows of W and a cluster's share of C; its warps share that out in turn.  Thread (g, t) of a warp has
// rows g and g + 8 of each 16 and 16 bytes of each, 32 (fp32: 16) values of C to the four t's.  The order of C in a product is free,
// so those bytes are used as the registers of two matrix instructions (k = 2t, 2t + 1, 2t + 8, 2t + 9) as they lie, with x
// the same way.  MT tiles of eight tokens.  fp32 multiplies on the FMA units.
// x comes from L2 once for every RT 16 rows: from 17 tokens on two.  bf16, us by itself: 1 x 1024, H = 4096 6.3 (8.4 MB: 1.3 at
// the copy bandwidth, and about 2.5 for a launch and its first loads), 32 tokens 8.4; 1 x 4096, H = 4096 11.3 (33.6 MB: 5.1), 32
// 18.1.  64 tokens in this way 29 and 53, where the tensor cores with K split take 12 and 18.  What 32 tokens wait for: a step's
// loads are issued together, and the next step's only when they have been multiplied.  fp32 in a graph, 1 / 8 tokens x 4096, H =
// 4096: 22.2 / 32.4 (67 MB: 10.2); nine, through the tensor cores with the weight split into planes, 58.8.
// The warps' sums meet in shared memory, the blocks' of a cluster in the shared memory of each, rows shared out.
template <typename T, int MT, bool Wide, typename TO>
struct Shape {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int V = 16 / sizeof(T), STEP = 4 * V, TOK = MT * 8, RT = MT >= 4 ? 2 : 1, ROWS = RT * 16;
  static constexpr int AHEAD = MT >= 4 ? 2 : 4;  // steps whose loads are under way together
};
template <typename T, int MT, bool Wide, typename TO>
__global__ void __launch_bounds__(WARPS * 32) few_kernel(const Args a) {
  typedef Shape<T, MT, Wide, TO> S;
  constexpr bool F32 = S::F32;
  constexpr int V = S::V, STEP = S::STEP, TOK = S::TOK, RT = S::RT, ROWS = S::ROWS, AHEAD = S::AHEAD;
  __shared__ float sums[WARPS][TOK][ROWS + 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int splits = a.splits, split = blockIdx.x % splits, h0 = blockIdx.x / splits * ROWS;  // (those blocks are a cluster)
  const int c0 = split * a.per, c1 = min(a.C, c0 + a.per);
  const T* w = static_cast<const T*>(a.w) + (long long)(h0 + g) * a.C;
  const T* x = static_cast<const T*>(a.x);
  float d[RT][MT][4] = {};                   // [tile]: (g, token 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1)
  float f[F32 ? 2 : 1][F32 ? TOK : 1] = {};  // fp32: the thread's part of (row, token)
  for (int c = c0 + warp * STEP * AHEAD; c < c1; c += WARPS * STEP * AHEAD) {
    Raw<T, V> ws[AHEAD][RT][2], xs[AHEAD][F32 ? 1 : MT];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int at = c + i * STEP + t * V;
#pragma unroll
      for (int r = 0; r < 2 * RT; ++r) ws[i][r / 2][r % 2] = load16<T, Wide>(h0 + g + 8 * r < a.H, w + 8LL * r * a.C, at, c1);
      if constexpr (!F32)
#pragma unroll
        for (int m = 0; m < MT; ++m) xs[i][m] = load16<T, Wide>(m * 8 + g < a.M, x + (m * 8 + g) * a.x_ld, at, c1);
    }
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int at = c + i * STEP + t * V;
        float p[V], q[V];
        unpack<T, V>(ws[i][0][0], p);
        unpack<T, V>(ws[i][0][1], q);
#pragma unroll
        for (int m = 0; m < TOK; ++m) {
          float v[V];
          unpack<T, V>(load16<T, Wide>(m < a.M, x + m * a.x_ld, at, c1), v);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            f[0][m] = fmaf(p[j], v[j], f[0][m]);
            f[1][m] = fmaf(q[j], v[j], f[1][m]);
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const uint32_t k[4] = {ws[i][r][0].w[2 * half], ws[i][r][1].w[2 * half], ws[i][r][0].w[2 * half + 1], ws[i][r][1].w[2 * half + 1]};
#pragma unroll
            for (int m = 0; m < MT; ++m) mma<T>(d[r][m], k, xs[i][m].w[2 * half], xs[i][m].w[2 * half + 1]);
          }
    }
  }
  if constexpr (F32) {
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int m = 0; m < TOK; ++m) {
        float v = f[r][m];
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        v += __shfl_xor_sync(0xffffffffu, v, 2);
        if (t == 0) sums[warp][m][g + 8 * r] = v;
      }
  } else {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[warp][m * 8 + 2 * t + i % 2][r * 16 + g + i / 2 * 8] = d[r][m][i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < TOK * ROWS; i += WARPS * 32) {
    const int m = i / ROWS, r = i % ROWS;
    float s = sums[0][m][r];
#pragma unroll
    for (int v = 1; v < WARPS; ++v) s += sums[v][m][r];
    if (splits > 1) sums[0][m][r] = s;
    else if (m < a.M && h0 + r < a.H) epi::finish<T, TO>(a.e, s, m, h0 + r, static_cast<TO*>(a.y) + m * a.y_ld + h0 + r);
  }
  if (splits == 1) return;
  tc::cluster_sync_all();
  for (int i = split * WARPS * 32 + threadIdx.x; i < TOK * ROWS; i += splits * WARPS * 32) {
    const int m = i / ROWS, r = i % ROWS;
    const uint32_t at = tc::smem_u32(&sums[0][m][r]);
    float s = 0.f;
    for (int k = 0; k < splits; ++k) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(tc::mapa_u32(at, k)));
      s += v;
    }
    if (m < a.M && h0 + r < a.H) epi::finish<T, TO>(a.e, s, m, h0 + r, static_cast<TO*>(a.y) + m * a.y_ld + h0 + r);
  }
  tc::cluster_sync_all();  // nobody leaves while its sums are read
}

template <typename T, int MT, bool Wide, typename TO>
int launch(Args a, cudaStream_t s) {
  typedef Shape<T, MT, Wide, TO> S;
  // Shares of C until there are two blocks an SM, each with the loads that its warps have under way together.
  const int tiles = ceil_div(a.H, S::ROWS);
  int splits = 1;
  while (splits < 8 && splits * tiles < 2 * sm_count() && a.C / (2 * splits) >= WARPS * S::STEP * S::AHEAD) splits *= 2;
  a.splits = splits;
  a.per = ceil_div(ceil_div(a.C, splits), S::V) * S::V;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits * tiles);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  HB_CUDA_OK(cudaLaunchKernelEx(&cfg, few_kernel<T, MT, Wide, TO>, a));
  count_launch(1);
  return HASTE_B200_OK;
}

template <typename T, typename TO>
int run(const Args& a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = a.C % V == 0 && a.x_ld % V == 0 && aligned(a.x, 16) && aligned(a.w, 16);
#define HB_FEW(MT) return wide ? launch<T, MT, true, TO>(a, s) : launch<T, MT, false, TO>(a, s)
  if constexpr (sizeof(T) == 4) {
    HB_FEW(1);
  } else {
    if (a.M <= 8) HB_FEW(1);
    if (a.M <= 16) HB_FEW(2);
    HB_FEW(4);
  }
#undef HB_FEW
}

}  // namespace few
}  // namespace hb
