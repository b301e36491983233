// Sums of per-block partial results, shared by the state space operators' backward passes.
#include "state_space.cuh"

namespace hb {
namespace ss {
namespace {

constexpr int kCols = 32, kRows = 32;

// 32 columns x 32 groups of rows: thread (r, c) adds rows r, r + 32, ... of its column, eight loads ahead,
// and the sums are added in order.  The partials were written just before and lie in L2.
__global__ void __launch_bounds__(kCols* kRows) sum_parts_kernel(const float* __restrict__ part, int P,
                                                                 long long stride, SumJobs jobs) {
  __shared__ float sums[kRows][kCols];
  const SumJob job = jobs.job[blockIdx.y];
  const int c = threadIdx.x % kCols, r = threadIdx.x / kCols;
  const int j = blockIdx.x * kCols + c;
  if (blockIdx.x * kCols >= job.width) return;
  const float* p = part + job.offset + j;
  float s = 0.f;
  if (j < job.width) {
    int i = r;
    for (; i + 7 * kRows < P; i += 8 * kRows) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = p[(i + k * kRows) * stride];
      s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    for (; i < P; i += kRows) s += p[i * stride];
  }
  sums[r][c] = s;
  __syncthreads();
  if (r != 0 || j >= job.width) return;
#pragma unroll 8
  for (int k = 1; k < kRows; ++k) s += sums[k][c];
  if (job.dtype == HASTE_B200_F32) static_cast<float*>(job.out)[j * job.stride] = s;
  else if (job.dtype == HASTE_B200_BF16) st(static_cast<__nv_bfloat16*>(job.out) + j * job.stride, s);
  else st(static_cast<__half*>(job.out) + j * job.stride, s);
}

}  // namespace

int sum_parts(const float* part, int P, long long stride, const SumJobs& jobs, cudaStream_t s) {
  int width = 0;
  for (int k = 0; k < jobs.n; ++k) width = jobs.job[k].width > width ? jobs.job[k].width : width;
  if (width == 0) return HASTE_B200_OK;
  sum_parts_kernel<<<dim3(ceil_div(width, kCols), jobs.n), kCols * kRows, 0, s>>>(part, P, stride, jobs);
  HB_LAUNCH_OK();
  count_launch(1);
  return HASTE_B200_OK;
}

}  // namespace ss
}  // namespace hb
