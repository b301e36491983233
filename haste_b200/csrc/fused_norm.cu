// Fused norm: argument checks, the size of its scratch and the choice of the storage type.
#include <algorithm>

#include "state_space.cuh"

namespace hb {
namespace norm {

using namespace ss;

template <typename T>
int run(const haste_b200_fused_norm& a, bool backward, cudaStream_t s);
extern template int run<float>(const haste_b200_fused_norm&, bool, cudaStream_t);
extern template int run<__nv_bfloat16>(const haste_b200_fused_norm&, bool, cudaStream_t);
extern template int run<__half>(const haste_b200_fused_norm&, bool, cudaStream_t);

namespace {

int check(const haste_b200_fused_norm& a, bool backward) {
  HB_REQUIRE(storage_dtype(a.dtype), "dtype");
  HB_REQUIRE(a.residual_dtype == HASTE_B200_F32 || a.residual_dtype == a.dtype, "residual_dtype");
  HB_REQUIRE(a.param_dtype == HASTE_B200_F32 || a.param_dtype == a.dtype, "param_dtype");
  HB_REQUIRE(a.T >= 0 && a.N >= 0, "T,N");
  HB_REQUIRE((long long)a.T * a.N < (1LL << 31) - 65536, "T*N too large");
  HB_REQUIRE(a.H >= 1 && a.H <= 8192, "H must be 1..8192");
  HB_REQUIRE(a.eps >= 0.f, "eps");
  for (const haste_b200_sequence* q : {&a.x, &a.gate, &a.residual, &a.y, &a.r, &a.dy, &a.dr, &a.dx, &a.dgate, &a.dresidual})
    HB_REQUIRE(strides_fit(a.T, *q), "a step's stride must be below 2^31 elements");
  HB_REQUIRE(!a.scale || a.residual.data || a.T == 0 || a.N == 0, "scale needs a residual");
  HB_REQUIRE(a.weight, "null pointer");
  HB_REQUIRE(aligned(a.stats, 8), "stats must be aligned to 8 bytes");
  if (backward) HB_REQUIRE(a.scratch && a.dweight, "null pointer");
  if (a.T == 0 || a.N == 0) return HASTE_B200_OK;
  HB_REQUIRE(a.x.data, "null pointer");
  if (backward) HB_REQUIRE(a.dy.data && a.stats, "null pointer");
  else HB_REQUIRE(a.y.data, "null pointer");
  return HASTE_B200_OK;
}

int dispatch(const haste_b200_fused_norm& a, bool backward, cudaStream_t s) {
  HB_TRY(check(a, backward));
  ProfScope p(PH_OTHER, s);
  if (a.dtype == HASTE_B200_F32) return run<float>(a, backward, s);
  if (a.dtype == HASTE_B200_BF16) return run<__nv_bfloat16>(a, backward, s);
  return run<__half>(a, backward, s);
}

}  // namespace

// Blocks of the backward pass, each of which leaves a row of partial sums: 512 threads an SM, what the registers
// allow (twice as many, in two waves: 192 us against 184).
int parts(const haste_b200_fused_norm& a) {
  const int per = a.H <= 4096 ? 8 : 16, th = a.H <= 128 ? 128 : ceil_div(ceil_div(a.H, per), 32) * 32;
  const int rows = a.H <= 64 ? 16 : a.H <= 128 ? 8 : 1;  // of a block side by side
  const int per_sm = std::max(1, std::min(16, 512 / th));
  return std::max(1, std::min(ceil_div((long long)a.T * a.N, rows), per_sm * sm_count()));
}

}  // namespace norm

int fused_norm_forward(const haste_b200_fused_norm& a, cudaStream_t s) { return norm::dispatch(a, false, s); }
int fused_norm_backward(const haste_b200_fused_norm& a, cudaStream_t s) { return norm::dispatch(a, true, s); }
long long fused_norm_scratch(const haste_b200_fused_norm& a) {
  if (a.T < 0 || a.N < 0 || a.H < 1 || a.H > 8192) return 0;
  return 3LL * norm::parts(a) * a.H;
}

}  // namespace hb
