// Gated linear recurrence: argument checks, scratch sizes and the choice of the storage type.
#include "gated_scan.cuh"

namespace hb {
namespace gated {

extern template int run<float>(const haste_b200_gated_scan&, bool, cudaStream_t);
extern template int run<__nv_bfloat16>(const haste_b200_gated_scan&, bool, cudaStream_t);
extern template int run<__half>(const haste_b200_gated_scan&, bool, cudaStream_t);

namespace {

int check(const haste_b200_gated_scan& a, bool backward) {
  HB_REQUIRE(storage_dtype(a.dtype), "dtype");
  HB_REQUIRE(a.T >= 0 && a.T <= (1 << 30) && a.N >= 0 && a.D >= 0 && a.D <= (1 << 30), "T,N,D");
  HB_REQUIRE((long long)a.N * a.D < (1LL << 31), "N*D too large");
  for (const haste_b200_sequence* q : {&a.x, &a.gate, &a.input_gate, &a.y, &a.dy, &a.dx, &a.dgate, &a.dinput_gate})
    HB_REQUIRE(strides_fit(a.T, *q), "a step's stride must be below 2^31 elements");
  HB_REQUIRE(aligned(a.scratch, 8), "scratch must be aligned to 8 bytes");
  if (a.N == 0 || a.D == 0) return HASTE_B200_OK;
  if (backward) HB_REQUIRE(!a.decay || (a.ddecay && a.scratch), "null pointer");
  if (a.T == 0) return HASTE_B200_OK;
  HB_REQUIRE(a.x.data && a.gate.data, "null pointer");
  if (backward) {
    HB_REQUIRE(a.checkpoints && a.dy.data && a.dx.data && a.dgate.data, "null pointer");
    HB_REQUIRE(a.scratch || gated_scan_scratch(a, true) == 0, "null pointer");
    HB_REQUIRE(!a.input_gate.data == !a.dinput_gate.data, "dinput_gate goes with input_gate");
  } else {
    HB_REQUIRE(a.y.data, "null pointer");
  }
  return HASTE_B200_OK;
}

int dispatch(const haste_b200_gated_scan& a, bool backward, cudaStream_t s) {
  HB_TRY(check(a, backward));
  if (a.N == 0 || a.D == 0) {  // (of no rows the decay's gradient is zero)
    if (backward && a.decay && a.ddecay && a.D > 0) HB_CUDA_OK(cudaMemsetAsync(a.ddecay, 0, (size_t)a.D * 4, s));
    return HASTE_B200_OK;
  }
  ProfScope p(backward ? PH_REC_BWD : PH_REC_FWD, s);
  if (a.dtype == HASTE_B200_F32) return run<float>(a, backward, s);
  if (a.dtype == HASTE_B200_BF16) return run<__nv_bfloat16>(a, backward, s);
  return run<__half>(a, backward, s);
}

}  // namespace
}  // namespace gated

int gated_scan_forward(const haste_b200_gated_scan& a, cudaStream_t s) { return gated::dispatch(a, false, s); }
int gated_scan_backward(const haste_b200_gated_scan& a, cudaStream_t s) { return gated::dispatch(a, true, s); }

long long gated_scan_scratch(const haste_b200_gated_scan& a, bool backward) {
  if (a.T < 0 || a.N <= 0 || a.D <= 0) return 0;
  const int pieces = gated::most_pieces(a, backward);
  const long long rows = (long long)a.N * a.D, ends = pieces > 1 ? 2 * pieces * rows : 0;
  return ends + (backward && a.decay ? pieces * rows : 0);
}
long long gated_scan_checkpoints(const haste_b200_gated_scan& a) {
  if (a.T <= 0 || a.N <= 0 || a.D <= 0) return 0;
  return (long long)ceil_div(a.T, gated::CKPT) * a.N * a.D;
}

}  // namespace hb
