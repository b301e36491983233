// Selective scan: argument checks, scratch sizes and the choice of the storage type.
#include <algorithm>

#include "selective_scan.cuh"

namespace hb {
namespace scan {

extern template int forward<float>(const haste_b200_selective_scan&, cudaStream_t);
extern template int forward<__nv_bfloat16>(const haste_b200_selective_scan&, cudaStream_t);
extern template int forward<__half>(const haste_b200_selective_scan&, cudaStream_t);
extern template int backward<float>(const haste_b200_selective_scan&, cudaStream_t);
extern template int backward<__nv_bfloat16>(const haste_b200_selective_scan&, cudaStream_t);
extern template int backward<__half>(const haste_b200_selective_scan&, cudaStream_t);

int check(const haste_b200_selective_scan& a, bool backward) {
  HB_REQUIRE(storage_dtype(a.dtype), "dtype");
  HB_REQUIRE(a.T >= 0 && a.T <= (1 << 30) && a.N >= 0 && a.D >= 0, "T,N,D");
  HB_REQUIRE(a.S >= 1 && a.S <= 128, "S must be 1..128");
  HB_REQUIRE(a.G >= 1 && a.D % a.G == 0, "G must divide D");
  HB_REQUIRE((long long)a.D * (a.S + 2) < (1LL << 31) && (long long)a.N * a.D < (1LL << 31), "N*D too large");
  HB_REQUIRE((long long)a.N * a.D * a.S < (1LL << 37), "N*D*S too large");
  for (const haste_b200_sequence* q : {&a.x, &a.dt, &a.z, &a.y, &a.B, &a.C, &a.dy, &a.dx, &a.ddt, &a.dz, &a.dB, &a.dC})
    HB_REQUIRE(strides_fit(a.T, *q), "a step's stride must be below 2^31 elements");
  if (a.N == 0 || a.D == 0) return HASTE_B200_OK;
  HB_REQUIRE(a.A, "null pointer");
  if (backward) HB_REQUIRE(a.dA && a.scratch, "null pointer");
  if (a.T == 0) return HASTE_B200_OK;
  HB_REQUIRE(a.x.data && a.dt.data && a.B.data && a.C.data, "null pointer");
  if (backward) {
    HB_REQUIRE(a.checkpoints && a.dy.data && a.dx.data && a.ddt.data && a.dB.data && a.dC.data, "null pointer");
    HB_REQUIRE(!a.z.data == !a.dz.data, "dz goes with z");
  } else {
    HB_REQUIRE(a.y.data, "null pointer");
  }
  return HASTE_B200_OK;
}

// Pieces of a sequence.  Walking it twice pays where whole sequences leave most SMs without work: below two
// blocks per SM, if at least three pieces of 64 steps or more come of it, as many as make five blocks per
// SM.  fp32 T=2000 N=1 D=1024 S=16, us: whole 132; pieces for 2, 3, 5, 8 blocks 42, 40, 38, 42; 32 steps at
// least 38, 128 40.  T=333 N=7 D=250 S=24: whole 27.4, in pieces 25.4.
int forward_pieces(const haste_b200_selective_scan& a) {
  const int CB = THREADS / lanes(a.S);
  const long long blocks = (long long)a.N * a.G * ceil_div(a.D / a.G, CB);
  if (blocks >= 2LL * sm_count()) return 1;
  const long long want = std::min(ceil_div(5LL * sm_count(), blocks), ceil_div(a.T, 64));
  return want < 3 ? 1 : (int)want;
}

}  // namespace scan

int selective_scan_forward(const haste_b200_selective_scan& a, cudaStream_t s) {
  HB_TRY(scan::check(a, false));
  if (a.N == 0 || a.D == 0) return HASTE_B200_OK;
  ProfScope p(PH_REC_FWD, s);
  if (a.dtype == HASTE_B200_F32) return scan::forward<float>(a, s);
  if (a.dtype == HASTE_B200_BF16) return scan::forward<__nv_bfloat16>(a, s);
  return scan::forward<__half>(a, s);
}

int selective_scan_backward(const haste_b200_selective_scan& a, cudaStream_t s) {
  HB_TRY(scan::check(a, true));
  if (a.N == 0 || a.D == 0) return HASTE_B200_OK;
  ProfScope p(PH_REC_BWD, s);
  if (a.dtype == HASTE_B200_F32) return scan::backward<float>(a, s);
  if (a.dtype == HASTE_B200_BF16) return scan::backward<__nv_bfloat16>(a, s);
  return scan::backward<__half>(a, s);
}

long long selective_scan_scratch(const haste_b200_selective_scan& a, bool backward) {
  if (a.T < 0 || a.N <= 0 || a.D <= 0 || a.S < 1 || a.S > 128 || a.G < 1 || a.D % a.G) return 0;
  if (backward) return scan::BwdShape(a).floats(a);
  const int J = scan::forward_pieces(a);
  return J > 1 ? (long long)J * a.N * a.D * (a.S + 1) : 0;
}

long long selective_scan_checkpoints(const haste_b200_selective_scan& a) {
  if (a.T <= 0 || a.N <= 0 || a.D <= 0 || a.S <= 0) return 0;
  return (long long)ceil_div(a.T, scan::CKPT) * a.N * a.D * a.S;
}

}  // namespace hb
