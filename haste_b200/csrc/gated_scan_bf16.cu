// The gated linear recurrence's kernels for __nv_bfloat16 sequences.
#include "gated_scan.cuh"

namespace hb {
namespace gated {
template int run<__nv_bfloat16>(const haste_b200_gated_scan&, bool, cudaStream_t);
}  // namespace gated
}  // namespace hb
