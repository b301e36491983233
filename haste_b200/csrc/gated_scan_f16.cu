// The gated linear recurrence's kernels for __half sequences.
#include "gated_scan.cuh"

namespace hb {
namespace gated {
template int run<__half>(const haste_b200_gated_scan&, bool, cudaStream_t);
}  // namespace gated
}  // namespace hb
