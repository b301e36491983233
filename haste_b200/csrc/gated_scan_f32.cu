// The gated linear recurrence's kernels for float sequences.
#include "gated_scan.cuh"

namespace hb {
namespace gated {
template int run<float>(const haste_b200_gated_scan&, bool, cudaStream_t);
}  // namespace gated
}  // namespace hb
