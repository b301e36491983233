// The fused norm's kernels for float sequences.
#include "fused_norm.cuh"

namespace hb {
namespace norm {
template int run<float>(const haste_b200_fused_norm&, bool, cudaStream_t);
}  // namespace norm
}  // namespace hb
