// The fused norm's kernels for __half sequences.
#include "fused_norm.cuh"

namespace hb {
namespace norm {
template int run<__half>(const haste_b200_fused_norm&, bool, cudaStream_t);
}  // namespace norm
}  // namespace hb
