// The fused norm's kernels for __nv_bfloat16 sequences.
#include "fused_norm.cuh"

namespace hb {
namespace norm {
template int run<__nv_bfloat16>(const haste_b200_fused_norm&, bool, cudaStream_t);
}  // namespace norm
}  // namespace hb
