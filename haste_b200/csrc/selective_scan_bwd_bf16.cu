// The selective scan's backward kernels for __nv_bfloat16 sequences.
#include "selective_scan_bwd.cuh"

namespace hb {
namespace scan {
template int backward<__nv_bfloat16>(const haste_b200_selective_scan&, cudaStream_t);
}  // namespace scan
}  // namespace hb
