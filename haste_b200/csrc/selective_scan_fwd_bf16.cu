// The selective scan's forward kernels for __nv_bfloat16 sequences.
#include "selective_scan_fwd.cuh"

namespace hb {
namespace scan {
template int forward<__nv_bfloat16>(const haste_b200_selective_scan&, cudaStream_t);
}  // namespace scan
}  // namespace hb
