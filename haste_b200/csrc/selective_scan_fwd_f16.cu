// The selective scan's forward kernels for __half sequences.
#include "selective_scan_fwd.cuh"

namespace hb {
namespace scan {
template int forward<__half>(const haste_b200_selective_scan&, cudaStream_t);
}  // namespace scan
}  // namespace hb
