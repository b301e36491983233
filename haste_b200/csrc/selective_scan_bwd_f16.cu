// The selective scan's backward kernels for __half sequences.
#include "selective_scan_bwd.cuh"

namespace hb {
namespace scan {
template int backward<__half>(const haste_b200_selective_scan&, cudaStream_t);
}  // namespace scan
}  // namespace hb
