// The selective scan's backward kernels for float sequences.
#include "selective_scan_bwd.cuh"

namespace hb {
namespace scan {
template int backward<float>(const haste_b200_selective_scan&, cudaStream_t);
}  // namespace scan
}  // namespace hb
