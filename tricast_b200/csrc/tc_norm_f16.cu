// The norm's kernels for one input type (compiled on its own to build in parallel).
#include "tc_norm.cuh"

namespace tc {
namespace norm {
void launch_f16(const Args &a, int elem, cudaStream_t s) { launch<__half>(a, elem, s); }
}  // namespace norm
}  // namespace tc
