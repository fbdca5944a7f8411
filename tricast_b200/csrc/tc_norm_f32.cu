// The norm's kernels for one input type (compiled on its own to build in parallel).
#include "tc_norm.cuh"

namespace tc {
namespace norm {
void launch_f32(const Args &a, int elem, cudaStream_t s) { launch<float>(a, elem, s); }
}  // namespace norm
}  // namespace tc
