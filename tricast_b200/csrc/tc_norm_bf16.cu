// The norm's kernels for one input type (compiled on its own to build in parallel).
#include "tc_norm.cuh"

namespace tc {
namespace norm {
void launch_bf16(const Args &a, int elem, cudaStream_t s) { launch<__nv_bfloat16>(a, elem, s); }
}  // namespace norm
}  // namespace tc
