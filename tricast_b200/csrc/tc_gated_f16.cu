// The gated activation's kernels for one input type (compiled on its own to build in parallel).
#include "tc_gated.cuh"

namespace tc {
namespace gated {
void launch_f16(const Args &a, int elem, cudaStream_t s) { launch<__half>(a, elem, s); }
}  // namespace gated
}  // namespace tc
