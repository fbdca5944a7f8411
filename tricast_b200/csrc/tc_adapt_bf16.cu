// The adapters' kernels for one type of weights (compiled on its own to build in parallel).
#include "tc_adapt.cuh"

namespace tc {
namespace adapt {
cudaError_t launch_bf16(const Args &a, cudaStream_t s) { return launch_as<__nv_bfloat16>(a, s); }
}  // namespace adapt
}  // namespace tc
