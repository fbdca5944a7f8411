// The chunk attention kernel for one cache scheme (compiled on its own to build in parallel).
#include "tc_attn_chunk.cuh"

namespace tc {
namespace attn {
int launch_chunk_none(const Args &a, float *parts, Stretch *stretches, int *status, int most, cudaStream_t s) {
  return chunk::launch_scheme<KV_NONE>(a, parts, stretches, status, most, s);
}
}  // namespace attn
}  // namespace tc
