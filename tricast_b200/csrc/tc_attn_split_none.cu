// The split attention kernel for one cache scheme (compiled on its own to build in parallel).
#include "tc_attn_split.cuh"

namespace tc {
namespace attn {
int launch_split_none(const Args &a, float *parts, int sms, cudaStream_t s) {
  return split::launch_scheme<KV_NONE>(a, parts, sms, s);
}
}  // namespace attn
}  // namespace tc
