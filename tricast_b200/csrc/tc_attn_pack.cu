// The chunk attention kernel over units laid out beforehand, and the kernel that lays them out.
#include "tc_attn_chunk.cuh"

namespace tc {
namespace attn {

size_t packed_unit_bytes(int dim) { return dim <= 64 ? chunk::Packed<64>::kBytes : chunk::Packed<128>::kBytes; }

int launch_packed(const Args &a, float *parts, Stretch *stretches, int *status, int most, unsigned char *packed, int max_units,
                  cudaStream_t s) {
  return a.c.scheme == KV_FP8_ROW    ? chunk::launch_packed<KV_FP8_ROW>(a, parts, stretches, status, most, packed, max_units, s)
         : a.c.scheme == KV_INT8_ROW ? chunk::launch_packed<KV_INT8_ROW>(a, parts, stretches, status, most, packed, max_units, s)
                                     : chunk::launch_packed<KV_MXFP4>(a, parts, stretches, status, most, packed, max_units, s);
}

}  // namespace attn
}  // namespace tc
