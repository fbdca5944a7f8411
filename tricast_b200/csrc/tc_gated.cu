// The C entry of the gated activation with an 8-bit output.
#include <string>

#include "tc_gated.cuh"

namespace tc {
namespace gated {
void launch_f32(const Args &a, int elem, cudaStream_t s);
void launch_bf16(const Args &a, int elem, cudaStream_t s);
void launch_f16(const Args &a, int elem, cudaStream_t s);
}  // namespace gated
}  // namespace tc

extern "C" int tc_gated_quantize(const void *gate, int64_t gate_stride, const void *up, int64_t up_stride, int32_t dtype,
                                 int64_t rows, int64_t K, int32_t activation, const tc_quant_spec *spec, void *codes, void *scale,
                                 tc_stream stream) {
  using namespace tc;
  if (rows == 0) return TC_OK;
  auto bad = [](const char *m) { return set_error(std::string("tc_gated_quantize: ") + m), (int)TC_INVALID_ARGUMENT; };
  if (rows < 0 || K <= 0 || rows >= (1ll << 40) / K) return bad("rows and K out of range");
  if (!gate || !up || !spec || !codes || !scale) return bad("null pointer");
  if (dtype < 0 || dtype > 2) return bad("unsupported dtype");
  if (activation < 0 || activation > 3) return bad("unknown activation");
  if (gate_stride < K || up_stride < K) return bad("row strides must be at least K");
  gated::Args a;
  int elem;
  const int st = cast8_spec(spec, K, "tc_gated_quantize", elem, a);
  if (st != TC_OK) return st;
  a.gate = gate;
  a.up = up;
  a.gate_stride = gate_stride;
  a.up_stride = up_stride;
  a.rows = rows;
  a.act = activation;
  a.codes = static_cast<unsigned char *>(codes);
  a.scale = scale;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == TC_F32) gated::launch_f32(a, elem, s);
  else if (dtype == TC_BF16) gated::launch_bf16(a, elem, s);
  else gated::launch_f16(a, elem, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(std::string("tc_gated_quantize: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  return TC_OK;
}
