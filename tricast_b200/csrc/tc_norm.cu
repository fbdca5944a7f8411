// The C entry of the norm with an 8-bit output.
#include <string>

#include "tc_norm.cuh"

namespace tc {
namespace norm {
void launch_f32(const Args &a, int elem, cudaStream_t s);
void launch_bf16(const Args &a, int elem, cudaStream_t s);
void launch_f16(const Args &a, int elem, cudaStream_t s);
}  // namespace norm
}  // namespace tc

extern "C" int tc_rms_norm_quantize(const void *x, const void *residual, int32_t dtype, int64_t rows, int64_t K,
                                    int64_t x_stride, int64_t residual_stride, const void *weight,
                                    int32_t weight_dtype, float eps, const tc_quant_spec *spec, void *codes,
                                    void *scale, void *residual_out, tc_stream stream) {
  using namespace tc;
  if (rows == 0) return TC_OK;
  auto bad = [](const char *m) { return set_error(std::string("tc_rms_norm_quantize: ") + m), (int)TC_INVALID_ARGUMENT; };
  if (rows < 0 || K <= 0 || rows >= (1ll << 40) / K) return bad("rows and K out of range");
  if (!x || !spec || !codes || !scale) return bad("null pointer");
  if (dtype < 0 || dtype > 2 || weight_dtype < 0 || weight_dtype > 2) return bad("unsupported dtype");
  if (x_stride < K || (residual && residual_stride < K)) return bad("row strides must be at least K");
  if (!(eps >= 0.0f)) return bad("eps must not be negative");
  norm::Args a;
  int elem;
  const int st = cast8_spec(spec, K, "tc_rms_norm_quantize", elem, a);
  if (st != TC_OK) return st;
  a.x = x;
  a.res = residual;
  a.w = weight;
  a.h = residual_out;
  a.codes = static_cast<unsigned char *>(codes);
  a.scale = scale;
  a.rows = rows;
  a.x_stride = x_stride;
  a.res_stride = residual_stride;
  a.w_dtype = weight_dtype;
  a.eps = eps;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == TC_F32) norm::launch_f32(a, elem, s);
  else if (dtype == TC_BF16) norm::launch_bf16(a, elem, s);
  else norm::launch_f16(a, elem, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(std::string("tc_rms_norm_quantize: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  return TC_OK;
}
