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
  auto no = [](const char *m) { return set_error(std::string("tc_rms_norm_quantize: ") + m), (int)TC_UNSUPPORTED; };
  if (rows < 0 || K <= 0 || rows >= (1ll << 40) / K) return bad("rows and K out of range");
  if (!x || !spec || !codes || !scale) return bad("null pointer");
  if (dtype < 0 || dtype > 2 || weight_dtype < 0 || weight_dtype > 2) return bad("unsupported dtype");
  if (x_stride < K || (residual && residual_stride < K)) return bad("row strides must be at least K");
  if (!(eps >= 0.0f)) return bad("eps must not be negative");
  const tc_format &f = spec->format;
  int elem;
  if (f.kind == 0 && f.is_signed && f.subnormals && f.ebits == 4 && f.mbits == 3 && f.bias == 7 && f.special == 1) elem = E8_E4M3;
  else if (f.kind == 0 && f.is_signed && f.subnormals && f.ebits == 5 && f.mbits == 2 && f.bias == 15 && f.special == 0) elem = E8_E5M2;
  else if (f.kind == 1 && f.bits == 8 && f.is_signed && f.symmetric && f.frac_bits == 0) elem = E8_INT8;
  else return no("elements must be fp8_e4m3, fp8_e5m2 or int8");
  if (spec->rounding != TC_RNE || !spec->saturate) return no("elements are rounded to nearest even, saturating");
  if (!spec->has_scale || spec->two_level || spec->zero_point) return no("one level of scales and no zero point");
  const tc_format &sf = spec->scale_format;
  const bool e8m0 = sf.kind == 2 && sf.ebits == 8 && sf.bias == 127 && spec->scale_method == M_POW2_FLOOR;
  const bool fp32 = sf.kind == 0 && sf.ebits == 8 && sf.mbits == 23 && spec->scale_method == M_ABSMAX;
  if ((!e8m0 && !fp32) || spec->scale_rounding != TC_RNE) return no("scales must be fp32 absmax or E8M0 pow2_floor");
  norm::Args a;
  if (spec->granularity == GRAN_ROW) a.group = 0;
  else if (spec->granularity == GRAN_GROUP && spec->group_size > 0) a.group = spec->group_size;
  else return no("scales are per row or per group");
  if (a.group == 0 || (int64_t)a.group > K) {
    if (K > 0x7FFFFFFFll) return bad("rows and K out of range");
    a.group = (int)K;
  }
  a.groups = (K + a.group - 1) / a.group;
  a.group_shift = 0;
  while ((1 << a.group_shift) < a.group && a.group_shift < 30) ++a.group_shift;
  a.x = x;
  a.res = residual;
  a.w = weight;
  a.h = residual_out;
  a.codes = static_cast<unsigned char *>(codes);
  a.scale = scale;
  a.rows = rows;
  a.K = K;
  a.x_stride = x_stride;
  a.res_stride = residual_stride;
  a.w_dtype = weight_dtype;
  a.e8m0 = e8m0;
  a.emax = fmt_emax_elem(f);
  a.max_elem = (float)fmt_max_normal(f);
  a.eps = eps;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == TC_F32) norm::launch_f32(a, elem, s);
  else if (dtype == TC_BF16) norm::launch_bf16(a, elem, s);
  else norm::launch_f16(a, elem, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(std::string("tc_rms_norm_quantize: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  return TC_OK;
}
