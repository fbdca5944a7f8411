// Low-rank adapters of many requests beside a shared projection:
//   out[t] = y[t] + gain[i] * B[i] (A[i] x[t]),  i = index[t]  (out[t] = y[t] where i names no adapter)
// x in 16 or 32 bits, or 8-bit codes with a scale a row; the products and their sum are fp32, out is rounded once.
#pragma once

#include "tc_mma16.cuh"
#include "tc_serve.cuh"

namespace tc {
namespace adapt {

// What x holds: a tc_dtype, or codes with scales.
enum { X_F32 = TC_F32, X_BF16 = TC_BF16, X_F16 = TC_F16, X_E4M3 = 3, X_E5M2 = 4, X_INT8 = 5 };

struct Args {
  const void *y, *x, *a, *b;  // y [tokens][n], x [tokens][k] with row strides; a [adapters][rank][k], b [adapters][n][rank]
  const float *x_scale, *gain;
  const int32_t *index;
  void *out;  // [tokens][n]
  int64_t tokens, k, n, y_stride, x_stride;
  int rank, adapters, y_dtype, x_kind, w_dtype, out_dtype;
};

__device__ __forceinline__ float x_at(const Args &a, int64_t i) {
  if (a.x_kind <= X_F16) return load_as_float(a.x, a.x_kind, i);
  const uint32_t c = static_cast<const unsigned char *>(a.x)[i];
  if (a.x_kind == X_INT8) return (float)(int8_t)c;
  return a.x_kind == X_E4M3 ? decode_e4m3(c) : __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E5M2)));
}

__device__ __forceinline__ void store_rounded(void *p, int dtype, int64_t i, float v) {
  if (dtype == TC_F32) static_cast<float *>(p)[i] = v;
  else if (dtype == TC_BF16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half *>(p)[i] = __float2half_rn(v);
}

}  // namespace adapt
}  // namespace tc
