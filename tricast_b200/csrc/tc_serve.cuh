// Shared device code of the serving operators (norm to 8 bits, paged cache, attention over it): 8- and
// 4-bit element encodings and their scales, with the results of the quantize kernels (tc_quant.cuh) bit
// for bit, NaN encodings of E5M2 aside (0x7F here).
#pragma once

#include <cuda_fp8.h>

#include "tc_common.cuh"

namespace tc {

enum { E8_E4M3 = 0, E8_E5M2 = 1, E8_INT8 = 2 };

// Magnitude maximum as bits: NaN sorts above Inf above every number, so a plain integer maximum
// propagates NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return f2u(v) & 0x7FFFFFFFu; }

// Group and row maxima are exact, so every warp or block order gives the same scale.
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xFFFFFFFFu, v); }

// absmax scale in fp32: RN(amax / max), the smallest fp32 where that is 0, the largest where amax is
// infinite, NaN where it is NaN, and 1 for an all-zero domain (amax_scale of tc_quant.cuh for an fp32 scale
// format).
__device__ __forceinline__ float absmax_scale(uint32_t amax_bits, float max_elem) {
  const float amax = u2f(amax_bits);
  const float s = __fdiv_rn(amax, max_elem);
  if (amax_bits == 0u) return 1.0f;
  if (amax_bits == kInf) return u2f(kInf - 1u);
  return s == 0.0f ? u2f(1u) : s;
}

// E8M0 code of 2**(floor(log2 amax) - emax), clamped to 2**-127 below; 0xFF (NaN) where amax is not
// finite. Subnormal and zero maxima lie below the clamp for every emax >= 1, so the exponent field alone
// decides.
__device__ __forceinline__ uint32_t pow2_code(uint32_t amax_bits, int emax) {
  if (amax_bits >= kInf) return 0xFFu;
  return (uint32_t)max((int)(amax_bits >> 23) - emax, 0);
}
// 2**(code - 127) and its reciprocal, both exact (2**-127 is an fp32 subnormal); NaN for 0xFF.
__device__ __forceinline__ float pow2_value(uint32_t code) {
  return code == 0xFFu ? u2f(kQNaN) : code == 0u ? u2f(0x00400000u) : u2f(code << 23);
}
__device__ __forceinline__ float pow2_inverse(uint32_t code) {
  return code == 0xFFu ? u2f(kQNaN) : code == 254u ? u2f(0x00400000u) : u2f((254u - code) << 23);
}

// 8-bit codes of a value already divided by its scale: round to nearest even, saturating.
template <int E>
__device__ __forceinline__ uint32_t encode8(float v) {
  if (E == E8_E4M3) return (uint32_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
  if (E == E8_E5M2) return (uint32_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E5M2);
  const float c = fminf(fmaxf(rintf(v), -127.0f), 127.0f);
  return v != v ? 0u : (uint32_t)(int)c & 0xFFu;
}

// 4-bit E2M1 code, ties to the even code, saturating at 6. NaN takes code 0 (its group's scale is NaN).
__device__ __forceinline__ uint32_t encode_e2m1(float v) {
  const float a = fabsf(v);
  uint32_t c = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
  return v != v ? 0u : c | ((f2u(v) >> 31) << 3);
}

// Value of an E2M1 code: exponent field 0 is the subnormal half step, the rest 2**(e - 1) * (1 + m / 2).
__device__ __forceinline__ float decode_e2m1(uint32_t c) {
  const uint32_t m = c & 7u;
  const float a = m < 2u ? 0.5f * (float)m : u2f((((m >> 1) + 126u) << 23) | ((m & 1u) << 22));
  return (c & 8u) ? -a : a;
}

__device__ __forceinline__ float decode_e4m3(uint32_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
}

// RN(x / s) for finite x without a division: with r = RN(1 / s) a quotient within an ulp or two is corrected
// twice by its exact remainder (Markstein's theorem: the second step rounds correctly. With s in [1, 2): r is off by 2**-25 at most, the
// first step's quotient by (1 + 2**-21) / 2 steps of its last place, so the second's sum by s (1 + 2**-21) 2**-26 steps; no quotient that is
// not a midpoint lies nearer to one than 2**-24 / s steps, which is more for s**2 (1 + 2**-21) < 4. The 2000 largest s, all that are not below
// that among them, were compared with the division for every x). s in
// [2**-100, 2**100]; quotients below 2**-60, which every format here rounds to 0, may lose bits. The remainder is taken
// negated: of q = x = -0 it is +0, and -0 * r + q keeps the sign.
__device__ __forceinline__ bool divides_fast(float s) { return s >= 7.888609052210118e-31f && s <= 1.2676506002282294e30f; }
__device__ __forceinline__ float divide_fast(float x, float s, float r) {
  float q = __fmul_rn(x, r);
  q = __fmaf_rn(-__fmaf_rn(q, s, -x), r, q);
  return __fmaf_rn(-__fmaf_rn(q, s, -x), r, q);
}

// Codes of two values of magnitude at most a hair above the format's largest (finite): low byte first.
template <int E>
__device__ __forceinline__ uint32_t encode8x2(float a, float b) {
  if (E == E8_INT8)  // the integer in the low bits of a + 1.5 * 2**23, rounded to nearest even by the addition
    return __byte_perm(f2u(__fadd_rn(a, 12582912.0f)), f2u(__fadd_rn(b, 12582912.0f)), 0x0040) & 0xFFFFu;
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, E == E8_E4M3 ? __NV_E4M3 : __NV_E5M2);
}

template <typename T>
struct Io;
template <>
struct Io<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Io<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Io<__half> {
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};

// Paged cache schemes (tc_kv_scheme).
enum { KV_NONE = 0, KV_FP8_ROW = 1, KV_INT8_ROW = 2, KV_MXFP4 = 3 };

struct KvCache {
  unsigned char *k, *v;    // [pages][kv_heads][page_size] rows of row_bytes
  unsigned char *ks, *vs;  // fp32 per row, or head_dim / 32 E8M0 bytes per row, or nullptr
  int64_t pages;
  int page_size, page_shift, heads, dim, row_bytes;
  int scheme, dtype;
  int scale_bytes;         // bytes of one row's scales
};

int kv_cache_check(const tc_kv_cache *c, KvCache &out);  // a tc_status; derives the layout

}  // namespace tc
