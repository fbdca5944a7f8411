// What the operators that end in 8-bit codes with scales (the norm, the gated activation) share: the specs they take,
// rows of a matrix eight elements at a time, and a scale from its domain's largest magnitude.
#pragma once

#include <cmath>
#include <string>

#include "tc_mma16.cuh"
#include "tc_quant.cuh"
#include "tc_serve.cuh"

namespace tc {

// An 8-bit output [rows][K] with a scale per row or per group of the row.
struct Cast8 {
  unsigned char *codes;
  void *scale;          // fp32, or E8M0 bytes
  int64_t K;
  int group;            // elements that share a scale (K for row scales)
  int group_shift;      // its logarithm where it is a power of two
  int64_t groups;       // per row
  int e8m0, emax;
  float max_elem;
};

// Fills in all but the pointers for rows of K elements, and which element format it is; a tc_status.
inline int cast8_spec(const tc_quant_spec *spec, int64_t K, const char *what, int &elem, Cast8 &a) {
  auto bad = [&](const char *m) { return set_error(std::string(what) + ": " + m), (int)TC_INVALID_ARGUMENT; };
  auto no = [&](const char *m) { return set_error(std::string(what) + ": " + m), (int)TC_UNSUPPORTED; };
  const tc_format &f = spec->format;
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
  a.K = K;
  a.e8m0 = e8m0;
  a.emax = fmt_emax_elem(f);
  a.max_elem = (float)fmt_max_normal(f);
  return TC_OK;
}

// Eight 16-bit elements as fp32.
template <typename T>
__device__ __forceinline__ void widen8(uint4 w, float (&v)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (Same<T, __nv_bfloat16>::value) {
      v[2 * k] = u2f(u[k] << 16);
      v[2 * k + 1] = u2f(u[k] & 0xFFFF0000u);
    } else {
      v[2 * k] = __half2float(__ushort_as_half((unsigned short)(u[k] & 0xFFFFu)));
      v[2 * k + 1] = __half2float(__ushort_as_half((unsigned short)(u[k] >> 16)));
    }
  }
}
// Eight elements as fp32, from 16-bit or fp32 memory at a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    widen8<T>(*reinterpret_cast<const uint4 *>(p), v);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack16<T>(v[0], v[1]), pack16<T>(v[2], v[3]), pack16<T>(v[4], v[5]), pack16<T>(v[6], v[7]));
  }
}

// max(m, |v|), NaN if either is.
__device__ __forceinline__ float max_abs(float m, float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
  return r;
}

// A scale from its domain's largest magnitude: what values are multiplied by (POW2) or divided by.
struct Scale {
  float s, r;   // the scale (absmax) and a reciprocal
  bool fast;    // finite, and divide_fast holds
  uint32_t code;
};
template <bool POW2>
__device__ __forceinline__ Scale make_scale(uint32_t top, const Cast8 &a) {
  Scale c;
  if (POW2) {
    c.code = pow2_code(top, a.emax);
    c.r = pow2_inverse(c.code);
    c.s = 0.0f;
    c.fast = c.code != 0xFFu;
  } else {
    c.s = absmax_scale(top, a.max_elem);
    c.fast = divides_fast(c.s);
    c.r = __frcp_rn(c.s);
    c.code = 0u;
  }
  return c;
}
template <bool POW2>
__device__ __forceinline__ void store_scale(const Cast8 &a, int64_t at, const Scale &c) {
  if (POW2) static_cast<unsigned char *>(a.scale)[at] = (unsigned char)c.code;
  else static_cast<float *>(a.scale)[at] = c.s;
}

}  // namespace tc
