// m16n8k16 tensor-core steps on 16-bit operands in registers, conversions of cached codes to fp16 pairs,
// and small power-of-two helpers of the attention kernels.
#pragma once

#include <cuda_fp8.h>

#include "tc_bulk.cuh"
#include "tc_common.cuh"

namespace tc {

template <typename A, typename B>
struct Same {
  static constexpr bool value = false;
};
template <typename A>
struct Same<A, A> {
  static constexpr bool value = true;
};

// Asynchronous copies that write zeros instead where `use` is false (the source is then not read).
__device__ __forceinline__ void cp_async16_or_zero(void *dst, const void *src, bool use) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(use ? 16u : 0u)
               : "memory");
}
__device__ __forceinline__ void cp_async4_or_zero(void *dst, const void *src, bool use) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(use ? 4u : 0u)
               : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// d += a * b, fp32 accumulation: a 16 x 16 (row), b 16 x 8 (column); fp16 or bf16 operands.
template <bool BF16>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 2**x to 2 ulp; 0 for -Inf and results below the normal range.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The same down to 2**-149.
__device__ __forceinline__ float exp2_wide(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Four codes to two pairs of fp16 values, exactly; the low code to the low half of the first.
__device__ __forceinline__ void e4m3x4_half2(uint32_t w, uint32_t &lo, uint32_t &hi) {
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
// Eight codes (code 0 in the low nibble) to four pairs.
__device__ __forceinline__ void e2m1x8_half2(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, a;\ncvt.rn.f16x2.e2m1x2 %1, b;\ncvt.rn.f16x2.e2m1x2 %2, c;\ncvt.rn.f16x2.e2m1x2 %3, d;\n}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// Bytes v + 128 picked by SEL from (bytes, 0x64 in every byte): fp16 1024 + (v + 128), less 1152.
template <int SEL>
__device__ __forceinline__ uint32_t int8x2_half2(uint32_t biased) {
  uint32_t r;
  asm("{\n.reg .b32 t;\nprmt.b32 t, %1, 0x64646464, %2;\nadd.rn.f16x2 %0, t, %3;\n}"
      : "=r"(r)
      : "r"(biased), "n"(SEL), "r"(0xE480E480u));  // -1152, -1152
  return r;
}

template <typename T>
__device__ __forceinline__ float half_bits_to_float(uint32_t h);
template <>
__device__ __forceinline__ float half_bits_to_float<__nv_bfloat16>(uint32_t h) {
  return u2f(h << 16);
}
template <>
__device__ __forceinline__ float half_bits_to_float<__half>(uint32_t h) {
  return __half2float(__ushort_as_half((unsigned short)h));
}
template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  return Same<T, __nv_bfloat16>::value ? pack_bf16(lo, hi) : pack_half(lo, hi);
}

// A power of two and its reciprocal that bring a row whose largest magnitude is `top` into
// [2**13, 2**14), so that fp16 holds it: elements down to 2**-27 of the largest keep 11 bits. Rows that are
// zero or not finite keep their scale.
struct Pow2 {
  float factor, inverse;
};
__device__ __forceinline__ Pow2 fp16_shift(float top) {
  const int field = (int)(f2u(top) >> 23);
  if (field == 0 || field == 255) return Pow2{1.0f, 1.0f};
  const int e = min(max(127 + 13 + 127 - field, 1), 253);  // field of 2**(13 - (field - 127))
  return Pow2{u2f((uint32_t)e << 23), u2f((uint32_t)(254 - e) << 23)};
}

// fp16 bits of 2**d, 0 below its subnormals (d <= 15).
__device__ __forceinline__ uint32_t half_pow2(int d) {
  return d >= -14 ? (uint32_t)(15 + d) << 10 : d >= -24 ? 1u << (24 + d) : 0u;
}

// E2M1 codes carry their group's scale relative to the row's largest, times 2**12: groups down to 2**-26 of
// the largest stay exact, and 6 * 2**12 fits fp16.
constexpr int kGroupShift = 12;

template <int N>
__device__ __forceinline__ void load_words(const unsigned char *src, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4 *>(src);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(src);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t *>(src);
  }
}

}  // namespace tc
