// Gated activation with an output in 8 bits with scales: what stands between a feed-forward block's two GEMMs.
//   y = act(gate) * up,  codes = cast(y / s), s from amax |y| per row or per group of the row
// in fp32. Activations: silu g / (1 + exp(-g)); gelu g Phi(g), the same value as g (1 + erf(g / sqrt 2)) / 2 without
// its cancellation; gelu_tanh g / (1 + exp(-2 z)), z = sqrt(2 / pi) (g + 0.044715 g**3), which is g (1 + tanh z) / 2; relu.
// (INT8 codes: the forms with erf and tanh, see gate8.)
//
// 8192 rows of 12288 gates and as many ups in fp32, to MXFP8: 143 us, 6.3 TB/s (139 for the bytes; DRAM 76% busy), gelu 153; with a scale
// a row 153, gelu 172; in bf16 106 and 104 (77 for the bytes), gelu 137 and 125, where relu with a scale a row takes 82: activation
// and cast bound it; groups of 128 with fp32 scales 135 (each lane divides for its group's). INT8 with a scale a row 181, in bf16 134
// (gelu 202 and 162: its functions' instructions). 333 rows of 1537 in bf16 3.1 to 3.5 us. Widths
// that no vector divides read single elements: 8192 x 12289 with a scale a row 297 us in bf16, 375 in fp32, MXFP8 160 and 235. Rows beyond
// 16384 with a scale a row are read twice: 3500 x 28672 259 and 399 us, where groups (106 and 142) are as fast as elsewhere.
#pragma once

#include "tc_cast8.cuh"

namespace tc {
namespace gated {

enum { ACT_SILU = 0, ACT_GELU = 1, ACT_GELU_TANH = 2, ACT_RELU = 3 };

struct Args : Cast8 {
  const void *gate, *up;
  int64_t rows, gate_stride, up_stride;
  int act;
};

constexpr int kThreads = 256;

// g / (1 + 2**t), t = -log2(e) times the logistic function's argument. The hardware's exponential and reciprocal are good to 2
// and 1 steps of fp32; t's rounding is |t| half steps of the exponential, at most half a step of g in the result, since
// |t| / (1 + 2**t) stays below 1 where 2**t is large. Both flush what is below 2**-126 to 0: the exponential stands beside 1, and a result
// that loses its factor this way is below 2**-119.
__device__ __forceinline__ float logistic(float g, float t) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(1.0f, exp2_fast(t))));
  return __fmul_rn(g, r);
}

// g Phi(g) = max(g, 0) - |g| Q(|g|), Q the normal distribution's upper tail: no cancellation on either side. Q(a) exp(a**2 / 2) is a
// polynomial of degree 8 in t = 1 / (1 + 0.3 a), as Hastings approximated it (1955), fitted here to the least relative error over
// [0, 14.5] (6e-8); behind that the exponential is 0. In fp32 the result is within 3 half steps of itself plus 2 of g, before the hardware's
// reciprocal and exponential (1 and 2 steps). Infinite gates give Inf and, as 0 * -Inf, NaN. CUDA's erfc took twice the time.
__device__ __forceinline__ float gelu(float g) {
  const float a = g > 20.0f ? 0.0f : fabsf(g);
  float t;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(__fmaf_rn(a, 0.3f, 1.0f)));
  float q = 0.0384073593f;
  q = __fmaf_rn(q, t, -0.169307336f);
  q = __fmaf_rn(q, t, 0.228951558f);
  q = __fmaf_rn(q, t, -0.076839447f);
  q = __fmaf_rn(q, t, 0.142765149f);
  q = __fmaf_rn(q, t, 0.094585903f);
  q = __fmaf_rn(q, t, 0.121945255f);
  q = __fmaf_rn(q, t, 0.119484209f);
  q = __fmaf_rn(q, t, 7.37236223e-06f);
  q = __fmul_rn(q, exp2_fast(__fmul_rn(__fmul_rn(a, a), -0.72134752f)));  // -log2(e) / 2
  return __fmaf_rn(-a, q, fmaxf(g, -0.0f));
}

__device__ __forceinline__ float largest8(const float (&y)[8]) {
  float m = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max_abs(m, y[e]);
  return m;
}

// act(g) * u of eight elements. INT8 codes are whole numbers up to 127, of which the last bits of y move one in some hundred
// thousands: for them (STEPS) y is what the formula gives with every step rounded by itself and CUDA's accurate functions.
template <bool STEPS>
__device__ __forceinline__ void gate8(float (&g)[8], const float (&u)[8], int act) {
  constexpr float kLog2E = 1.44269504f;
  if (STEPS && act == ACT_SILU) {
    if (largest8(g) <= 64.0f) {
      // The quotient by divide_fast, d = 1 + exp(-g) below 2**93. Its reciprocal has to be the correctly rounded one, and one Newton step
      // from the hardware's gives that for every d in [1, 2**94): compared with __frcp_rn for all 2**23 significands at each exponent.
      // The divisions are then those of the formula: a remainder is exact for quotients down to 2**-104 (g / d has multiples of its last
      // place times d's, 2**-149 at least), and gates that small have d = 2, whose half is rounded once.
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = __fadd_rn(1.0f, expf(-g[e]));
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
        r = __fmaf_rn(__fmaf_rn(-d, r, 1.0f), r, r);
        g[e] = divide_fast(g[e], d, r);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = __fdiv_rn(g[e], __fadd_rn(1.0f, expf(-g[e])));
    }
  } else if (STEPS && act == ACT_GELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = __fmul_rn(__fmul_rn(0.5f, g[e]), __fadd_rn(1.0f, erff(__fmul_rn(g[e], 0.70710678f))));
  } else if (STEPS && act == ACT_GELU_TANH) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float z = __fmul_rn(0.79788456f, __fadd_rn(g[e], __fmul_rn(__fmul_rn(__fmul_rn(0.044715f, g[e]), g[e]), g[e])));
      g[e] = __fmul_rn(__fmul_rn(0.5f, g[e]), __fadd_rn(1.0f, tanhf(z)));
    }
  } else if (act == ACT_SILU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = logistic(g[e], __fmul_rn(g[e], -kLog2E));
  } else if (act == ACT_GELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = gelu(g[e]);
  } else if (act == ACT_GELU_TANH) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float z = __fmul_rn(0.79788456f, __fmaf_rn(__fmul_rn(__fmul_rn(0.044715f, g[e]), g[e]), g[e], g[e]));
      g[e] = logistic(g[e], __fmul_rn(z, -2.0f * kLog2E));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(g[e]));
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) g[e] = __fmul_rn(g[e], u[e]);
}

// Eight codes; values beyond the format's largest need encode8's clamp: only a power-of-two scale leaves them.
template <int E, bool POW2>
__device__ __forceinline__ uint2 encode_all(const float (&y)[8], const Scale &sc) {
  uint32_t q[4];
  if (sc.fast && !(POW2 && E == E8_INT8)) {
    auto quotient = [&](float v) { return POW2 ? __fmul_rn(v, sc.r) : divide_fast(v, sc.s, sc.r); };
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = encode8x2<E>(quotient(y[2 * k]), quotient(y[2 * k + 1]));
  } else {
    auto slow = [&](float v) { return encode8<E>(POW2 ? __fmul_rn(v, sc.r) : __fdiv_rn(v, sc.s)); };
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = slow(y[2 * k]) | (slow(y[2 * k + 1]) << 8);
  }
  return make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
}

// Eight neighbouring elements from c on, zeros behind the row.
template <typename T, bool VEC>
__device__ __forceinline__ void fetch8(const T *p, int64_t c, int64_t K, float (&v)[8]) {
  if (VEC) {
    if (c < K) load8(p + c, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < K) v[e] = Io<T>::get(p[c + e]);
  }
}
template <bool VEC>
__device__ __forceinline__ void put8(unsigned char *p, int64_t c, int64_t K, uint2 q) {
  if (VEC) {
    if (c < K) *reinterpret_cast<uint2 *>(p + c) = q;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < K) p[c + e] = (unsigned char)((e < 4 ? q.x : q.y) >> (8 * (e & 3)));
  }
}

// Groups of 16 to 256 elements, a power of two: 2 to 32 lanes of 8 elements each, and nothing is shared beyond them. Threads walk over
// the matrix with every row filled up to whole groups (`width` vectors), so a group's lanes are neighbours in a warp.
template <typename T, int E, bool VEC, bool POW2>
__global__ void __launch_bounds__(kThreads) group_kernel(Args a, int64_t width) {
  const int64_t step = (int64_t)gridDim.x * kThreads, start = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t rows_a_step = step / width, rest = step - rows_a_step * width;
  int64_t r = start / width, v = start - r * width;
  constexpr bool AHEAD = VEC && sizeof(T) == 2;  // as in held_kernel
  uint4 next[2];
  auto ahead = [&](int64_t r, int64_t c) {
    if constexpr (AHEAD) {
      next[0] = next[1] = make_uint4(0u, 0u, 0u, 0u);
      if (r < a.rows && c < a.K) {
        next[0] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.gate) + r * a.gate_stride + c);
        next[1] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.up) + r * a.up_stride + c);
      }
    }
  };
  ahead(r, v * 8);
  // A warp's lanes go on together: some may be behind the last row.
  for (int64_t base = start - (threadIdx.x & 31); base < a.rows * width; base += step) {
    const bool real = r < a.rows;
    const int64_t c = v * 8, row = r;
    float y[8], u[8];
    if constexpr (AHEAD) {
      widen8<T>(next[0], y);
      widen8<T>(next[1], u);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = u[e] = 0.0f;
      if (real) {
        fetch8<T, VEC>(static_cast<const T *>(a.gate) + r * a.gate_stride, c, a.K, y);
        fetch8<T, VEC>(static_cast<const T *>(a.up) + r * a.up_stride, c, a.K, u);
      }
    }
    r += rows_a_step;
    v += rest;
    if (v >= width) v -= width, ++r;
    ahead(r, v * 8);
    gate8<E == E8_INT8>(y, u, a.act);
    uint32_t top = abs_bits(largest8(y));
    for (int k = a.group >> 4; k; k >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, k));
    const Scale sc = make_scale<POW2>(top, a);
    if (real && c < a.K) {
      if ((c & (a.group - 1)) == 0) store_scale<POW2>(a, row * a.groups + (c >> a.group_shift), sc);
      put8<VEC>(a.codes + row * a.K, c, a.K, encode_all<E, POW2>(y, sc));
    }
  }
}

// One scale a row, which a block's registers hold: NV vectors of 8 neighbouring elements a thread. Vectors of 16-bit elements are small
// enough to hold the next row's too: its loads are under way while this row's maximum is agreed on and its codes are written.
template <typename T, int E, int NV, bool VEC, bool POW2>
__global__ void __launch_bounds__(1024) held_kernel(Args a) {
  constexpr bool AHEAD = VEC && sizeof(T) == 2;
  __shared__ uint32_t tops[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warps = blockDim.x >> 5, threads = blockDim.x;
  int flip = 0;  // the two halves of the exchange buffer alternate, so one barrier a row suffices
  uint4 next[AHEAD ? NV : 1][2];
  auto ahead = [&](int64_t r) {
    if constexpr (AHEAD) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int64_t c = (int64_t)(tid + i * threads) * 8;
        next[i][0] = next[i][1] = make_uint4(0u, 0u, 0u, 0u);
        if (r < a.rows && c < a.K) {
          next[i][0] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.gate) + r * a.gate_stride + c);
          next[i][1] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.up) + r * a.up_stride + c);
        }
      }
    }
  };
  ahead(blockIdx.x);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, flip ^= 1) {
    float y[NV][8], u[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (AHEAD) {
        widen8<T>(next[i][0], y[i]);
        widen8<T>(next[i][1], u[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = u[i][e] = 0.0f;
        const int64_t c = (int64_t)(tid + i * threads) * 8;
        fetch8<T, VEC>(static_cast<const T *>(a.gate) + r * a.gate_stride, c, a.K, y[i]);
        fetch8<T, VEC>(static_cast<const T *>(a.up) + r * a.up_stride, c, a.K, u[i]);
      }
    }
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      gate8<E == E8_INT8>(y[i], u[i], a.act);
      m = max_abs(m, largest8(y[i]));
    }
    ahead(r + gridDim.x);
    const uint32_t top = warp_max(abs_bits(m));
    if (lane == 0) tops[flip][tid >> 5] = top;
    __syncthreads();
    const Scale sc = make_scale<POW2>(warp_max(lane < warps ? tops[flip][lane] : 0u), a);
    if (tid == 0) store_scale<POW2>(a, r, sc);
#pragma unroll
    for (int i = 0; i < NV; ++i) put8<VEC>(a.codes + r * a.K, (int64_t)(tid + i * threads) * 8, a.K, encode_all<E, POW2>(y[i], sc));
  }
}

// One block a row, any length, alignment and group: the row is read once per group for its maximum and again for its
// codes (from L1 / L2). A warp takes a group; row scales have one group, which the block shares.
template <typename T, int E>
__global__ void __launch_bounds__(kThreads) row_kernel(Args a) {
  __shared__ uint32_t top;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T *gate = static_cast<const T *>(a.gate) + r * a.gate_stride, *up = static_cast<const T *>(a.up) + r * a.up_stride;
    const bool shared_group = a.groups == 1;
    if (threadIdx.x == 0) top = 0u;
    __syncthreads();
    const int64_t step = shared_group ? 8 * kThreads : 256;
    for (int64_t g = shared_group ? 0 : warp; g < a.groups; g += shared_group ? 1 : kThreads / 32) {
      const int64_t lo = g * a.group, hi = min(lo + (int64_t)a.group, a.K);
      const int64_t first = lo + 8 * (shared_group ? threadIdx.x : lane);
      auto y_at = [&](int64_t c, float (&y)[8]) {
        float u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = u[e] = 0.0f;
        fetch8<T, false>(gate, c, hi, y);
        fetch8<T, false>(up, c, hi, u);
        gate8<E == E8_INT8>(y, u, a.act);
      };
      float y[8];
      uint32_t m = 0u;
      for (int64_t c = first; c < hi; c += step) {
        y_at(c, y);
        m = max(m, abs_bits(largest8(y)));
      }
      m = warp_max(m);
      if (shared_group) {
        if (lane == 0) atomicMax(&top, m);
        __syncthreads();
        m = top;
      }
      const Scale p = make_scale<true>(m, a), s = make_scale<false>(m, a);
      if (first == lo) a.e8m0 ? store_scale<true>(a, r * a.groups + g, p) : store_scale<false>(a, r * a.groups + g, s);
      for (int64_t c = first; c < hi; c += step) {
        y_at(c, y);
        put8<false>(a.codes + r * a.K, c, hi, a.e8m0 ? encode_all<E, true>(y, p) : encode_all<E, false>(y, s));
      }
    }
    __syncthreads();
  }
}

template <typename T, int E, bool VEC, bool POW2>
static void launch_scale(const Args &a, bool lanes, cudaStream_t s) {
  if (lanes) {
    const int64_t width = a.groups * (a.group / 8), blocks = (a.rows * width + kThreads - 1) / kThreads, most = (int64_t)sm_count() * 8;
    group_kernel<T, E, VEC, POW2><<<(unsigned)(blocks < most ? blocks : most), kThreads, 0, s>>>(a, width);
  } else {
    const int64_t vectors = (a.K + 7) / 8;
    // One vector a thread up to 512, two beyond; whole warps, so that at most one of them is partly idle.
    const int threads = (int)(((vectors <= 512 ? vectors : (vectors + 1) / 2) + 31) / 32 * 32);
    const int64_t most = (int64_t)sm_count() * (2048 / threads);
    const unsigned grid = (unsigned)(a.rows < most ? a.rows : most);
    if (vectors <= 512) held_kernel<T, E, 1, VEC, POW2><<<grid, threads, 0, s>>>(a);
    else held_kernel<T, E, 2, VEC, POW2><<<grid, threads, 0, s>>>(a);
  }
  count_launch();
}

template <typename T, int E>
static void launch_elem(const Args &a, cudaStream_t s) {
  auto aligned = [](const void *p, size_t n) { return (uintptr_t)p % n == 0; };
  const bool vec = a.K % 8 == 0 && a.gate_stride % 8 == 0 && a.up_stride % 8 == 0 && aligned(a.gate, 16) && aligned(a.up, 16) &&
                   aligned(a.codes, 8);
  const bool lanes = a.groups > 1 && a.group >= 16 && a.group <= 256 && (a.group & (a.group - 1)) == 0;
  if (lanes || (a.groups == 1 && a.K <= 16384)) {
    if (vec) a.e8m0 ? launch_scale<T, E, true, true>(a, lanes, s) : launch_scale<T, E, true, false>(a, lanes, s);
    else a.e8m0 ? launch_scale<T, E, false, true>(a, lanes, s) : launch_scale<T, E, false, false>(a, lanes, s);
  } else {
    const int64_t most = (int64_t)sm_count() * 8;
    row_kernel<T, E><<<(unsigned)(a.rows < most ? a.rows : most), kThreads, 0, s>>>(a);
    count_launch();
  }
}

template <typename T>
static void launch(const Args &a, int elem, cudaStream_t s) {
  if (elem == E8_E4M3) launch_elem<T, E8_E4M3>(a, s);
  else if (elem == E8_E5M2) launch_elem<T, E8_E5M2>(a, s);
  else launch_elem<T, E8_INT8>(a, s);
}

}  // namespace gated
}  // namespace tc
