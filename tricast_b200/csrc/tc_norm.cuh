// Root-mean-square norm with the residual's addition and an output in 8 bits with scales:
//   h = x + residual,  y = h / sqrt(mean(h**2) + eps) * weight,  codes = cast(y / s), s from amax |y|
// per row or per group of the row. h and y stay in fp32; h is rounded once where it is stored.
#pragma once

#include "tc_cast8.cuh"

namespace tc {
namespace norm {

struct Args : Cast8 {
  const void *x, *res, *w;
  void *h;
  int64_t rows, x_stride, res_stride;
  int w_dtype;
  float eps;
};

constexpr int kThreads = 256;

__device__ __forceinline__ float block_sum(float v, float *part) {
  for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.0f;
  for (int i = 0; i < kThreads / 32; ++i) t += part[i];
  __syncthreads();
  return t;
}

// One block a row, any length, alignment and group: the row is read once for the sum of squares, and again per
// group for its maximum and its codes (from L1 / L2). A warp takes a group; row scales have one group,
// which the block shares.
template <typename T, int E>
__global__ void __launch_bounds__(kThreads) row_kernel(Args a) {
  __shared__ float part[kThreads / 32];
  __shared__ uint32_t top;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
    const T *res = a.res ? static_cast<const T *>(a.res) + r * a.res_stride : nullptr;
    T *ho = a.h ? static_cast<T *>(a.h) + r * a.K : nullptr;
    auto h_at = [&](int64_t c) {
      const float v = Io<T>::get(x[c]);
      return res ? __fadd_rn(v, Io<T>::get(res[c])) : v;
    };
    float ss = 0.0f;
    for (int64_t c = threadIdx.x; c < a.K; c += kThreads) {
      const float h = h_at(c);
      ss = __fmaf_rn(h, h, ss);
    }
    const float mean = __fdiv_rn(block_sum(ss, part), (float)a.K);
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(mean, a.eps)));
    auto y_at = [&](int64_t c) {
      const float v = __fmul_rn(h_at(c), inv);
      return a.w ? __fmul_rn(v, load_as_float(a.w, a.w_dtype, c)) : v;
    };
    const bool shared_group = a.groups == 1;
    if (threadIdx.x == 0) top = 0u;
    __syncthreads();
    const int64_t step = shared_group ? kThreads : 32;
    for (int64_t g = shared_group ? 0 : warp; g < a.groups; g += shared_group ? 1 : kThreads / 32) {
      const int64_t lo = g * a.group, hi = min(lo + (int64_t)a.group, a.K);
      const int64_t first = lo + (shared_group ? threadIdx.x : lane);
      uint32_t m = 0u;
      for (int64_t c = first; c < hi; c += step) m = max(m, abs_bits(y_at(c)));
      m = warp_max(m);
      if (shared_group) {
        if (lane == 0) atomicMax(&top, m);
        __syncthreads();
        m = top;
      }
      const uint32_t sc = a.e8m0 ? pow2_code(m, a.emax) : 0u;
      const float s = a.e8m0 ? pow2_inverse(sc) : absmax_scale(m, a.max_elem);
      if (first == lo) {
        if (a.e8m0) static_cast<unsigned char *>(a.scale)[r * a.groups + g] = (unsigned char)sc;
        else static_cast<float *>(a.scale)[r * a.groups + g] = s;
      }
      for (int64_t c = first; c < hi; c += step) {
        const float y = y_at(c);
        a.codes[r * a.K + c] = (unsigned char)encode8<E>(a.e8m0 ? __fmul_rn(y, s) : __fdiv_rn(y, s));
      }
    }
    if (ho) {
      // After every read of the row by this block: the caller may pass x or the residual as h.
      __syncthreads();
      for (int64_t c = threadIdx.x; c < a.K; c += kThreads) ho[c] = Io<T>::put(h_at(c));
    }
    __syncthreads();
  }
}

// One block a row that its registers hold, read once and written once. A thread has NV vectors
// of 8 neighbouring elements (VEC 8; vector v of the row is thread v % threads's), or 8 NV single ones where rows
// are not aligned (VEC 1). A group's maximum stays inside a warp: 2 to 32 lanes (VEC 8), or exactly a warp
// (VEC 1, groups of 32); a row's goes through shared memory, like the sum of squares. Aligned 16-bit rows are
// fetched a row ahead, so that HBM works while a row is waited for and encoded. 16384 rows of 8192 bf16 elements and
// as many residuals, to MXFP8: 197 us, 4.8 TB/s, with a scale a row 212 us; 777 of 4093 (single elements) 16 us; one
// of 4096 2.6 us. The large case keeps 70% of issue slots and 55% of DRAM's cycles busy: the cast and the block-wide
// reductions between the loads bound it. Single elements spill (64 to 876 bytes a thread, under the 64 registers of 1024 threads).
template <typename T, int E, int NV, int VEC, bool GROUPED, bool POW2>
__global__ void __launch_bounds__(1024) held_kernel(Args a) {
  constexpr bool kAhead = VEC == 8 && sizeof(T) == 2;
  __shared__ float part[2][32];
  __shared__ uint32_t tops[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warps = blockDim.x >> 5, threads = blockDim.x;
  const int K = (int)a.K;
  // Element of vector i; single ones follow at a distance of a block.
  auto at = [&](int i, int e) { return VEC == 8 ? (tid + i * threads) * 8 : tid + (8 * i + e) * threads; };
  uint4 ahead_x[kAhead ? NV : 1], ahead_r[kAhead ? NV : 1];
  auto fetch = [&](int64_t r) {
    const T *x = static_cast<const T *>(a.x) + r * a.x_stride, *res = static_cast<const T *>(a.res) + r * a.res_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (at(i, 0) < K) {
        ahead_x[kAhead ? i : 0] = *reinterpret_cast<const uint4 *>(x + at(i, 0));
        if (a.res) ahead_r[kAhead ? i : 0] = *reinterpret_cast<const uint4 *>(res + at(i, 0));
      }
  };
  if (kAhead && blockIdx.x < a.rows) fetch(blockIdx.x);
  int flip = 0;  // the two halves of the exchange buffers alternate, so one barrier an exchange suffices
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, flip ^= 1) {
    const T *x = static_cast<const T *>(a.x) + r * a.x_stride, *res = static_cast<const T *>(a.res) + r * a.res_stride;
    float v[NV][8];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = w[e] = 0.0f;
      if (VEC == 8) {
        if (at(i, 0) < K) {
          load8(kAhead ? reinterpret_cast<const T *>(&ahead_x[kAhead ? i : 0]) : x + at(i, 0), v[i]);
          if (a.res) load8(kAhead ? reinterpret_cast<const T *>(&ahead_r[kAhead ? i : 0]) : res + at(i, 0), w);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (at(i, e) < K) {
            v[i][e] = Io<T>::get(x[at(i, e)]);
            if (a.res) w[e] = Io<T>::get(res[at(i, e)]);
          }
      }
      if (a.res)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = __fadd_rn(v[i][e], w[e]);
    }
    if (kAhead && r + gridDim.x < a.rows) fetch(r + gridDim.x);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __fmaf_rn(v[i][e], v[i][e], ss);
#pragma unroll
    for (int m = 16; m; m >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, m);
    if (lane == 0) part[flip][tid >> 5] = ss;
    if (a.h) {  // beside the wait for the other warps
      T *h = static_cast<T *>(a.h) + r * a.K;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (VEC == 8) {
          if (at(i, 0) < K) store8(h + at(i, 0), v[i]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (at(i, e) < K) h[at(i, e)] = Io<T>::put(v[i][e]);
        }
      }
    }
    __syncthreads();
    ss = lane < warps ? part[flip][lane] : 0.0f;
#pragma unroll
    for (int m = 16; m; m >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, m);
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)K), a.eps)));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = 1.0f;
        v[i][e] = __fmul_rn(v[i][e], inv);
      }
      if (a.w) {
        if (VEC == 8) {
          if (at(i, 0) < K) {
            if (a.w_dtype == TC_F32) load8(static_cast<const float *>(a.w) + at(i, 0), w);
            else if (a.w_dtype == TC_BF16) load8(static_cast<const __nv_bfloat16 *>(a.w) + at(i, 0), w);
            else load8(static_cast<const __half *>(a.w) + at(i, 0), w);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (at(i, e) < K) w[e] = load_as_float(a.w, a.w_dtype, at(i, e));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = __fmul_rn(v[i][e], w[e]);
      }
    }
    Scale sc;
    if (!GROUPED) {
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max_abs(m, v[i][e]);
      const uint32_t top = warp_max(abs_bits(m));
      if (lane == 0) tops[flip][tid >> 5] = top;
      __syncthreads();
      sc = make_scale<POW2>(warp_max(lane < warps ? tops[flip][lane] : 0u), a);
      if (tid == 0) store_scale<POW2>(a, r, sc);
    }
    // Values beyond the format's largest need encode8's clamp: only a power-of-two scale leaves them.
    auto quotient = [&](float y) { return POW2 ? __fmul_rn(y, sc.r) : divide_fast(y, sc.s, sc.r); };
    auto slow = [&](float y) { return encode8<E>(POW2 ? __fmul_rn(y, sc.r) : __fdiv_rn(y, sc.s)); };
    unsigned char *codes = a.codes + r * a.K;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (VEC == 8) {
        const int c = at(i, 0);
        if (GROUPED) {
          float m = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) m = max_abs(m, v[i][e]);
          uint32_t top = abs_bits(m);
          for (int k = a.group >> 4; k; k >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, k));
          sc = make_scale<POW2>(top, a);
          if (c < K && (c & (a.group - 1)) == 0) store_scale<POW2>(a, r * a.groups + (c >> a.group_shift), sc);
        }
        uint32_t q[4];
        if (sc.fast && !(POW2 && E == E8_INT8)) {
#pragma unroll
          for (int k = 0; k < 4; ++k) q[k] = encode8x2<E>(quotient(v[i][2 * k]), quotient(v[i][2 * k + 1]));
        } else {
#pragma unroll 1
          for (int k = 0; k < 4; ++k) q[k] = 0u;
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e >> 1] |= slow(v[i][e]) << (8 * (e & 1));
        }
        if (c < K) *reinterpret_cast<uint2 *>(codes + c) = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = at(i, e);
          if (GROUPED) {  // groups of 32: a warp's elements
            sc = make_scale<POW2>(warp_max(abs_bits(v[i][e])), a);
            if (lane == 0 && c < K) store_scale<POW2>(a, r * a.groups + (c >> 5), sc);
          }
          const uint32_t q = sc.fast && !(POW2 && E == E8_INT8) ? encode8x2<E>(quotient(v[i][e]), 0.0f) : slow(v[i][e]);
          if (c < K) codes[c] = (unsigned char)q;
        }
      }
    }
  }
}

template <typename T, int E, int VEC, bool GROUPED, bool POW2>
static void launch_held(const Args &a, cudaStream_t s) {
  // A vector a thread while that makes 512 of them, then two: short rows spread over more SMs' latency, long
  // ones keep more bytes in flight a thread. 16384 rows of 8192 (bf16, residual, scale a row): 512 threads of two
  // vectors 212 us, 1024 of one 233; one row of 4096: 512 of one 2.7 us, 256 of two 3.3 (16384 rows 110 and 105).
  const int64_t vectors = (a.K + 7) / 8;
  int threads = 64;
  while (threads < 512 && threads < vectors) threads *= 2;
  while (threads < 1024 && threads * 2 < vectors) threads *= 2;
  const int64_t most = (int64_t)sm_count() * (2048 / threads);
  const unsigned grid = (unsigned)(a.rows < most ? a.rows : most);
  if (vectors <= threads) held_kernel<T, E, 1, VEC, GROUPED, POW2><<<grid, threads, 0, s>>>(a);
  else held_kernel<T, E, 2, VEC, GROUPED, POW2><<<grid, threads, 0, s>>>(a);
  count_launch();
}

template <typename T, int E, int VEC>
static void launch_mode(const Args &a, cudaStream_t s) {
  if (a.groups == 1) a.e8m0 ? launch_held<T, E, VEC, false, true>(a, s) : launch_held<T, E, VEC, false, false>(a, s);
  else a.e8m0 ? launch_held<T, E, VEC, true, true>(a, s) : launch_held<T, E, VEC, true, false>(a, s);
}

template <typename T, int E>
static void launch_elem(const Args &a, cudaStream_t s) {
  auto aligned = [](const void *p, size_t n) { return (uintptr_t)p % n == 0; };
  const bool vec = a.K % 8 == 0 && a.x_stride % 8 == 0 && (!a.res || a.res_stride % 8 == 0) && aligned(a.x, 16) &&
                   aligned(a.res, 16) && aligned(a.w, 16) && aligned(a.h, 16) && aligned(a.codes, 8);
  const bool lanes = a.group >= 16 && a.group <= 256 && (a.group & (a.group - 1)) == 0;
  if (vec && a.K <= 16384 && (a.groups == 1 || lanes)) {
    launch_mode<T, E, 8>(a, s);
  } else if (a.K <= 16384 && (a.groups == 1 || a.group == 32)) {
    launch_mode<T, E, 1>(a, s);
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

}  // namespace norm
}  // namespace tc
