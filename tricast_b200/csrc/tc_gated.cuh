// Gated activation with an output in 8 bits with scales: what stands between a feed-forward block's two GEMMs.
//   y = act(gate) * up,  codes = cast(y / s), s from amax |y| per row or per group of the row
// in fp32. Activations: silu g / (1 + exp(-g)); gelu g * erfc(-g / sqrt 2) / 2, the same value as g (1 + erf) / 2 without
// its cancellation; gelu_tanh g / (1 + exp(-2 z)), z = sqrt(2 / pi) (g + 0.044715 g**3), which is g (1 + tanh z) / 2; relu.
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

__device__ __forceinline__ float activate(float g, int act) {
  if (act == ACT_SILU) return __fdiv_rn(g, __fadd_rn(1.0f, expf(-g)));
  if (act == ACT_GELU) return __fmul_rn(__fmul_rn(0.5f, g), erfcf(__fmul_rn(g, -0.70710678f)));
  if (act == ACT_GELU_TANH) {
    const float z = __fmul_rn(0.79788456f, __fmaf_rn(__fmul_rn(__fmul_rn(0.044715f, g), g), g, g));
    return __fdiv_rn(g, __fadd_rn(1.0f, expf(__fmul_rn(-2.0f, z))));
  }
  return g > 0.0f ? g : g != g ? g : 0.0f;
}

// One block a row, any length, alignment and group: the row is read once per group for its maximum and again for its
// codes (from L1 / L2). A warp takes a group; row scales have one group, which the block shares.
template <typename T, int E>
__global__ void __launch_bounds__(kThreads) row_kernel(Args a) {
  __shared__ uint32_t top;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T *gate = static_cast<const T *>(a.gate) + r * a.gate_stride, *up = static_cast<const T *>(a.up) + r * a.up_stride;
    auto y_at = [&](int64_t c) { return __fmul_rn(activate(Io<T>::get(gate[c]), a.act), Io<T>::get(up[c])); };
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
    __syncthreads();
  }
}

template <typename T, int E>
static void launch_elem(const Args &a, cudaStream_t s) {
  const int64_t most = (int64_t)sm_count() * 8;
  row_kernel<T, E><<<(unsigned)(a.rows < most ? a.rows : most), kThreads, 0, s>>>(a);
  count_launch();
}

template <typename T>
static void launch(const Args &a, int elem, cudaStream_t s) {
  if (elem == E8_E4M3) launch_elem<T, E8_E4M3>(a, s);
  else if (elem == E8_E5M2) launch_elem<T, E8_E5M2>(a, s);
  else launch_elem<T, E8_INT8>(a, s);
}

}  // namespace gated
}  // namespace tc
