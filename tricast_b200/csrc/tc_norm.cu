// Root-mean-square norm with the residual's addition and an output in 8 bits with scales:
//   h = x + residual,  y = h / sqrt(mean(h**2) + eps) * weight,  codes = cast(y / s), s from amax |y|
// per row or per group of the row. h and y stay in fp32; h is rounded once where it is stored.
#include <cmath>
#include <string>

#include "tc_quant.cuh"
#include "tc_serve.cuh"

namespace tc {
namespace norm {

struct Args {
  const void *x, *res, *w;
  void *h;
  unsigned char *codes;
  void *scale;          // fp32, or E8M0 bytes
  int64_t rows, K, x_stride, res_stride;
  int group;            // elements that share a scale (K for row scales)
  int64_t groups;       // per row
  int w_dtype;
  int e8m0, emax;
  float max_elem, eps;
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

// One block a row, any length and alignment: the row is read once for the sum of squares, and again per
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

template <typename T>
static void launch(const Args &a, int elem, cudaStream_t s) {
  const int64_t most = (int64_t)sm_count() * 8;
  const unsigned grid = (unsigned)(a.rows < most ? a.rows : most);
  if (elem == E8_E4M3) row_kernel<T, E8_E4M3><<<grid, kThreads, 0, s>>>(a);
  else if (elem == E8_E5M2) row_kernel<T, E8_E5M2><<<grid, kThreads, 0, s>>>(a);
  else row_kernel<T, E8_INT8><<<grid, kThreads, 0, s>>>(a);
  count_launch();
}

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
  if (dtype == TC_F32) norm::launch<float>(a, elem, s);
  else if (dtype == TC_BF16) norm::launch<__nv_bfloat16>(a, elem, s);
  else norm::launch<__half>(a, elem, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(std::string("tc_rms_norm_quantize: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  return TC_OK;
}
