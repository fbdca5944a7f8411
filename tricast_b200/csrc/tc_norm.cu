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

// Eight elements as fp32, from 16-bit or fp32 memory at a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const unsigned short lo = (unsigned short)(u[k] & 0xFFFFu), hi = (unsigned short)(u[k] >> 16);
      v[2 * k] = Io<T>::get(*reinterpret_cast<const T *>(&lo));
      v[2 * k + 1] = Io<T>::get(*reinterpret_cast<const T *>(&hi));
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
  T h[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) h[k] = Io<T>::put(v[k]);
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(h[0], h[1], h[2], h[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(h[4], h[5], h[6], h[7]);
  } else {
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      u[k] = (uint32_t)*reinterpret_cast<unsigned short *>(&h[2 * k]) | ((uint32_t)*reinterpret_cast<unsigned short *>(&h[2 * k + 1]) << 16);
    *reinterpret_cast<uint4 *>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// One block a row that its registers hold, read once and written once: bound by HBM. A thread has NV vectors
// of 8 neighbouring elements (VEC 8; vector v of the row is thread v % threads's), or 8 NV single ones where rows
// are not aligned (VEC 1). A group's maximum stays inside a warp: 2 to 32 lanes (VEC 8), or exactly a warp
// (VEC 1, groups of 32); a row's goes through shared memory, like the sum of squares.
template <typename T, int E, int NV, int VEC>
__global__ void __launch_bounds__(1024) held_kernel(Args a) {
  __shared__ float part[2][32];
  __shared__ uint32_t tops[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warps = blockDim.x >> 5;
  const int K = (int)a.K;
  const bool row_scale = a.groups == 1;
  const int lanes = VEC == 8 ? a.group / 8 : 32;  // that share a group
  int flip = 0;  // the two halves of the exchange buffers alternate, so one barrier an exchange suffices
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, flip ^= 1) {
    const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
    const T *res = a.res ? static_cast<const T *>(a.res) + r * a.res_stride : nullptr;
    float v[NV][8];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
      if (VEC == 8) {
        const int c = (tid + i * blockDim.x) * 8;
        if (c < K) load8(x + c, v[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = tid + (8 * i + e) * blockDim.x;
          if (c < K) v[i][e] = Io<T>::get(x[c]);
        }
      }
    }
    if (res) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (VEC == 8) {
          const int c = (tid + i * blockDim.x) * 8;
          if (c < K) {
            float w[8];
            load8(res + c, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = __fadd_rn(v[i][e], w[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int c = tid + (8 * i + e) * blockDim.x;
            if (c < K) v[i][e] = __fadd_rn(v[i][e], Io<T>::get(res[c]));
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __fmaf_rn(v[i][e], v[i][e], ss);
    for (int m = 16; m; m >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, m);
    if (lane == 0) part[flip][tid >> 5] = ss;
    if (a.h) {  // beside the wait for the other warps
      T *h = static_cast<T *>(a.h) + r * a.K;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (VEC == 8) {
          const int c = (tid + i * blockDim.x) * 8;
          if (c < K) store8(h + c, v[i]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int c = tid + (8 * i + e) * blockDim.x;
            if (c < K) h[c] = Io<T>::put(v[i][e]);
          }
        }
      }
    }
    __syncthreads();
    ss = lane < warps ? part[flip][lane] : 0.0f;
    for (int m = 16; m; m >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, m);
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)K), a.eps)));
    uint32_t row_top = 0u;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.0f;
      if (a.w) {
        if (VEC == 8) {
          const int c = (tid + i * blockDim.x) * 8;
          if (c < K) {
            if (a.w_dtype == TC_F32) load8(static_cast<const float *>(a.w) + c, w);
            else if (a.w_dtype == TC_BF16) load8(static_cast<const __nv_bfloat16 *>(a.w) + c, w);
            else load8(static_cast<const __half *>(a.w) + c, w);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int c = tid + (8 * i + e) * blockDim.x;
            if (c < K) w[e] = load_as_float(a.w, a.w_dtype, c);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] = __fmul_rn(v[i][e], inv);
        if (a.w) v[i][e] = __fmul_rn(v[i][e], w[e]);
        row_top = max(row_top, abs_bits(v[i][e]));
      }
    }
    float s = 1.0f, rs = 1.0f;
    bool fast = true;
    if (row_scale) {
      row_top = warp_max(row_top);
      if (lane == 0) tops[flip][tid >> 5] = row_top;
      __syncthreads();
      row_top = warp_max(lane < warps ? tops[flip][lane] : 0u);
      if (a.e8m0) {
        const uint32_t code = pow2_code(row_top, a.emax);
        rs = pow2_inverse(code);
        fast = code != 0xFFu;
        if (tid == 0) static_cast<unsigned char *>(a.scale)[r] = (unsigned char)code;
      } else {
        s = absmax_scale(row_top, a.max_elem);
        fast = divides_fast(s);
        rs = __fdiv_rn(1.0f, s);
        if (tid == 0) static_cast<float *>(a.scale)[r] = s;
      }
    }
    unsigned char *codes = a.codes + r * a.K;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c0 = VEC == 8 ? (tid + i * blockDim.x) * 8 : tid + 8 * i * blockDim.x;
      if (VEC == 8) {
        if (!row_scale) {
          uint32_t top = 0u;
#pragma unroll
          for (int e = 0; e < 8; ++e) top = max(top, abs_bits(v[i][e]));
          for (int m = lanes >> 1; m; m >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, m));
          const bool first = c0 < K && (c0 / 8) % lanes == 0;
          const int64_t at = r * a.groups + c0 / a.group;
          if (a.e8m0) {
            const uint32_t code = pow2_code(top, a.emax);
            rs = pow2_inverse(code);
            fast = code != 0xFFu;
            if (first) static_cast<unsigned char *>(a.scale)[at] = (unsigned char)code;
          } else {
            s = absmax_scale(top, a.max_elem);
            fast = divides_fast(s);
            rs = __fdiv_rn(1.0f, s);
            if (first) static_cast<float *>(a.scale)[at] = s;
          }
        }
        uint32_t q[4];
        if (fast) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float y0 = v[i][2 * k], y1 = v[i][2 * k + 1];
            if (a.e8m0 && E == E8_INT8) {  // the scale of a power of two may leave values beyond the largest
              q[k] = encode8<E>(__fmul_rn(y0, rs)) | (encode8<E>(__fmul_rn(y1, rs)) << 8);
            } else {
              q[k] = a.e8m0 ? encode8x2<E>(__fmul_rn(y0, rs), __fmul_rn(y1, rs))
                            : encode8x2<E>(divide_fast(y0, s, rs), divide_fast(y1, s, rs));
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t two[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
              two[e] = encode8<E>(a.e8m0 ? __fmul_rn(v[i][2 * k + e], rs) : __fdiv_rn(v[i][2 * k + e], s));
            q[k] = two[0] | (two[1] << 8);
          }
        }
        if (c0 < K) *reinterpret_cast<uint2 *>(codes + c0) = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = c0 + e * (int)blockDim.x;
          if (!row_scale) {  // groups of 32: a warp's elements
            const uint32_t top = warp_max(abs_bits(v[i][e]));
            const int64_t at = r * a.groups + c / 32;
            if (a.e8m0) {
              const uint32_t code = pow2_code(top, a.emax);
              rs = pow2_inverse(code);
              if (lane == 0 && c < K) static_cast<unsigned char *>(a.scale)[at] = (unsigned char)code;
            } else {
              s = absmax_scale(top, a.max_elem);
              if (lane == 0 && c < K) static_cast<float *>(a.scale)[at] = s;
            }
          }
          if (c < K) codes[c] = (unsigned char)encode8<E>(a.e8m0 ? __fmul_rn(v[i][e], rs) : __fdiv_rn(v[i][e], s));
        }
      }
    }
  }
}

template <typename T, int E, int VEC>
static void launch_held(const Args &a, cudaStream_t s) {
  // Threads for about two vectors each, so that a row's latency is short and several rows share an SM; the
  // longest rows take four. (16384 x 8192 bf16: FIXME)
  const int64_t vectors = (a.K + 7) / 8;
  int threads = 64;
  while (threads < 1024 && threads * 2 < vectors) threads *= 2;
  const int64_t most = (int64_t)sm_count() * (2048 / threads);
  const unsigned grid = (unsigned)(a.rows < most ? a.rows : most);
  const int nv = (int)((vectors + threads - 1) / threads);
  if (nv <= 1) held_kernel<T, E, 1, VEC><<<grid, threads, 0, s>>>(a);
  else if (nv <= 2) held_kernel<T, E, 2, VEC><<<grid, threads, 0, s>>>(a);
  else held_kernel<T, E, 4, VEC><<<grid, threads, 0, s>>>(a);
  count_launch();
}

template <typename T, int E>
static void launch_elem(const Args &a, cudaStream_t s) {
  auto aligned = [](const void *p, size_t n) { return (uintptr_t)p % n == 0; };
  const bool vec = a.K % 8 == 0 && a.x_stride % 8 == 0 && (!a.res || a.res_stride % 8 == 0) && aligned(a.x, 16) &&
                   aligned(a.res, 16) && aligned(a.w, 16) && aligned(a.h, 16) && aligned(a.codes, 8);
  const bool pow2_lanes = a.group % 8 == 0 && a.group <= 256 && (a.group & (a.group - 1)) == 0;
  if (vec && a.K <= 32768 && (a.groups == 1 || pow2_lanes)) {
    launch_held<T, E, 8>(a, s);
  } else if (a.K <= 32768 && (a.groups == 1 || a.group == 32)) {
    launch_held<T, E, 1>(a, s);
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
