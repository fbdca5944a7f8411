// Low-rank adapters: the C entry, and the plain kernel for every type, size and alignment.
#include <string>

#include "tc_adapt.cuh"

namespace tc {
namespace adapt {

constexpr int kPlainRank = 1024;

// A block a token: a warp a row of A, then a thread an output.
__global__ void __launch_bounds__(256) plain_kernel(Args a) {
  __shared__ float h[kPlainRank];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const int i = a.index[t];
    const bool some = i >= 0 && i < a.adapters;
    if (some) {
      float s = a.x_scale ? a.x_scale[t] : 1.0f;
      if (a.gain) s = __fmul_rn(s, a.gain[i]);
      for (int r = warp; r < a.rank; r += 8) {
        float v = 0.0f;
        for (int64_t c = lane; c < a.k; c += 32)
          v = __fmaf_rn(x_at(a, t * a.x_stride + c), load_as_float(a.a, a.w_dtype, ((int64_t)i * a.rank + r) * a.k + c), v);
        for (int m = 16; m; m >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xFFFFFFFFu, v, m));
        if (lane == 0) h[r] = __fmul_rn(v, s);
      }
    }
    __syncthreads();
    for (int64_t c = threadIdx.x; c < a.n; c += 256) {
      float v = 0.0f;
      if (some)
        for (int r = 0; r < a.rank; ++r) v = __fmaf_rn(h[r], load_as_float(a.b, a.w_dtype, ((int64_t)i * a.n + c) * a.rank + r), v);
      store_rounded(a.out, a.out_dtype, t * a.n + c, __fadd_rn(load_as_float(a.y, a.y_dtype, t * a.y_stride + c), v));
    }
    __syncthreads();
  }
}

template <typename T, int NG, int RW, bool VEC>
static cudaError_t launch_tiles(Args a, cudaStream_t s) {
  const int rows = (a.rank + RW - 1) / RW * RW, row_blocks = rows / RW;
  const size_t bytes = (size_t)kWarps / row_blocks * 8 * NG * rows * sizeof(float) + (size_t)3 * 8 * NG * (rows + 8) * sizeof(uint16_t) +
                       (Same<T, __half>::value ? (size_t)8 * NG * rows * sizeof(float) : 0);
  cudaError_t e = cudaFuncSetAttribute(tile_kernel<T, NG, RW, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.tokens + a.tile - 1) / a.tile * a.blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, tile_kernel<T, NG, RW, VEC>, a);
}

template <typename T>
static cudaError_t launch_as(Args a, cudaStream_t s) {
  auto aligned = [](const void *p, size_t n) { return (uintptr_t)p % n == 0; };
  const int y16 = a.y_dtype == TC_F32 ? 4 : 8;
  const bool vec = a.k % 8 == 0 && a.n % 8 == 0 && a.rank % (a.rank <= 16 ? 4 : 8) == 0 && a.x_stride % 8 == 0 &&
                   a.y_stride % y16 == 0 && aligned(a.x, a.x_kind <= X_F16 ? 16 : 8) && aligned(a.y, 16) && aligned(a.a, 16) &&
                   aligned(a.b, 16) && aligned(a.out, 16);
  // Few tokens: tiles of at most 8, as small as the card has clusters of 8 blocks for. Many: tiles of 32.
  const int sms = sm_count();
  const bool few = a.tokens <= 8 * (int64_t)sms / 4;
  if (few) {
    a.tile = 1;
    while (a.tile < 8 && (a.tokens + a.tile - 1) / a.tile * 8 > sms) a.tile *= 2;
  } else {
    a.tile = 32;
  }
  a.blocks = 1;
  while (a.blocks < 8 && (a.tokens + a.tile - 1) / a.tile * a.blocks * 2 <= (few ? 1 : 4) * sms) a.blocks *= 2;
  if (few) {
    if (a.rank <= 16) return vec ? launch_tiles<T, 1, 16, true>(a, s) : launch_tiles<T, 1, 16, false>(a, s);
    return vec ? launch_tiles<T, 1, 32, true>(a, s) : launch_tiles<T, 1, 32, false>(a, s);
  }
  if (a.rank <= 16) return vec ? launch_tiles<T, 4, 16, true>(a, s) : launch_tiles<T, 4, 16, false>(a, s);
  return vec ? launch_tiles<T, 4, 32, true>(a, s) : launch_tiles<T, 4, 32, false>(a, s);
}

}  // namespace adapt
}  // namespace tc

extern "C" int tc_low_rank_add(const void *y, int32_t y_dtype, int64_t y_stride, const void *x, int32_t x_kind, int64_t x_stride,
                               const float *x_scale, int64_t tokens, int64_t k, int64_t n, const void *a, const void *b,
                               int32_t w_dtype, int32_t adapters, int32_t rank, const float *gain, const int32_t *index, void *out,
                               int32_t out_dtype, tc_stream stream) {
  using namespace tc;
  if (tokens == 0 || n == 0) return TC_OK;
  auto bad = [](const char *m) { return set_error(std::string("tc_low_rank_add: ") + m), (int)TC_INVALID_ARGUMENT; };
  if (tokens < 0 || k < 0 || n < 0 || adapters < 0 || tokens >= (1ll << 31) || n >= (1ll << 31) || k >= (1ll << 31))
    return bad("sizes out of range");
  if (rank < 1 || rank > adapt::kPlainRank) return bad("rank must be in [1, 1024]");
  if (x_kind < 0 || x_kind > adapt::X_INT8 || y_dtype < 0 || y_dtype > 2 || w_dtype < 0 || w_dtype > 2 || out_dtype < 0 ||
      out_dtype > 2)
    return bad("unsupported dtype");
  if (!y || !index || !out || (k && !x) || (adapters && k && (!a || !b))) return bad("null pointer");
  if (x_kind > adapt::X_F16 && !x_scale) return bad("codes need scales");
  if (y_stride < n || x_stride < k) return bad("row strides must be at least the row's length");
  adapt::Args g{y, x, a, b, x_scale, gain, index, out, tokens, k, n, y_stride, x_stride, rank, adapters, y_dtype, x_kind, w_dtype, out_dtype, 0, 0};
  if (k == 0) g.adapters = 0;  // nothing to add
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  // MMAs take operands of one 16-bit type, which holds 8-bit codes exactly; the rest goes element by element.
  if (w_dtype != TC_F32 && (x_kind == w_dtype || x_kind > adapt::X_F16) && rank <= adapt::kMaxRank) {
    e = w_dtype == TC_BF16 ? adapt::launch_as<__nv_bfloat16>(g, s) : adapt::launch_as<__half>(g, s);
  } else {
    const int64_t most = (int64_t)sm_count() * 8;
    adapt::plain_kernel<<<(unsigned)(tokens < most ? tokens : most), 256, 0, s>>>(g);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return set_error(std::string("tc_low_rank_add: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  count_launch();
  return TC_OK;
}
