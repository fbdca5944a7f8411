// Low-rank adapters: the C entry, and the plain kernel for every type, size and alignment.
#include <string>

#include "tc_adapt.cuh"

namespace tc {
namespace adapt {

constexpr int kMaxRank = 1024;

// A block a token: a warp a row of A, then a thread an output.
__global__ void __launch_bounds__(256) plain_kernel(Args a) {
  __shared__ float h[kMaxRank];
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
  if (rank < 1 || rank > adapt::kMaxRank) return bad("rank must be in [1, 1024]");
  if (x_kind < 0 || x_kind > adapt::X_INT8 || y_dtype < 0 || y_dtype > 2 || w_dtype < 0 || w_dtype > 2 || out_dtype < 0 ||
      out_dtype > 2)
    return bad("unsupported dtype");
  if (!y || !index || !out || (k && !x) || (adapters && k && (!a || !b))) return bad("null pointer");
  if (x_kind > adapt::X_F16 && !x_scale) return bad("codes need scales");
  if (y_stride < n || x_stride < k) return bad("row strides must be at least the row's length");
  adapt::Args g{y, x, a, b, x_scale, gain, index, out, tokens, k, n, y_stride, x_stride, rank, adapters, y_dtype, x_kind, w_dtype, out_dtype};
  if (k == 0) g.adapters = 0;  // nothing to add
  const int64_t most = (int64_t)sm_count() * 8;
  adapt::plain_kernel<<<(unsigned)(tokens < most ? tokens : most), 256, 0, (cudaStream_t)stream>>>(g);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(std::string("tc_low_rank_add: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  count_launch();
  return TC_OK;
}
