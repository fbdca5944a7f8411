// Low-rank adapters: the C entry, and the plain kernel for every type, size and alignment.
#include <string>

#include "tc_adapt.cuh"

namespace tc {
namespace adapt {

constexpr int kPlainRank = 1024;

// A block a token: a warp a row of A, then a thread an output. 4096 -> 4096, rank 16, all fp32: one token 36 us, 64 38, 8192 1340; rank 200 in
// bf16, 64 tokens 824: every block reads its adapter itself, in single elements. It serves what the tensor cores do not take, not speed.
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

cudaError_t launch_bf16(const Args &a, cudaStream_t s);
cudaError_t launch_f16(const Args &a, cudaStream_t s);

// y and out of 32 bits or of the weights' type.
static bool on_tensor_cores(int x_kind, int w_dtype, int rank, int y_dtype, int out_dtype) {
  auto fits = [&](int d) { return d == TC_F32 || d == w_dtype; };
  return w_dtype != TC_F32 && (x_kind == w_dtype || x_kind > X_F16) && fits(y_dtype) && fits(out_dtype) && rank <= kMaxRank;
}

}  // namespace adapt
}  // namespace tc

// h in up to three parts of 16 bits, and a factor a token.
extern "C" size_t tc_low_rank_add_workspace(int64_t tokens, int32_t x_kind, int32_t w_dtype, int32_t rank, int32_t y_dtype,
                                            int32_t out_dtype) {
  using namespace tc;
  if (rank < 1 || tokens <= adapt::few_tokens() || !adapt::on_tensor_cores(x_kind, w_dtype, rank, y_dtype, out_dtype)) return 0;
  return (size_t)tokens * ((size_t)adapt::rank_rows(rank) * 3 * sizeof(uint16_t) + sizeof(float));
}

extern "C" int tc_low_rank_add(const void *y, int32_t y_dtype, int64_t y_stride, const void *x, int32_t x_kind, int64_t x_stride,
                               const float *x_scale, int64_t tokens, int64_t k, int64_t n, const void *a, const void *b,
                               int32_t w_dtype, int32_t adapters, int32_t rank, const float *gain, const int32_t *index, void *out,
                               int32_t out_dtype, void *workspace, size_t workspace_bytes, tc_stream stream) {
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
  adapt::Args g{y, x, a, b, x_scale, gain, index, out, tokens, k, n, y_stride, x_stride, rank, adapters, y_dtype, x_kind, w_dtype, out_dtype, 0, 0,
                nullptr, nullptr};
  if (k == 0) g.adapters = 0;  // nothing to add
  if (const size_t need = tc_low_rank_add_workspace(tokens, x_kind, w_dtype, rank, y_dtype, out_dtype)) {
    if (!workspace || workspace_bytes < need) return set_error("tc_low_rank_add: workspace too small"), TC_WORKSPACE_TOO_SMALL;
    if ((uintptr_t)workspace % 16) return bad("workspace must be 16-byte aligned");
    g.parts = static_cast<uint16_t *>(workspace);
    g.factors = reinterpret_cast<float *>(g.parts + (size_t)tokens * adapt::rank_rows(rank) * 3);
  }
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  // MMAs take operands of one 16-bit type, which holds 8-bit codes exactly; the rest goes element by element.
  if (adapt::on_tensor_cores(x_kind, w_dtype, rank, y_dtype, out_dtype)) {
    e = w_dtype == TC_BF16 ? adapt::launch_bf16(g, s) : adapt::launch_f16(g, s);
  } else {
    const int64_t most = (int64_t)sm_count() * 8;
    adapt::plain_kernel<<<(unsigned)(tokens < most ? tokens : most), 256, 0, s>>>(g);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return set_error(std::string("tc_low_rank_add: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  count_launch();
  return TC_OK;
}
