// The C entry of sampling.
#include <string>

#include "tc_sample.cuh"

namespace tc {
namespace sample {

constexpr int64_t kMaxVocab = 1 << 23;  // histograms add 12-bit parts of 2**20 weights a block in 32 bits
constexpr int64_t kMaxHeld = 53248;     // weights that a block's shared memory holds beside the rest

template <typename T, bool HELD>
static cudaError_t launch_as(const Args &a, cudaStream_t s) {
  const size_t bytes = HELD ? (size_t)a.part * sizeof(float) : 0;
  // The attribute belongs to the kernel, which other host threads may be launching with stretches of another length: always the largest.
  if (HELD) {
    const cudaError_t e = cudaFuncSetAttribute(sample_kernel<T, HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)(kMaxHeld * sizeof(float)));
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * a.blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, HELD>, a);
}

template <typename T>
static cudaError_t launch(Args a, cudaStream_t s) {
  // Stretches short enough for two blocks an SM, and more of them while the card is not full and they stay long enough to be worth it.
  // Measured with 1, 2, 4 and 8 blocks a row, us, bf16, top-k 50 and top-p 0.9: one row of 4096 11.2, 11.6, 11.5, 10.8, of 8192 12.5, 12.4, 12.3,
  // 10.9, of 32000 19.9, 15.1, 13.4, 11.6; 37 rows of 2000 10.4, 10.9, 14.2, 19.3, of 16000 15.4, 13.4, 15.2, 20.2; 296 rows of 16000 21, 33,
  // 60, 92, of 32000 41, 40, 68, 103, of 60000 2, 4 and 8 blocks 80, 84, 118 (without filters 66, 61, 88). The second condition
  // lets a row more than fill the card: from 37 to 148 rows half as many blocks are faster (74 rows of 32000 16.6 in 2, 26.1 in the 4 it takes).
  a.blocks = 1;
  while (a.blocks < 8 && (a.vocab > 23552 * (int64_t)a.blocks ||
                          (a.rows * a.blocks <= sm_count() && a.vocab > 4096 * (int64_t)a.blocks)))
    a.blocks *= 2;
  a.part = (int)(((a.vocab + 8 + a.blocks - 1) / a.blocks + 127) / 128 * 128);  // positions begin up to 7 elements before the row
  return a.part <= kMaxHeld ? launch_as<T, true>(a, s) : launch_as<T, false>(a, s);
}

}  // namespace sample
}  // namespace tc

extern "C" int tc_sample_tokens(const void *logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t stride, const float *uniform,
                                const float *temperature, float all_temperature, const int32_t *top_k, int32_t all_top_k,
                                const float *top_p, float all_top_p, const float *min_p, float all_min_p, int64_t *tokens,
                                float *logprobs, tc_stream stream) {
  using namespace tc;
  if (rows == 0) return TC_OK;
  auto bad = [](const char *m) { return set_error(std::string("tc_sample_tokens: ") + m), (int)TC_INVALID_ARGUMENT; };
  if (rows < 0 || rows > (1 << 27) || vocab < 1 || vocab > sample::kMaxVocab)
    return bad("rows and vocab out of range (at most 2**27 and 2**23)");
  if (dtype < 0 || dtype > 2) return bad("unsupported dtype");
  if (!logits || !uniform || !tokens) return bad("null pointer");
  if (rows > 1 && stride < vocab) return bad("the row stride must be at least vocab");
  sample::Args a{logits, rows, vocab, stride, uniform, temperature, top_p, min_p, top_k, all_temperature, all_top_p, all_min_p,
                 all_top_k, tokens, logprobs, 1, 0};
  cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = dtype == TC_F32    ? sample::launch<float>(a, s)
                        : dtype == TC_BF16 ? sample::launch<__nv_bfloat16>(a, s)
                                           : sample::launch<__half>(a, s);
  if (e != cudaSuccess) return set_error(std::string("tc_sample_tokens: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  count_launch();
  return TC_OK;
}
