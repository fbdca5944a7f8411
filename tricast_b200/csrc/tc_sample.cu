// The C entry of sampling.
#include <string>

#include "tc_sample.cuh"

namespace tc {
namespace sample {

template <typename T>
static cudaError_t launch(const Args &a, cudaStream_t s) {
  const int blocks = a.vocab >= 16384 ? 8 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, a);
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
  if (rows < 0 || rows > (1 << 27) || vocab < 1 || vocab > 0x7FFFFFFFll) return bad("rows and vocab out of range");
  if (dtype < 0 || dtype > 2) return bad("unsupported dtype");
  if (!logits || !uniform || !tokens) return bad("null pointer");
  if (rows > 1 && stride < vocab) return bad("the row stride must be at least vocab");
  sample::Args a{logits, rows, vocab, stride, uniform, temperature, top_p, min_p, top_k, all_temperature, all_top_p, all_min_p,
                 all_top_k, tokens, logprobs};
  cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = dtype == TC_F32    ? sample::launch<float>(a, s)
                        : dtype == TC_BF16 ? sample::launch<__nv_bfloat16>(a, s)
                                           : sample::launch<__half>(a, s);
  if (e != cudaSuccess) return set_error(std::string("tc_sample_tokens: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  count_launch();
  return TC_OK;
}
