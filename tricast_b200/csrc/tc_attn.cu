// Attention of new tokens over a paged, quantized cache: the C entry, and the plain kernel.
#include <cmath>
#include <string>

#include "tc_attn.cuh"

namespace tc {
namespace attn {

constexpr int kThreads = 256;

// Element d of a cached row, in fp32.
template <typename T>
__device__ __forceinline__ float cached(const KvCache &c, const unsigned char *codes, const unsigned char *scales, int d) {
  if (c.scheme == KV_NONE) return Io<T>::get(reinterpret_cast<const T *>(codes)[d]);
  if (c.scheme == KV_MXFP4) return __fmul_rn(decode_e2m1((codes[d >> 1] >> (4 * (d & 1))) & 15u), pow2_value(scales[d >> 5]));
  const float s = *reinterpret_cast<const float *>(scales);
  return __fmul_rn(c.scheme == KV_FP8_ROW ? decode_e4m3(codes[d]) : (float)(signed char)codes[d], s);
}

// A warp a (new token, query head): lanes over the head's elements, one key at a time, with the running
// maximum and sum of the softmax. Every type, scheme and head size; all arithmetic in fp32.
template <typename T>
__global__ void __launch_bounds__(kThreads) plain_kernel(Args a) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = a.total_q * a.heads;
  for (int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); r < rows;
       r += (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t token = r / a.heads;
    const int head = (int)(r % a.heads);
    // The last sequence whose first token is not after this one (idle sequences share their start with
    // the next one).
    int b = 0;
    if (a.cu) {
      int hi = a.batch;
      while (b + 1 < hi) {
        const int mid = (b + hi) >> 1;
        if (a.cu[mid] <= token) b = mid;
        else hi = mid;
      }
    } else {
      b = (int)token;
    }
    const Seq s = sequence(a, b);
    if (token < s.q0 || token >= s.q0 + s.n) continue;
    int lo, hi;
    visible(a, s, (int)(token - s.q0), lo, hi);
    const T *qp = static_cast<const T *>(a.q) + token * a.q_tok + head * a.q_head;
    float q[8], o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 32 * i;
      q[i] = d < a.c.dim ? Io<T>::get(qp[d]) : 0.0f;
      o[i] = 0.0f;
    }
    float top = -INFINITY, total = 0.0f;
    const int kvh = head / a.group;
    for (int p = lo; p < hi; ++p) {
      const int page = a.table[b * a.table_stride + (p >> a.c.page_shift)];
      if (page < 0 || page >= a.c.pages) continue;
      const int64_t row = (((int64_t)page * a.c.heads + kvh) << a.c.page_shift) + (p & (a.c.page_size - 1));
      const unsigned char *kc = a.c.k + row * a.c.row_bytes, *ks = a.c.ks + row * a.c.scale_bytes;
      const unsigned char *vc = a.c.v + row * a.c.row_bytes, *vs = a.c.vs + row * a.c.scale_bytes;
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d < a.c.dim) dot = __fmaf_rn(q[i], cached<T>(a.c, kc, ks, d), dot);
      }
      for (int m = 16; m; m >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, m);
      dot *= a.scale;
      if (dot == -INFINITY) continue;  // exp2 of it is 0 whatever the maximum
      const float now = fmaxf(top, dot), keep = exp2f(top - now), w = exp2f(dot - now);
      top = now;
      total = __fmaf_rn(total, keep, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d < a.c.dim) o[i] = __fmaf_rn(w, cached<T>(a.c, vc, vs, d), o[i] * keep);
      }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 32 * i;
      if (d < a.c.dim) static_cast<T *>(a.out)[r * a.c.dim + d] = Io<T>::put(o[i] * inv);
    }
    if (a.lse && lane == 0) a.lse[r] = total == 0.0f ? -INFINITY : (top + log2f(total)) * 0.69314718055994531f;
  }
}

int launch_split_none(const Args &a, float *parts, int most, cudaStream_t s);
int launch_split_fp8(const Args &a, float *parts, int most, cudaStream_t s);
int launch_split_int8(const Args &a, float *parts, int most, cudaStream_t s);
int launch_split_mxfp4(const Args &a, float *parts, int most, cudaStream_t s);

// Blocks of the split kernel: as many as run at once.
static int split_blocks(const KvCache &c) {
  return sm_count() * (c.scheme == KV_NONE && split_width(c.dim) == 256 ? 1 : 2);
}

static int launch_split(const Args &a, float *parts, cudaStream_t s) {
  const int most = split_blocks(a.c);
  const int st = a.c.scheme == KV_NONE       ? launch_split_none(a, parts, most, s)
                 : a.c.scheme == KV_FP8_ROW  ? launch_split_fp8(a, parts, most, s)
                 : a.c.scheme == KV_INT8_ROW ? launch_split_int8(a, parts, most, s)
                                             : launch_split_mxfp4(a, parts, most, s);
  if (st != TC_OK) return st;
  if (a.c.dtype == TC_BF16) join_kernel<__nv_bfloat16, 16, 64><<<most - 1, 256, 0, s>>>(a, parts, split_width(a.c.dim), most);
  else join_kernel<__half, 16, 64><<<most - 1, 256, 0, s>>>(a, parts, split_width(a.c.dim), most);
  count_launch();
  return TC_OK;
}

}  // namespace attn
}  // namespace tc

extern "C" size_t tc_paged_attention_workspace(const tc_kv_cache *cache, int32_t q_heads, int64_t total_q, int32_t batch,
                                               int32_t max_q_len) {
  using namespace tc;
  KvCache c;
  if (kv_cache_check(cache, c) != TC_OK || c.dtype == TC_F32) return 0;
  return 2 * (size_t)attn::split_blocks(c) * attn::partial_floats(16, attn::split_width(c.dim)) * sizeof(float);
}

extern "C" int tc_paged_attention(const tc_kv_cache *cache, const void *q, int64_t q_token_stride, int64_t q_head_stride,
                                  int64_t total_q, int32_t q_heads, const int32_t *block_table, int64_t table_stride,
                                  int32_t max_pages, const int32_t *seq_lens, const int32_t *cu_q, int32_t batch,
                                  int32_t max_q_len, float scale, int32_t causal, int32_t window, void *out, float *lse,
                                  void *workspace, size_t workspace_bytes, tc_stream stream) {
  using namespace tc;
  attn::Args a;
  const int st = kv_cache_check(cache, a.c);
  if (st != TC_OK) return st;
  auto bad = [](const char *m) { return set_error(std::string("tc_paged_attention: ") + m), (int)TC_INVALID_ARGUMENT; };
  if (total_q == 0 || batch == 0) return TC_OK;
  if (!q || !block_table || !seq_lens || !out) return bad("null pointer");
  if (total_q < 0 || total_q > 0x7FFFFFFFll || batch < 0 || max_pages < 0 || max_q_len < 1) return bad("sizes out of range");
  if (!cu_q && total_q != batch) return bad("without cu_q every sequence has one new token");
  if (q_heads < 1 || q_heads % cache->kv_heads) return bad("query heads must be a multiple of the cache's");
  if (!std::isfinite(scale)) return bad("scale must be finite");
  if (window < 0 || (window && !causal)) return bad("a window must be positive and needs causal");
  if (((int64_t)max_pages << a.c.page_shift) > (1ll << 30)) return bad("contexts are limited to 2**30 tokens");
  if (total_q * q_heads > 0x7FFFFFFFll) return bad("queries are limited to 2**31 - 1 rows");
  a.q = q;
  a.q_tok = q_token_stride;
  a.q_head = q_head_stride;
  a.total_q = total_q;
  a.heads = q_heads;
  a.group = q_heads / cache->kv_heads;
  a.table = block_table;
  a.table_stride = table_stride;
  a.max_pages = max_pages;
  a.lens = seq_lens;
  a.cu = cu_q;
  a.batch = batch;
  a.max_q = cu_q ? max_q_len : 1;
  a.scale = (float)((double)scale * 1.4426950408889634);
  a.causal = causal;
  a.window = window;
  a.out = out;
  a.lse = lse;
  cudaStream_t s = (cudaStream_t)stream;
  if (a.c.dtype == TC_F32) {
    const int64_t want = (total_q * q_heads + 7) / 8, most = (int64_t)sm_count() * 8;
    attn::plain_kernel<float><<<(unsigned)(want < most ? want : most), attn::kThreads, 0, s>>>(a);
    count_launch();
  } else {
    if (!workspace || workspace_bytes < tc_paged_attention_workspace(cache, q_heads, total_q, batch, max_q_len))
      return set_error("tc_paged_attention: workspace too small"), TC_WORKSPACE_TOO_SMALL;
    const int r = attn::launch_split(a, static_cast<float *>(workspace), s);
    if (r != TC_OK) return r;
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(std::string("tc_paged_attention: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  return TC_OK;
}
