// Attention of new tokens over a paged, quantized cache: the C entry, and the plain kernel.
#include <cmath>
#include <string>

#include "tc_attn.cuh"

namespace tc {
namespace attn {

constexpr int kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads) plain_kernel(Args a) {
  plain_rows<T>(a, (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), (int64_t)gridDim.x * (kThreads / 32));
}

int launch_split_none(const Args &a, float *parts, int sms, cudaStream_t s);
int launch_split_fp8(const Args &a, float *parts, int sms, cudaStream_t s);
int launch_split_int8(const Args &a, float *parts, int sms, cudaStream_t s);
int launch_split_mxfp4(const Args &a, float *parts, int most, cudaStream_t s);

int launch_chunk_none(const Args &a, float *parts, Stretch *stretches, int *status, int most, cudaStream_t s);
int launch_chunk_fp8(const Args &a, float *parts, Stretch *stretches, int *status, int most, cudaStream_t s);
int launch_chunk_int8(const Args &a, float *parts, Stretch *stretches, int *status, int most, cudaStream_t s);
int launch_chunk_mxfp4(const Args &a, float *parts, Stretch *stretches, int *status, int most, cudaStream_t s);

int launch_packed(const Args &a, float *parts, Stretch *stretches, int *status, int most, unsigned char *packed, int max_units,
                  cudaStream_t s);
size_t packed_unit_bytes(int dim);

static int launch_split(const Args &a, float *parts, cudaStream_t s) {
  const int sms = sm_count();
  return a.c.scheme == KV_NONE       ? launch_split_none(a, parts, sms, s)
         : a.c.scheme == KV_FP8_ROW  ? launch_split_fp8(a, parts, sms, s)
         : a.c.scheme == KV_INT8_ROW ? launch_split_int8(a, parts, sms, s)
                                     : launch_split_mxfp4(a, parts, sms, s);
}

// From kChunkRows query rows of a key / value head the chunk kernel's tiles of 128 rows pay, unless the call is
// small. Split against chunk kernel, us, 8 heads of 128 over fp8: 16 sequences of 2048 keys 60 and 82 (32 rows), 93 and
// 85 (64 rows), 126 and 86 (96); 16 of 8192 141 and 202, 253 and 206, 364 and 207; one of 16384 52 and 59 (64 rows), 78
// and 61 (128), 128 and 76 (256); one of 2048 32 and 33 (128), 38 and 39 (256), 69 and 57 (768). The rule is at its worst
// for one long sequence of 65 to 255 rows, where the split kernel's 78 us stand against 61.
constexpr int64_t kChunkRows = 65, kChunkTotalRows = 256;
static bool use_chunk(const KvCache &c, int group, int batch, int64_t max_q) {
  const int64_t rows = max_q * group;
  return c.dim <= 128 && rows >= kChunkRows && rows * batch >= kChunkTotalRows;
}

static size_t split_bytes(const KvCache &c) {
  // At most four blocks an SM of 8 rows, or as many rows in fewer blocks (split::Shape).
  return 2 * (size_t)sm_count() * 4 * partial_floats(16, split_width(c.dim)) * sizeof(float) + (size_t)sm_count() * 4 * sizeof(Stretch);
}
static size_t chunk_parts(const KvCache &c) {
  return 2 * (size_t)sm_count() * partial_floats(256, split_width(c.dim)) * sizeof(float);
}
static size_t chunk_bytes(const KvCache &c) {
  const size_t n = chunk_parts(c) + (size_t)sm_count() * (sizeof(Stretch) + sizeof(int));
  return (n + 127) / 128 * 128;
}

// Whether the chunk kernel's operands are laid out once, before it, and not by every row tile again: for quantized
// caches (the others need no conversion), from kPackRows query rows of a key / value head on, while the tables'
// width bounds the room it takes by kPackBytes. Laid out by every tile against once (fp8, 8 heads of 128): 512 rows
// over one sequence of 16384 keys 98 and 105 us, over sixteen of 2048 181 and 185; 768 rows 123 and 119, 248 and 229;
// 1024 rows 149 and 143, 315 and 271; 2048 rows 241 and 201, 518 and 421.
constexpr int64_t kPackRows = 768;
constexpr size_t kPackBytes = (size_t)1 << 29;
static int pack_units(const KvCache &c, int max_pages) {
  const int64_t n = (((int64_t)max_pages << c.page_shift) + 127) / 128;
  return (int)(n < 1 ? 1 : n);
}
static size_t pack_bytes(const KvCache &c, int group, int batch, int64_t max_q, int max_pages) {
  if (c.scheme == KV_NONE || max_q * group < kPackRows) return 0;
  const double n = (double)batch * c.heads * pack_units(c, max_pages) * (double)packed_unit_bytes(c.dim);
  return n <= (double)kPackBytes ? (size_t)n : 0;
}

static int launch_chunk(const Args &a, void *workspace, cudaStream_t s) {
  const int most = sm_count();
  float *parts = static_cast<float *>(workspace);
  Stretch *stretches = reinterpret_cast<Stretch *>(static_cast<char *>(workspace) + chunk_parts(a.c));
  int *status = reinterpret_cast<int *>(stretches + most);
  const int st = pack_bytes(a.c, a.group, a.batch, a.max_q, a.max_pages)
                     ? launch_packed(a, parts, stretches, status, most, static_cast<unsigned char *>(workspace) + chunk_bytes(a.c),
                                     pack_units(a.c, a.max_pages), s)
                 : a.c.scheme == KV_NONE     ? launch_chunk_none(a, parts, stretches, status, most, s)
                 : a.c.scheme == KV_FP8_ROW  ? launch_chunk_fp8(a, parts, stretches, status, most, s)
                 : a.c.scheme == KV_INT8_ROW ? launch_chunk_int8(a, parts, stretches, status, most, s)
                                             : launch_chunk_mxfp4(a, parts, stretches, status, most, s);
  if (st != TC_OK) return st;
  // Few items are cut into many parts each (see join_kernel).
  const double items = (double)a.batch * a.c.heads * (((double)a.max_q * a.group + 255) / 256);
  if (items * 4 <= most)
    return a.c.dtype == TC_BF16 ? launch_join<__nv_bfloat16, 256, 16>(a, parts, stretches, most, status, s)
                                : launch_join<__half, 256, 16>(a, parts, stretches, most, status, s);
  return a.c.dtype == TC_BF16 ? launch_join<__nv_bfloat16, 256, 64>(a, parts, stretches, most, status, s)
                              : launch_join<__half, 256, 64>(a, parts, stretches, most, status, s);
}

}  // namespace attn
}  // namespace tc

extern "C" size_t tc_paged_attention_workspace(const tc_kv_cache *cache, int32_t q_heads, int64_t total_q, int32_t batch,
                                               int32_t max_q_len, int32_t max_pages) {
  using namespace tc;
  KvCache c;
  if (kv_cache_check(cache, c) != TC_OK || c.dtype == TC_F32) return 0;
  if (q_heads < c.heads || q_heads % c.heads) return 0;
  const int group = q_heads / c.heads;
  if (attn::use_chunk(c, group, batch, max_q_len)) return attn::chunk_bytes(c) + attn::pack_bytes(c, group, batch, max_q_len, max_pages);
  return attn::split_bytes(c);
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
  if (total_q == 0) return TC_OK;
  if (!q || !out || (batch > 0 && ((!block_table && max_pages) || !seq_lens))) return bad("null pointer");
  if ((uintptr_t)out % 16 || (uintptr_t)workspace % 16) return bad("out and workspace must be 16-byte aligned");
  if (total_q < 0 || total_q > 0x7FFFFFFFll || batch < 0 || max_pages < 0 || max_q_len < 1) return bad("sizes out of range");
  if (!cu_q && total_q != batch) return bad("without cu_q every sequence has one new token");
  if (q_heads < 1 || q_heads % cache->kv_heads) return bad("query heads must be a multiple of the cache's");
  // The kernels take it times log2(e).
  if (!std::isfinite((float)((double)scale * 1.4426950408889634))) return bad("scale must be finite, with room for a factor log2(e)");
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
  if (a.c.dtype == TC_F32 || batch == 0) {
    const int64_t want = (total_q * q_heads + 7) / 8, most = (int64_t)sm_count() * 8;
    const unsigned grid = (unsigned)(want < most ? want : most);
    if (a.c.dtype == TC_F32) attn::plain_kernel<float><<<grid, attn::kThreads, 0, s>>>(a);
    else if (a.c.dtype == TC_BF16) attn::plain_kernel<__nv_bfloat16><<<grid, attn::kThreads, 0, s>>>(a);
    else attn::plain_kernel<__half><<<grid, attn::kThreads, 0, s>>>(a);
    count_launch();
  } else {
    if (!workspace || workspace_bytes < tc_paged_attention_workspace(cache, q_heads, total_q, batch, a.max_q, max_pages))
      return set_error("tc_paged_attention: workspace too small"), TC_WORKSPACE_TOO_SMALL;
    const int r = attn::use_chunk(a.c, a.group, a.batch, a.max_q) ? attn::launch_chunk(a, workspace, s)
                                                         : attn::launch_split(a, static_cast<float *>(workspace), s);
    if (r != TC_OK) return r;
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(std::string("tc_paged_attention: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  return TC_OK;
}
