// Paged key / value cache, quantized as it is written and read back: one scale (or one set of E8M0 group
// scales) per token and head, so that a token is written without touching its neighbours.
#include <string>

#include "tc_serve.cuh"

namespace tc {

int kv_cache_check(const tc_kv_cache *c, KvCache &o) {
  auto bad = [](const char *m) { return set_error(std::string("paged cache: ") + m), (int)TC_INVALID_ARGUMENT; };
  if (!c || !c->k || !c->v) return bad("null pointer");
  if (c->scheme < KV_NONE || c->scheme > KV_MXFP4) return bad("unknown scheme");
  if (c->dtype < 0 || c->dtype > 2) return bad("unsupported dtype");
  if (c->scheme != KV_NONE && (!c->k_scale || !c->v_scale)) return bad("null scale pointer");
  if (c->page_size < 8 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return bad("page_size must be a power of two in [8, 256]");
  if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % (c->scheme == KV_MXFP4 ? 32 : 16))
    return bad("head_dim must be a multiple of 16 (mxfp4: 32) in [16, 256]");
  if (c->kv_heads < 1 || c->kv_heads > 65535) return bad("kv_heads out of range");
  if (c->num_pages < 1 || c->num_pages > 0x7FFFFFFFll) return bad("num_pages out of range");
  o.k = static_cast<unsigned char *>(c->k);
  o.v = static_cast<unsigned char *>(c->v);
  o.ks = static_cast<unsigned char *>(c->k_scale);
  o.vs = static_cast<unsigned char *>(c->v_scale);
  o.pages = c->num_pages;
  o.page_size = c->page_size;
  o.page_shift = 0;
  while ((1 << o.page_shift) < o.page_size) ++o.page_shift;
  o.heads = c->kv_heads;
  o.dim = c->head_dim;
  o.scheme = c->scheme;
  o.dtype = c->dtype;
  o.row_bytes = c->scheme == KV_NONE ? o.dim * (c->dtype == TC_F32 ? 4 : 2) : c->scheme == KV_MXFP4 ? o.dim / 2 : o.dim;
  o.scale_bytes = c->scheme == KV_NONE ? 0 : c->scheme == KV_MXFP4 ? o.dim / 32 : 4;
  if (((uintptr_t)o.k | (uintptr_t)o.v) % 16) return bad("codes must be 16-byte aligned");
  if (c->scheme != KV_NONE && ((uintptr_t)o.ks | (uintptr_t)o.vs) % 4)
    return bad("scales must be 4-byte aligned");
  return TC_OK;
}

namespace kvc {

struct Move {
  KvCache c;
  void *k, *v;  // [tokens][heads][dim] with token and head strides (elements)
  int64_t k_tok, k_head, v_tok, v_head;
  const int64_t *slots;
  int64_t tokens;
};

constexpr int kThreads = 256;

// Row index of (slot, head) in the pool; -1 for a slot outside it (padding tokens have slot -1).
__device__ __forceinline__ int64_t pool_row(const KvCache &c, int64_t slot, int head) {
  if (slot < 0 || slot >= (c.pages << c.page_shift)) return -1;
  return (((slot >> c.page_shift) * c.heads + head) << c.page_shift) + (slot & (c.page_size - 1));
}

// A warp a row (token, head, side).
template <typename T, int S>
__global__ void __launch_bounds__(kThreads) write_kernel(Move m) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = m.tokens * m.c.heads * 2;
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < rows;
       i += (int64_t)gridDim.x * (kThreads / 32)) {
    const int side = (int)(i & 1);
    const int64_t token = (i >> 1) / m.c.heads;
    const int head = (int)((i >> 1) % m.c.heads);
    const int64_t row = pool_row(m.c, m.slots[token], head);
    if (row < 0) continue;
    const T *x = side ? static_cast<const T *>(m.v) + token * m.v_tok + head * m.v_head
                      : static_cast<const T *>(m.k) + token * m.k_tok + head * m.k_head;
    unsigned char *codes = (side ? m.c.v : m.c.k) + row * m.c.row_bytes;
    unsigned char *scales = (side ? m.c.vs : m.c.ks) + row * m.c.scale_bytes;
    if (S == KV_NONE) {
      for (int d = lane; d < m.c.dim; d += 32) reinterpret_cast<T *>(codes)[d] = x[d];
    } else if (S == KV_MXFP4) {
      for (int d = lane; d < m.c.dim; d += 32) {
        const float v = Io<T>::get(x[d]);
        const uint32_t sc = pow2_code(warp_max(abs_bits(v)), 2);
        const uint32_t c = encode_e2m1(__fmul_rn(v, pow2_inverse(sc)));
        const uint32_t next = __shfl_down_sync(0xFFFFFFFFu, c, 1);
        if (!(lane & 1)) codes[d >> 1] = (unsigned char)(c | (next << 4));
        if (lane == 0) scales[d >> 5] = (unsigned char)sc;
      }
    } else {
      uint32_t top = 0u;
      for (int d = lane; d < m.c.dim; d += 32) top = max(top, abs_bits(Io<T>::get(x[d])));
      const float s = absmax_scale(warp_max(top), S == KV_FP8_ROW ? 448.0f : 127.0f);
      if (lane == 0) *reinterpret_cast<float *>(scales) = s;
      for (int d = lane; d < m.c.dim; d += 32)
        codes[d] = (unsigned char)encode8<S == KV_FP8_ROW ? E8_E4M3 : E8_INT8>(__fdiv_rn(Io<T>::get(x[d]), s));
    }
  }
}

// Value of element d of a pool row, in fp32: code * scale with one rounding (exact for mxfp4).
template <typename T, int S>
__device__ __forceinline__ float element(const unsigned char *codes, const unsigned char *scales, int d) {
  if (S == KV_NONE) return Io<T>::get(reinterpret_cast<const T *>(codes)[d]);
  if (S == KV_MXFP4) return __fmul_rn(decode_e2m1((codes[d >> 1] >> (4 * (d & 1))) & 15u), pow2_value(scales[d >> 5]));
  const float s = *reinterpret_cast<const float *>(scales);
  return __fmul_rn(S == KV_FP8_ROW ? decode_e4m3(codes[d]) : (float)(signed char)codes[d], s);
}

template <typename T, int S>
__global__ void __launch_bounds__(kThreads) read_kernel(Move m) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = m.tokens * m.c.heads * 2;
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < rows;
       i += (int64_t)gridDim.x * (kThreads / 32)) {
    const int side = (int)(i & 1);
    const int64_t token = (i >> 1) / m.c.heads;
    const int head = (int)((i >> 1) % m.c.heads);
    const int64_t row = pool_row(m.c, m.slots[token], head);
    T *x = side ? static_cast<T *>(m.v) + token * m.v_tok + head * m.v_head
                : static_cast<T *>(m.k) + token * m.k_tok + head * m.k_head;
    const unsigned char *codes = (side ? m.c.v : m.c.k) + (row < 0 ? 0 : row) * m.c.row_bytes;
    const unsigned char *scales = (side ? m.c.vs : m.c.ks) + (row < 0 ? 0 : row) * m.c.scale_bytes;
    for (int d = lane; d < m.c.dim; d += 32) x[d] = Io<T>::put(row < 0 ? 0.0f : element<T, S>(codes, scales, d));
  }
}

template <typename T, int S>
static void launch(const Move &m, bool write, cudaStream_t s) {
  const int64_t want = (m.tokens * m.c.heads * 2 + kThreads / 32 - 1) / (kThreads / 32), most = (int64_t)sm_count() * 8;
  const unsigned grid = (unsigned)(want < most ? want : most);
  if (write) write_kernel<T, S><<<grid, kThreads, 0, s>>>(m);
  else read_kernel<T, S><<<grid, kThreads, 0, s>>>(m);
  count_launch();
}

template <typename T>
static void by_scheme(const Move &m, bool write, cudaStream_t s) {
  if (m.c.scheme == KV_NONE) launch<T, KV_NONE>(m, write, s);
  else if (m.c.scheme == KV_FP8_ROW) launch<T, KV_FP8_ROW>(m, write, s);
  else if (m.c.scheme == KV_INT8_ROW) launch<T, KV_INT8_ROW>(m, write, s);
  else launch<T, KV_MXFP4>(m, write, s);
}

static int move(const char *what, const tc_kv_cache *cache, const int64_t *slots, int64_t tokens, void *k, int64_t k_tok,
                int64_t k_head, void *v, int64_t v_tok, int64_t v_head, bool write, tc_stream stream) {
  Move m;
  const int st = kv_cache_check(cache, m.c);
  if (st != TC_OK) return st;
  if (tokens == 0) return TC_OK;
  if (tokens < 0 || tokens >= (1ll << 32) || !slots || !k || !v) {
    set_error(std::string(what) + ": bad argument");
    return TC_INVALID_ARGUMENT;
  }
  m.k = k;
  m.v = v;
  m.k_tok = k_tok;
  m.k_head = k_head;
  m.v_tok = v_tok;
  m.v_head = v_head;
  m.slots = slots;
  m.tokens = tokens;
  cudaStream_t s = (cudaStream_t)stream;
  if (m.c.dtype == TC_F32) by_scheme<float>(m, write, s);
  else if (m.c.dtype == TC_BF16) by_scheme<__nv_bfloat16>(m, write, s);
  else by_scheme<__half>(m, write, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(std::string(what) + ": " + cudaGetErrorString(e)), TC_CUDA_ERROR;
  return TC_OK;
}

}  // namespace kvc
}  // namespace tc

extern "C" int tc_kv_write(const tc_kv_cache *cache, const void *k, int64_t k_token_stride, int64_t k_head_stride,
                           const void *v, int64_t v_token_stride, int64_t v_head_stride, const int64_t *slots,
                           int64_t tokens, tc_stream stream) {
  return tc::kvc::move("tc_kv_write", cache, slots, tokens, const_cast<void *>(k), k_token_stride, k_head_stride,
                       const_cast<void *>(v), v_token_stride, v_head_stride, true, stream);
}

extern "C" int tc_kv_read(const tc_kv_cache *cache, const int64_t *slots, int64_t tokens, void *k, void *v,
                          tc_stream stream) {
  const int64_t head = cache ? cache->head_dim : 0, token = cache ? head * cache->kv_heads : 0;
  return tc::kvc::move("tc_kv_read", cache, slots, tokens, k, token, head, v, token, head, false, stream);
}
