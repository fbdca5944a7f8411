// Paged key / value cache, quantized as it is written and read back: one scale (or one set of E8M0 group
// scales) per token and head, so that a token is written without touching its neighbours.
#include <string>

#include "tc_mma16.cuh"
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
  uint32_t rows;  // tokens * heads * 2
};

constexpr int kThreads = 256;

// Row index of (slot, head) in the pool; -1 for a slot outside it (padding tokens have slot -1).
__device__ __forceinline__ int64_t pool_row(const KvCache &c, int64_t slot, int head) {
  if (slot < 0 || slot >= (c.pages << c.page_shift)) return -1;
  return (((slot >> c.page_shift) * c.heads + head) << c.page_shift) + (slot & (c.page_size - 1));
}

constexpr int kOwn = 16;  // elements a lane: what finding a row costs is shared by them

// A lane's elements as they are stored; whole 16-byte words where rows start at such boundaries (VEC).
template <typename T>
struct Held {
  uint32_t w[kOwn * sizeof(T) / 4];
};
template <typename T, bool VEC>
__device__ __forceinline__ void fetch(const T *x, Held<T> &h) {
  if (VEC) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(Held<T>) / 16; ++k) {
      const uint4 v = reinterpret_cast<const uint4 *>(x)[k];
      h.w[4 * k] = v.x, h.w[4 * k + 1] = v.y, h.w[4 * k + 2] = v.z, h.w[4 * k + 3] = v.w;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < kOwn; ++k) h.w[k] = reinterpret_cast<const uint32_t *>(x)[k];
  } else {
    const unsigned short *u = reinterpret_cast<const unsigned short *>(x);
#pragma unroll
    for (int k = 0; k < kOwn / 2; ++k) h.w[k] = (uint32_t)u[2 * k] | ((uint32_t)u[2 * k + 1] << 16);
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store(T *x, const Held<T> &h) {
  if (VEC) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(Held<T>) / 16; ++k)
      reinterpret_cast<uint4 *>(x)[k] = make_uint4(h.w[4 * k], h.w[4 * k + 1], h.w[4 * k + 2], h.w[4 * k + 3]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < kOwn; ++k) reinterpret_cast<uint32_t *>(x)[k] = h.w[k];
  } else {
    unsigned short *u = reinterpret_cast<unsigned short *>(x);
#pragma unroll
    for (int k = 0; k < kOwn; ++k) u[k] = (unsigned short)(h.w[k >> 1] >> (16 * (k & 1)));
  }
}
template <typename T>
__device__ __forceinline__ float element_of(const Held<T> &h, int e) {
  if constexpr (sizeof(T) == 4) return u2f(h.w[e]);
  else if constexpr (Same<T, __nv_bfloat16>::value) return u2f(e & 1 ? h.w[e >> 1] & 0xFFFF0000u : h.w[e >> 1] << 16);
  else return __half2float(__ushort_as_half((unsigned short)(h.w[e >> 1] >> (16 * (e & 1)))));
}
// Bits of the largest magnitude as fp32: the order of the bits is that of the magnitudes in every type, NaN on
// top, so 16-bit ones are compared two at a time as they are.
template <typename T>
__device__ __forceinline__ uint32_t top_of(const Held<T> &h) {
  uint32_t m = 0u;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < kOwn; ++k) m = max(m, h.w[k] & 0x7FFFFFFFu);
    return m;
  } else {
#pragma unroll
    for (int k = 0; k < kOwn / 2; ++k) m = __vmaxu2(m, h.w[k] & 0x7FFF7FFFu);
    m = max(m & 0xFFFFu, m >> 16);
    if constexpr (Same<T, __nv_bfloat16>::value) return m << 16;
    else return f2u(__half2float(__ushort_as_half((unsigned short)m))) & 0x7FFFFFFFu;
  }
}

// The item (token, head, side) of a group of lanes that hold a row, 16 elements each. Rows follow one another by
// head within a token and side, so a warp's reads are whole lines.
struct RowOf {
  int64_t row;  // in the pool, -1 for none
  uint32_t token;
  int head, side;
};
__device__ __forceinline__ RowOf row_of(const Move &m, uint32_t i) {
  RowOf r{-1, 0u, 0, 0};
  if (i >= m.rows) return r;
  const uint32_t rest = i / (uint32_t)m.c.heads;
  r.head = (int)(i - rest * m.c.heads);
  r.side = (int)(rest & 1u);
  r.token = rest >> 1;
  r.row = pool_row(m.c, m.slots[r.token], r.head);
  return r;
}

// LANES (a power of two, at most 16) lanes a row of at most 16 LANES elements; VEC: rows start at 16-byte
// boundaries. A row is read once and written once, kFlight rows a group of lanes in flight. 32768 tokens of 8 heads of
// 128 in bf16 to E4M3, keys and values: 53.6 us, 3.8 TB/s; 71% of issue slots busy (finding rows, maxima, conversions),
// 38% of DRAM's cycles.
template <typename T>
constexpr int flight() {
  return sizeof(T) == 4 ? 2 : 4;
}
template <typename T, int S, int LANES, bool VEC>
__global__ void __launch_bounds__(kThreads) write_kernel(Move m) {
  constexpr int kFlight = flight<T>();
  const int lane = threadIdx.x % LANES, d0 = lane * kOwn;
  const uint32_t groups = gridDim.x * (kThreads / LANES), first = blockIdx.x * (kThreads / LANES);
  const bool have = d0 < m.c.dim;
  // Every lane of a block goes round equally often: the lanes of a row exchange values.
  for (uint32_t b0 = first; b0 < m.rows; b0 += groups * kFlight) {
    const uint32_t i0 = b0 + threadIdx.x / LANES;
    RowOf r[kFlight];
    Held<T> h[kFlight];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      r[f] = row_of(m, i0 + f * groups);
      if (!have) r[f].row = -1;
#pragma unroll
      for (int k = 0; k < (int)sizeof(Held<T>) / 4; ++k) h[f].w[k] = 0u;
      if (r[f].row >= 0)
        fetch<T, VEC>((r[f].side ? static_cast<const T *>(m.v) + r[f].token * m.v_tok + r[f].head * m.v_head
                                 : static_cast<const T *>(m.k) + r[f].token * m.k_tok + r[f].head * m.k_head) + d0, h[f]);
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      unsigned char *codes = (r[f].side ? m.c.v : m.c.k) + r[f].row * m.c.row_bytes;
      unsigned char *scales = (r[f].side ? m.c.vs : m.c.ks) + r[f].row * m.c.scale_bytes;
      const bool live = r[f].row >= 0;
      if (S == KV_NONE) {
        if (live) store<T, true>(reinterpret_cast<T *>(codes) + d0, h[f]);
        continue;
      }
      uint32_t top = top_of<T>(h[f]);
      // A row's lanes, or the two that share 32 elements.
#pragma unroll
      for (int k = 1; k < (S == KV_MXFP4 ? 2 : LANES); k <<= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, k));
      if (S == KV_MXFP4) {
        const uint32_t sc = pow2_code(top, 2);
        const float inv = pow2_inverse(sc);
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < kOwn; ++e) w[e >> 3] |= encode_e2m1(__fmul_rn(element_of<T>(h[f], e), inv)) << (4 * (e & 7));
        if (live) {
          *reinterpret_cast<uint2 *>(codes + d0 / 2) = make_uint2(w[0], w[1]);
          if ((lane & 1) == 0) scales[d0 / 32] = (unsigned char)sc;
        }
      } else {
        constexpr int E = S == KV_FP8_ROW ? E8_E4M3 : E8_INT8;
        const float s = absmax_scale(top, E == E8_E4M3 ? 448.0f : 127.0f);
        uint32_t q[4];
        if (divides_fast(s)) {
          const float rs = __frcp_rn(s);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = divide_fast(element_of<T>(h[f], 4 * k + e), s, rs);
            q[k] = encode8x2<E>(v[0], v[1]) | (encode8x2<E>(v[2], v[3]) << 16);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            q[k] = 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) q[k] |= encode8<E>(__fdiv_rn(element_of<T>(h[f], 4 * k + e), s)) << (8 * e);
          }
        }
        if (live) {
          *reinterpret_cast<uint4 *>(codes + d0) = make_uint4(q[0], q[1], q[2], q[3]);
          if (lane == 0) *reinterpret_cast<float *>(scales) = s;
        }
      }
    }
  }
}

// The same lanes: code * scale in fp32, rounded once to T (exact for mxfp4 in fp32 and bf16). 50021 tokens of 8 heads
// of 128 from INT8: 80 us, 3.9 TB/s; warps wait for loads, slot, then codes and scale (12.6 of 19 cycles an instruction).
template <typename T, int S, int LANES, bool VEC>
__global__ void __launch_bounds__(kThreads) read_kernel(Move m) {
  constexpr int kFlight = flight<T>();
  const int lane = threadIdx.x % LANES, d0 = lane * kOwn;
  const uint32_t groups = gridDim.x * (kThreads / LANES);
  if (d0 >= m.c.dim) return;
  for (uint32_t i0 = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES; i0 < m.rows; i0 += groups * kFlight) {
    RowOf r[kFlight];
    Held<T> h[kFlight];
    uint4 c[kFlight];
    float sc[kFlight];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      r[f] = row_of(m, i0 + f * groups);
      c[f] = make_uint4(0, 0, 0, 0);
      sc[f] = 0.0f;
#pragma unroll
      for (int k = 0; k < (int)sizeof(Held<T>) / 4; ++k) h[f].w[k] = 0u;
      if (r[f].row >= 0) {
        const unsigned char *codes = (r[f].side ? m.c.v : m.c.k) + r[f].row * m.c.row_bytes;
        const unsigned char *scales = (r[f].side ? m.c.vs : m.c.ks) + r[f].row * m.c.scale_bytes;
        if (S == KV_NONE) {
          fetch<T, true>(reinterpret_cast<const T *>(codes) + d0, h[f]);
        } else if (S == KV_MXFP4) {
          const uint2 w = *reinterpret_cast<const uint2 *>(codes + d0 / 2);
          c[f].x = w.x, c[f].y = w.y;
          sc[f] = pow2_value(scales[d0 / 32]);
        } else {
          c[f] = *reinterpret_cast<const uint4 *>(codes + d0);
          sc[f] = *reinterpret_cast<const float *>(scales);
        }
      }
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      if (i0 + f * groups >= m.rows) continue;
      T *x = (r[f].side ? static_cast<T *>(m.v) + r[f].token * m.v_tok + r[f].head * m.v_head
                        : static_cast<T *>(m.k) + r[f].token * m.k_tok + r[f].head * m.k_head) + d0;
      if (S != KV_NONE && r[f].row >= 0) {
        const uint32_t w[4] = {c[f].x, c[f].y, c[f].z, c[f].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float v[4];
          if (S == KV_MXFP4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = decode_e2m1((w[k >> 1] >> (4 * (4 * (k & 1) + e))) & 15u);
          } else if (S == KV_FP8_ROW) {
            uint32_t lo, hi;
            e4m3x4_half2(w[k], lo, hi);
            v[0] = half_bits_to_float<__half>(lo & 0xFFFFu), v[1] = half_bits_to_float<__half>(lo >> 16);
            v[2] = half_bits_to_float<__half>(hi & 0xFFFFu), v[3] = half_bits_to_float<__half>(hi >> 16);
          } else {
            // 2**23 + (v + 128) from the byte, less 2**23 + 128.
            const uint32_t u = w[k] ^ 0x80808080u;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __fsub_rn(u2f(__byte_perm(u, 0x4B000000u, 0x7440 + e)), 8388736.0f);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = __fmul_rn(v[e], sc[f]);
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) h[f].w[4 * k + e] = f2u(v[e]);
          } else {
            h[f].w[2 * k] = pack16<T>(v[0], v[1]);
            h[f].w[2 * k + 1] = pack16<T>(v[2], v[3]);
          }
        }
      }
      store<T, VEC>(x, h[f]);
    }
  }
}

template <typename T, int S, int LANES>
static void launch_lanes(const Move &m, bool write, cudaStream_t s) {
  const int64_t per = kThreads / LANES, want = (m.rows + per - 1) / per, most = (int64_t)sm_count() * 8;
  const unsigned grid = (unsigned)(want < most ? want : most);
  const int64_t strides = m.k_tok | m.k_head | m.v_tok | m.v_head;
  const bool vec = ((uintptr_t)m.k | (uintptr_t)m.v) % 16 == 0 && (strides * (int64_t)sizeof(T)) % 16 == 0;
  if (write) {
    if (vec) write_kernel<T, S, LANES, true><<<grid, kThreads, 0, s>>>(m);
    else write_kernel<T, S, LANES, false><<<grid, kThreads, 0, s>>>(m);
  } else {
    if (vec) read_kernel<T, S, LANES, true><<<grid, kThreads, 0, s>>>(m);
    else read_kernel<T, S, LANES, false><<<grid, kThreads, 0, s>>>(m);
  }
  count_launch();
}

template <typename T, int S>
static void launch(const Move &m, bool write, cudaStream_t s) {
  if (m.c.dim <= 32) launch_lanes<T, S, 2>(m, write, s);
  else if (m.c.dim <= 64) launch_lanes<T, S, 4>(m, write, s);
  else if (m.c.dim <= 128) launch_lanes<T, S, 8>(m, write, s);
  else launch_lanes<T, S, 16>(m, write, s);
}

template <typename T>
static void by_scheme(const Move &m, bool write, cudaStream_t s) {
  if (m.c.scheme == KV_NONE) launch<T, KV_NONE>(m, write, s);
  else if (m.c.scheme == KV_FP8_ROW) launch<T, KV_FP8_ROW>(m, write, s);
  else if (m.c.scheme == KV_INT8_ROW) launch<T, KV_INT8_ROW>(m, write, s);
  else launch<T, KV_MXFP4>(m, write, s);
}

static int64_t c_size(int dtype) { return dtype == TC_F32 ? 4 : 2; }

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
  m.k_tok = k_tok;
  m.k_head = k_head;
  m.v_tok = v_tok;
  m.v_head = v_head;
  cudaStream_t s = (cudaStream_t)stream;
  // Rows are counted in 32 bits: calls of more than 2**30 take several launches.
  const int64_t most = (1ll << 30) / (2 * m.c.heads), size = c_size(m.c.dtype);
  for (int64_t at = 0; at < tokens; at += most) {
    m.k = static_cast<char *>(k) + at * k_tok * size;
    m.v = static_cast<char *>(v) + at * v_tok * size;
    m.slots = slots + at;
    m.tokens = tokens - at < most ? tokens - at : most;
    m.rows = (uint32_t)(m.tokens * m.c.heads * 2);
    if (m.c.dtype == TC_F32) by_scheme<float>(m, write, s);
    else if (m.c.dtype == TC_BF16) by_scheme<__nv_bfloat16>(m, write, s);
    else by_scheme<__half>(m, write, s);
  }
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
