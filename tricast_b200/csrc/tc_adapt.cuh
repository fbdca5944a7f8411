// Low-rank adapters of many requests beside a shared projection:
//   out[t] = y[t] + gain[i] * B[i] (A[i] x[t]),  i = index[t]  (out[t] = y[t] where i names no adapter)
// x in 16 or 32 bits, or 8-bit codes with a scale a row; the products and their sum are fp32, out is rounded once.
//
// Measured: one token 4096 -> 6144, rank 16, fp32 to bf16 6.3 us; 64 tokens with as many adapters 4096 -> 4096, rank 32 12.6 us (5.5 for
// the bytes: waits for loads that follow one another, index, then A, then B); 8192 tokens of E4M3 codes 4096 -> 12288 157 us (4.1 TB/s;
// 98 for the bytes): 31 the first kernel, whose issue slots are 53% busy with widening codes and MMAs while loads are waited for, 124
// the second, 16 warps an SM that wait for y. Rank 32 194 us, rank 64 282. Tokens whose adapters alternate cost their products each: 374 us
// (360 with sums whose order goes by the number of adapters in the tile).
#pragma once

#include <cooperative_groups.h>

#include "tc_mma16.cuh"
#include "tc_serve.cuh"

namespace tc {
namespace adapt {

namespace cg = cooperative_groups;

// What x holds: a tc_dtype, or codes with scales.
enum { X_F32 = TC_F32, X_BF16 = TC_BF16, X_F16 = TC_F16, X_E4M3 = 3, X_E5M2 = 4, X_INT8 = 5 };

constexpr int kThreads = 256, kWarps = kThreads / 32, kMaxRank = 128;

struct Args {
  const void *y, *x, *a, *b;  // y [tokens][n], x [tokens][k] with row strides; a [adapters][rank][k], b [adapters][n][rank]
  const float *x_scale, *gain;
  const int32_t *index;
  void *out;  // [tokens][n]
  int64_t tokens, k, n, y_stride, x_stride;
  int rank, adapters, y_dtype, x_kind, w_dtype, out_dtype;
  int tile;    // tokens of a cluster, or of a block of the first kernel of two
  int blocks;  // of a cluster
  // Workspace of the two kernels: h in parts of 16 bits [tokens][terms][rows], and fp16's factors [tokens].
  uint16_t *parts;
  float *factors;
};

__host__ __device__ __forceinline__ int rank_rows(int rank) { return rank <= 16 ? 16 : (rank + 31) / 32 * 32; }

__device__ __forceinline__ float x_at(const Args &a, int64_t i) {
  if (a.x_kind <= X_F16) return load_as_float(a.x, a.x_kind, i);
  const uint32_t c = static_cast<const unsigned char *>(a.x)[i];
  if (a.x_kind == X_INT8) return (float)(int8_t)c;
  return a.x_kind == X_E4M3 ? decode_e4m3(c) : __half2float(__ushort_as_half((unsigned short)(c << 8)));
}

__device__ __forceinline__ void store_rounded(void *p, int dtype, int64_t i, float v) {
  if (dtype == TC_F32) static_cast<float *>(p)[i] = v;
  else if (dtype == TC_BF16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half *>(p)[i] = __float2half_rn(v);
}

// Eight codes as pairs of T: every code of 8 bits is exact in both 16-bit types.
template <typename T>
__device__ __forceinline__ uint4 widen(uint2 c, int kind) {
  uint32_t r[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t w = h ? c.y : c.x;
    if (kind == X_INT8) {
      const uint32_t u = w ^ 0x80808080u;  // 2**23 + 128 + v as fp32, less 2**23 + 128
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __fsub_rn(u2f(0x4B000000u | ((u >> (8 * e)) & 255u)), 8388736.0f);
      r[2 * h] = pack16<T>(v[0], v[1]), r[2 * h + 1] = pack16<T>(v[2], v[3]);
    } else {
      uint32_t lo, hi;
      if (kind == X_E4M3) e4m3x4_half2(w, lo, hi);
      else lo = __byte_perm(w, 0u, 0x1404), hi = __byte_perm(w, 0u, 0x3424);  // E5M2 is the upper byte of fp16
      if constexpr (Same<T, __nv_bfloat16>::value) {
        const float2 a = __half22float2(*reinterpret_cast<__half2 *>(&lo)), b = __half22float2(*reinterpret_cast<__half2 *>(&hi));
        lo = pack_bf16(a.x, a.y), hi = pack_bf16(b.x, b.y);
      }
      r[2 * h] = lo, r[2 * h + 1] = hi;
    }
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// N elements of 16 bits from p[at] on (N 4 or 8), zeros from `end` on.
template <int N, bool VEC>
__device__ __forceinline__ void load16(const uint16_t *p, int64_t at, int64_t end, uint32_t (&w)[N / 2]) {
  if (VEC) {
    if (at < end) {
      if constexpr (N == 8) {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p + at));
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p + at));
        w[0] = v.x, w[1] = v.y;
      }
    } else {
#pragma unroll
      for (int k = 0; k < N / 2; ++k) w[k] = 0u;
    }
  } else {
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      const uint32_t lo = at + 2 * k < end ? p[at + 2 * k] : 0u, hi = at + 2 * k + 1 < end ? p[at + 2 * k + 1] : 0u;
      w[k] = lo | (hi << 16);
    }
  }
}

// Eight elements of x[row] from k on, as they are: pairs of T, or codes in the first two words.
template <bool CODES, bool VEC>
__device__ __forceinline__ void load_x(const Args &a, int64_t row, int64_t k, uint32_t (&w)[4]) {
  if constexpr (!CODES) {
    load16<8, VEC>(static_cast<const uint16_t *>(a.x) + row * a.x_stride, k, a.k, w);
  } else {
    w[0] = w[1] = 0u;
    const unsigned char *p = static_cast<const unsigned char *>(a.x) + row * a.x_stride + k;
    if (VEC) {
      if (k < a.k) {
        const uint2 c = __ldg(reinterpret_cast<const uint2 *>(p));
        w[0] = c.x, w[1] = c.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k + e < a.k) w[e >> 2] |= (uint32_t)p[e] << (8 * (e & 3));
    }
  }
}

// Eight numbers of y[row] from n0 on: as they are in memory (y_floats widens them), or one by one.
template <bool VEC>
__device__ __forceinline__ void load_y(const Args &a, int64_t row, int64_t n0, int valid, uint4 (&u)[2], float (&v)[8]) {
  const int64_t at = row * a.y_stride + n0;
  if (VEC) {
    if (valid <= 0) return;
    if (a.y_dtype == TC_F32) {
      const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const float *>(a.y) + at);
      u[0] = __ldg(p), u[1] = __ldg(p + 1);
    } else {
      u[0] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.y) + at));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) v[e] = load_as_float(a.y, a.y_dtype, at + e);
  }
}
template <bool VEC>
__device__ __forceinline__ void y_floats(int dtype, const uint4 (&x)[2], float (&v)[8]) {
  if (!VEC) return;
  const uint32_t u[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
  if (dtype == TC_F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = u2f(u[e]);
  } else if (dtype == TC_BF16) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[2 * e] = u2f(u[e] << 16), v[2 * e + 1] = u2f(u[e] & 0xFFFF0000u);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[e]));
      v[2 * e] = f.x, v[2 * e + 1] = f.y;
    }
  }
}
template <bool VEC>
__device__ __forceinline__ void store_out(void *out, int dtype, int64_t at, int valid, const float (&v)[8]) {
  if (VEC) {
    if (valid <= 0) return;
    if (dtype == TC_F32) {
      float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(out) + at);
      p[0] = make_float4(v[0], v[1], v[2], v[3]), p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else if (dtype == TC_BF16) {
      *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out) + at) =
          make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    } else {
      *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out) + at) =
          make_uint4(pack_half(v[0], v[1]), pack_half(v[2], v[3]), pack_half(v[4], v[5]), pack_half(v[6], v[7]));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) store_rounded(out, dtype, at + e, v[e]);
  }
}

// The tokens of a tile and their adapters.
template <int NG>
struct Tile {
  int index[8 * NG], adapters[8 * NG];
  uint32_t members[8 * NG];  // of each distinct adapter, the groups of 8 tokens that it has
  int distinct;
  uint32_t peak[8 * NG];     // fp16: of each token, the largest |h| that is finite

  // One warp.
  __device__ __forceinline__ void fill(const Args &a, int64_t t0, int tokens) {
    constexpr int kEach = (8 * NG + 31) / 32;
    const int lane = threadIdx.x & 31;
    int mine[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int t = lane + 32 * i;
      mine[i] = t < tokens ? a.index[t0 + t] : -1;
      if (mine[i] >= a.adapters) mine[i] = -1;
      if (t < 8 * NG) index[t] = max(mine[i], -1), peak[t] = 0u;
    }
    int n = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      unsigned open;
      while ((open = __ballot_sync(0xFFFFFFFFu, mine[i] >= 0))) {
        const int v = __shfl_sync(0xFFFFFFFFu, mine[i], __ffs(open) - 1);
        uint32_t groups = 0u;
#pragma unroll
        for (int o = i; o < kEach; ++o) {
          const unsigned same = __ballot_sync(0xFFFFFFFFu, mine[o] == v);
#pragma unroll
          for (int b = 0; b < 4; ++b) groups |= ((same >> (8 * b)) & 255u ? 1u : 0u) << (4 * o + b);
          if (mine[o] == v) mine[o] = -1;
        }
        if (lane == 0) adapters[n] = v, members[n] = groups;
        ++n;
      }
    }
    if (lane == 0) distinct = n;
  }
};

// How many warps share a sum over k: as many as there are for every adapter (one at least) and block of RW rows of A. The sum itself
// is always cut into the slots that a single adapter has, which its warps take in turn: how many adapters a tile holds changes no token's bits.
__device__ __forceinline__ int splits_of(int count, int row_blocks) {
  int splits = kWarps;
  while (splits > 1 && splits * count * row_blocks > kWarps) splits >>= 1;
  return splits;
}

// Sums over the elements [32 c0, 32 c1) of x of a tile's tokens, each with its own adapter's rows: part [token][rows].
// m16n8k16 MMAs with A's rows in rows and tokens in columns, so a single token wastes none of A's traffic; operands go from memory to
// registers as vectors of 16 bytes, which the order of k inside a product allows: any, as long as both operands have the
// same. The distinct adapters are taken one by one, and a token's result is stored by its own only, so what is not
// finite in an adapter stays with its tokens.
template <typename T, int NG, int RW, bool CODES, bool VEC>
__device__ __forceinline__ void sum_rows(const Args &a, const Tile<NG> &tile, int64_t t0, int tokens, int64_t c0, int64_t c1, float *part) {
  constexpr int kTokens = 8 * NG, kRowTiles = RW / 16;
  constexpr bool kBf16 = Same<T, __nv_bfloat16>::value;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const uint16_t *A = static_cast<const uint16_t *>(a.a);
  const int rows = RW == 16 ? 16 : rank_rows(a.rank), row_blocks = RW == 16 ? 1 : rows / RW, count = tile.distinct;
  const int splits = splits_of(count, row_blocks), slots = splits_of(1, row_blocks);
  const int first = (int)c0, end = (int)c1;  // below 2**26
  for (int item = warp; item < count * row_blocks * splits; item += kWarps) {
    const int s = item % splits, rb = item / splits % row_blocks, j = item / splits / row_blocks;
    const int who = tile.adapters[j];
    const uint32_t has = tile.members[j];
    float acc[NG][kRowTiles][4];
    auto clear = [&] {
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r) acc[i][r][0] = acc[i][r][1] = acc[i][r][2] = acc[i][r][3] = 0.0f;
    };
    clear();
    constexpr int kAtOnce = !VEC ? 1 : NG == 2 ? 2 : RW == 16 ? 4 : 2;  // steps whose loads are on their way together
    int slot = s, c = first + s;
    while (slot < slots) {
      uint32_t w[kAtOnce][kRowTiles][2][4], x[kAtOnce][NG][4];
      int of[kAtOnce];     // the slot of each step, and whether it is its slot's last (an empty slot has one step, of zeros)
      bool last[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int64_t k = (int64_t)c * 32 + q * 8;
        const bool live = slot < slots && c < end;
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = rb * RW + r * 16 + h * 8 + g;
            load16<8, VEC>(A + ((int64_t)who * a.rank + row) * a.k, k, live && row < a.rank ? a.k : 0, w[u][r][h]);
          }
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          x[u][i][0] = x[u][i][1] = x[u][i][2] = x[u][i][3] = 0u;
          if (live && (has >> i & 1u) && i * 8 + g < tokens) load_x<CODES, VEC>(a, t0 + i * 8 + g, k, x[u][i]);
        }
        of[u] = slot;
        c += slots;
        last[u] = c >= end;
        if (last[u]) slot += splits, c = first + slot;
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (of[u] >= slots) break;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          if (!(has >> i & 1u)) continue;
          if (CODES) {  // after every load is on its way
            const uint4 v = widen<T>(make_uint2(x[u][i][0], x[u][i][1]), a.x_kind);
            x[u][i][0] = v.x, x[u][i][1] = v.y, x[u][i][2] = v.z, x[u][i][3] = v.w;
          }
#pragma unroll
          for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t f[4] = {w[u][r][0][2 * h], w[u][r][1][2 * h], w[u][r][0][2 * h + 1], w[u][r][1][2 * h + 1]};
              mma16<kBf16>(acc[i][r], f, x[u][i][2 * h], x[u][i][2 * h + 1]);
            }
        }
        if (!last[u]) continue;
#pragma unroll
        for (int i = 0; i < NG; ++i)
          if (has >> i & 1u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int t = i * 8 + q * 2 + e;
              if (tile.index[t] == who)
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r) {
                  float *to = part + ((int64_t)of[u] * kTokens + t) * rows + rb * RW + r * 16 + g;
                  to[0] = acc[i][r][e], to[8] = acc[i][r][2 + e];
                }
            }
        clear();
      }
    }
  }
  __syncthreads();
  for (int e = tid; e < kTokens * rows; e += kThreads) {
    float v = 0.0f;
    for (int s = 0; s < slots; ++s) v = __fadd_rn(v, part[s * kTokens * rows + e]);
    part[e] = v;
  }
}
// Floats of `part`, its splits included.
__host__ __device__ __forceinline__ size_t part_floats(int ng, int rw, int rows) { return (size_t)(kWarps / (rows / rw)) * 8 * ng * rows; }

// Of a number's magnitude the bits, 0 of what is not finite: what the power of two of fp16 parts goes by.
__device__ __forceinline__ uint32_t finite_bits(float v) { return abs_bits(v) < 0x7F800000u ? abs_bits(v) : 0u; }

// h in parts of 16 bits, each the rounded rest of the one before, `apart` elements from one another.
template <typename T>
__device__ __forceinline__ void split_parts(float v, int terms, uint16_t *to, int apart) {
  for (int p = 0; p < terms; ++p) {
    const uint32_t h = pack16<T>(v, 0.0f) & 0xFFFFu;
    to[p * apart] = (uint16_t)h;
    const float back = half_bits_to_float<T>(h);
    v = fabsf(back) < INFINITY ? __fsub_rn(v, back) : 0.0f;  // what is not finite stands in the first part
  }
}

// d = the products of one adapter's 64 columns (w: of its B the rows n0 + 2 k + h, n0 a lane's own) with eight tokens' h, a part
// after the other.
template <typename T, int RW>
__device__ __forceinline__ void multiply(const uint32_t (&w)[4][2][RW / 8], const uint32_t (&h)[RW / 8], float (&d)[4][4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int st = 0; st < RW / 16; ++st) {
      const uint32_t f[4] = {w[k][0][2 * st], w[k][1][2 * st], w[k][0][2 * st + 1], w[k][1][2 * st + 1]};
      mma16<Same<T, __nv_bfloat16>::value>(d[k], f, h[2 * st], h[2 * st + 1]);
    }
}
template <int RW>
__device__ __forceinline__ void load_h(const uint16_t *from, uint32_t (&h)[RW / 8]) {
  if constexpr (RW == 32) {
    const uint4 v = *reinterpret_cast<const uint4 *>(from);
    h[0] = v.x, h[1] = v.y, h[2] = v.z, h[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2 *>(from);
    h[0] = v.x, h[1] = v.y;
  }
}
template <int RW, bool VEC>
__device__ __forceinline__ void load_rows(const Args &a, int who, int64_t n0, int valid, int kc, int q, uint32_t (&w)[4][2][RW / 8]) {
  const uint16_t *from = static_cast<const uint16_t *>(a.b) + ((int64_t)who * a.n + n0) * a.rank;
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      load16<RW / 4, VEC>(from + (2 * k + h) * a.rank, kc * 32 + q * (RW / 4), 2 * k + h < valid ? a.rank : 0, w[k][h]);
}
// The sums of one of a lane's two tokens, on top of its y.
__device__ __forceinline__ void take(const float (&d)[4][4], int e, float factor, float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) v[2 * k] = __fmaf_rn(d[k][e], factor, v[2 * k]), v[2 * k + 1] = __fmaf_rn(d[k][2 + e], factor, v[2 * k + 1]);
}

// Few tokens: both products in one kernel. A cluster takes a tile of up to 8 tokens; its blocks share the sums over k, add them up through
// distributed shared memory, and share the columns of out. h = A x is fp32 and enters the second product in parts
// of 16 bits: two where out has 16 bits (2**-16 of h is left out), three where it has 32; fp16 parts are taken of h times a power of two, a
// token's own, that brings its largest to 2**13. The rows of B that come first are asked for before h is there.
template <typename T, int RW, bool CODES, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) tile_kernel(Args a) {
  constexpr int kTokens = 8;
  constexpr bool kBf16 = Same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(16) unsigned char dynamic[];
  __shared__ Tile<1> tile;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int blocks = a.blocks, rank = (int)cluster.block_rank();
  const int64_t t0 = (int64_t)(blockIdx.x / blocks) * a.tile;
  const int tokens = (int)min((int64_t)a.tile, a.tokens - t0);
  if (warp == 0) tile.fill(a, t0, tokens);
  __syncthreads();
  const int count = tile.distinct, rows = RW == 16 ? 16 : rank_rows(a.rank), row_blocks = RW == 16 ? 1 : rows / RW;
  const int row_stride = rows + 8;                     // of h's parts: rows of 16 bytes more, against bank conflicts
  float *part = reinterpret_cast<float *>(dynamic);    // [splits][kTokens][rows]
  uint16_t *parts = reinterpret_cast<uint16_t *>(part + part_floats(1, RW, rows));
  float *full = reinterpret_cast<float *>(parts + 3 * kTokens * row_stride);  // fp16: h
  const int terms = a.out_dtype == TC_F32 ? 3 : 2;

  // Columns: a warp takes 64 at a time, a lane 8 neighbouring ones of two tokens.
  const int64_t columns = (a.n + 63) / 64, share = (columns + blocks - 1) / blocks, c1 = min(share * (rank + 1), columns);
  int64_t c = share * rank + warp;
  uint32_t w[4][2][RW / 8];
  uint4 u[2][2];
  float v[2][8];
  auto valid_at = [&](int64_t column) { return (int)min(max(a.n - column * 64 - g * 8, (int64_t)0), (int64_t)8); };
  auto ask_rows = [&](int64_t column, int j) {
    if (row_blocks == 1 && column < c1 && j < count) load_rows<RW, VEC>(a, tile.adapters[j], column * 64 + g * 8, valid_at(column), 0, q, w);
  };
  auto ask_y = [&](int64_t column) {
    if (column < c1)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        load_y<VEC>(a, t0 + q * 2 + e, column * 64 + g * 8, q * 2 + e < tokens ? valid_at(column) : 0, u[e], v[e]);
  };
  ask_y(c);
  ask_rows(c, 0);

  if (count) {
    const int64_t chunks = (a.k + 31) / 32, each = (chunks + blocks - 1) / blocks, k0 = min(each * rank, chunks);
    sum_rows<T, 1, RW, CODES, VEC>(a, tile, t0, tokens, k0, min(k0 + each, chunks), part);
    cluster.sync();
    for (int e = tid; e < kTokens * rows; e += kThreads) {
      const int t = e / rows, r = e - t * rows, who = tile.index[t];
      float x = 0.0f;
      if (who >= 0 && r < a.rank) {  // 0 behind the rank: there A's zeros would make NaN of an infinite x
        for (int b = 0; b < blocks; ++b) x = __fadd_rn(x, *cluster.map_shared_rank(part + e, b));
        float f = a.x_scale ? a.x_scale[t0 + t] : 1.0f;
        if (a.gain) f = __fmul_rn(f, a.gain[who]);
        x = __fmul_rn(x, f);
      }
      if (kBf16) split_parts<T>(x, terms, parts + t * row_stride + r, kTokens * row_stride);
      else full[e] = x, atomicMax(&tile.peak[t], finite_bits(x));
    }
    __syncthreads();
    if (!kBf16) {
      for (int e = tid; e < kTokens * rows; e += kThreads) {
        const int t = e / rows;
        split_parts<T>(__fmul_rn(full[e], fp16_shift(u2f(tile.peak[t])).factor), terms, parts + t * row_stride + e - t * rows,
                       kTokens * row_stride);
      }
      __syncthreads();
    }
  }

  const int who0 = tile.index[q * 2], who1 = tile.index[q * 2 + 1];
  for (; c < c1; c += kWarps) {
    const int64_t n0 = c * 64 + g * 8;
    const int valid = valid_at(c);
    float y[2][8];
    y_floats<VEC>(a.y_dtype, u[0], v[0]), y_floats<VEC>(a.y_dtype, u[1], v[1]);
#pragma unroll
    for (int k = 0; k < 8; ++k) y[0][k] = v[0][k], y[1][k] = v[1][k];
    ask_y(c + kWarps);
    for (int j = 0; j < count; ++j) {
      const int who = tile.adapters[j];
      float d[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) d[k][0] = d[k][1] = d[k][2] = d[k][3] = 0.0f;
      for (int kc = 0; kc < row_blocks; ++kc) {
        if (row_blocks > 1) load_rows<RW, VEC>(a, who, n0, valid, kc, q, w);
        for (int p = 0; p < terms; ++p) {
          uint32_t h[RW / 8];
          load_h<RW>(parts + (p * kTokens + g) * row_stride + kc * 32 + q * (RW / 4), h);
          multiply<T, RW>(w, h, d);
        }
      }
      if (j + 1 < count) ask_rows(c, j + 1);
      else ask_rows(c + kWarps, 0);
      if (who0 == who) take(d, 0, kBf16 ? 1.0f : fp16_shift(u2f(tile.peak[q * 2])).inverse, y[0]);
      if (who1 == who) take(d, 1, kBf16 ? 1.0f : fp16_shift(u2f(tile.peak[q * 2 + 1])).inverse, y[1]);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) store_out<VEC>(a.out, a.out_dtype, (t0 + q * 2 + e) * a.n + n0, q * 2 + e < tokens ? valid : 0, y[e]);
  }
  if (count) cluster.sync();  // the other blocks may still read this one's sums
}

// Many tokens, in two kernels. h first: a cluster a tile of tokens, whose blocks share the sums over k, and then the tokens.
template <typename T, int NG, int RW, bool CODES, bool VEC>
__global__ void __launch_bounds__(kThreads, RW == 16 ? 4 : 3) down_kernel(Args a) {
  constexpr int kTokens = 8 * NG;
  constexpr bool kBf16 = Same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(16) unsigned char dynamic[];
  __shared__ Tile<NG> tile;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, blocks = a.blocks, rank = (int)cluster.block_rank();
  const int64_t t0 = (int64_t)(blockIdx.x / blocks) * kTokens;
  const int tokens = (int)min((int64_t)kTokens, a.tokens - t0);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid < 32) tile.fill(a, t0, tokens);
  __syncthreads();
  if (tile.distinct == 0) return;  // nobody reads the tile's h
  const int rows = RW == 16 ? 16 : rank_rows(a.rank), terms = a.out_dtype == TC_F32 ? 3 : 2;
  float *part = reinterpret_cast<float *>(dynamic);
  const int64_t chunks = (a.k + 31) / 32, each = (chunks + blocks - 1) / blocks, c0 = min(each * rank, chunks);
  sum_rows<T, NG, RW, CODES, VEC>(a, tile, t0, tokens, c0, min(c0 + each, chunks), part);
  cluster.sync();
  auto sum = [&](int e, int t, int who) {
    float v = 0.0f;
    for (int b = 0; b < blocks; ++b) v = __fadd_rn(v, *cluster.map_shared_rank(part + e, b));
    float f = a.x_scale ? a.x_scale[t0 + t] : 1.0f;
    if (a.gain) f = __fmul_rn(f, a.gain[who]);
    return __fmul_rn(v, f);
  };
  const int warp = tid >> 5, lane = tid & 31;
  for (int t = rank * kWarps + warp; t < tokens; t += blocks * kWarps) {  // a warp a token
    const int who = tile.index[t];
    if (who < 0) continue;
    float v[kMaxRank / 32];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxRank / 32; ++i) {
      const int r = lane + 32 * i;
      v[i] = r < a.rank ? sum(t * rows + r, t, who) : 0.0f;  // as above
      if (!kBf16) top = fmaxf(top, u2f(finite_bits(v[i])));
    }
    float factor = 1.0f;
    if (!kBf16) {
      const Pow2 p = fp16_shift(u2f(warp_max(f2u(top))));
      factor = p.factor;
      if (lane == 0) a.factors[t0 + t] = p.inverse;
    }
#pragma unroll
    for (int i = 0; i < kMaxRank / 32; ++i)
      if (lane + 32 * i < rows) split_parts<T>(__fmul_rn(v[i], factor), terms, a.parts + (t0 + t) * terms * rows + lane + 32 * i, rows);
  }
  cluster.sync();  // the other blocks may still read this one's sums
}

// Then out, with tokens in the MMAs' rows and columns of out in their columns: a warp takes 32 columns and a run of tokens, a lane 8
// neighbouring columns of two tokens of each sixteen, so that four lanes read and write a token's columns side by side (with columns in the
// rows, as above, every quarter of a warp touched four lines at a time, and L1 was the fullest resource). The rows of B stay in
// registers as long as the adapter does; y and the adapters of the next sixteen tokens are on their way while these are computed. Y, O: y and out have 32 bits (else 16). In bf16 with 16 bits out, y is
// what the products are added to in the MMAs, whatever adapters the sixteen have; otherwise it is added in fp32 behind them.
template <typename T, int RW, bool Y, bool O, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) up_kernel(Args a) {
  constexpr bool kBf16 = Same<T, __nv_bfloat16>::value;
  constexpr int kTerms = O ? 3 : 2, kWords = RW / 8;
  constexpr bool kOnY = kBf16 && !O;
  const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int64_t columns = (a.n + 31) / 32, item = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int64_t run = item / columns, base = (item - run * columns) * 32, n0 = base + q * 8, t0 = run * a.tile;
  if (t0 >= a.tokens) return;
  int left = (int)min((int64_t)a.tile, a.tokens - t0);
  const int valid = (int)min(max(a.n - n0, (int64_t)0), (int64_t)8);
  const int rows = RW == 16 ? 16 : rank_rows(a.rank), row_blocks = RW == 16 ? 1 : rows / RW;
  int64_t token = t0 + g;  // this lane's first; the other one stands 8 behind it
  const int32_t *index = a.index + token;
  int64_t y_at = token * a.y_stride + n0, out_at = token * a.n + n0;
  const uint16_t *parts = a.parts + token * kTerms * rows + q * (RW / 4);
  // Beyond 32 ranks the rows of B stand in shared memory, a lane's own pieces of 16 bytes side by side with the other lanes'.
  extern __shared__ __align__(16) unsigned char dynamic[];
  uint4 *kept = reinterpret_cast<uint4 *>(dynamic) + (size_t)(threadIdx.x >> 5) * row_blocks * 4 * 32 + lane;
  uint32_t w[4][kWords], h[kTerms][2][kWords];
  int loaded = -1, who[2];
  uint4 u[2][Y ? 2 : 1];
  float v[2][VEC ? 1 : 8];
  auto ask = [&](int64_t y_from, const int32_t *from, int tokens) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool real = g + 8 * e < tokens;
      who[e] = real ? __ldg(from + 8 * e) : -1;
      const int64_t at = y_from + 8 * e * a.y_stride;
      if constexpr (!VEC) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[e][k] = real && k < valid ? load_as_float(a.y, a.y_dtype, at + k) : 0.0f;
      } else if (real && valid > 0) {
        if constexpr (Y) {
          const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const float *>(a.y) + at);
          u[e][0] = __ldg(p), u[e][1] = __ldg(p + 1);
        } else {
          u[e][0] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.y) + at));
        }
      }
    }
  };
  auto load_parts = [&](const uint16_t *from, int tokens, uint32_t (&x)[kTerms][2][kWords]) {
#pragma unroll
    for (int p = 0; p < kTerms; ++p)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (g + 8 * e < tokens) load_h<RW>(from + (8 * e * kTerms + p) * rows, x[p][e]);
  };
  // Of one adapter's B the rows of this lane's column of each MMA: column c of the j-th is the warp's 8 (c / 2) + 2 j + c % 2.
  auto load_b = [&](int i, int kc) {
    const int64_t column = base + (g >> 1) * 8 + (g & 1);
    const uint16_t *from = static_cast<const uint16_t *>(a.b) + ((int64_t)i * a.n + column) * a.rank;
#pragma unroll
    for (int j = 0; j < 4; ++j) load16<RW / 4, VEC>(from + 2 * j * a.rank, kc * 32 + q * (RW / 4), column + 2 * j < a.n ? a.rank : 0, w[j]);
  };
#pragma unroll
  for (int p = 0; p < kTerms; ++p)
#pragma unroll
    for (int k = 0; k < kWords; ++k) h[p][0][k] = h[p][1][k] = 0u;
  ask(y_at, index, left);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the first kernel's h
  if (row_blocks == 1) load_parts(parts, left, h);
  for (; left > 0; left -= 16) {
    float y[2][8];
    int mine[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mine[e] = (unsigned)who[e] < (unsigned)a.adapters ? who[e] : -1;
      if constexpr (!VEC) {
#pragma unroll
        for (int k = 0; k < 8; ++k) y[e][k] = v[e][k];
      } else if constexpr (Y) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          y[e][4 * k] = u2f(u[e][k].x), y[e][4 * k + 1] = u2f(u[e][k].y), y[e][4 * k + 2] = u2f(u[e][k].z), y[e][4 * k + 3] = u2f(u[e][k].w);
      } else {
        const uint32_t x[4] = {u[e][0].x, u[e][0].y, u[e][0].z, u[e][0].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) y[e][2 * k] = half_bits_to_float<T>(x[k] & 0xFFFFu), y[e][2 * k + 1] = half_bits_to_float<T>(x[k] >> 16);
      }
    }
    y_at += 16 * a.y_stride, index += 16;
    ask(y_at, index, left - 16);

    float d[4][4];
    // The products of one adapter with the sixteen tokens, on top of d, a part of h after the other.
    auto multiply_parts = [&](const uint32_t (&x)[kTerms][2][kWords]) {
#pragma unroll
      for (int p = 0; p < kTerms; ++p)
#pragma unroll
        for (int st = 0; st < RW / 16; ++st) {
          const uint32_t f[4] = {x[p][0][2 * st], x[p][1][2 * st], x[p][0][2 * st + 1], x[p][1][2 * st + 1]};
#pragma unroll
          for (int j = 0; j < 4; ++j) mma16<kBf16>(d[j], f, w[j][2 * st], w[j][2 * st + 1]);
        }
    };
    auto products = [&](int i) {
      if (row_blocks == 1) {
        if (loaded != i) load_b(i, 0);
        multiply_parts(h);
      } else if constexpr (RW == 32) {
        for (int kc = 0; kc < row_blocks; ++kc) {
          uint4 *piece = kept + kc * 4 * 32;
          if (loaded != i) {
            load_b(i, kc);
#pragma unroll
            for (int j = 0; j < 4; ++j) piece[j * 32] = make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint4 x = piece[j * 32];
              w[j][0] = x.x, w[j][1] = x.y, w[j][2] = x.z, w[j][3] = x.w;
            }
          }
          uint32_t x[kTerms][2][kWords];
#pragma unroll
          for (int p = 0; p < kTerms; ++p)
#pragma unroll
            for (int k = 0; k < kWords; ++k) x[p][0][k] = x[p][1][k] = 0u;
          load_parts(parts + kc * 32, left, x);
          multiply_parts(x);
        }
      }
      loaded = i;
    };
    const int one = __shfl_sync(0xFFFFFFFFu, mine[0], 0);
    if (kOnY && one >= 0 && __all_sync(0xFFFFFFFFu, mine[0] == one && mine[1] == one)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j][0] = y[0][2 * j], d[j][1] = y[0][2 * j + 1], d[j][2] = y[1][2 * j], d[j][3] = y[1][2 * j + 1];
      products(one);
#pragma unroll
      for (int j = 0; j < 4; ++j) y[0][2 * j] = d[j][0], y[0][2 * j + 1] = d[j][1], y[1][2 * j] = d[j][2], y[1][2 * j + 1] = d[j][3];
    } else {
      unsigned open[2] = {__ballot_sync(0xFFFFFFFFu, mine[0] >= 0), __ballot_sync(0xFFFFFFFFu, mine[1] >= 0)};
      while (open[0] | open[1]) {
        const int i = open[0] ? __shfl_sync(0xFFFFFFFFu, mine[0], __ffs(open[0]) - 1) : __shfl_sync(0xFFFFFFFFu, mine[1], __ffs(open[1]) - 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          d[j][0] = d[j][1] = d[j][2] = d[j][3] = 0.0f;
          if (kOnY) d[j][0] = y[0][2 * j], d[j][1] = y[0][2 * j + 1], d[j][2] = y[1][2 * j], d[j][3] = y[1][2 * j + 1];
        }
        products(i);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (kOnY && mine[e] == i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) y[e][2 * j] = d[j][2 * e], y[e][2 * j + 1] = d[j][2 * e + 1];
          } else if (mine[e] == i) {
            const float factor = kBf16 ? 1.0f : a.factors[token + 8 * e];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              y[e][2 * j] = __fmaf_rn(d[j][2 * e], factor, y[e][2 * j]), y[e][2 * j + 1] = __fmaf_rn(d[j][2 * e + 1], factor, y[e][2 * j + 1]);
          }
          open[e] &= ~__ballot_sync(0xFFFFFFFFu, mine[e] == i);
        }
      }
    }
    parts += 16 * kTerms * rows;
    if (row_blocks == 1) load_parts(parts, left - 16, h);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      store_out<VEC>(a.out, O ? TC_F32 : kBf16 ? TC_BF16 : TC_F16, out_at + 8 * e * a.n, g + 8 * e < left ? valid : 0, y[e]);
    out_at += 16 * a.n, token += 16;
  }
}

static cudaLaunchConfig_t config(int64_t blocks, size_t bytes, cudaStream_t s, cudaLaunchAttribute *attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = attr ? 1 : 0;
  return cfg;
}

template <typename K>
static cudaError_t room(K kernel, size_t bytes) {
  return bytes > 48 << 10 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) : cudaSuccess;
}

template <typename T, int RW, bool CODES, bool VEC>
static cudaError_t launch_tiles(const Args &a, cudaStream_t s) {
  const int rows = rank_rows(a.rank);
  const size_t bytes = part_floats(1, RW, rows) * sizeof(float) + (size_t)3 * 8 * (rows + 8) * sizeof(uint16_t) +
                       (Same<T, __half>::value ? (size_t)8 * rows * sizeof(float) : 0);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  const cudaLaunchConfig_t cfg = config((a.tokens + a.tile - 1) / a.tile * a.blocks, bytes, s, &attr);
  const cudaError_t e = room(tile_kernel<T, RW, CODES, VEC>, bytes);
  return e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, tile_kernel<T, RW, CODES, VEC>, a);
}

constexpr int kDownGroups = 2;  // of 8 tokens, a block of the first kernel

template <typename T, int RW, bool CODES, bool VEC>
static cudaError_t launch_two(Args a, cudaStream_t s) {
  const size_t bytes = part_floats(kDownGroups, RW, rank_rows(a.rank)) * sizeof(float);
  cudaError_t e = room(down_kernel<T, kDownGroups, RW, CODES, VEC>, bytes);
  if (e != cudaSuccess) return e;
  const int64_t tiles = (a.tokens + 8 * kDownGroups - 1) / (8 * kDownGroups);
  a.blocks = 1;
  while (a.blocks < 8 && tiles * a.blocks < 4 * (int64_t)sm_count()) a.blocks *= 2;  // a wave: four an SM
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = config(tiles * a.blocks, bytes, s, &attr);
  e = cudaLaunchKernelEx(&cfg, down_kernel<T, kDownGroups, RW, CODES, VEC>, a);
  if (e != cudaSuccess) return e;
  count_launch();
  const int64_t columns = (a.n + 31) / 32;
  a.tile = 128;
  while (a.tile > 16 && (a.tokens + a.tile - 1) / a.tile * columns < 48 * (int64_t)sm_count()) a.tile /= 2;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  const int row_blocks = rank_rows(a.rank) / RW;
  const size_t kept = row_blocks > 1 ? (size_t)kWarps * row_blocks * 4 * 512 : 0;
  cfg = config(((a.tokens + a.tile - 1) / a.tile * columns + kWarps - 1) / kWarps, kept, s, &attr);
  auto up = [&](auto kernel) {
    const cudaError_t r = room(kernel, kept);
    return r != cudaSuccess ? r : cudaLaunchKernelEx(&cfg, kernel, a);
  };
  if (!VEC) {  // any type of y
    return a.out_dtype == TC_F32 ? up(up_kernel<T, RW, false, true, false>)
                                 : up(up_kernel<T, RW, false, false, false>);
  }
  if (a.y_dtype == TC_F32)
    return a.out_dtype == TC_F32 ? up(up_kernel<T, RW, true, true, true>)
                                 : up(up_kernel<T, RW, true, false, true>);
  return a.out_dtype == TC_F32 ? up(up_kernel<T, RW, false, true, true>)
                               : up(up_kernel<T, RW, false, false, true>);
}

// Up to this many tokens one kernel does both products: a little less than what clusters of 8 blocks with 8 tokens each hold when the
// card is full. One and two kernels, us, 4096 -> 4096, rank 16, fp32 to bf16: runs of 6 adapters, 64 tokens 7.4 and 7.4, 160 8.2 and 7.9,
// 256 8.3 and 8.1, 296 13.0 and 9.0; an adapter of 64 a token, 64 tokens 8.3 and 25, 160 18 and 27, 256 19 and 31, 296 33 and 32, 400 31 and 39,
// 600 55 and 48.
inline int64_t few_tokens() { return (int64_t)sm_count() * 7 / 4; }

template <typename T, bool CODES>
static cudaError_t launch_two_as(const Args &a, bool vec, cudaStream_t s) {
  if (a.rank <= 16) return vec ? launch_two<T, 16, CODES, true>(a, s) : launch_two<T, 16, CODES, false>(a, s);
  return vec ? launch_two<T, 32, CODES, true>(a, s) : launch_two<T, 32, CODES, false>(a, s);
}
template <typename T, bool CODES>
static cudaError_t launch_tiles_as(const Args &a, bool vec, cudaStream_t s) {
  if (a.rank <= 16) return vec ? launch_tiles<T, 16, CODES, true>(a, s) : launch_tiles<T, 16, CODES, false>(a, s);
  return vec ? launch_tiles<T, 32, CODES, true>(a, s) : launch_tiles<T, 32, CODES, false>(a, s);
}

template <typename T>
static cudaError_t launch_as(Args a, cudaStream_t s) {
  auto aligned = [](const void *p, size_t n) { return (uintptr_t)p % n == 0; };
  const int y16 = a.y_dtype == TC_F32 ? 4 : 8;
  const bool vec = a.k % 8 == 0 && a.n % 8 == 0 && a.rank % (a.rank <= 16 ? 4 : 8) == 0 && a.x_stride % 8 == 0 &&
                   a.y_stride % y16 == 0 && aligned(a.x, a.x_kind <= X_F16 ? 16 : 8) && aligned(a.y, 16) && aligned(a.a, 16) &&
                   aligned(a.b, 16) && aligned(a.out, 16);
  const bool codes = a.x_kind > X_F16;
  if (a.tokens > few_tokens()) return codes ? launch_two_as<T, true>(a, vec, s) : launch_two_as<T, false>(a, vec, s);
  // Tiles of at most 8 tokens, as small as the card holds clusters of 8 blocks for (two blocks an SM): tokens that share a tile
  // wait for one another's adapters. 4096 -> 4096, rank 32, us: 64 tokens with as many adapters, tiles of 1 by clusters of 4 11.0 and of
  // 8 14.9, of 2 by 4 13.6 and by 8 10.8, of 4 by 8 15.8; of one adapter tiles of 2 by 8 8.4, of 8 by 8 7.3; 32 tokens, tiles of 1 by 4
  // 9.5 and by 8 7.9, of 2 by 8 10.5; one token by 2, 4 and 8 9.7, 6.9 and 5.5 (rank 16).
  const int room = 2 * sm_count();
  a.tile = 1;
  while (a.tile < 8 && (a.tokens + a.tile - 1) / a.tile * 8 > room) a.tile *= 2;
  a.blocks = 1;
  while (a.blocks < 8 && (a.tokens + a.tile - 1) / a.tile * a.blocks * 2 <= room) a.blocks *= 2;
  return codes ? launch_tiles_as<T, true>(a, vec, s) : launch_tiles_as<T, false>(a, vec, s);
}

}  // namespace adapt
}  // namespace tc
