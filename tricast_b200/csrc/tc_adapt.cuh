// Low-rank adapters of many requests beside a shared projection:
//   out[t] = y[t] + gain[i] * B[i] (A[i] x[t]),  i = index[t]  (out[t] = y[t] where i names no adapter)
// x in 16 or 32 bits, or 8-bit codes with a scale a row; the products and their sum are fp32, out is rounded once.
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
  int tile;    // tokens of a cluster
  int blocks;  // of a cluster
};

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

// Eight elements of x[row] from k on.
template <typename T, bool VEC>
__device__ __forceinline__ void load_x(const Args &a, int64_t row, int64_t k, uint32_t (&w)[4]) {
  if (a.x_kind <= X_F16) {
    load16<8, VEC>(static_cast<const uint16_t *>(a.x) + row * a.x_stride, k, a.k, w);
  } else {
    uint2 c = make_uint2(0u, 0u);
    const unsigned char *p = static_cast<const unsigned char *>(a.x) + row * a.x_stride + k;
    if (VEC) {
      if (k < a.k) c = __ldg(reinterpret_cast<const uint2 *>(p));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k + e < a.k) (e < 4 ? c.x : c.y) |= (uint32_t)p[e] << (8 * (e & 3));
    }
    const uint4 v = widen<T>(c, a.x_kind);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
}

// Eight numbers of y or out, as they are in memory (fp32 in all of `u`, 16 bits in its first half).
template <bool VEC>
__device__ __forceinline__ void load_y(const void *y, int dtype, int64_t at, int valid, uint32_t (&u)[8]) {
  if (VEC) {
    if (valid <= 0) return;
    if (dtype == TC_F32) {
      const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const float *>(y) + at);
      const uint4 a = __ldg(p), b = __ldg(p + 1);
      u[0] = a.x, u[1] = a.y, u[2] = a.z, u[3] = a.w, u[4] = b.x, u[5] = b.y, u[6] = b.z, u[7] = b.w;
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(y) + at));
      u[0] = a.x, u[1] = a.y, u[2] = a.z, u[3] = a.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) u[e] = f2u(load_as_float(y, dtype, at + e));
  }
}
template <bool VEC>
__device__ __forceinline__ void y_floats(int dtype, const uint32_t (&u)[8], float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t half = (u[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
    v[e] = !VEC || dtype == TC_F32 ? u2f(u[e]) : dtype == TC_BF16 ? u2f(half << 16) : __half2float(__ushort_as_half((unsigned short)half));
  }
}
template <bool VEC>
__device__ __forceinline__ void store_out(void *out, int dtype, int64_t at, int valid, const float (&v)[8]) {
  if (VEC) {
    if (valid <= 0) return;
    if (dtype == TC_F32) {
      float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(out) + at);
      p[0] = make_float4(v[0], v[1], v[2], v[3]), p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = dtype == TC_BF16 ? pack_bf16(v[2 * e], v[2 * e + 1]) : pack_half(v[2 * e], v[2 * e + 1]);
      *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out) + at) = make_uint4(u[0], u[1], u[2], u[3]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) store_rounded(out, dtype, at + e, v[e]);
  }
}

// A cluster takes a tile of up to 8 NG tokens; its blocks share the sums over k, add them up through distributed shared memory, and
// share the columns of out. Both products run on m16n8k16 MMAs with weights in rows and tokens in columns, so a single token
// wastes none of the weights' traffic; operands go from memory to registers as vectors of 16 bytes (8 where a row of B has
// 16 ranks or fewer: RW), which the order of k inside a product allows: any, as long as both operands have the same.
// The tile's distinct adapters are taken in turn, each for the tokens that name it; a column's result is
// selected, not added, so what is not finite in an adapter stays with its tokens. h = A x is fp32 and enters the second
// product in parts of 16 bits, each the rounded rest of the one before: two where out has 16 bits (2**-16 of h is left out), three
// where it has 32. fp16 parts are taken of h times a power of two, a token's own, that brings its largest to 2**13.
template <typename T, int NG, int RW, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) tile_kernel(Args a) {
  constexpr int kTokens = 8 * NG, kRowTiles = RW / 16;
  constexpr bool kBf16 = Same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(16) unsigned char dynamic[];
  __shared__ int index[kTokens], adapters[kTokens];
  __shared__ uint32_t members[kTokens];  // of each distinct adapter, the groups of 8 tokens that it has
  __shared__ int distinct;
  __shared__ uint32_t peak[kTokens];     // fp16: of each token, the largest |h|
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int blocks = a.blocks, rank = (int)cluster.block_rank();
  const int64_t t0 = (int64_t)(blockIdx.x / blocks) * a.tile;
  const int tokens = (int)min((int64_t)a.tile, a.tokens - t0);
  const uint16_t *A = static_cast<const uint16_t *>(a.a), *B = static_cast<const uint16_t *>(a.b);

  if (warp == 0) {
    int mine[(kTokens + 31) / 32];
#pragma unroll
    for (int i = 0; i < (kTokens + 31) / 32; ++i) {
      const int t = lane + 32 * i;
      mine[i] = t < tokens ? a.index[t0 + t] : -1;
      if (mine[i] >= a.adapters) mine[i] = -1;
      if (t < kTokens) index[t] = max(mine[i], -1), peak[t] = 0u;
    }
    int n = 0;
#pragma unroll
    for (int i = 0; i < (kTokens + 31) / 32; ++i) {
      unsigned open;
      while ((open = __ballot_sync(0xFFFFFFFFu, mine[i] >= 0))) {
        const int v = __shfl_sync(0xFFFFFFFFu, mine[i], __ffs(open) - 1);
        uint32_t groups = 0u;
#pragma unroll
        for (int o = i; o < (kTokens + 31) / 32; ++o) {
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
  __syncthreads();
  const int count = distinct;

  const int rows = (a.rank + RW - 1) / RW * RW;        // of h, filled up with zeros
  const int row_blocks = rows / RW;
  int splits = kWarps;                                 // warps that share a sum over k
  while (splits > 1 && splits * count * row_blocks > kWarps) splits >>= 1;
  float *part = reinterpret_cast<float *>(dynamic);    // [splits][kTokens][rows]
  const int row_stride = rows + 8;                     // of h's parts: rows of 16 bytes more, against bank conflicts
  uint16_t *parts = reinterpret_cast<uint16_t *>(dynamic + (size_t)kWarps / row_blocks * kTokens * rows * sizeof(float));
  const int terms = a.out_dtype == TC_F32 ? 3 : 2;
  float *full = reinterpret_cast<float *>(parts + 3 * kTokens * row_stride);  // fp16: h
  auto split = [&](float v, int t, int r) {
    for (int p = 0; p < terms; ++p) {
      const uint32_t h = pack16<T>(v, 0.0f) & 0xFFFFu;
      parts[(p * kTokens + t) * row_stride + r] = (uint16_t)h;
      const float back = half_bits_to_float<T>(h);
      v = fabsf(back) < INFINITY ? __fsub_rn(v, back) : 0.0f;  // what is not finite stands in the first part
    }
  };

  if (count) {
    const int64_t chunks = (a.k + 31) / 32, each = (chunks + blocks - 1) / blocks;
    const int64_t c0 = min(each * rank, chunks), c1 = min(c0 + each, chunks);
    for (int item = warp; item < count * row_blocks * splits; item += kWarps) {
      const int s = item % splits, rb = item / splits % row_blocks, j = item / splits / row_blocks;
      const int who = adapters[j];
      const uint32_t groups = members[j];
      float acc[NG][kRowTiles][4];
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r) acc[i][r][0] = acc[i][r][1] = acc[i][r][2] = acc[i][r][3] = 0.0f;
#pragma unroll 2
      for (int64_t c = c0 + s; c < c1; c += splits) {
        const int64_t k = c * 32 + q * 8;
        uint32_t w[kRowTiles][2][4], x[NG][4];
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = rb * RW + r * 16 + h * 8 + g;
            load16<8, VEC>(A + ((int64_t)who * a.rank + row) * a.k, k, row < a.rank ? a.k : 0, w[r][h]);
          }
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0u;
          if ((groups >> i & 1u) && i * 8 + g < tokens) load_x<T, VEC>(a, t0 + i * 8 + g, k, x[i]);
        }
#pragma unroll
        for (int i = 0; i < NG; ++i)
          if (groups >> i & 1u)
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t f[4] = {w[r][0][2 * h], w[r][1][2 * h], w[r][0][2 * h + 1], w[r][1][2 * h + 1]};
                mma16<kBf16>(acc[i][r], f, x[i][2 * h], x[i][2 * h + 1]);
              }
      }
#pragma unroll
      for (int i = 0; i < NG; ++i)
        if (groups >> i & 1u)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int t = i * 8 + q * 2 + e;
            if (index[t] == who)
#pragma unroll
              for (int r = 0; r < kRowTiles; ++r) {
                float *to = part + ((int64_t)s * kTokens + t) * rows + rb * RW + r * 16 + g;
                to[0] = acc[i][r][e], to[8] = acc[i][r][2 + e];
              }
          }
    }
    __syncthreads();
    for (int e = tid; e < kTokens * rows; e += kThreads) {
      float v = 0.0f;
      for (int s = 0; s < splits; ++s) v = __fadd_rn(v, part[s * kTokens * rows + e]);
      part[e] = v;
    }
    cluster.sync();
    for (int e = tid; e < kTokens * rows; e += kThreads) {
      const int t = e / rows, r = e - t * rows, who = index[t];
      float v = 0.0f;
      if (who >= 0) {
        for (int b = 0; b < blocks; ++b) v = __fadd_rn(v, *cluster.map_shared_rank(part + e, b));
        float f = a.x_scale ? a.x_scale[t0 + t] : 1.0f;
        if (a.gain) f = __fmul_rn(f, a.gain[who]);
        v = __fmul_rn(v, f);
      }
      if (kBf16) split(v, t, r);
      else full[e] = v, atomicMax(&peak[t], abs_bits(v));
    }
    __syncthreads();
    if (!kBf16) {
      for (int e = tid; e < kTokens * rows; e += kThreads) {
        const int t = e / rows;
        split(__fmul_rn(full[e], fp16_shift(u2f(peak[t])).factor), t, e - t * rows);
      }
      __syncthreads();
    }
  }

  // Columns: a warp takes 64 at a time, a lane 8 neighbouring ones of two tokens.
  const int64_t chunks = (a.n + 63) / 64, each = (chunks + blocks - 1) / blocks;
  const int64_t c1 = min(each * (rank + 1), chunks);
  for (int64_t c = each * rank + warp; c < c1; c += kWarps) {
    const int64_t n0 = c * 64 + g * 8;
    const int valid = (int)min(max(a.n - n0, (int64_t)0), (int64_t)8);
    uint32_t w[4][2][RW / 8];  // the rows n0 + 2 i + h of one adapter
    int loaded = -1;
    auto load_rows = [&](int who, int kc) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t row = n0 + 2 * i + h;
          load16<RW / 4, VEC>(B + ((int64_t)who * a.n + row) * a.rank, kc * 32 + q * (RW / 4), row < a.n ? a.rank : 0, w[i][h]);
        }
    };
    for (int i = 0; i < NG; ++i) {
      if (i * 8 >= tokens) break;
      uint32_t u[2][8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = i * 8 + q * 2 + e;
        load_y<VEC>(a.y, a.y_dtype, (t0 + t) * a.y_stride + n0, t < tokens ? valid : 0, u[e]);
      }
      float sum[2][8];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[e][k] = 0.0f;
      const int who0 = index[i * 8 + q * 2], who1 = index[i * 8 + q * 2 + 1];
      for (int j = 0; j < count; ++j) {
        if (!(members[j] >> i & 1u)) continue;
        const int who = adapters[j];
        float d[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) d[k][0] = d[k][1] = d[k][2] = d[k][3] = 0.0f;
        for (int kc = 0; kc < row_blocks; ++kc) {
          if (row_blocks > 1 || loaded != who) load_rows(who, kc);
          for (int p = 0; p < terms; ++p) {
            uint32_t h[RW / 8];
            const uint16_t *from = parts + (p * kTokens + i * 8 + g) * row_stride + kc * 32 + q * (RW / 4);
            if constexpr (RW == 32) {
              const uint4 v = *reinterpret_cast<const uint4 *>(from);
              h[0] = v.x, h[1] = v.y, h[2] = v.z, h[3] = v.w;
            } else {
              const uint2 v = *reinterpret_cast<const uint2 *>(from);
              h[0] = v.x, h[1] = v.y;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int st = 0; st < RW / 16; ++st) {
                const uint32_t f[4] = {w[k][0][2 * st], w[k][1][2 * st], w[k][0][2 * st + 1], w[k][1][2 * st + 1]};
                mma16<kBf16>(d[k], f, h[2 * st], h[2 * st + 1]);
              }
          }
        }
        loaded = who;
        if (!kBf16) {
          const float f0 = fp16_shift(u2f(peak[i * 8 + q * 2])).inverse, f1 = fp16_shift(u2f(peak[i * 8 + q * 2 + 1])).inverse;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            d[k][0] = __fmul_rn(d[k][0], f0), d[k][2] = __fmul_rn(d[k][2], f0), d[k][1] = __fmul_rn(d[k][1], f1), d[k][3] = __fmul_rn(d[k][3], f1);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (who0 == who) sum[0][2 * k] = d[k][0], sum[0][2 * k + 1] = d[k][2];
          if (who1 == who) sum[1][2 * k] = d[k][1], sum[1][2 * k + 1] = d[k][3];
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = i * 8 + q * 2 + e;
        float v[8];
        y_floats<VEC>(a.y_dtype, u[e], v);
        if ((e ? who1 : who0) >= 0)
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = __fadd_rn(v[k], sum[e][k]);
        store_out<VEC>(a.out, a.out_dtype, (t0 + t) * a.n + n0, t < tokens ? valid : 0, v);
      }
    }
  }
  if (count) cluster.sync();  // the other blocks may still read this one's sums
}

}  // namespace adapt
}  // namespace tc
