// Attention of few query rows over a long paged cache (decode steps, drafted tokens): bound by the bytes of
// the codes, which are read once.
//
// A block takes a stretch of the work line (tc_attn.cuh) in items of 8 or 16 query rows and units of 64 keys,
// 16 for each of its four warps. A warp runs alone through its keys: asynchronous copies bring 16 rows of K and V
// codes into its own ring of shared-memory stages, several steps ahead, and codes go from there to registers as
// the left operands of m16n8k16 MMAs, keys and elements in rows and queries in columns, so that 8 query rows fill
// them: S^T = K Q^T and O^T = V^T P^T. No step needs another warp or a transposed copy:
//  - K has one key a row. The order of the summed index is free as long as Q has the same, so lane t of a quad
//    reads 16 contiguous bytes of its key and Q is laid out to match.
//  - V^T has one element a row, the keys summed over: a register holds one element of two keys. Lane g reads the
//    same bytes of four keys and interleaves them; the order of V's elements is free too, so its bytes are
//    contiguous again (rows g and g + 8 of MMA i are elements g * DP / 8 + 2 i and + 1).
//  - P^T is S^T transposed by 8 x 8 (movmatrix).
// Codes are exact in fp16 (E4M3, INT8, E2M1 times a power of two), so scales stay out of the products: a key's
// scale multiplies its score, a value's scale its weight. Q is scaled per row by a power of two into fp16's
// range. Weights are relative to a reference that follows a row's largest product of weight and value scale
// (tc_attn.cuh) only when it has risen by more than 2**8, so a step votes once and reduces nothing. Unquantized rows use their own type; bf16 ones get bf16 weights. A weight is rounded once, to the
// 16 bits of its product, and the sum it is divided by is taken before that in fp32: with the result's own rounding
// an output over a cache of its own type (fp16 ones over any) is off by 1.4 to 1.6 times what rounding it alone would
// give. Weights in two parts would undo that for twice the MMAs of the values.
//
// 64 sequences of up to 8192 keys, 8 heads of 128 over E4M3, 4 query heads each: 133 us, 4.9 TB/s of codes (57% of issue
// slots, 62% of DRAM's cycles busy). 16 sequences of up to 4000 keys and 4 new tokens over bf16: 44 us, 3.1 TB/s. One of
// 1025 keys: 13.5 us, start, one unit and join.
#pragma once

#include <atomic>
#include <cmath>
#include <string>

#include "tc_attn.cuh"
#include "tc_mma16.cuh"

namespace tc {
namespace attn {
namespace split {

constexpr int kStep = 16, kWarps = 4, kKeys = kStep * kWarps, kThreads = kWarps * 32;

template <int S, int DP, int NR>
struct Shape {
  static constexpr int kRows = 8 * NR;
  static constexpr int kRowBytes = S == KV_NONE ? 2 * DP : S == KV_MXFP4 ? DP / 2 : DP;  // a row in a stage
  static constexpr int kScaleBytes = S == KV_NONE ? 0 : S == KV_MXFP4 ? DP / 32 : 4;
  static constexpr int kSide = kStep * kRowBytes;
  static constexpr int kScales = (kStep * kScaleBytes + 15) / 16 * 16;
  static constexpr int kStage = 2 * kSide + 2 * kScales + 16;  // K codes, V codes, K scales, V scales, key mask
  // Blocks an SM: as many as the registers allow (outputs and queries take DP / 2 * NR of a thread's), and the
  // ring as deep as they fit its 227 KB: it covers HBM's latency.
  static constexpr int kRegs = DP * NR <= 64 ? 4 : DP * NR <= 128 ? 4 : DP * NR <= 256 ? 2 : 1;
  static constexpr int kRoom = kRowBytes <= 128 ? 4 : kRowBytes <= 256 ? 2 : 1;
  static constexpr int kBlocks = kRegs < kRoom ? kRegs : kRoom;
  static constexpr int kFit = (kBlocks == 4 ? 54 : kBlocks == 2 ? 108 : 200) * 1024 / (kWarps * kStage);
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kMerge = kWarps * kRows * DP * 4;  // the warps' outputs, over the ring
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
  static constexpr int kLaneBytes = kRowBytes >= 64 ? 16 : kRowBytes / 4;  // of K, a lane and chunk
  static constexpr int kChunks = kRowBytes / (4 * kLaneBytes);
  static constexpr int kLaneDims = kLaneBytes * DP / kRowBytes;
  static constexpr int kKSteps = DP / 16;
  static constexpr int kVBytes = kRowBytes / 8;  // of V, a lane
  static constexpr int kVPart = kVBytes > 16 ? 16 : kVBytes;
};

// 16-byte granule i of a stage side, swizzled so that reads along a key and across keys spread over the banks.
__device__ __forceinline__ int granule(int i) { return i ^ ((i >> 3) & 7); }

// An 8 x 8 matrix of 16-bit elements as the MMAs hold it, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

// PAD: head_dim is below DP (the general, slower addressing).
template <typename T, int S, int DP, int NR, bool PAD>
__global__ void __launch_bounds__(kThreads, Shape<S, DP, NR>::kBlocks) split_kernel(Args a, float *parts, Stretch *stretches, int most) {
  using P = Shape<S, DP, NR>;
  constexpr int kRows = P::kRows;
  using W = Work<kRows, kKeys>;
  constexpr bool kBf16 = S == KV_NONE && Same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Item first;
  __shared__ float merge_top[kWarps][kRows], merge_sum[kWarps][kRows];
  __shared__ int left_out[kWarps];  // whether the warp's products leave an odd key's values out
  constexpr bool kSharedQ = DP * NR > 256;  // Q does not fit the registers
  __shared__ uint4 qfrag[kSharedQ ? P::kKSteps * 32 : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const KvCache &c = a.c;
  unsigned char *ring = smem + warp * P::kStages * P::kStage;
  // Columns past head_dim are never copied to: they are zeros.
  auto clear = [&]() {
    for (int i = lane; i < P::kStages * P::kStage / 16; i += 32) reinterpret_cast<uint4 *>(ring)[i] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  };
  if (warp == 0) {
    const Stretch mine = W::stretch(a, blockIdx.x, most);
    if (lane == 0) {
      first = mine.first;
      stretches[blockIdx.x] = mine;
    }
  }
  if (PAD) clear();
  __syncthreads();
  let_next_start();
  Item it = first;
  if (it.n == 0) return;
  const int cpr = c.row_bytes / 16, dim = PAD ? c.dim : DP, row_bytes = PAD ? c.row_bytes : P::kRowBytes;
  const int scale_bytes = PAD ? c.scale_bytes : P::kScaleBytes;
  // Where this lane's operands lie in a stage side (the swizzle makes a table of it; rows 8 further are a constant
  // away where 8 rows are whole swizzle periods).
  constexpr bool kWide = P::kRowBytes >= 128;
  auto k_at = [&](int nt, int ch) {
    const int at = ((kWide ? 0 : nt * 8) + g) * P::kRowBytes + (ch * 4 + t) * P::kLaneBytes;
    return 16 * granule(at / 16) + at % 16 + (kWide ? nt * 8 * P::kRowBytes : 0);
  };
  auto v_at = [&](int k, int part) {
    const int at = (2 * t + (k & 1) + (kWide ? 0 : 8 * (k >> 1))) * P::kRowBytes + g * P::kVBytes + part * 16;
    return 16 * granule(at / 16) + at % 16 + (kWide ? 8 * (k >> 1) * P::kRowBytes : 0);
  };
  int koff[kWide ? 1 : 2][P::kChunks], voff[kWide ? 2 : 4][P::kVBytes / P::kVPart];
#pragma unroll
  for (int nt = 0; nt < (kWide ? 1 : 2); ++nt)
#pragma unroll
    for (int ch = 0; ch < P::kChunks; ++ch) koff[nt][ch] = k_at(nt, ch);
#pragma unroll
  for (int k = 0; k < (kWide ? 2 : 4); ++k)
#pragma unroll
    for (int part = 0; part < P::kVBytes / P::kVPart; ++part) voff[k][part] = v_at(k, part);
  const uint32_t flip_q = a.scale < 0.0f ? 0x80008000u : 0u;  // the scale's sign goes into Q
  const bool qvec = ((uintptr_t)a.q | (uintptr_t)(a.q_tok * 2) | (uintptr_t)(a.q_head * 2)) % 16 == 0;

  while (true) {
    const Seq s = sequence(a, it.b);
    int lo, hi;
    W::keys(a, s, it.tile, lo, hi);
    const int key0 = lo + it.at * kKeys + warp * kStep;
    const int key1 = min(lo + (it.at + it.n) * kKeys, hi);
    const int steps = key1 > key0 ? (key1 - key0 + kKeys - 1) / kKeys : 0;
    const int *table = a.table + (int64_t)it.b * a.table_stride;

    // Page of the half (8 keys: a page's least) of step i, -1 past the keys.
    auto page_at = [&](int i, int half) {
      const int p = key0 + i * kKeys + 8 * half;
      return p < key1 ? table[p >> c.page_shift] : -1;
    };
    auto issue = [&](int i, int slot, int pg0, int pg1) {
      unsigned char *st = ring + slot * P::kStage;
      const int p0 = key0 + i * kKeys;
      const int n = min(kStep, key1 - p0);
      const bool ok0 = pg0 >= 0 && pg0 < c.pages, ok1 = pg1 >= 0 && pg1 < c.pages;
      const int64_t row0 = ok0 ? (((int64_t)pg0 * c.heads + it.head) << c.page_shift) + (p0 & (c.page_size - 1)) : 0;
      const int64_t row1 = ok1 ? (((int64_t)pg1 * c.heads + it.head) << c.page_shift) + ((p0 + 8) & (c.page_size - 1)) : 0;
      const uint32_t valid = (ok0 ? (1u << min(n, 8)) - 1u : 0u) | (ok1 ? ((1u << max(n - 8, 0)) - 1u) << 8 : 0u);
      const bool all = valid == 0xFFFFu;
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const unsigned char *src = side ? c.v : c.k;
        unsigned char *dst = st + side * P::kSide;
        // Granule lane + 32 j of the 16 rows, which are contiguous by halves.
        constexpr int kCount = P::kSide / 16, kHalf = kCount / 2;
        if (!PAD) {
          const unsigned char *s0 = src + row0 * row_bytes + lane * 16, *s1 = src + (row1 - 8) * row_bytes + lane * 16;
          unsigned char *d = dst + 16 * granule(lane), *dx = dst + 16 * (granule(lane) ^ 4);
          if (all) {
#pragma unroll
            for (int j = 0; j < (kCount + 31) / 32; ++j) {
              const bool second = kHalf >= 32 ? 32 * j >= kHalf : lane + 32 * j >= kHalf;
              if (kCount >= 32 || lane < kCount) cp_async16((j & 1 ? dx : d) + 512 * j, (second ? s1 : s0) + 512 * j);
            }
          } else {
#pragma unroll
            for (int j = 0; j < (kCount + 31) / 32; ++j) {
              const bool second = kHalf >= 32 ? 32 * j >= kHalf : lane + 32 * j >= kHalf;
              const int r = (lane + 32 * j) / (P::kRowBytes / 16);
              if (kCount >= 32 || lane < kCount) {
                const bool use = (valid >> r) & 1u;
                cp_async16_or_zero((j & 1 ? dx : d) + 512 * j, use ? (second ? s1 : s0) + 512 * j : src, use);
              }
            }
          }
        } else {
          for (int i16 = lane; i16 < kStep * cpr; i16 += 32) {
            const int r = i16 / cpr, ch = i16 - r * cpr;
            const bool use = (valid >> r) & 1u;
            cp_async16_or_zero(dst + 16 * granule(r * (P::kRowBytes / 16) + ch),
                               use ? src + ((r >> 3 ? row1 : row0) + (r & 7)) * row_bytes + 16 * ch : src, use);
          }
        }
        if (S != KV_NONE) {
          // The scales of 8 rows are contiguous and 4-byte aligned, whatever one row's count.
          const unsigned char *ss = side ? c.vs : c.ks;
          unsigned char *sd = st + 2 * P::kSide + side * P::kScales;
          const int words = 2 * scale_bytes;
#pragma unroll
          for (int w = lane; w < 2 * words; w += 32) {
            const bool half = w >= words, use = half ? ok1 && n > 8 : ok0;
            cp_async4_or_zero(sd + 4 * w, use ? ss + (half ? row1 : row0) * scale_bytes + 4 * (w - (half ? words : 0)) : ss, use);
          }
        }
      }
      if (lane == 0) *reinterpret_cast<uint32_t *>(st + P::kStage - 16) = valid;
    };

    int pre0 = -1, pre1 = -1;  // the pages of the next step to issue, fetched a step before they are needed
    for (int i = 0; i < P::kStages - 1; ++i) {
      if (i < steps) issue(i, i, page_at(i, 0), page_at(i, 1));
      cp_async_commit();
    }
    if (P::kStages - 1 < steps) {
      pre0 = page_at(P::kStages - 1, 0);
      pre1 = page_at(P::kStages - 1, 1);
    }

    // Q: lane (g, t) holds rows g (and g + 8) at the dims its K bytes cover; rows past the last are zero.
    const int rows = s.n * a.group;
    uint32_t qf[P::kKSteps][2 * NR];
    float qmul[NR][2];  // of rows 8 r + 2 t and + 1, whose scores this lane gets
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
      const int r = it.tile * kRows + g + 8 * nr, tok = min(r, rows - 1) / a.group;
      const T *qp = static_cast<const T *>(a.q) + (s.q0 + tok) * a.q_tok + (it.head * a.group + r % a.group) * a.q_head;
      float big = 0.0f;
#pragma unroll
      for (int ch = 0; ch < P::kChunks; ++ch)
#pragma unroll
        for (int e = 0; e < P::kLaneDims; e += 8) {
          const int d = (ch * 4 + t) * P::kLaneDims + e;
          uint32_t w[4] = {0u, 0u, 0u, 0u};
          if (r < rows && d < dim) {
            if (qvec) {
              load_words<4>(reinterpret_cast<const unsigned char *>(qp + d), w);
            } else {
              const unsigned short *u = reinterpret_cast<const unsigned short *>(qp + d);
#pragma unroll
              for (int k = 0; k < 4; ++k) w[k] = (uint32_t)u[2 * k] | ((uint32_t)u[2 * k + 1] << 16);
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            qf[(ch * P::kLaneDims + e) / 4 + (k >> 1)][2 * nr + (k & 1)] = w[k] ^ flip_q;
            big = fmaxf(big, fmaxf(fabsf(half_bits_to_float<T>(w[k] & 0xFFFFu)), fabsf(half_bits_to_float<T>(w[k] >> 16))));
          }
        }
      float mul = a.scale == 0.0f ? 1.1754943508222875e-38f : fabsf(a.scale);  // scores vanish but keep -Inf
      if (S != KV_NONE) {
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
        const Pow2 f = fp16_shift(big);
        mul *= f.inverse;
#pragma unroll
        for (int k = 0; k < P::kKSteps; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t w = qf[k][2 * nr + e];
            qf[k][2 * nr + e] = pack_half(half_bits_to_float<T>(w & 0xFFFFu) * f.factor, half_bits_to_float<T>(w >> 16) * f.factor);
          }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) qmul[nr][e] = __shfl_sync(0xFFFFFFFFu, mul, 4 * (2 * t + e));
    }
    if constexpr (kSharedQ) {  // the last item's readers passed its closing barrier
      if (warp == 0)
#pragma unroll
        for (int k = 0; k < P::kKSteps; ++k) qfrag[k * 32 + lane] = make_uint4(qf[k][0], qf[k][1], qf[k][2], qf[k][3]);
      __syncthreads();
    }
    // Keys that the lane's rows see, and those that every row of the tile sees.
    int all_lo, all_hi, unused;
    visible(a, s, it.tile * kRows / a.group, unused, all_hi);
    visible(a, s, (min((it.tile + 1) * kRows, rows) - 1) / a.group, all_lo, unused);

    float o[DP / 16][NR][4];  // elements g * DP / 8 + 2 i + (e >> 1), rows 8 nr + 2 t + (e & 1)
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][nr][e] = 0.0f;
    // ref: the base-2 logarithm that a row's weights are relative to, far below everything before the first key; sum:
    // of this lane's weights. vfield: the largest exponent field of a value scale so far, seen or not: it says when a
    // reference may have to move, and the keys that the row sees say where to.
    float ref[NR][2], sum[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ref[nr][e] = -3e38f;
        sum[nr][e] = 0.0f;
      }
    int vfield = S == KV_NONE ? 127 : 0;
    if (lane == 0) left_out[warp] = 0;

    for (int i = 0, slot = 0; i < steps; ++i, slot = slot + 1 == P::kStages ? 0 : slot + 1) {
      if (i + P::kStages - 1 < steps) {
        issue(i + P::kStages - 1, slot == 0 ? P::kStages - 1 : slot - 1, pre0, pre1);
        pre0 = page_at(i + P::kStages, 0);
        pre1 = page_at(i + P::kStages, 1);
      }
      cp_async_commit();
      cp_async_wait<P::kStages - 1>();
      __syncwarp();
      const unsigned char *st = ring + slot * P::kStage;
      const unsigned char *kscales = st + 2 * P::kSide, *vscales = kscales + P::kScales;
      const uint32_t valid = *reinterpret_cast<const uint32_t *>(st + P::kStage - 16);
      const int p0 = key0 + i * kKeys;

      // Scores: x[nr][e] is key g + 8 (e >> 1), row 8 nr + 2 t + (e & 1).
      float x[NR][4], vscale[2] = {1.0f, 1.0f};
      int vbig[2] = {0, 0};
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[nr][e] = 0.0f;
      {
        int kbig[2] = {0, 0};
        float kscale[2] = {1.0f, 1.0f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = g + 8 * h;
          if (S == KV_MXFP4) {
#pragma unroll
            for (int q = 0; q < P::kScaleBytes; ++q)
              if (q < scale_bytes) {
                kbig[h] = max(kbig[h], (int)kscales[key * scale_bytes + q]);
                vbig[h] = max(vbig[h], (int)vscales[key * scale_bytes + q]);
              }
            kscale[h] = pow2_value(kbig[h]) * (1.0f / (1 << kGroupShift));
            vscale[h] = pow2_value(vbig[h]) * (1.0f / (1 << kGroupShift));
          } else if (S != KV_NONE) {
            kscale[h] = reinterpret_cast<const float *>(kscales)[key];
            vscale[h] = reinterpret_cast<const float *>(vscales)[key];
          }
        }
#pragma unroll
        for (int ch = 0; ch < P::kChunks; ++ch) {
          uint32_t w[2][P::kLaneBytes / 4], gmul[2] = {0u, 0u};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            load_words<P::kLaneBytes / 4>(st + koff[kWide ? 0 : h][ch] + (kWide ? h * 8 * P::kRowBytes : 0), w[h]);
            if (S == KV_MXFP4) {
              const int grp = (ch * 4 + t) * P::kLaneDims / 32;
              if (grp < scale_bytes)
                gmul[h] = half_pow2((int)kscales[(g + 8 * h) * scale_bytes + grp] - kbig[h] + kGroupShift) * 0x10001u;
            }
          }
#pragma unroll
          for (int k = 0; k < P::kLaneDims / 4; ++k) {
            uint32_t ka[4];  // key g, key g + 8 at the first two elements, then at the next two
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (S == KV_NONE) {
                ka[h] = w[h][(2 * k) % (P::kLaneBytes / 4)];
                ka[2 + h] = w[h][(2 * k + 1) % (P::kLaneBytes / 4)];
              } else if (S == KV_MXFP4) {
                uint32_t v[4];
                e2m1x8_half2(w[h][(k >> 1) % (P::kLaneBytes / 4)], v);
                ka[h] = mul_half2(v[2 * (k & 1)], gmul[h]);
                ka[2 + h] = mul_half2(v[2 * (k & 1) + 1], gmul[h]);
              } else if (S == KV_FP8_ROW) {
                e4m3x4_half2(w[h][k % (P::kLaneBytes / 4)], ka[h], ka[2 + h]);
              } else {
                const uint32_t u = w[h][k % (P::kLaneBytes / 4)] ^ 0x80808080u;
                ka[h] = int8x2_half2<0x4140>(u);
                ka[2 + h] = int8x2_half2<0x4342>(u);
              }
            }
            const int ks = ch * (P::kLaneDims / 4) + k;
            if constexpr (kSharedQ) {
              const uint4 q4 = qfrag[ks * 32 + lane];
              mma16<kBf16>(x[0], ka, q4.x, q4.y);
              mma16<kBf16>(x[NR - 1], ka, q4.z, q4.w);
            } else {
#pragma unroll
              for (int nr = 0; nr < NR; ++nr) mma16<kBf16>(x[nr], ka, qf[ks][2 * nr], qf[ks][2 * nr + 1]);
            }
          }
        }
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[nr][e] = x[nr][e] * kscale[e >> 1] * qmul[nr][e & 1];
      }
      const bool whole = valid == 0xFFFFu && p0 >= all_lo && p0 + kStep <= all_hi;
      if (!whole) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            int lo_r, hi_r;
            visible(a, s, min(it.tile * kRows + 8 * nr + 2 * t + r, rows - 1) / a.group, lo_r, hi_r);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int key = g + 8 * h;
              if (!((valid >> key) & 1u) || p0 + key < lo_r || p0 + key >= hi_r) x[nr][2 * h + r] = -INFINITY;
            }
          }
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (!((valid >> (g + 8 * h)) & 1u)) vscale[h] = 0.0f;
      }
      uint32_t odd_keys = 0u;  // keys whose values the products leave out (tc_attn.cuh)
      if (S == KV_NONE && !whole) {
        // Rows of the step differ in what they see: a value that is not finite must not reach the others.
        for (int r = 0; r < kStep; ++r) {
          bool bad = false;
          for (int w = lane; w < P::kRowBytes / 4; w += 32) {
            const int at = r * P::kRowBytes + 4 * w;
            bad |= not_finite2<T>(*reinterpret_cast<const uint32_t *>(st + P::kSide + 16 * granule(at / 16) + at % 16));
          }
          if (__any_sync(0xFFFFFFFFu, bad)) odd_keys |= 1u << r;
        }
        if (odd_keys && lane == 0) left_out[warp] = 1;
      }

      // May a row's reference have to move?
      bool any = false;
      const float above = kHeadroom - lift_of(vfield);
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int r = 0; r < 2; ++r) any |= fmaxf(x[nr][r], x[nr][2 + r]) > ref[nr][r] + above;
      if (S != KV_NONE) {
#pragma unroll
        for (int h = 0; h < 2; ++h) any |= (int)(f2u(vscale[h]) >> 23) > vfield;  // odd ones too
      }
      if (__any_sync(0xFFFFFFFFu, any)) {
        float lift[2] = {0.0f, 0.0f};
        if (S != KV_NONE) {
          uint32_t f = 0u, zeros = 0u;  // zeros: of this lane's two keys
          if ((S == KV_FP8_ROW || S == KV_INT8_ROW) &&
              __any_sync(0xFFFFFFFFu, f2u(vscale[0]) == kOneScale || f2u(vscale[1]) == kOneScale)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t bits = 0u;
              for (int k = t; k < P::kRowBytes / 4; k += 4) {
                const int at = (g + 8 * h) * P::kRowBytes + 4 * k;
                bits |= nonzero_codes<S>(*reinterpret_cast<const uint32_t *>(st + P::kSide + 16 * granule(at / 16) + at % 16));
              }
              bits |= __shfl_xor_sync(0xFFFFFFFFu, bits, 1);
              bits |= __shfl_xor_sync(0xFFFFFFFFu, bits, 2);
              if (bits == 0u && f2u(vscale[h]) == kOneScale) zeros |= 1u << h;
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t v = f2u(vscale[h]);
            // What rows see of an odd key's values is added at the end; in the products they count as 0 (where the
            // scale is NaN so are the codes).
            if (odd_scale(v)) {
              odd_keys |= 1u << (g + 8 * h);
              vscale[h] = 0.0f;
              lift[h] = (float)kOddLift;
            } else if ((zeros >> h) & 1u) {
              vscale[h] = 0.0f;
              lift[h] = (float)kLeastLift;
            } else {
              f = max(f, v >> 23);
              lift[h] = lift_of((int)(v >> 23));
            }
          }
          odd_keys = __reduce_or_sync(0xFFFFFFFFu, odd_keys);
          vfield = max(vfield, (int)warp_max(f));
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (lift[h] >= lift_of(vfield) - kNarrow) lift[h] = fmaxf(lift[h], lift_of(vfield));
        }
        float keep[NR][2];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float top = fmaxf(x[nr][r] + lift[0], x[nr][2 + r] + lift[1]);
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, k));
            const float next = top > ref[nr][r] + kHeadroom ? ceilf(top) - kBelow : ref[nr][r];
            keep[nr][r] = exp2_wide(ref[nr][r] - next);
            ref[nr][r] = next;
            sum[nr][r] *= keep[nr][r];
          }
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
          for (int nr = 0; nr < NR; ++nr)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[k][nr][e] *= keep[nr][e & 1];
        if (odd_keys && lane == 0) left_out[warp] = 1;
      }
      uint32_t pf[NR][2];  // P^T: keys 2 t, 2 t + 1 (and + 8) of row g
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float p[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            p[r] = exp2_fast(x[nr][2 * h + r] - ref[nr][r]);
            sum[nr][r] += p[r];
            if (S != KV_NONE) p[r] *= vscale[h];
          }
          pf[nr][h] = transpose8x8(kBf16 ? pack_bf16(p[0], p[1]) : pack_half(p[0], p[1]));
        }

      // O^T += V^T P^T. Keys of the operand: 2 t, 2 t + 1, then 2 t + 8, 2 t + 9.
      uint32_t vm0 = 0u, vm1 = 0u;
      if (S == KV_MXFP4) {
        const int grp = g * (DP / 8) / 32;
        uint32_t mul[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = 2 * t + (k & 1) + 8 * (k >> 1);
          const int big = __shfl_sync(0xFFFFFFFFu, k >> 1 ? vbig[1] : vbig[0], 4 * (2 * t + (k & 1)));
          mul[k] = grp < scale_bytes ? half_pow2((int)vscales[key * scale_bytes + grp] - big + kGroupShift) : 0u;
        }
        vm0 = mul[0] | (mul[1] << 16);
        vm1 = mul[2] | (mul[3] << 16);
      }
#pragma unroll
      for (int part = 0; part < P::kVBytes / P::kVPart; ++part) {
        uint32_t w[4][P::kVPart / 4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = 2 * t + (k & 1) + 8 * (k >> 1);
          load_words<P::kVPart / 4>(st + P::kSide + voff[kWide ? k & 1 : k][part] + (kWide ? 8 * (k >> 1) * P::kRowBytes : 0), w[k]);
          if (odd_keys)
#pragma unroll
            for (int q = 0; q < P::kVPart / 4; ++q)
              if ((odd_keys >> key) & 1u) w[k][q] = 0u;
        }
#pragma unroll
        for (int q = 0; q < P::kVPart / 4; ++q) {
          auto add = [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
            const uint32_t va[4] = {a0, a1, a2, a3};
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) mma16<kBf16>(o[i][nr], va, pf[nr][0], pf[nr][1]);
          };
          if (S == KV_NONE) {
            add((part * 16 + q * 4) / 4, __byte_perm(w[0][q], w[1][q], 0x5410), __byte_perm(w[0][q], w[1][q], 0x7632),
                __byte_perm(w[2][q], w[3][q], 0x5410), __byte_perm(w[2][q], w[3][q], 0x7632));
          } else if (S == KV_MXFP4) {
            // Bytes of one nibble from each of two keys: even elements, odd elements.
            uint32_t e0[4], d0[4], e1[4], d1[4];
            e2m1x8_half2((w[0][q] & 0x0F0F0F0Fu) | ((w[1][q] & 0x0F0F0F0Fu) << 4), e0);
            e2m1x8_half2(((w[0][q] >> 4) & 0x0F0F0F0Fu) | (w[1][q] & 0xF0F0F0F0u), d0);
            e2m1x8_half2((w[2][q] & 0x0F0F0F0Fu) | ((w[3][q] & 0x0F0F0F0Fu) << 4), e1);
            e2m1x8_half2(((w[2][q] >> 4) & 0x0F0F0F0Fu) | (w[3][q] & 0xF0F0F0F0u), d1);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              add(part * 16 + q * 4 + k, mul_half2(e0[k], vm0), mul_half2(d0[k], vm0), mul_half2(e1[k], vm1), mul_half2(d1[k], vm1));
          } else {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t ab = __byte_perm(w[0][q], w[1][q], k ? 0x7362 : 0x5140);
              const uint32_t cd = __byte_perm(w[2][q], w[3][q], k ? 0x7362 : 0x5140);
              uint32_t h[4];
              if (S == KV_FP8_ROW) {
                e4m3x4_half2(ab, h[0], h[1]);
                e4m3x4_half2(cd, h[2], h[3]);
              } else {
                const uint32_t u0 = ab ^ 0x80808080u, u1 = cd ^ 0x80808080u;
                h[0] = int8x2_half2<0x4140>(u0);
                h[1] = int8x2_half2<0x4342>(u0);
                h[2] = int8x2_half2<0x4140>(u1);
                h[3] = int8x2_half2<0x4342>(u1);
              }
              add((part * 16 + q * 4) / 2 + k, h[0], h[1], h[2], h[3]);
            }
          }
        }
      }
      __syncwarp();  // the stage may be filled again
    }

    // The warps' results become one.
    cp_async_wait_all();
    __syncthreads();
    float *mo = reinterpret_cast<float *>(smem) + warp * kRows * DP;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) sum[nr][r] += __shfl_xor_sync(0xFFFFFFFFu, sum[nr][r], k);
        if (g == 0) {
          merge_top[warp][8 * nr + 2 * t + r] = sum[nr][r] == 0.0f ? -INFINITY : ref[nr][r];
          merge_sum[warp][8 * nr + 2 * t + r] = sum[nr][r];
        }
      }
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          mo[(g * (DP / 8) + 2 * k + (e >> 1)) * kRows + 8 * nr + 2 * t + (e & 1)] = o[k][nr][e];
    __syncwarp();
    if (left_out[warp]) {
      // The values of odd keys in fp32, to the rows that see them; a row's score of the key is worked out again.
      uint32_t gone = 0u;  // rows that nothing changes any more: all NaN
      for (int in = 0; in < kRows; ++in)
        if (merge_sum[warp][in] != merge_sum[warp][in]) gone |= 1u << in;
      for (int i = 0; i < steps; ++i) {
        const int mine = key0 + i * kKeys + lane, pg = lane < kStep && mine < key1 ? table[mine >> c.page_shift] : -1;
        const int64_t own = pg >= 0 && pg < c.pages ? (((int64_t)pg * c.heads + it.head) << c.page_shift) + (mine & (c.page_size - 1)) : -1;
        if (S == KV_NONE) {  // only where rows differ in what they see
          int lo_r, hi_r, unused;
          visible(a, s, it.tile * kRows / a.group, unused, hi_r);
          visible(a, s, (min((it.tile + 1) * kRows, rows) - 1) / a.group, lo_r, unused);
          const int p0 = key0 + i * kKeys;
          if (__ballot_sync(0xFFFFFFFFu, own >= 0) == 0xFFFFu && p0 >= lo_r && p0 + kStep <= hi_r) continue;
        }
        for (uint32_t odd = __ballot_sync(0xFFFFFFFFu, own >= 0 && odd_values<T, S>(c, own)); odd; odd &= odd - 1) {
          const int from = __ffs(odd) - 1, at = key0 + i * kKeys + from;
          const int64_t row = __shfl_sync(0xFFFFFFFFu, own, from);
          for (int in = 0; in < kRows && it.tile * kRows + in < rows; ++in) {
            const int r = it.tile * kRows + in;
            int row_lo, row_hi;
            visible(a, s, r / a.group, row_lo, row_hi);
            if (at < row_lo || at >= row_hi || ((gone >> in) & 1u)) continue;
            const T *qp = static_cast<const T *>(a.q) + (s.q0 + r / a.group) * a.q_tok + (it.head * a.group + r % a.group) * a.q_head;
            float dot = 0.0f;
            for (int d = lane; d < dim; d += 32)
              dot = __fmaf_rn(Io<T>::get(qp[d]), cached<T>(c, c.k + row * row_bytes, c.ks + row * scale_bytes, d), dot);
            for (int k = 16; k; k >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, k);
            const float w = exp2_wide(dot * a.scale - merge_top[warp][in]);
            bool nan = true;
            for (int d = lane; d < dim; d += 32) {
              const float sum = __fmaf_rn(w, cached<T>(c, c.v + row * row_bytes, c.vs + row * scale_bytes, d), mo[d * kRows + in]);
              mo[d * kRows + in] = sum;
              nan = nan && sum != sum;
            }
            if (__all_sync(0xFFFFFFFFu, nan)) gone |= 1u << in;
          }
        }
      }
    }
    __syncthreads();
    const bool done = it.at == 0 && it.n == it.units;
    float *part = parts + (size_t)(2 * blockIdx.x + (it.at > 0 ? 0 : 1)) * partial_floats(kRows, DP);
    const int row = threadIdx.x % kRows;
    float m = merge_top[0][row];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, merge_top[w][row]);
    float weight[kWarps], total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      weight[w] = merge_top[w][row] == -INFINITY ? 0.0f : exp2_wide(merge_top[w][row] - m);
      total += merge_sum[w][row] * weight[w];
    }
    const int r = it.tile * kRows + row;
    const int64_t out_row = (s.q0 + r / a.group) * a.heads + it.head * a.group + r % a.group;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    for (int d = threadIdx.x / kRows; d < dim; d += kThreads / kRows) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        if (weight[w] != 0.0f) v += reinterpret_cast<const float *>(smem)[(w * DP + d) * kRows + row] * weight[w];
      if (!done) part[(2 + d) * kRows + row] = v;
      else if (r < rows) static_cast<T *>(a.out)[out_row * dim + d] = Io<T>::put(v * inv);
    }
    if (threadIdx.x < kRows) {
      if (!done) {
        part[row] = m;
        part[kRows + row] = total;
      } else if (a.lse && r < rows) {
        a.lse[out_row] = total == 0.0f ? -INFINITY : (m + log2f(total)) * 0.69314718055994531f;
      }
    }
    __syncthreads();
    if (it.left == 0) return;
    if (PAD) clear();
    W::next(a, it);
  }
}

template <typename T, int S, int DP, int NR, bool PAD>
int launch(const Args &a, float *parts, int sms, cudaStream_t s) {
  using P = Shape<S, DP, NR>;
  static_assert(P::kStages >= 2, "the ring holds the step at hand and the next");
  auto kern = split_kernel<T, S, DP, NR, PAD>;
  static std::atomic<uint64_t> ready[2];  // devices whose shared-memory limit is raised
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return set_error(std::string("tc_paged_attention: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  if (dev >= 128 || !((ready[dev >> 6].load(std::memory_order_relaxed) >> (dev & 63)) & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, P::kSmem);
    if (e != cudaSuccess) return set_error(std::string("tc_paged_attention: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
    if (dev < 128) ready[dev >> 6].fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
  }
  const int most = sms * P::kBlocks;
  Stretch *stretches = reinterpret_cast<Stretch *>(parts + 2 * (size_t)most * partial_floats(8 * NR, DP));
  kern<<<most, kThreads, P::kSmem, s>>>(a, parts, stretches, most);
  count_launch();
  return launch_join<T, 8 * NR>(a, parts, stretches, most, nullptr, s);
}

template <typename T, int S, int DP>
int launch_rows(const Args &a, float *parts, int sms, cudaStream_t s) {
  const bool pad = a.c.dim != DP;
  if ((int64_t)a.max_q * a.group <= 8)
    return pad ? launch<T, S, DP, 1, true>(a, parts, sms, s) : launch<T, S, DP, 1, false>(a, parts, sms, s);
  return pad ? launch<T, S, DP, 2, true>(a, parts, sms, s) : launch<T, S, DP, 2, false>(a, parts, sms, s);
}

template <int S>
int launch_scheme(const Args &a, float *parts, int sms, cudaStream_t s) {
  const bool bf16 = a.c.dtype == TC_BF16;
  if (a.c.dim <= 64) return bf16 ? launch_rows<__nv_bfloat16, S, 64>(a, parts, sms, s) : launch_rows<__half, S, 64>(a, parts, sms, s);
  if (a.c.dim <= 128) return bf16 ? launch_rows<__nv_bfloat16, S, 128>(a, parts, sms, s) : launch_rows<__half, S, 128>(a, parts, sms, s);
  return bf16 ? launch_rows<__nv_bfloat16, S, 256>(a, parts, sms, s) : launch_rows<__half, S, 256>(a, parts, sms, s);
}

}  // namespace split
}  // namespace attn
}  // namespace tc
