// Attention of few query rows over a long paged cache (decode steps, drafted tokens): bound by the bytes of
// the codes, which are read once.
//
// A block takes a stretch of the work line (tc_attn.cuh) in items of 16 query rows, one tensor-core tile,
// and units of 64 keys, 16 for each of its four warps. A warp runs alone through its keys: asynchronous
// copies bring 16 rows of K and V codes into its own ring of shared-memory stages, several steps ahead, and
// codes go from there to registers as the operands of m16n8k16 MMAs. No step needs another warp or a
// transposed copy:
//  - K is the MMA's B operand with one key a column. The order of the summed index is free as long as Q has
//    the same, so lane t of a quad reads 16 contiguous bytes of its key and Q is laid out to match.
//  - V is the B operand with the keys summed over: a register holds one element of two keys. Lane g reads
//    the same bytes of four keys and interleaves them; the order of V's columns is free too, so its bytes
//    are contiguous again (column n of MMA tile j is dim n * DP / 8 + j).
// Codes are exact in fp16 (E4M3, INT8, E2M1 times a power of two), so scales stay out of the products: a
// key's scale multiplies its score, a value's scale its weight. Q is scaled per row by a power of two into
// fp16's range. Weights are fp16 too, as p * scale * 2**14 / T with T the power of two of the largest scale
// so far: 11 bits down to 2**-28 of the largest product. Unquantized rows use their own type; bf16 ones get
// bf16 weights.
#pragma once

#include <atomic>
#include <cmath>
#include <string>

#include "tc_attn.cuh"
#include "tc_mma16.cuh"

namespace tc {
namespace attn {
namespace split {

constexpr int kRows = 16, kStep = 16, kWarps = 4, kKeys = kStep * kWarps, kThreads = kWarps * 32;
using W = Work<kRows, kKeys>;

template <int S, int DP>
struct Shape {
  static constexpr int kRowBytes = S == KV_NONE ? 2 * DP : S == KV_MXFP4 ? DP / 2 : DP;  // a row in a stage
  static constexpr int kScaleBytes = S == KV_NONE ? 0 : S == KV_MXFP4 ? DP / 32 : 4;
  static constexpr int kSide = kStep * kRowBytes;
  static constexpr int kScales = (kStep * kScaleBytes + 15) / 16 * 16;
  static constexpr int kStage = 2 * kSide + 2 * kScales + 16;  // K codes, V codes, K scales, V scales, key mask
  // As deep as two blocks fit an SM with (one for unquantized rows of 256): the ring covers HBM's latency.
  static constexpr int kBlocks = S == KV_NONE && DP == 256 ? 1 : 2;
  static constexpr int kFit = (kBlocks == 1 ? 200 : 104) * 1024 / (kWarps * kStage);
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

// A 16-bit element whose exponent is all ones.
template <typename T>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
  const uint32_t m = Same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u;
  return (w & m) == m || ((w >> 16) & m) == m;
}

// PAD: head_dim is below DP (the general, slower addressing).
template <typename T, int S, int DP, bool PAD>
__global__ void __launch_bounds__(kThreads, Shape<S, DP>::kBlocks) split_kernel(Args a, float *parts, int most) {
  using P = Shape<S, DP>;
  constexpr bool kBf16 = S == KV_NONE && Same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Item first;
  __shared__ float merge_top[kWarps][kRows], merge_sum[kWarps][kRows];
  __shared__ uint4 qfrag[DP == 256 ? P::kKSteps * 32 : 1];  // Q of wide heads does not fit the registers
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const KvCache &c = a.c;
  unsigned char *ring = smem + warp * P::kStages * P::kStage;
  // Columns past head_dim are never copied to: they are zeros.
  auto clear = [&]() {
    for (int i = lane; i < P::kStages * P::kStage / 16; i += 32) reinterpret_cast<uint4 *>(ring)[i] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  };
  if (warp == 0) {
    const int64_t total = W::total(a);
    const int n = W::blocks(total, most);
    Item it{0, 0, 0, 0, 0, 0, 0};
    if ((int)blockIdx.x < n) {
      const int64_t u0 = W::start(total, blockIdx.x, n), u1 = W::start(total, blockIdx.x + 1, n);
      it = W::find(a, u0);
      it.n = (int)min((int64_t)(it.units - it.at), u1 - u0);
      it.left = u1 - u0 - it.n;
    }
    if (lane == 0) first = it;
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

    // Q: lane (g, t) holds rows g and g + 8 at the dims its K bytes cover; rows past the last are zero.
    const int rows = s.n * a.group;
    uint32_t qf[P::kKSteps][4];
    float qmul[2];
    int tok[2];
#pragma unroll
    for (int hrow = 0; hrow < 2; ++hrow) {
      const int r = it.tile * kRows + g + 8 * hrow;
      tok[hrow] = min(r, rows - 1) / a.group;
      const T *qp = static_cast<const T *>(a.q) + (s.q0 + tok[hrow]) * a.q_tok + (it.head * a.group + r % a.group) * a.q_head;
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
            qf[(ch * P::kLaneDims + e) / 4 + (k >> 1)][hrow + 2 * (k & 1)] = w[k];
            big = fmaxf(big, fmaxf(fabsf(half_bits_to_float<T>(w[k] & 0xFFFFu)), fabsf(half_bits_to_float<T>(w[k] >> 16))));
          }
        }
      qmul[hrow] = a.scale;
      if (S != KV_NONE) {
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
        const Pow2 f = fp16_shift(big);
        qmul[hrow] = a.scale * f.inverse;
#pragma unroll
        for (int k = 0; k < P::kKSteps; ++k)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const uint32_t w = qf[k][hrow + e];
            qf[k][hrow + e] = pack_half(half_bits_to_float<T>(w & 0xFFFFu) * f.factor, half_bits_to_float<T>(w >> 16) * f.factor);
          }
      }
    }
    if (DP == 256) {  // the last item's readers passed its closing barrier
      if (warp == 0)
#pragma unroll
        for (int k = 0; k < P::kKSteps; ++k) qfrag[DP == 256 ? k * 32 + lane : 0] = make_uint4(qf[k][0], qf[k][1], qf[k][2], qf[k][3]);
      __syncthreads();
    }
    // Keys that rows g and g + 8 see, and those that every row of the tile sees.
    int see_lo[2], see_hi[2], all_lo, all_hi, unused;
#pragma unroll
    for (int hrow = 0; hrow < 2; ++hrow) visible(a, s, tok[hrow], see_lo[hrow], see_hi[hrow]);
    visible(a, s, it.tile * kRows / a.group, unused, all_hi);
    visible(a, s, (min((it.tile + 1) * kRows, rows) - 1) / a.group, all_lo, unused);

    float o[DP / 8][4];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
    int vfield = 254;  // exponent field of 2**14 / T (what the weights are multiplied by)

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

      // Scores: x[nt][e] is key nt * 8 + 2 t + (e & 1), row g + 8 (e >> 1).
      float x[2][4], vscale[2][2];
      int vbig[2][2];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const int r = nt * 8 + g;
        int big = 0;
        if (S == KV_MXFP4) {
#pragma unroll
          for (int q = 0; q < P::kScaleBytes; ++q)
            if (q < scale_bytes) big = max(big, (int)kscales[r * scale_bytes + q]);
        }
#pragma unroll
        for (int ch = 0; ch < P::kChunks; ++ch) {
          uint32_t w[P::kLaneBytes / 4], gmul = 0u;
          load_words<P::kLaneBytes / 4>(st + koff[kWide ? 0 : nt][ch] + (kWide ? nt * 8 * P::kRowBytes : 0), w);
          if (S == KV_MXFP4) {
            const int grp = (ch * 4 + t) * P::kLaneDims / 32;
            if (grp < scale_bytes) gmul = half_pow2((int)kscales[r * scale_bytes + grp] - big + kGroupShift) * 0x10001u;
          }
#pragma unroll
          for (int k = 0; k < P::kLaneDims / 4; ++k) {
            uint32_t b0, b1, h[4];
            if (S == KV_NONE) {
              b0 = w[(2 * k) % (P::kLaneBytes / 4)];
              b1 = w[(2 * k + 1) % (P::kLaneBytes / 4)];
            } else if (S == KV_MXFP4) {
              e2m1x8_half2(w[(k >> 1) % (P::kLaneBytes / 4)], h);
              b0 = mul_half2(h[2 * (k & 1)], gmul);
              b1 = mul_half2(h[2 * (k & 1) + 1], gmul);
            } else if (S == KV_FP8_ROW) {
              e4m3x4_half2(w[k % (P::kLaneBytes / 4)], b0, b1);
            } else {
              const uint32_t u = w[k % (P::kLaneBytes / 4)] ^ 0x80808080u;
              b0 = int8x2_half2<0x4140>(u);
              b1 = int8x2_half2<0x4342>(u);
            }
            const int ks = ch * (P::kLaneDims / 4) + k;
            if (DP == 256) {
              const uint4 q4 = qfrag[DP == 256 ? ks * 32 + lane : 0];
              const uint32_t qa[4] = {q4.x, q4.y, q4.z, q4.w};
              mma16<kBf16>(acc, qa, b0, b1);
            } else {
              mma16<kBf16>(acc, qf[ks], b0, b1);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = nt * 8 + 2 * t + e;
          float ks = 1.0f;
          vscale[nt][e] = 1.0f;
          if (S == KV_MXFP4) {
            int bk = 0, bv = 0;
#pragma unroll
            for (int q = 0; q < P::kScaleBytes; ++q)
              if (q < scale_bytes) {
                bk = max(bk, (int)kscales[key * scale_bytes + q]);
                bv = max(bv, (int)vscales[key * scale_bytes + q]);
              }
            ks = pow2_value(bk) * (1.0f / (1 << kGroupShift));
            vscale[nt][e] = pow2_value(bv);
            vbig[nt][e] = bv;
          } else if (S != KV_NONE) {
            ks = reinterpret_cast<const float *>(kscales)[key];
            vscale[nt][e] = reinterpret_cast<const float *>(vscales)[key];
          }
          x[nt][e] = acc[e] * ks * qmul[0];
          x[nt][e + 2] = acc[e + 2] * ks * qmul[1];
        }
      }
      const bool whole = valid == 0xFFFFu && p0 >= all_lo && p0 + kStep <= all_hi;
      if (!whole) {
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = nt * 8 + 2 * t + (e & 1);
            const bool there = (valid >> key) & 1u;
            if (!there || p0 + key < see_lo[e >> 1] || p0 + key >= see_hi[e >> 1]) x[nt][e] = -INFINITY;
            if (e < 2 && !there) vscale[nt][e] = 0.0f;
          }
      }

      // Running maxima and sums; keep[] scales what the sums hold, okeep[] what the outputs hold.
      float keep[2], okeep[2];
      bool moved = false;
#pragma unroll
      for (int hrow = 0; hrow < 2; ++hrow) {
        float m = fmaxf(fmaxf(x[0][2 * hrow], x[0][2 * hrow + 1]), fmaxf(x[1][2 * hrow], x[1][2 * hrow + 1]));
        m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
        m = fmaxf(m, top[hrow]);
        keep[hrow] = okeep[hrow] = m == top[hrow] ? 1.0f : exp2_fast(top[hrow] - m);
        moved |= m != top[hrow];
        top[hrow] = m;
      }
      uint32_t nan_keys = 0u;  // keys whose V scale is NaN
      float vmul = 16384.0f;
      if (S != KV_NONE) {
        int f = 0;
        bool nan = false;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int v = (int)(f2u(vscale[nt][e]) >> 23);
            nan |= v >= 255;
            f = max(f, v >= 255 ? 0 : v);
          }
        f = max(f, __shfl_xor_sync(0xFFFFFFFFu, f, 1));
        f = max(f, __shfl_xor_sync(0xFFFFFFFFu, f, 2));
        const int field = min(vfield, 268 - f);  // 2**(14 - (f - 127)), at most 2**127
        if (field != vfield) {
          const float down = u2f((uint32_t)max(127 + field - vfield, 0) << 23);
          okeep[0] *= down;
          okeep[1] *= down;
          moved = true;
          vfield = field;
        }
        vmul = u2f((uint32_t)vfield << 23);
        if (__any_sync(0xFFFFFFFFu, nan)) {
          // Rare. A NaN scale comes with NaN codes, which would reach rows that do not see the key as
          // 0 * NaN: such codes count as 0 below, and the weight carries the NaN.
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if ((f2u(vscale[nt][e]) >> 23) >= 255) nan_keys |= 1u << (nt * 8 + 2 * t + e);
          nan_keys = __reduce_or_sync(0xFFFFFFFFu, nan_keys);
        }
      } else if (!whole) {
        // Rows of the step differ in what they see: a value that is not finite must not reach the others.
        // Its whole row counts as 0 and the weights of the rows that see it become NaN.
        for (int r = 0; r < kStep; ++r) {
          bool bad = false;
          for (int w = lane; w < P::kRowBytes / 4; w += 32) {
            const int at = r * P::kRowBytes + 4 * w;
            bad |= not_finite2<T>(*reinterpret_cast<const uint32_t *>(st + P::kSide + 16 * granule(at / 16) + at % 16));
          }
          if (__any_sync(0xFFFFFFFFu, bad)) nan_keys |= 1u << r;
        }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if ((nan_keys >> (nt * 8 + 2 * t + e)) & 1u) vscale[nt][e] = u2f(kQNaN);
      }
      uint32_t pf[4];
#pragma unroll
      for (int hrow = 0; hrow < 2; ++hrow) {
        const float ref = top[hrow] == -INFINITY ? 0.0f : top[hrow];
        sum[hrow] *= keep[hrow];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          float p[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            p[e] = exp2_fast(x[nt][2 * hrow + e] - ref);
            sum[hrow] += p[e];
            if (S != KV_NONE) p[e] = p[e] == 0.0f ? 0.0f : p[e] * (vscale[nt][e] * vmul);
            else if (!kBf16) p[e] *= vmul;
            if (S == KV_NONE && nan_keys && p[e] != 0.0f) p[e] *= vscale[nt][e];
          }
          pf[2 * nt + hrow] = kBf16 ? pack_bf16(p[0], p[1]) : pack_half(p[0], p[1]);
        }
      }
      if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
        for (int j = 0; j < DP / 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j][e] *= okeep[e >> 1];
      }

      // O += P V. Keys of the operand: 2 t, 2 t + 1 (b0), 2 t + 8, 2 t + 9 (b1).
      uint32_t vm0 = 0u, vm1 = 0u;
      if (S == KV_MXFP4) {
        const int grp = g * (DP / 8) / 32;
        if (grp < scale_bytes) {
          uint32_t m[2][2];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              m[nt][e] = half_pow2((int)vscales[(nt * 8 + 2 * t + e) * scale_bytes + grp] - vbig[nt][e] + kGroupShift);
          vm0 = m[0][0] | (m[0][1] << 16);
          vm1 = m[1][0] | (m[1][1] << 16);
        }
      }
#pragma unroll
      for (int part = 0; part < P::kVBytes / P::kVPart; ++part) {
        uint32_t w[4][P::kVPart / 4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = 2 * t + (k & 1) + 8 * (k >> 1);
          load_words<P::kVPart / 4>(st + P::kSide + voff[kWide ? k & 1 : k][part] + (kWide ? 8 * (k >> 1) * P::kRowBytes : 0), w[k]);
          if (nan_keys)
#pragma unroll
            for (int q = 0; q < P::kVPart / 4; ++q)
              if ((nan_keys >> key) & 1u) w[k][q] = 0u;
        }
#pragma unroll
        for (int q = 0; q < P::kVPart / 4; ++q) {
          if (S == KV_NONE) {
            const int j = (part * 16 + q * 4) / 2;
            mma16<kBf16>(o[j], pf, __byte_perm(w[0][q], w[1][q], 0x5410), __byte_perm(w[2][q], w[3][q], 0x5410));
            mma16<kBf16>(o[j + 1], pf, __byte_perm(w[0][q], w[1][q], 0x7632), __byte_perm(w[2][q], w[3][q], 0x7632));
          } else if (S == KV_MXFP4) {
            const int j = (part * 16 + q * 4) * 2;
            // Bytes of one nibble from each of two keys: even elements, odd elements.
            const uint32_t e0 = (w[0][q] & 0x0F0F0F0Fu) | ((w[1][q] & 0x0F0F0F0Fu) << 4);
            const uint32_t d0 = ((w[0][q] >> 4) & 0x0F0F0F0Fu) | (w[1][q] & 0xF0F0F0F0u);
            const uint32_t e1 = (w[2][q] & 0x0F0F0F0Fu) | ((w[3][q] & 0x0F0F0F0Fu) << 4);
            const uint32_t d1 = ((w[2][q] >> 4) & 0x0F0F0F0Fu) | (w[3][q] & 0xF0F0F0F0u);
            uint32_t h0[4], h1[4];
            e2m1x8_half2(e0, h0);
            e2m1x8_half2(e1, h1);
#pragma unroll
            for (int k = 0; k < 4; ++k) mma16<false>(o[j + 2 * k], pf, mul_half2(h0[k], vm0), mul_half2(h1[k], vm1));
            e2m1x8_half2(d0, h0);
            e2m1x8_half2(d1, h1);
#pragma unroll
            for (int k = 0; k < 4; ++k) mma16<false>(o[j + 2 * k + 1], pf, mul_half2(h0[k], vm0), mul_half2(h1[k], vm1));
          } else {
            const int j = part * 16 + q * 4;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t ab = __byte_perm(w[0][q], w[1][q], k ? 0x7362 : 0x5140);
              const uint32_t cd = __byte_perm(w[2][q], w[3][q], k ? 0x7362 : 0x5140);
              if (S == KV_FP8_ROW) {
                uint32_t h[4];
                e4m3x4_half2(ab, h[0], h[1]);
                e4m3x4_half2(cd, h[2], h[3]);
                mma16<false>(o[j + 2 * k], pf, h[0], h[2]);
                mma16<false>(o[j + 2 * k + 1], pf, h[1], h[3]);
              } else {
                const uint32_t u0 = ab ^ 0x80808080u, u1 = cd ^ 0x80808080u;
                mma16<false>(o[j + 2 * k], pf, int8x2_half2<0x4140>(u0), int8x2_half2<0x4140>(u1));
                mma16<false>(o[j + 2 * k + 1], pf, int8x2_half2<0x4342>(u0), int8x2_half2<0x4342>(u1));
              }
            }
          }
        }
      }
      __syncwarp();  // the stage may be filled again
    }

    // The warps' results become one.
    cp_async_wait_all();
    __syncthreads();
    float undo = S == KV_NONE ? (kBf16 ? 1.0f : 1.0f / 16384.0f) : 1.0f / u2f((uint32_t)vfield << 23);
    if (S == KV_MXFP4) undo *= 1.0f / (1 << kGroupShift);
    float *mo = reinterpret_cast<float *>(smem) + warp * kRows * DP;
#pragma unroll
    for (int hrow = 0; hrow < 2; ++hrow) {
      sum[hrow] += __shfl_xor_sync(0xFFFFFFFFu, sum[hrow], 1);
      sum[hrow] += __shfl_xor_sync(0xFFFFFFFFu, sum[hrow], 2);
      if (t == 0) {
        merge_top[warp][g + 8 * hrow] = top[hrow];
        merge_sum[warp][g + 8 * hrow] = sum[hrow];
      }
    }
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) mo[((2 * t + (e & 1)) * (DP / 8) + j) * kRows + g + 8 * (e >> 1)] = o[j][e] * undo;
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
      weight[w] = merge_top[w][row] == -INFINITY && merge_sum[w][row] == 0.0f ? 0.0f : exp2_fast(merge_top[w][row] - m);
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

template <typename T, int S, int DP, bool PAD>
int launch_pad(const Args &a, float *parts, int most, cudaStream_t s) {
  using P = Shape<S, DP>;
  auto kern = split_kernel<T, S, DP, PAD>;
  static std::atomic<uint64_t> ready[2];  // devices whose shared-memory limit is raised
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return set_error(std::string("tc_paged_attention: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  if (dev >= 128 || !((ready[dev >> 6].load(std::memory_order_relaxed) >> (dev & 63)) & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, P::kSmem);
    if (e != cudaSuccess) return set_error(std::string("tc_paged_attention: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
    if (dev < 128) ready[dev >> 6].fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
  }
  kern<<<most, kThreads, P::kSmem, s>>>(a, parts, most);
  count_launch();
  return TC_OK;
}

template <typename T, int S, int DP>
int launch(const Args &a, float *parts, int most, cudaStream_t s) {
  return a.c.dim == DP ? launch_pad<T, S, DP, false>(a, parts, most, s) : launch_pad<T, S, DP, true>(a, parts, most, s);
}

template <int S>
int launch_scheme(const Args &a, float *parts, int most, cudaStream_t s) {
  const bool bf16 = a.c.dtype == TC_BF16;
  if (a.c.dim <= 64) return bf16 ? launch<__nv_bfloat16, S, 64>(a, parts, most, s) : launch<__half, S, 64>(a, parts, most, s);
  if (a.c.dim <= 128) return bf16 ? launch<__nv_bfloat16, S, 128>(a, parts, most, s) : launch<__half, S, 128>(a, parts, most, s);
  return bf16 ? launch<__nv_bfloat16, S, 256>(a, parts, most, s) : launch<__half, S, 256>(a, parts, most, s);
}

}  // namespace split
}  // namespace attn
}  // namespace tc
