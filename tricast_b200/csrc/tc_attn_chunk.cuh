// Attention of a chunk of new tokens over a paged cache: bound by the tensor cores and by the softmax's
// exponentials beside them.
//
// A block takes a stretch of the work line (tc_attn.cuh) in items of 256 query rows, two tiles of 128, and
// units of 128 keys. Its warps have roles, joined by mbarriers:
//  - producers (4 warps) read the codes of a unit, a step ahead in registers, and write them as 16-bit
//    operands into swizzled shared memory (K and V, two stages each), with the keys' scales beside them;
//  - one thread issues the tcgen05 MMAs: S = Q K^T of each tile into TMEM, O += P V with P read from TMEM;
//  - two groups of 4 warps, one a tile, a thread a row: S to P by the running softmax, P over the
//    columns of S it has read. One tile's softmax runs under the other's MMAs.
// TMEM: S of the two tiles (128 columns each, P over their first 64), O of the two (DP columns each).
//
// Codes are exact in fp16 and their scales stay out of the products, as in the split kernel: a key's scale
// multiplies its score, a value's its weight. Weights are kept relative to a reference that follows a row's
// maximum only when it has risen by more than 2**8 (O in TMEM is rescaled then, rarely), and to the largest
// value scale so far, so that they stay below 2**15: P = exp2(x - ref) * scale with
// ref = maximum - 6 + log2(T). The sum takes the weights before the value's scale and before their rounding.
#pragma once

#include <atomic>
#include <cmath>
#include <string>

#include "tc_attn.cuh"
#include "tc_tcgen05.cuh"

namespace tc {
namespace attn {
namespace chunk {

constexpr int kTile = 128, kRows = 2 * kTile, kKeys = 128, kSlots = 4;
constexpr int kSoftmaxWarps = 8, kProducerWarps = 4, kThreads = (kSoftmaxWarps + kProducerWarps + 1) * 32;
using W = Work<kRows, kKeys>;

template <int DP>
struct Shape {
  static constexpr int kOperand = kTile * DP * 2;  // bytes of a Q, K or V tile
  static constexpr int kHalves = DP / 64;          // 128-byte wide swizzled blocks of 128 rows
  static constexpr int kSmem = 6 * kOperand + 1024;
};

// What the softmax needs of a unit's keys.
struct __align__(16) KeySlot {
  float k[kKeys], v[kKeys];
  uint32_t valid[4];
  int vfield[4];  // largest exponent field of the value scales, by quarter
};

// 16 bytes (8 elements) of row r, granule q of a tile: 128-byte rows in blocks of 128, swizzled.
__device__ __forceinline__ uint32_t tile_at(int r, int q) {
  return (uint32_t)((q >> 3) * (kTile * 128) + r * 128 + (((q & 7) ^ (r & 7)) << 4));
}

// Shared-memory descriptors of a 128-byte-swizzled tile. K-major (rows along M or N): 8-row groups 1024
// bytes apart. MN-major (rows along K, 64 elements of N each): the next 64 of N a block (16 KB) further,
// 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Bits of a unit's 32 keys from 32 * part that a row seeing [lo, hi) (relative to the unit) sees.
__device__ __forceinline__ uint32_t range_bits(int lo, int hi, int part) {
  const int l = min(max(lo - 32 * part, 0), 32), h = min(max(hi - 32 * part, 0), 32);
  const uint32_t below_h = h == 32 ? 0xFFFFFFFFu : (1u << h) - 1u;
  const uint32_t below_l = l == 32 ? 0xFFFFFFFFu : (1u << l) - 1u;
  return below_h & ~below_l;
}

struct Barriers {
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], slot[kSlots], qfull[2], sfull[2], pfull[2], ofull[2], drain;
};

// Bounds of an item that every role derives alike.
struct Part {
  Seq s;
  int rows;            // of the sequence's heads on this key head
  bool two;            // the second tile has rows
  int64_t key0, key1;  // keys of the part
  int steps;
  int all_lo, all_hi;  // keys that every row sees
};
__device__ __forceinline__ Part part_of(const Args &a, const Item &it) {
  Part p;
  p.s = sequence(a, it.b);
  p.rows = p.s.n * a.group;
  p.two = p.rows > it.tile * kRows + kTile;
  int lo, hi, unused;
  W::keys(a, p.s, it.tile, lo, hi);
  p.key0 = (int64_t)lo + (int64_t)it.at * kKeys;
  p.key1 = min((int64_t)lo + (int64_t)(it.at + it.n) * kKeys, (int64_t)hi);
  p.steps = it.n;
  visible(a, p.s, it.tile * kRows / a.group, unused, p.all_hi);
  visible(a, p.s, (min((it.tile + 1) * kRows, p.rows) - 1) / a.group, p.all_lo, unused);
  return p;
}

// ---------------------------------------------------------------- producers
template <typename T, int S, int DP>
__device__ __forceinline__ bool produce(const Args &a, Item it, unsigned char *ks, unsigned char *vs, KeySlot *slots,
                                        Barriers &bar, int polls) {
  constexpr int kRowBytes = S == KV_NONE ? 2 * DP : S == KV_MXFP4 ? DP / 2 : DP;
  constexpr int kCpr = kRowBytes / 16;                      // 16-byte chunks of a row
  constexpr int kOwn = kCpr * kKeys / (kProducerWarps * 32);  // chunks a thread and side
  constexpr int kOut = S == KV_NONE ? 1 : S == KV_MXFP4 ? 4 : 2;  // granules of a chunk
  const KvCache &c = a.c;
  const int warp = (threadIdx.x >> 5) - kSoftmaxWarps, lane = threadIdx.x & 31, key = warp * 32 + lane;
  uint32_t step = 0;

  // A warp's chunks lie in its 32 keys, in four blocks of 8 rows: chunk i of a lane.
  auto block_of = [&](int i) { return kCpr >= 4 ? i / (kCpr / 4) : 2 * i + (lane >> 4); };
  auto chunk_of = [&](int i) { return kCpr >= 4 ? (i % (kCpr / 4)) * 4 + (lane >> 3) : (lane >> 3) & 1; };

  while (true) {
    const Part p = part_of(a, it);
    const int *table = a.table + (int64_t)it.b * a.table_stride;
    // Page of this lane's key, and with it the row: -1 for a key that is not there.
    auto page_at = [&](int j) {
      const int64_t at = p.key0 + (int64_t)j * kKeys + key;
      return j < p.steps && at < p.key1 ? table[at >> c.page_shift] : -1;
    };
    auto row_at = [&](int j, int pg) -> int64_t {
      if (pg < 0 || pg >= c.pages) return -1;
      const int64_t at = p.key0 + (int64_t)j * kKeys + key;
      return (((int64_t)pg * c.heads + it.head) << c.page_shift) + (at & (c.page_size - 1));
    };
    // Row of lane 8 i's key, as every lane of the warp needs it: rows of a block of 8 are adjacent.
    auto block_row = [&](int64_t row, int blk) { return __shfl_sync(0xFFFFFFFFu, row, 8 * blk + (lane & 7)); };

    uint4 kreg[S == KV_NONE ? 1 : kOwn], vreg[S == KV_NONE ? 1 : kOwn];
    uint32_t kword[2] = {0u, 0u}, vword[2] = {0u, 0u};  // this key's scales as they are stored
    auto load = [&](const unsigned char *codes, int64_t row, uint4 *reg) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int64_t r = block_row(row, block_of(i));
        const int ch = chunk_of(i);
        reg[S == KV_NONE ? 0 : i] = r >= 0 && ch * 16 < c.row_bytes
                                        ? __ldg(reinterpret_cast<const uint4 *>(codes + r * c.row_bytes + ch * 16))
                                        : make_uint4(0, 0, 0, 0);
      }
    };
    auto load_scale = [&](const unsigned char *scales, int64_t row, uint32_t (&w)[2]) {
      w[0] = w[1] = 0u;
      if (row < 0) return;
      if (S == KV_MXFP4) {
#pragma unroll
        for (int q = 0; q < DP / 32; ++q)
          if (q < c.scale_bytes) w[0] |= (uint32_t)scales[row * c.scale_bytes + q] << (8 * q);
      } else if (S != KV_NONE) {
        w[0] = *reinterpret_cast<const uint32_t *>(scales + row * 4);
      }
    };
    // Largest group exponent of a key (mxfp4).
    auto biggest = [&](uint32_t w) {
      int big = 0;
#pragma unroll
      for (int q = 0; q < DP / 32; ++q) big = max(big, (int)((w >> (8 * q)) & 0xFFu));
      return big;
    };
    auto convert = [&](const uint4 *reg, uint32_t scale_word, bool dead, unsigned char *dst) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int blk = block_of(i), ch = chunk_of(i), r = warp * 32 + blk * 8 + (lane & 7);
        const uint4 in = reg[S == KV_NONE ? 0 : i];
        const uint32_t w[4] = {in.x, in.y, in.z, in.w};
        uint32_t h[4 * kOut];
        if (S == KV_MXFP4) {
          const uint32_t sw = __shfl_sync(0xFFFFFFFFu, scale_word, 8 * blk + (lane & 7));
          const uint32_t mul = half_pow2((int)((sw >> (8 * ch)) & 0xFFu) - biggest(sw) + kGroupShift) * 0x10001u;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t e[4];
            e2m1x8_half2(w[q], e);
#pragma unroll
            for (int k = 0; k < 4; ++k) h[(4 * q + k) % (4 * kOut)] = mul_half2(e[k], mul);
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (S == KV_FP8_ROW) {
              h[(2 * q) % (4 * kOut)] = e4m3x2_half2(w[q] & 0xFFFFu);
              h[(2 * q + 1) % (4 * kOut)] = e4m3x2_half2(w[q] >> 16);
            } else {
              h[(2 * q) % (4 * kOut)] = int8x2_half2<0x4140>(w[q] ^ 0x80808080u);
              h[(2 * q + 1) % (4 * kOut)] = int8x2_half2<0x4342>(w[q] ^ 0x80808080u);
            }
          }
        }
        // A key with a NaN scale has NaN codes, which would reach rows that do not see it as 0 * NaN: they
        // count as 0, and the scale carries the NaN.
        const bool zero = S == KV_FP8_ROW && __shfl_sync(0xFFFFFFFFu, (int)dead, 8 * blk + (lane & 7));
#pragma unroll
        for (int g = 0; g < kOut; ++g)
          *reinterpret_cast<uint4 *>(dst + tile_at(r, ch * kOut + g)) =
              zero ? make_uint4(0, 0, 0, 0)
                   : make_uint4(h[(4 * g) % (4 * kOut)], h[(4 * g + 1) % (4 * kOut)], h[(4 * g + 2) % (4 * kOut)],
                                h[(4 * g + 3) % (4 * kOut)]);
      }
    };
    // Unquantized rows go straight to shared memory.
    auto copy = [&](const unsigned char *codes, int64_t row, bool skip, unsigned char *dst) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int blk = block_of(i), ch = chunk_of(i), r = warp * 32 + blk * 8 + (lane & 7);
        const int64_t from = block_row(skip ? -1 : row, blk);
        const bool use = from >= 0 && ch * 16 < c.row_bytes;
        cp_async16_or_zero(dst + tile_at(r, ch), codes + (use ? from : 0) * c.row_bytes + (use ? ch * 16 : 0), use);
      }
    };
    // The key's entry of the unit's slot; true where its V row must count as zeros.
    auto put_slot = [&](int j, int64_t row) {
      KeySlot &sl = slots[(step + j) % kSlots];
      float k = 1.0f, v = 1.0f;
      bool dead = false;
      if (S == KV_MXFP4) {
        k = pow2_value((uint32_t)biggest(kword[0])) * (1.0f / (1 << kGroupShift));
        v = pow2_value((uint32_t)biggest(vword[0])) * (1.0f / (1 << kGroupShift));
      } else if (S != KV_NONE) {
        k = u2f(kword[0]);
        v = u2f(vword[0]);
        dead = v != v;
      } else {
        const int64_t p0 = p.key0 + (int64_t)j * kKeys;
        if (row >= 0 && !(p0 >= p.all_lo && p0 + kKeys <= p.all_hi)) {
          // Rows differ in what they see: a value that is not finite must not reach the others. The whole
          // V row counts as 0 and the weights of the rows that see it become NaN.
          const uint32_t m = Same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u;
          for (int d = 0; d < c.row_bytes / 4; ++d) {
            const uint32_t w = reinterpret_cast<const uint32_t *>(c.v + row * c.row_bytes)[d];
            dead |= (w & m) == m || ((w >> 16) & m) == m;
          }
          if (dead) v = u2f(kQNaN);
        }
      }
      if (row < 0) k = v = 0.0f;
      sl.k[key] = k;
      sl.v[key] = v;
      const uint32_t valid = __ballot_sync(0xFFFFFFFFu, row >= 0);
      const int f = (int)((f2u(v) >> 23) & 0xFFu);
      const int top = (int)__reduce_max_sync(0xFFFFFFFFu, (uint32_t)(f == 255 ? 0 : f));
      if (lane == 0) {
        sl.valid[warp] = valid;
        sl.vfield[warp] = top;
      }
      return dead;
    };

    int64_t row = row_at(0, page_at(0));
    int page = page_at(1);
    if (S != KV_NONE) {
      load_scale(c.ks, row, kword);
      load_scale(c.vs, row, vword);
      load(c.k, row, kreg);
      load(c.v, row, vreg);
      for (int j = 0; j < p.steps; ++j) {
        const uint32_t n = step + j, st = n & 1, ph = (n >> 1) & 1;
        const int64_t next = row_at(j + 1, page);
        page = page_at(j + 2);
        if (!mbar_wait_sleep(&bar.kempty[st], ph ^ 1, polls)) return false;
        const bool dead = put_slot(j, row);
        convert(kreg, kword[0], false, ks + st * Shape<DP>::kOperand);
        fence_async_proxy();
        mbar_arrive(&bar.kfull[st]);
        mbar_arrive(&bar.slot[n % kSlots]);
        const uint32_t vw = vword[0];
        load(c.k, next, kreg);
        load_scale(c.ks, next, kword);
        load_scale(c.vs, next, vword);
        if (!mbar_wait_sleep(&bar.vempty[st], ph ^ 1, polls)) return false;
        convert(vreg, vw, dead, vs + st * Shape<DP>::kOperand);
        fence_async_proxy();
        mbar_arrive(&bar.vfull[st]);
        load(c.v, next, vreg);
        row = next;
      }
    } else {
      bool dead = false;
      if (!mbar_wait_sleep(&bar.kempty[step & 1], ((step >> 1) & 1) ^ 1, polls)) return false;
      copy(c.k, row, false, ks + (step & 1) * Shape<DP>::kOperand);
      cp_async_commit();
      dead = put_slot(0, row);
      if (!mbar_wait_sleep(&bar.vempty[step & 1], ((step >> 1) & 1) ^ 1, polls)) return false;
      copy(c.v, row, dead, vs + (step & 1) * Shape<DP>::kOperand);
      cp_async_commit();
      for (int j = 0; j < p.steps; ++j) {
        const uint32_t n = step + j, st = n & 1, nst = (n + 1) & 1, nph = ((n + 1) >> 1) & 1;
        const int64_t next = row_at(j + 1, page);
        page = page_at(j + 2);
        const bool more = j + 1 < p.steps;
        if (more) {
          if (!mbar_wait_sleep(&bar.kempty[nst], nph ^ 1, polls)) return false;
          copy(c.k, next, false, ks + nst * Shape<DP>::kOperand);
        }
        cp_async_commit();
        cp_async_wait<2>();
        fence_async_proxy();
        mbar_arrive(&bar.kfull[st]);
        mbar_arrive(&bar.slot[n % kSlots]);
        if (more) {
          dead = put_slot(j + 1, next);
          if (!mbar_wait_sleep(&bar.vempty[nst], nph ^ 1, polls)) return false;
          copy(c.v, next, dead, vs + nst * Shape<DP>::kOperand);
        }
        cp_async_commit();
        cp_async_wait<2>();
        fence_async_proxy();
        mbar_arrive(&bar.vfull[st]);
        row = next;
      }
      cp_async_wait_all();
    }
    step += (uint32_t)p.steps;
    if (it.left == 0) return true;
    W::next(a, it);
  }
}

// ---------------------------------------------------------------- MMA issue (one thread)
template <bool BF16, int DP>
__device__ __forceinline__ bool multiply(const Args &a, Item it, uint32_t qs, uint32_t ks, uint32_t vs, uint32_t tmem,
                                         Barriers &bar, int polls, bool &issued) {
  constexpr uint32_t kType = BF16 ? (1u << 7) | (1u << 10) : 0u;
  constexpr uint32_t kQk = (1u << 4) | kType | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
  constexpr uint32_t kPv = (1u << 4) | kType | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
  uint32_t step = 0, items[2] = {0u, 0u}, psteps[2] = {0u, 0u};
  while (true) {
    const Part p = part_of(a, it);
    const int tiles = p.two ? 2 : 1;
    auto qk = [&](int t, uint32_t n) {
      const uint32_t k0 = ks + (n & 1) * Shape<DP>::kOperand, q0 = qs + t * Shape<DP>::kOperand;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint32_t off = (k >> 2) * (kTile * 128) + (k & 3) * 32;
        tc5::mma_f16_ss(tmem + t * 128, desc_sw128(q0 + off, 16), desc_sw128(k0 + off, 16), kQk, k > 0);
      }
      issued = true;
      tc5::mma_commit(&bar.sfull[t]);
    };
    for (int t = 0; t < tiles; ++t)
      if (!mbar_wait_sleep(&bar.qfull[t], items[t]++ & 1, polls)) return false;
    if (!mbar_wait(&bar.kfull[step & 1], (step >> 1) & 1, polls)) return false;
    tc5::fence_after_sync();
    for (int t = 0; t < tiles; ++t) qk(t, step);
    tc5::mma_commit(&bar.kempty[step & 1]);
    for (int j = 0; j < p.steps; ++j) {
      const uint32_t n = step + j;
      const bool more = j + 1 < p.steps;
      for (int t = 0; t < tiles; ++t) {
        if (!mbar_wait(&bar.pfull[t], psteps[t]++ & 1, polls)) return false;
        if (t == 0 && !mbar_wait(&bar.vfull[n & 1], (n >> 1) & 1, polls)) return false;
        tc5::fence_after_sync();
        const uint32_t v0 = vs + (n & 1) * Shape<DP>::kOperand;
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          tc5::mma_f16_ts(tmem + 256 + t * DP, tmem + t * 128 + k * 8, desc_sw128(v0 + k * 2048, kTile * 128), kPv,
                          j > 0 || k > 0);
        if (t == tiles - 1) tc5::mma_commit(&bar.vempty[n & 1]);
        if (more) {
          if (t == 0) {
            if (!mbar_wait(&bar.kfull[(n + 1) & 1], ((n + 1) >> 1) & 1, polls)) return false;
            tc5::fence_after_sync();
          }
          qk(t, n + 1);
          if (t == tiles - 1) tc5::mma_commit(&bar.kempty[(n + 1) & 1]);
        } else {
          tc5::mma_commit(&bar.ofull[t]);
        }
      }
    }
    step += (uint32_t)p.steps;
    if (it.left == 0) return true;
    W::next(a, it);
  }
}

// ---------------------------------------------------------------- softmax (a thread a row)
template <typename T, int S, int DP>
__device__ __forceinline__ bool softmax(const Args &a, Item it, unsigned char *qs, const KeySlot *slots, uint32_t tmem,
                                        Barriers &bar, int polls, float *parts) {
  constexpr bool kBf16 = S == KV_NONE && Same<T, __nv_bfloat16>::value;
  const int t = threadIdx.x >> 7, row = threadIdx.x & 127;
  const uint32_t lanes = (uint32_t)((threadIdx.x >> 5) & 3) << 21;  // this warp's 32 lanes of TMEM, bits 16 up
  const uint32_t ts = tmem + lanes + t * 128, to = tmem + lanes + 256 + t * DP;
  unsigned char *q0 = qs + t * Shape<DP>::kOperand;
  const bool qvec = ((uintptr_t)a.q | (uintptr_t)(a.q_tok * 2) | (uintptr_t)(a.q_head * 2)) % 16 == 0;
  uint32_t step = 0, ssteps = 0, items = 0;
  while (true) {
    const Part p = part_of(a, it);
    if (t == 0 || p.two) {
      const int r = it.tile * kRows + t * kTile + row;
      const int tok = min(r, p.rows - 1) / a.group;
      const int head = it.head * a.group + r % a.group;
      // Q: the row as 16-bit operand; over quantized caches scaled by a power of two into fp16.
      float qmul = a.scale;
      {
        const T *qp = static_cast<const T *>(a.q) + (p.s.q0 + tok) * a.q_tok + head * a.q_head;
        uint32_t w[DP / 2];
#pragma unroll
        for (int g = 0; g < DP / 8; ++g) {
          uint32_t x[4] = {0u, 0u, 0u, 0u};
          if (r < p.rows && 8 * g < a.c.dim) {
            if (qvec) {
              load_words<4>(reinterpret_cast<const unsigned char *>(qp + 8 * g), x);
            } else {
              const unsigned short *u = reinterpret_cast<const unsigned short *>(qp + 8 * g);
#pragma unroll
              for (int k = 0; k < 4; ++k) x[k] = (uint32_t)u[2 * k] | ((uint32_t)u[2 * k + 1] << 16);
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) w[4 * g + k] = x[k];
        }
        if (S != KV_NONE) {
          float big = 0.0f;
#pragma unroll
          for (int k = 0; k < DP / 2; ++k)
            big = fmaxf(big, fmaxf(fabsf(half_bits_to_float<T>(w[k] & 0xFFFFu)), fabsf(half_bits_to_float<T>(w[k] >> 16))));
          const Pow2 f = fp16_shift(big);
          qmul *= f.inverse;
#pragma unroll
          for (int k = 0; k < DP / 2; ++k)
            w[k] = pack_half(half_bits_to_float<T>(w[k] & 0xFFFFu) * f.factor, half_bits_to_float<T>(w[k] >> 16) * f.factor);
        }
#pragma unroll
        for (int g = 0; g < DP / 8; ++g)
          *reinterpret_cast<uint4 *>(q0 + tile_at(row, g)) = make_uint4(w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]);
        fence_async_proxy();
        tc5::fence_before_sync();
        mbar_arrive(&bar.qfull[t]);
      }
      int see_lo, see_hi;
      visible(a, p.s, tok, see_lo, see_hi);
      const uint64_t qmul2 = pack2(qmul, qmul);
      float top = -INFINITY;  // maximum that ref follows
      float ref = 0.0f;       // base-2 logarithm that weights are relative to
      uint64_t sum2 = 0ull;
      int vfield = kBf16 ? 127 : 0;  // exponent field of T
      for (int j = 0; j < p.steps; ++j) {
        const uint32_t n = step + j;
        const KeySlot &sl = slots[n % kSlots];
        if (!mbar_wait_sleep(&bar.slot[n % kSlots], (n / kSlots) & 1, polls)) return false;
        if (!mbar_wait(&bar.sfull[t], ssteps++ & 1, polls)) return false;
        tc5::fence_after_sync();
        const int64_t p0 = p.key0 + (int64_t)j * kKeys;
        const bool whole = p0 >= p.all_lo && p0 + kKeys <= p.all_hi &&
                           (sl.valid[0] & sl.valid[1] & sl.valid[2] & sl.valid[3]) == 0xFFFFFFFFu;
        const int lo = (int)max(min((int64_t)see_lo - p0, (int64_t)kKeys), (int64_t)0);
        const int hi = (int)max(min((int64_t)see_hi - p0, (int64_t)kKeys), (int64_t)0);

        // The maximum of the row's scores.
        float m = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t x[32];
          tc5::tmem_ld32(ts + 32 * q, x);
          const uint32_t bits = whole ? 0xFFFFFFFFu : sl.valid[q] & range_bits(lo, hi, q);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float v[4] = {u2f(x[i]), u2f(x[i + 1]), u2f(x[i + 2]), u2f(x[i + 3])};
            if (S != KV_NONE) {
              const float4 k4 = *reinterpret_cast<const float4 *>(&sl.k[32 * q + i]);
              unpack2(mul2(pack2(v[0], v[1]), pack2(k4.x, k4.y)), v[0], v[1]);
              unpack2(mul2(pack2(v[2], v[3]), pack2(k4.z, k4.w)), v[2], v[3]);
            }
            if (!whole) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!((bits >> (i + e)) & 1u)) v[e] = qmul >= 0.0f ? -INFINITY : INFINITY;
            }
            if (qmul >= 0.0f) m = fmaxf(m, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
            else m = fmaxf(m, -fminf(fminf(v[0], v[1]), fminf(v[2], v[3])));
          }
        }
        m = m == -INFINITY ? m : m * fabsf(qmul);
        // The reference moves when the maximum has risen by more than 2**8 (or from nothing), and when
        // a larger value scale comes.
        int field = vfield;
        if (!kBf16) field = max(max(field, max(sl.vfield[0], sl.vfield[1])), max(sl.vfield[2], sl.vfield[3]));
        const bool up = m > top + 8.0f || (top == -INFINITY && m != -INFINITY);
        if (__any_sync(0xFFFFFFFFu, up) || field != vfield) {
          const float now = up ? m : top;
          // exp2(x - ref) <= 2**(8 + 6) / T, at most 2**(8 + 100).
          const float next = (now == -INFINITY ? 0.0f : now) - fminf(6.0f + (127.0f - (float)field), 100.0f);
          const float keep = top == -INFINITY ? 0.0f : exp2_fast(ref - next);
          top = now;
          ref = next;
          vfield = field;
          sum2 = mul2(sum2, pack2(keep, keep));
          if (j > 0) {
#pragma unroll
            for (int q = 0; q < DP / 32; ++q) {
              uint32_t x[32];
              tc5::tmem_ld32(to + 32 * q, x);
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = f2u(u2f(x[i]) * keep);
              tc5::tmem_st32(to + 32 * q, x);
            }
          }
        }
        const uint64_t nref2 = pack2(-ref, -ref);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t x[32], w[16];
          tc5::tmem_ld32(ts + 32 * q, x);
          const uint32_t bits = whole ? 0xFFFFFFFFu : sl.valid[q] & range_bits(lo, hi, q);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            uint64_t y0 = pack2(u2f(x[i]), u2f(x[i + 1])), y1 = pack2(u2f(x[i + 2]), u2f(x[i + 3]));
            if (S != KV_NONE) {
              const float4 k4 = *reinterpret_cast<const float4 *>(&sl.k[32 * q + i]);
              y0 = mul2(y0, pack2(k4.x, k4.y));
              y1 = mul2(y1, pack2(k4.z, k4.w));
            }
            y0 = fma2(y0, qmul2, nref2);
            y1 = fma2(y1, qmul2, nref2);
            float v[4];
            unpack2(y0, v[0], v[1]);
            unpack2(y1, v[2], v[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[e] = exp2_fast(v[e]);
              if (!whole && !((bits >> (i + e)) & 1u)) v[e] = 0.0f;
            }
            y0 = pack2(v[0], v[1]);
            y1 = pack2(v[2], v[3]);
            sum2 = add2(sum2, add2(y0, y1));
            if (S != KV_NONE || !whole) {
              const float4 v4 = *reinterpret_cast<const float4 *>(&sl.v[32 * q + i]);
              unpack2(mul2(y0, pack2(v4.x, v4.y)), v[0], v[1]);
              unpack2(mul2(y1, pack2(v4.z, v4.w)), v[2], v[3]);
              if (!whole) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (!((bits >> (i + e)) & 1u)) v[e] = 0.0f;  // whatever the scale
              }
            }
            w[i / 2] = kBf16 ? pack_bf16(v[0], v[1]) : pack_half(v[0], v[1]);
            w[i / 2 + 1] = kBf16 ? pack_bf16(v[2], v[3]) : pack_half(v[2], v[3]);
          }
          tc5::tmem_st16(ts + 16 * q, w);
        }
        tc5::tmem_wait_st();
        tc5::fence_before_sync();
        mbar_arrive(&bar.pfull[t]);
      }
      // The item's part is done.
      if (!mbar_wait_sleep(&bar.ofull[t], items++ & 1, polls)) return false;
      tc5::fence_after_sync();
      float sum, s1;
      unpack2(sum2, sum, s1);
      sum += s1;
      const bool done = it.at == 0 && it.n == it.units;
      float *part = parts + (size_t)(2 * blockIdx.x + (it.at > 0 ? 0 : 1)) * partial_floats(kRows, DP) + t * kTile + row;
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      const int64_t out_row = (p.s.q0 + tok) * a.heads + head;
#pragma unroll
      for (int q = 0; q < DP / 32; ++q) {
        uint32_t x[32];
        tc5::tmem_ld32(to + 32 * q, x);
        if (!done) {
#pragma unroll
          for (int i = 0; i < 32; ++i) part[(2 + 32 * q + i) * kRows] = u2f(x[i]);
        } else if (r < p.rows) {
          T *o = static_cast<T *>(a.out) + out_row * a.c.dim + 32 * q;
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            if (32 * q + i < a.c.dim) {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                w[k] = sum == 0.0f ? 0u : pack16<T>(u2f(x[i + 2 * k]) * inv, u2f(x[i + 2 * k + 1]) * inv);
              *reinterpret_cast<uint4 *>(o + i) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
      }
      if (!done) {
        part[0] = sum == 0.0f ? -INFINITY : ref;
        part[kRows] = sum;
      } else if (a.lse && r < p.rows) {
        a.lse[out_row] = sum == 0.0f ? -INFINITY : (ref + log2f(sum)) * 0.69314718055994531f;
      }
      tc5::fence_before_sync();
    }
    step += (uint32_t)p.steps;
    if (it.left == 0) return true;
    W::next(a, it);
  }
}

template <typename T, int S, int DP>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(Args a, float *parts, int *status, int most, int polls) {
  constexpr bool kBf16 = S == KV_NONE && Same<T, __nv_bfloat16>::value;
  extern __shared__ unsigned char raw[];
  __shared__ KeySlot slots[kSlots];
  __shared__ __align__(8) Barriers bar;
  __shared__ Item first;
  __shared__ uint32_t tmem_base;
  __shared__ int failed;
  unsigned char *smem = raw + (1024 - (smem_addr(raw) & 1023)) % 1024;  // the swizzle is of address bits
  unsigned char *qs = smem, *ks = qs + 2 * Shape<DP>::kOperand, *vs = ks + 2 * Shape<DP>::kOperand;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == kSoftmaxWarps) {
    const int64_t total = W::total(a);
    const int n = W::blocks(total, most);
    Item it{0, 0, 0, 0, 0, 0, 0};
    if ((int)blockIdx.x < n) {
      const int64_t u0 = W::start(total, blockIdx.x, n), u1 = W::start(total, blockIdx.x + 1, n);
      it = W::find(a, u0);
      it.n = (int)min((int64_t)(it.units - it.at), u1 - u0);
      it.left = u1 - u0 - it.n;
    }
    if (lane == 0) {
      first = it;
      failed = 0;
    }
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.kfull[i], kProducerWarps * 32);
      mbar_init(&bar.vfull[i], kProducerWarps * 32);
      mbar_init(&bar.kempty[i], 1);
      mbar_init(&bar.vempty[i], 1);
      mbar_init(&bar.qfull[i], kTile);
      mbar_init(&bar.pfull[i], kTile);
      mbar_init(&bar.sfull[i], 1);
      mbar_init(&bar.ofull[i], 1);
    }
    for (int i = 0; i < kSlots; ++i) mbar_init(&bar.slot[i], kProducerWarps * 32);
    mbar_init(&bar.drain, 1);
    fence_barrier_init();
  }
  if (warp == 1) tc5::tmem_alloc(&tmem_base, 512);
  tc5::fence_before_sync();
  __syncthreads();
  tc5::fence_after_sync();
  const Item it = first;
  const uint32_t tmem = tmem_base;
  if (it.n > 0) {
    bool ok = true;
    if (warp < kSoftmaxWarps) {
      ok = softmax<T, S, DP>(a, it, qs, slots, tmem, bar, polls, parts);
    } else if (warp < kSoftmaxWarps + kProducerWarps) {
      ok = produce<T, S, DP>(a, it, ks, vs, slots, bar, polls);
      cp_async_wait_all();
    } else if (lane == 0) {
      bool issued = false;
      ok = multiply<kBf16, DP>(a, it, smem_addr(qs), smem_addr(ks), smem_addr(vs), tmem, bar, polls, issued);
      if (issued) {
        // No MMA may be in flight when the block's shared memory and TMEM go.
        tc5::mma_commit(&bar.drain);
        mbar_wait_sleep(&bar.drain, 0);
      }
    }
    if (!ok) failed = 1;
  }
  tc5::fence_before_sync();
  __syncthreads();
  tc5::fence_after_sync();
  if (warp == 1) tc5::tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0) status[blockIdx.x] = failed;
}

template <typename T, int S, int DP>
int launch(const Args &a, float *parts, int *status, int most, cudaStream_t s) {
  auto kern = chunk_kernel<T, S, DP>;
  static std::atomic<uint64_t> ready[2];  // devices whose shared-memory limit is raised
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return set_error(std::string("tc_paged_attention: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  if (dev >= 128 || !((ready[dev >> 6].load(std::memory_order_relaxed) >> (dev & 63)) & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP>::kSmem);
    if (e != cudaSuccess) return set_error(std::string("tc_paged_attention: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
    if (dev < 128) ready[dev >> 6].fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
  }
  kern<<<most, kThreads, Shape<DP>::kSmem, s>>>(a, parts, status, most, wait_polls());
  count_launch();
  return TC_OK;
}

template <int S>
int launch_scheme(const Args &a, float *parts, int *status, int most, cudaStream_t s) {
  const bool bf16 = a.c.dtype == TC_BF16;
  if (a.c.dim <= 64)
    return bf16 ? launch<__nv_bfloat16, S, 64>(a, parts, status, most, s) : launch<__half, S, 64>(a, parts, status, most, s);
  return bf16 ? launch<__nv_bfloat16, S, 128>(a, parts, status, most, s) : launch<__half, S, 128>(a, parts, status, most, s);
}

}  // namespace chunk
}  // namespace attn
}  // namespace tc
