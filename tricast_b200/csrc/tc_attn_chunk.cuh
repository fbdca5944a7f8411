// Attention of a chunk of new tokens over a paged cache: bound by the tensor cores and by the softmax's
// exponentials beside them.
//
// A block takes a stretch of the work line (tc_attn.cuh) in items of 256 query rows, two tiles of 128, and
// units of 128 keys. Its warps have roles, joined by mbarriers:
//  - producers (7 warps) take the quarters of K and V tiles in turn: the codes of 32 keys, fetched into registers
//    a turn ahead, become 16-bit operands in swizzled shared memory (K and V, two stages each), with the
//    keys' scales beside them. Where many row tiles read the same keys, pack_kernel has laid the operands out
//    beforehand and one thread fetches them by bulk copies: conversions and stores for every tile cost 300 of
//    1450 us below;
//  - one warp issues the tcgen05 MMAs: S = Q K^T of each tile into TMEM, O += P V with P read from TMEM;
//  - two groups of 4 warps, one a tile, a warp 32 rows: S to P by the running softmax, P over the columns
//    of S it has read, half a unit at a time. One tile's softmax runs under the other's MMAs.
// TMEM: S of the two tiles (128 columns each, P of a half over the half's first 32), O of the two (DP columns each).
//
// 4096 new tokens at the end of 16384, 32 query and 8 key heads of 128, E4M3, causal: 952 to 983 us, 979 to 1010 TFLOP/s,
// 61 to 63% of the measured bf16 peak (1056 us a call among others with inputs of their own, 56%). The MMAs with
// everything but the weights' arithmetic take 730 us; a unit's 256 x 128
// exponentials are 2048 cycles of the 4500 a unit takes, and the two do not overlap fully: a tile's next scores
// wait for its weights. Scores in halves of 64 keys, so that they need not, took more MMAs of the same price each
// and gained nothing; two issuing warps lost 6%.
//
// Codes are exact in fp16 and their scales stay out of the products, as in the split kernel: a key's scale
// multiplies its score, a value's its weight. Weights are kept relative to a reference that follows a row's
// largest product of weight and value scale (tc_attn.cuh) only when it has risen by more than 2**8 (O in TMEM is
// rescaled then, rarely), so that the products stay below 2**15. The sum takes the weights before the value's scale
// and before their rounding.
#pragma once

#include <atomic>
#include <cmath>
#include <string>

#include "tc_attn.cuh"
#include "tc_tcgen05.cuh"

namespace tc {
namespace attn {
namespace chunk {

constexpr int kTile = 128, kRows = 2 * kTile, kKeys = 128, kHalf = kKeys / 2, kSlots = 4;
constexpr int kSoftmaxWarps = 8, kProducerWarps = 7, kThreads = 512;  // and one warp for the MMA thread
// Registers a thread: 128 at launch; 256 * 160 + 256 * 96 = 512 * 128. Over packed units one warp stands in for the
// producers, in a group of four with the MMA thread's: 168 at launch; 256 * 208 + 128 * 88 = 384 * 168.
constexpr int kPackedThreads = 384;
constexpr int softmax_regs(bool packed) { return packed ? 208 : 160; }
constexpr int other_regs(bool packed) { return packed ? 88 : 96; }
using W = Work<kRows, kKeys>;

template <int DP>
struct Shape {
  static constexpr int kOperand = kTile * DP * 2;  // bytes of a Q, K or V tile
  static constexpr int kHalves = DP / 64;          // 128-byte wide swizzled blocks of 128 rows
  static constexpr int kSmem = 6 * kOperand + 1024;
};

// What the softmax needs of a unit's keys.
constexpr int kOdd = 0x7FFFFFFF;
struct __align__(16) KeySlot {
  float k[kKeys], v[kKeys];
  uint32_t valid[4];  // keys that are there
  uint32_t dead[4];   // keys whose scale is not a number: it is 1 here, and the rows that see them become NaN
  // Largest and least exponent field of the value scales, by quarter (0 and 255: none). A key whose values the products
  // leave out (tc_attn.cuh) has the scale -0 here, and makes its quarter's largest kOdd, which no reference is low enough
  // for; one whose values are zeros has the scale 0, and counts in neither.
  int top[4], low[4];
};

// What pack_kernel leaves of a unit: the K and V tiles as they lie in shared memory, then the slot.
constexpr int KV_PACKED = 100;  // in place of a scheme: the kernel over such units
template <int DP>
struct Packed {
  static constexpr int kSlot = 2 * Shape<DP>::kOperand;
  static constexpr int kBytes = kSlot + (int)(sizeof(KeySlot) + 127) / 128 * 128;
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

// Pairs of fp32: one instruction where two would issue.
using F2 = uint64_t;
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(F2 v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 16 bytes that L1 need not keep: what shared memory leaves of it holds the few spilled registers.
__device__ __forceinline__ uint4 load_once(const unsigned char *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__device__ __forceinline__ void st_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Bits of a unit's 32 keys from 32 * part that a row seeing [lo, hi) (relative to the unit) sees.
__device__ __forceinline__ uint32_t range_bits(int lo, int hi, int part) {
  const int l = min(max(lo - 32 * part, 0), 32), h = min(max(hi - 32 * part, 0), 32);
  const uint32_t below_h = h == 32 ? 0xFFFFFFFFu : (1u << h) - 1u;
  const uint32_t below_l = l == 32 ? 0xFFFFFFFFu : (1u << l) - 1u;
  return below_h & ~below_l;
}

// One arrival for the warp, after what its threads have done: every thread's arrival costs about 20 cycles, one
// after the other.
__device__ __forceinline__ void warp_arrive(uint64_t *bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Waits by a whole warp, whose threads go on together or give up together.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, int polls) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, polls));
}
__device__ __forceinline__ bool warp_wait_sleep(uint64_t *bar, uint32_t parity, int polls) {
  return __all_sync(0xFFFFFFFFu, mbar_wait_sleep(bar, parity, polls));
}

// The same value in every thread of the warp, known to be.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xFFFFFFFFu, v, 0); }

struct Barriers {
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], slot[kSlots], qfull[2], sfull[2], pfull[2][2], pvdone[2], ofull[2], drain;
};

// Bounds of an item that every role derives alike.
struct Part {
  Seq s;
  int rows;            // of the sequence's heads on this key head
  bool two;            // the second tile has rows
  int key0, key1;      // keys of the part
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
  p.key0 = lo + it.at * kKeys;
  p.key1 = min(lo + (it.at + it.n) * kKeys, hi);
  p.steps = it.n;
  visible(a, p.s, it.tile * kRows / a.group, unused, p.all_hi);
  visible(a, p.s, (min((it.tile + 1) * kRows, p.rows) - 1) / a.group, p.all_lo, unused);
  return p;
}

// What a warp knows of its item, kept in shared memory: registers are for what every step needs.
struct Stash {
  Item it;
  Part p;
  bool odd;  // the products left values out (of an item of the softmax, over a quantized cache)
};
// The stash is written by one lane and read by all; the barriers keep the compiler from holding copies.
__device__ __forceinline__ void put(Stash &st, const Item &it, const Part &p) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    st.it = it;
    st.p = p;
    st.odd = false;
  }
  __syncwarp();
}

// ---------------------------------------------------------------- codes to operands
// Largest group exponent of a key (mxfp4), whose scales are the bytes of a word.
template <int DP>
__device__ __forceinline__ int biggest(uint32_t w) {
  int big = 0;
#pragma unroll
  for (int q = 0; q < DP / 32; ++q) big = max(big, (int)((w >> (8 * q)) & 0xFFu));
  return big;
}
// What a group's elements are multiplied by, twice, for a key of this largest exponent.
__device__ __forceinline__ uint32_t group_mul(uint32_t exponent, int big) {
  return half_pow2((int)exponent - big + kGroupShift) * 0x10001u;
}
// Eight 16-bit elements: granule g of 16 bytes of codes.
template <int S>
__device__ __forceinline__ void granule(const uint32_t (&w)[4], int g, uint32_t mul, uint32_t (&h)[4]) {
  if (S == KV_MXFP4) {
    e2m1x8_half2(w[g % 4], h);
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = mul_half2(h[k], mul);
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t v = w[(2 * g + k) % 4];
      if (S == KV_FP8_ROW) {
        e4m3x4_half2(v, h[2 * k], h[2 * k + 1]);
      } else {
        h[2 * k] = int8x2_half2<0x4140>(v ^ 0x80808080u);
        h[2 * k + 1] = int8x2_half2<0x4342>(v ^ 0x80808080u);
      }
    }
  }
}
// A quarter's entries of its unit's slot, a lane a key: its row in the cache (-1: it is not there) and its scales' words.
template <int S, int DP>
__device__ __forceinline__ void put_keys(const KvCache &c, KeySlot &sl, int quarter, int64_t row, uint32_t kw, uint32_t vw) {
  const int lane = threadIdx.x & 31;
  const bool there = row >= 0;
  float k = 1.0f, v = 1.0f;
  if (S == KV_MXFP4) {
    k = pow2_value((uint32_t)biggest<DP>(kw)) * (1.0f / (1 << kGroupShift));
    v = pow2_value((uint32_t)biggest<DP>(vw)) * (1.0f / (1 << kGroupShift));
  } else if (S != KV_NONE) {
    k = u2f(kw);
    v = u2f(vw);
  }
  const bool dead = k != k;
  const bool odd = there && odd_scale(f2u(v));
  if (!there || dead) k = 1.0f;
  k = k == 0.0f ? 1.1754943508222875e-38f : k;  // a slot that was never written: scores of 0, hidden ones still -Inf
  if (!there) v = 1.0f;
  bool zeros = false;
  if ((S == KV_FP8_ROW || S == KV_INT8_ROW) && there && vw == kOneScale) {
    uint32_t bits = 0u;
    for (int d = 0; d < c.row_bytes; d += 16) {
      uint32_t w[4];
      load_words<4>(c.v + row * c.row_bytes + d, w);
      bits |= nonzero_codes<S>(w[0] | w[1] | w[2] | w[3]);
    }
    zeros = bits == 0u;
  }
  if (zeros) v = 0.0f;
  if (odd) v = -0.0f;
  sl.k[32 * quarter + lane] = k;
  sl.v[32 * quarter + lane] = v;
  const uint32_t valid = __ballot_sync(0xFFFFFFFFu, there), dead_keys = __ballot_sync(0xFFFFFFFFu, there && dead);
  const int top = (int)__reduce_max_sync(0xFFFFFFFFu, odd ? (unsigned)kOdd : there ? f2u(v) >> 23 : 0u);
  const int low = (int)__reduce_min_sync(0xFFFFFFFFu, there && !odd && !zeros ? f2u(v) >> 23 : 255u);
  if (lane == 0) {
    sl.valid[quarter] = valid;
    sl.dead[quarter] = dead_keys;
    sl.top[quarter] = top;
    sl.low[quarter] = low;
  }
}
// The word of a row's scales.
template <int S, int DP>
__device__ __forceinline__ uint32_t scale_word(const KvCache &c, const unsigned char *scales, int64_t row) {
  uint32_t w = 0u;
  if (S == KV_MXFP4) {
#pragma unroll
    for (int q = 0; q < DP / 32; ++q)
      if (q < c.scale_bytes) w |= (uint32_t)scales[row * c.scale_bytes + q] << (8 * q);
  } else if (S != KV_NONE) {
    w = *reinterpret_cast<const uint32_t *>(scales + row * 4);
  }
  return w;
}

// ---------------------------------------------------------------- producers
// A job is 32 keys (a quarter) of a unit's K or V: job 8 u + 4 side + quarter of the block's unit u. A warp
// takes every seventh.
struct Job {
  int page;    // of this lane's key, -1 for a key that is not there
  int at;      // its position
  int head;
  bool mixed;  // the item's rows differ in which of the unit's keys they see
};

template <typename T, int S, int DP>
__device__ __forceinline__ bool produce(const Args &a, unsigned char *ks, unsigned char *vs, KeySlot *slots, Stash &mine,
                                        Barriers &bar, int polls, volatile int &left_out) {
  constexpr int kRowBytes = S == KV_NONE ? 2 * DP : S == KV_MXFP4 ? DP / 2 : DP;
  constexpr int kCpr = kRowBytes / 16;                            // 16-byte chunks of a row
  constexpr int kOwn = kCpr;                                      // chunks a lane and job
  constexpr int kOut = S == KV_NONE ? 1 : S == KV_MXFP4 ? 4 : 2;  // granules of a chunk
  // A job is four blocks of 8 rows; a warp's access covers 8 rows by 64 bytes (16 by 32 where a row has no
  // more), so that neither the reads nor the swizzled writes collide.
  constexpr int kBlocks = kCpr >= 4 ? 4 : 2;  // that a lane has chunks in
  const KvCache &c = a.c;
  const int warp = (threadIdx.x >> 5) - kSoftmaxWarps, lane = threadIdx.x & 31;
  const int chunk0 = kCpr >= 4 ? lane >> 3 : (lane >> 3) & 1;
  const bool fits = c.dim == DP;

  // The stash holds the item that the jobs being looked up belong to; base is its first unit in the block's count.
  uint32_t base = 0;
  bool over = false;
  auto look = [&](uint32_t job) {
    Job r{-1, 0, 0, false};
    const uint32_t unit = job >> 3;
    while (!over && unit >= base + (uint32_t)mine.p.steps) {
      base += (uint32_t)mine.p.steps;
      Item it = mine.it;
      if (it.left == 0) {
        over = true;
      } else {
        W::next(a, it);
        put(mine, it, part_of(a, it));
      }
    }
    if (over) return r;
    const int p0 = mine.p.key0 + (int)(unit - base) * kKeys, at = p0 + 32 * (int)(job & 3) + lane;
    if (at < mine.p.key1) {
      const int pg = a.table[(int64_t)mine.it.b * a.table_stride + (at >> c.page_shift)];
      r.page = pg < c.pages ? pg : -1;
    }
    r.at = at;
    r.head = mine.it.head;
    r.mixed = !(p0 >= mine.p.all_lo && p0 + kKeys <= mine.p.all_hi);
    return r;
  };
  // Row of key `in` of the job, whose page is pg >= 0.
  auto row_at = [&](const Job &r, int pg, int in) -> int64_t {
    return (((int64_t)pg * c.heads + r.head) << c.page_shift) + ((r.at - lane + in) & (c.page_size - 1));
  };
  auto key_of = [&](int blk) { return 8 * (kCpr >= 4 ? blk : 2 * blk + (lane >> 4)) + (lane & 7); };
  // Chunk i is chunk chunk0 + cstep(i) of key key_of(bstep(i)).
  auto bstep = [&](int i) { return kCpr >= 4 ? i / (kCpr / 4) : i; };
  auto cstep = [&](int i) { return kCpr >= 4 ? (i % (kCpr / 4)) * 4 : 0; };
  auto load_scale = [&](const unsigned char *scales, const Job &r) {
    return r.page >= 0 ? scale_word<S, DP>(c, scales, row_at(r, r.page, lane)) : 0u;
  };
  // Where rows of a job differ in what they see, a V row of an unquantized cache that is not finite must not
  // reach the others: the products take it as 0.
  auto not_finite = [&](const Job &r) { return r.mixed && r.page >= 0 && odd_values<T, S>(c, row_at(r, r.page, lane)); };
  // The keys' entries of the unit's slot.
  auto put_slot = [&](uint32_t job, const Job &r, uint32_t kw, uint32_t vw) {
    put_keys<S, DP>(c, slots[(job >> 3) % kSlots], job & 3, r.page >= 0 ? row_at(r, r.page, lane) : -1, kw, vw);
    if (S == KV_NONE && not_finite(r)) left_out = 1;
  };
  auto wait_empty = [&](uint32_t job) {
    const uint32_t unit = job >> 3, st = unit & 1, parity = ((unit >> 1) & 1) ^ 1;
    return warp_wait_sleep((job & 4) ? &bar.vempty[st] : &bar.kempty[st], parity, polls);
  };
  auto arrive_full = [&](uint32_t job) {
    const uint32_t unit = job >> 3, st = unit & 1;
    fence_async_proxy();
    warp_arrive((job & 4) ? &bar.vfull[st] : &bar.kfull[st]);
    if (!(job & 4) && (threadIdx.x & 31) == 0) mbar_arrive(&bar.slot[unit % kSlots]);
  };

  uint32_t job = (uint32_t)warp;
  Job now = look(job);
  if (over) return true;  // a stretch of one unit has a job for every warp: not taken
  if constexpr (S != KV_NONE) {
    uint4 buf[kOwn];
    int64_t off[kBlocks];
    uint32_t kword = 0u, vword = 0u;
    // Where the lane's chunks of a job begin; -1 for a key that is not there.
    auto find_rows = [&](const Job &r) {
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int pg = __shfl_sync(0xFFFFFFFFu, r.page, key_of(b));
        off[b] = pg >= 0 ? row_at(r, pg, key_of(b)) * c.row_bytes + chunk0 * 16 : -1;
      }
    };
    // Chunk i: 16 bytes of codes. `full`: every key of the job is there, and heads fill the rows.
    auto load = [&](const unsigned char *codes, bool full, int i) {
      const int64_t at = off[bstep(i)];
      if (full) return load_once(codes + at + 16 * cstep(i));
      uint4 v = make_uint4(0, 0, 0, 0);
      if (at >= 0 && 16 * (chunk0 + cstep(i)) < c.row_bytes) v = load_once(codes + at + 16 * cstep(i));
      return v;
    };
    // Chunk i as 16-bit granules into a tile (a shared-memory address).
    auto convert = [&](const uint4 in, uint32_t word, uint32_t dead_keys, uint32_t dst, int i) {
      const int key = key_of(bstep(i));
      const uint32_t w[4] = {in.x, in.y, in.z, in.w};
      uint32_t mul = 0u;
      if (S == KV_MXFP4) {
        const uint32_t sw = __shfl_sync(0xFFFFFFFFu, word, key);
        mul = group_mul((sw >> (8 * chunk0)) & 0xFFu, biggest<DP>(sw));
      }
#pragma unroll
      for (int g = 0; g < kOut; ++g) {
        uint32_t h[4];
        granule<S>(w, g, mul, h);
        // A key with a NaN value scale has NaN codes, which would be 0 * NaN for every row: they count as 0.
        if (S == KV_FP8_ROW && dead_keys && ((dead_keys >> key) & 1u)) h[0] = h[1] = h[2] = h[3] = 0u;
        // Granule q of the key's row, what depends on the lane apart from what depends on i.
        const int q0 = chunk0 * kOut + g, qi = cstep(i) * kOut;
        st_shared16(dst + (uint32_t)(((qi >> 3) + (q0 >> 3)) * (kTile * 128) + key * 128 + (((q0 & 7) ^ (lane & 7)) << 4)), h[0],
                    h[1], h[2], h[3]);
      }
    };

    Job next = look(job + kProducerWarps);
    bool over1 = over;
    find_rows(now);
    {
      const bool full = fits && __all_sync(0xFFFFFFFFu, now.page >= 0);
      if (!(job & 4)) kword = load_scale(c.ks, now);
      vword = load_scale(c.vs, now);
#pragma unroll
      for (int i = 0; i < kOwn; ++i) buf[i] = load((job & 4) ? c.v : c.k, full, i);
    }
    while (true) {
      // now: its codes arrive in buf; next: its page arrives.
      if (!wait_empty(job)) return false;
      const uint32_t kw = kword, vw = vword;
      if (!(job & 4)) put_slot(job, now, kw, vw);
      const uint32_t dead = S == KV_FP8_ROW && (job & 4) ? __ballot_sync(0xFFFFFFFFu, (vw & 0x7FFFFFFFu) > kInf) : 0u;
      const uint32_t st = (job >> 3) & 1, ahead = job + kProducerWarps;
      const uint32_t dst = smem_addr((job & 4) ? vs : ks) + st * Shape<DP>::kOperand + (job & 3) * 32 * 128;
      const unsigned char *codes = (ahead & 4) ? c.v : c.k;
      const bool full = fits && __all_sync(0xFFFFFFFFu, next.page >= 0);
      if (!over1) {
        find_rows(next);
        if (!(ahead & 4)) kword = load_scale(c.ks, next);
        vword = load_scale(c.vs, next);
      }
      const uint32_t word = (job & 4) ? vw : kw;
      if (!over1 && full) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          convert(buf[i], word, dead, dst, i);
          buf[i] = load(codes, true, i);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          convert(buf[i], word, dead, dst, i);
          if (!over1) buf[i] = load(codes, false, i);
        }
      }
      arrive_full(job);
      if (over1) return true;
      now = next;
      job = ahead;
      next = look(job + kProducerWarps);
      over1 = over;
    }
  } else {
    // Unquantized rows go straight to shared memory.
    auto copy = [&](uint32_t j, const Job &r) {
      if (!(j & 4)) put_slot(j, r, 0u, 0u);
      const int use_page = (j & 4) && not_finite(r) ? -1 : r.page;
      const unsigned char *codes = (j & 4) ? c.v : c.k;
      unsigned char *dst = ((j & 4) ? vs : ks) + ((j >> 3) & 1) * Shape<DP>::kOperand;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int key = key_of(bstep(i)), ch = chunk0 + cstep(i);
        const int pg = __shfl_sync(0xFFFFFFFFu, use_page, key);
        const bool use = pg >= 0 && ch * 16 < c.row_bytes;
        cp_async16_or_zero(dst + tile_at(32 * (j & 3) + key, ch), use ? codes + row_at(r, pg, key) * c.row_bytes + ch * 16 : codes, use);
      }
      cp_async_commit();
    };
    if (!wait_empty(job)) return false;
    copy(job, now);
    while (true) {
      const uint32_t ahead = job + kProducerWarps;
      now = look(ahead);
      if (!over) {
        if (!wait_empty(ahead)) return false;
        copy(ahead, now);
        cp_async_wait<1>();
      } else {
        cp_async_wait<0>();
      }
      arrive_full(job);
      if (over) return true;
      job = ahead;
    }
  }
}

// ---------------------------------------------------------------- packed units (one thread)
// Brings the units that pack_kernel has laid out: what the producers make, three bulk copies a unit.
template <int DP>
__device__ __forceinline__ bool fetch(const Args &a, Item it, const unsigned char *packed, int max_units, unsigned char *ks,
                                      unsigned char *vs, KeySlot *slots, Barriers &bar, int polls) {
  uint32_t step = 0, nk = 0, nv = 0;  // units whose K (and slot), whose V copies are on their way
  bool ok = true;
  while (ok) {
    const Part p = part_of(a, it);
    const unsigned char *from = packed + ((int64_t)(it.b * a.c.heads + it.head) * max_units + p.key0 / kKeys) * Packed<DP>::kBytes;
    for (uint32_t n = step; n < step + (uint32_t)p.steps; ++n, from += Packed<DP>::kBytes) {
      const uint32_t st = n & 1, parity = ((n >> 1) & 1) ^ 1;
      if (!(ok = mbar_wait_sleep(&bar.kempty[st], parity, polls))) break;
      mbar_expect_tx(&bar.kfull[st], Shape<DP>::kOperand);
      bulk_g2s(ks + st * Shape<DP>::kOperand, from, Shape<DP>::kOperand, &bar.kfull[st]);
      mbar_expect_tx(&bar.slot[n % kSlots], sizeof(KeySlot));
      bulk_g2s(&slots[n % kSlots], from + Packed<DP>::kSlot, sizeof(KeySlot), &bar.slot[n % kSlots]);
      ++nk;
      if (!(ok = mbar_wait_sleep(&bar.vempty[st], parity, polls))) break;
      mbar_expect_tx(&bar.vfull[st], Shape<DP>::kOperand);
      bulk_g2s(vs + st * Shape<DP>::kOperand, from + Shape<DP>::kOperand, Shape<DP>::kOperand, &bar.vfull[st]);
      ++nv;
    }
    step += (uint32_t)p.steps;
    if (it.left == 0) break;
    W::next(a, it);
  }
  // The block's shared memory stays until the copies are in. A K copy is in before the unit after the next is asked for;
  // nothing says so of a slot, which is waited for while its barrier is its own.
  for (uint32_t k = nk > 2 ? nk - 2 : 0; k < nk; ++k) mbar_wait_sleep(&bar.kfull[k & 1], (k >> 1) & 1);
  for (uint32_t k = nk > kSlots ? nk - kSlots : 0; k < nk; ++k) mbar_wait_sleep(&bar.slot[k % kSlots], (k / kSlots) & 1);
  for (uint32_t k = nv > 2 ? nv - 2 : 0; k < nv; ++k) mbar_wait_sleep(&bar.vfull[k & 1], (k >> 1) & 1);
  return ok;
}

// ---------------------------------------------------------------- MMA issue (one warp)
// The warp stays together and one of its threads issues: what the instructions take in uniform registers is then
// prepared once. A lone thread in a branch of its own took about 110 cycles an MMA.
template <bool BF16, int DP>
__device__ __forceinline__ bool multiply(const Args &a, Item it, uint32_t qs, uint32_t ks, uint32_t vs, uint32_t tmem,
                                         Barriers &bar, int polls, bool &issued) {
  constexpr uint32_t kType = BF16 ? (1u << 7) | (1u << 10) : 0u;
  constexpr uint32_t kQk = (1u << 4) | kType | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
  constexpr uint32_t kPv = (1u << 4) | kType | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
  uint32_t step = 0, items[2] = {0u, 0u}, psteps[2] = {0u, 0u};
  while (true) {
    const Part p = part_of(a, it);
    const int tiles = uniform(p.two ? 2 : 1), steps = uniform(p.steps);
    // Scores of a unit; `then`: its keys are done with.
    auto qk = [&](int t, uint32_t n, bool then) {
      const uint64_t dk = desc_sw128(ks + (n & 1) * Shape<DP>::kOperand, 16);
      const uint64_t dq = desc_sw128(qs + t * Shape<DP>::kOperand, 16);
      const uint32_t d = tmem + t * 128;
      issued = true;
      if (tc5::elect_one()) {
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint64_t off = ((k >> 2) * (kTile * 128) + (k & 3) * 32) >> 4;
          tc5::mma_f16_ss(d, dq + off, dk + off, kQk, k > 0);
        }
        tc5::mma_commit(&bar.sfull[t]);
        if (then) tc5::mma_commit(&bar.kempty[n & 1]);
      }
      __syncwarp();
    };
    for (int t = 0; t < tiles; ++t)
      if (!warp_wait_sleep(&bar.qfull[t], items[t]++ & 1, polls)) return false;
    if (!warp_wait(&bar.kfull[step & 1], (step >> 1) & 1, polls)) return false;
    tc5::fence_after_sync();
    for (int t = 0; t < tiles; ++t) qk(t, step, t == tiles - 1);
    for (int j = 0; j < steps; ++j) {
      const uint32_t n = step + j;
      const uint64_t dv = desc_sw128(vs + (n & 1) * Shape<DP>::kOperand, kTile * 128);
      const bool more = j + 1 < steps;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (t >= tiles) break;
        const bool last = t == tiles - 1;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!warp_wait(&bar.pfull[t][half], psteps[t] & 1, polls)) return false;
          if (t == 0 && half == 0 && !warp_wait(&bar.vfull[n & 1], (n >> 1) & 1, polls)) return false;
          tc5::fence_after_sync();
          const uint32_t d = tmem + 256 + t * DP, w = tmem + t * 128 + half * kHalf;
          if (tc5::elect_one()) {
#pragma unroll
            for (int k = 0; k < kHalf / 16; ++k)
              tc5::mma_f16_ts(d, w + k * 8, dv + (half * (kHalf / 16) + k) * (2048 >> 4), kPv, j > 0 || half > 0 || k > 0);
            tc5::mma_commit(&bar.pvdone[t]);
            if (half && last) tc5::mma_commit(&bar.vempty[n & 1]);
            if (half && !more) tc5::mma_commit(&bar.ofull[t]);
          }
          __syncwarp();
        }
        ++psteps[t];
        if (more) {
          if (t == 0) {
            if (!warp_wait(&bar.kfull[(n + 1) & 1], ((n + 1) >> 1) & 1, polls)) return false;
            tc5::fence_after_sync();
          }
          qk(t, n + 1, last);
        }
      }
    }
    step += (uint32_t)steps;
    if (it.left == 0) return true;
    W::next(a, it);
  }
}

// ---------------------------------------------------------------- softmax (a warp 32 rows)
// A step of the softmax covers half a unit. A warp's 32 rows are held as MMA fragments: thread (g, t) has columns
// 8 j + 2 t, + 1 of rows 16 h + 8 e + g, rows 2 h + e of its four. A key's scale then serves four rows: what the
// scales take of shared memory's bandwidth, which the MMAs need, is a quarter of a thread a row's.
constexpr int kPairs = kHalf / 8;
using Rows = F2[4][kPairs];  // [row][j]: two neighbouring columns

// As they come from TMEM: asked for, and there after `arrived`, through which they pass.
struct Raw {
  uint32_t a[kHalf / 2], b[kHalf / 2];
};
__device__ __forceinline__ void ask(uint32_t ts, Raw &r) {
  tc5::tmem_ld_frag64(ts, r.a);
  tc5::tmem_ld_frag64(ts + (16u << 16), r.b);
}
__device__ __forceinline__ void arrived(Raw &r) {
  tc5::tmem_wait_ld_frag(r.a);
  tc5::tmem_wait_ld_frag(r.b);
}
__device__ __forceinline__ void rows_of(const Raw &r, Rows &x) {
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    x[0][j] = pack2(u2f(r.a[4 * j]), u2f(r.a[4 * j + 1]));
    x[1][j] = pack2(u2f(r.a[4 * j + 2]), u2f(r.a[4 * j + 3]));
    x[2][j] = pack2(u2f(r.b[4 * j]), u2f(r.b[4 * j + 1]));
    x[3][j] = pack2(u2f(r.b[4 * j + 2]), u2f(r.b[4 * j + 3]));
  }
}

// Scores that a row does not see become -Inf, those of keys that are not numbers NaN. Rows see keys [lo, hi)
// of the half; there and dead are its keys' bits. A bit test and a select an element.
__device__ __forceinline__ void mask_rows(Rows &x, const uint32_t *there, const uint32_t *dead, int t, const int (&lo)[4],
                                          const int (&hi)[4]) {
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const uint32_t keys = there[part], bad = dead[part] >> (2 * t);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t in = (keys & range_bits(lo[r], hi[r], part)) >> (2 * t);
#pragma unroll
      for (int j = 0; j < kPairs / 2; ++j) {
        float v0, v1;
        F2 &pair = x[r][part * (kPairs / 2) + j];
        unpack2(pair, v0, v1);
        v0 = (bad & (1u << (8 * j))) ? u2f(kQNaN) : v0;
        v1 = (bad & (2u << (8 * j))) ? u2f(kQNaN) : v1;
        v0 = (in & (1u << (8 * j))) ? v0 : -INFINITY;
        v1 = (in & (2u << (8 * j))) ? v1 : -INFINITY;
        pair = pack2(v0, v1);
      }
    }
  }
}

// P = exp2(score * key scale * qmul - ref) * value scale as packed pairs, this thread's sums of P before the
// value's scale, and its largest scores (before qmul). Everything in one pass: the products and maxima issue
// under the exponentials, which bound it (16 a cycle and SM).
template <int S, bool BF16>
__device__ __forceinline__ void weights(const Rows &x, const float *ks, const float *vs, int t, const float (&qmul)[4],
                                        const float (&ref)[4], uint32_t (&p)[2][kHalf / 4], F2 (&sum2)[4], float (&m)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) m[r] = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    F2 k2, v2;
    if (S != KV_NONE) {
      k2 = *reinterpret_cast<const F2 *>(ks + 8 * j + 2 * t);
      v2 = *reinterpret_cast<const F2 *>(vs + 8 * j + 2 * t);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      F2 y = x[r][j];
      if (S != KV_NONE) y = mul2(y, k2);
      float v0, v1;
      unpack2(y, v0, v1);
      m[r] = fmaxf(fmaxf(m[r], v0), v1);
      unpack2(fma2(y, pack2(qmul[r], qmul[r]), pack2(-ref[r], -ref[r])), v0, v1);
      y = pack2(exp2_fast(v0), exp2_fast(v1));
      sum2[r] = j ? add2(sum2[r], y) : y;
      if (S != KV_NONE) y = mul2(y, v2);
      unpack2(y, v0, v1);
      p[r >> 1][2 * j + (r & 1)] = BF16 ? pack_bf16(v0, v1) : pack_half(v0, v1);
    }
  }
}

// This thread's largest x + lift of a half's keys that each of its rows sees, by every key's own lift: eight columns
// of scores at a time, read again.
__device__ __forceinline__ void highest(const Args &a, const Stash &mine, const KeySlot &sl, int half, int tile, int p0, bool whole,
                                        uint32_t ts, const float (&qm)[4], float (&m)[4]) {
  const int lane = threadIdx.x & 31, g4 = lane >> 2, t4 = lane & 3, row0 = 32 * ((threadIdx.x >> 5) & 3);
  int lo[4], hi[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lo[i] = 0, hi[i] = kKeys;
    if (!whole) {
      visible(a, mine.p.s, min(mine.it.tile * kRows + tile * kTile + row0 + 8 * i + g4, mine.p.rows - 1) / a.group, lo[i], hi[i]);
      lo[i] -= p0, hi[i] -= p0;
    }
    m[i] = -INFINITY;
  }
#pragma unroll 1
  for (int j = 0; j < kPairs; ++j) {
    uint32_t s[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) tc5::tmem_ld_frag8(ts + (h ? 16u << 16 : 0u) + kHalf * half + 8 * j, s[h]);
    tc5::tmem_wait_ld<4>(s[0]);
    tc5::tmem_wait_ld<4>(s[1]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int key = kHalf * half + 8 * j + 2 * t4 + e;
      const bool there = ((sl.valid[key >> 5] & ~sl.dead[key >> 5]) >> (key & 31)) & 1u;
      const float k = sl.k[key], lift = f2u(sl.v[key]) == 0x80000000u ? (float)kOddLift : lift_of((int)(f2u(sl.v[key]) >> 23));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (there && key >= lo[i] && key < hi[i]) m[i] = fmaxf(m[i], u2f(s[i >> 1][2 * (i & 1) + e]) * k * qm[i] + lift);
    }
  }
}

// Adds what the products left out: the values of odd keys, in fp32, to the outputs of the rows that see them. A thread
// works out the scores of one row of its warp's 32 again, from Q as it lies in shared memory. Rare, and a call of its own:
// inlined it took the softmax loop 8% of its time. 2 us a warp and key.
template <typename T, int S, int DP>
__device__ __noinline__ void add_odd(const Args &a, const Stash &mine, const unsigned char *q0, int tile, uint32_t to, float4 qm4, float4 ref4) {
  constexpr bool kBf16 = S == KV_NONE && Same<T, __nv_bfloat16>::value;
  const float qm[4] = {qm4.x, qm4.y, qm4.z, qm4.w}, ref[4] = {ref4.x, ref4.y, ref4.z, ref4.w};
  const KvCache c = a.c;
  const int lane = threadIdx.x & 31, g4 = lane >> 2, t4 = lane & 3, row0 = 32 * ((threadIdx.x >> 5) & 3);
  const int head = mine.it.head, key0 = mine.p.key0, key1 = mine.p.key1, all_lo = mine.p.all_lo, all_hi = mine.p.all_hi;
  const int *table = a.table + (int64_t)mine.it.b * a.table_stride;
  auto row_of = [&](int at) -> int64_t {
    const int page = table[at >> c.page_shift];
    return page < 0 || page >= c.pages ? -1 : (((int64_t)page * c.heads + head) << c.page_shift) + (at & (c.page_size - 1));
  };
  // Of this thread's row; `below` is NaN for one that nothing changes any more.
  float qmul = 0.0f, below = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float q = __shfl_sync(0xFFFFFFFFu, qm[i], 4 * (lane & 7)), r = __shfl_sync(0xFFFFFFFFu, ref[i], 4 * (lane & 7));
    if (lane >> 3 == i) qmul = q, below = r;
  }
  int lo, hi;
  visible(a, mine.p.s, min(mine.it.tile * kRows + tile * kTile + row0 + lane, mine.p.rows - 1) / a.group, lo, hi);
#pragma unroll 1
  for (int at0 = key0; at0 < key1; at0 += 32) {
    if (!__any_sync(0xFFFFFFFFu, below == below && lo < at0 + 32 && hi > at0)) continue;
    const int64_t own = at0 + lane < key1 ? row_of(at0 + lane) : -1;
    const int unit = at0 - (at0 - key0) % kKeys;
    if (S == KV_NONE && unit >= all_lo && unit + kKeys <= all_hi) continue;  // every row sees the unit
    uint32_t odd = __ballot_sync(0xFFFFFFFFu, own >= 0 && odd_values<T, S>(c, own));
#pragma unroll 1
    for (; odd; odd &= odd - 1) {
      const int at = at0 + __ffs(odd) - 1;
      const int64_t row = __shfl_sync(0xFFFFFFFFu, own, at - at0);
      const bool sees = at >= lo && at < hi && below == below;
      const uint32_t who = __ballot_sync(0xFFFFFFFFu, sees);
      if (who == 0u) continue;
      float k[DP / 32], v[DP / 32];  // elements lane + 32 i of the key's rows
      bool nan = true;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        const int d = lane + 32 * i;
        k[i] = v[i] = 0.0f;
        if (d < c.dim) {
          k[i] = cached<T>(c, c.k + row * c.row_bytes, c.ks + row * c.scale_bytes, d);
          v[i] = cached<T>(c, c.v + row * c.row_bytes, c.vs + row * c.scale_bytes, d);
          nan = nan && v[i] != v[i];
        }
      }
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll 8
        for (int d = 0; d < 32; d += 2) {
          const int at2 = 32 * i + d;  // zeros past head_dim, in Q too
          const uint32_t q = *reinterpret_cast<const uint32_t *>(q0 + tile_at(row0 + lane, at2 >> 3) + 2 * (at2 & 7));
          dot = __fmaf_rn(kBf16 ? half_bits_to_float<__nv_bfloat16>(q & 0xFFFFu) : half_bits_to_float<__half>(q & 0xFFFFu), __shfl_sync(0xFFFFFFFFu, k[i], d), dot);
          dot = __fmaf_rn(kBf16 ? half_bits_to_float<__nv_bfloat16>(q >> 16) : half_bits_to_float<__half>(q >> 16), __shfl_sync(0xFFFFFFFFu, k[i], d + 1), dot);
        }
      const float weight = exp2_wide(dot * qmul - below);
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __shfl_sync(0xFFFFFFFFu, weight, 8 * i + g4);
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        float part[8];  // columns 8 k + 2 t + e of the 32
#pragma unroll
        for (int e = 0; e < 8; ++e) part[e] = __shfl_sync(0xFFFFFFFFu, v[i], 8 * (e >> 1) + 2 * t4 + (e & 1));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t out = to + (h ? 16u << 16 : 0u) + 32 * i;
          uint32_t o[16];
          tc5::tmem_ld_frag32(out, o);
          tc5::tmem_wait_ld_frag(o);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int r = 2 * h + ((e >> 1) & 1);
            const float sum = __fmaf_rn(w[r], part[2 * (e >> 2) + (e & 1)], u2f(o[e]));
            o[e] = (who >> (8 * r + g4)) & 1u ? f2u(sum) : o[e];
          }
          tc5::tmem_st_frag32(out, o);
        }
      }
      tc5::tmem_wait_st();
      if (__all_sync(0xFFFFFFFFu, nan) && sees) below = u2f(kQNaN);  // nothing but NaN is left of the row
    }
  }
}

// Multiplies the outputs so far by a power of two a row.
template <int DP>
__device__ __forceinline__ void rescale(const float (&keep)[4], uint32_t to) {
#pragma unroll 1
  for (int i = 0; i < 2 * (DP / 32); ++i) {
    const int h = i & 1;
    const float k0 = h ? keep[2] : keep[0], k1 = h ? keep[3] : keep[1];
    const uint32_t at = to + (h ? 16u << 16 : 0u) + 32 * (i >> 1);
    uint32_t o[16];
    tc5::tmem_ld_frag32(at, o);
    tc5::tmem_wait_ld_frag(o);
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = f2u(u2f(o[e]) * ((e & 2) ? k1 : k0));
    tc5::tmem_st_frag32(at, o);
  }
}

template <typename T, int S, int DP>
__device__ __forceinline__ bool softmax(const Args &a, unsigned char *qs, const KeySlot *slots, Stash &mine, uint32_t tmem,
                                        Barriers &bar, int polls, float *parts, volatile int &left_out) {
  constexpr bool kBf16 = S == KV_NONE && Same<T, __nv_bfloat16>::value;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, t4 = lane & 3;
  const int t = warp >> 2, row0 = 32 * (warp & 3);  // a warp reaches the 32 TMEM lanes of its index
  const uint32_t ts = tmem + ((uint32_t)row0 << 16) + t * 128, to = tmem + ((uint32_t)row0 << 16) + 256 + t * DP;
  unsigned char *q0 = qs + t * Shape<DP>::kOperand;
  const bool qvec = ((uintptr_t)a.q | (uintptr_t)(a.q_tok * 2) | (uintptr_t)(a.q_head * 2)) % 16 == 0;
  uint32_t step = 0, ssteps = 0, items = 0;
  while (true) {
    if (t == 0 || mine.p.two) {
      // Q: a thread a row, as 16-bit operand; over quantized caches scaled by a power of two into fp16. The
      // sign of the scale goes into Q; a scale of 0 is replaced by one whose scores vanish but keep -Inf.
      float qmul = a.scale == 0.0f ? 1.1754943508222875e-38f : fabsf(a.scale);
      {
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
        const Part p = mine.p;
        const Item it = mine.it;
        const int first = it.tile * kRows + t * kTile + row0;  // the warp's first row
        const int r = first + lane, tok = min(r, p.rows - 1) / a.group;
        const T *qp = static_cast<const T *>(a.q) + (p.s.q0 + tok) * a.q_tok + (it.head * a.group + min(r, p.rows - 1) % a.group) * a.q_head;
        // Every thread reads, a row that is not there its neighbour's: without branches the loads go out together.
        uint32_t w[DP / 2];
#pragma unroll
        for (int g = 0; g < DP / 8; ++g) {
          const int at = min(8 * g, a.c.dim - 8);
          uint32_t x[4];
          if (qvec) {
            load_words<4>(reinterpret_cast<const unsigned char *>(qp + at), x);
          } else {
            const unsigned short *u = reinterpret_cast<const unsigned short *>(qp + at);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = (uint32_t)u[2 * k] | ((uint32_t)u[2 * k + 1] << 16);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) w[4 * g + k] = x[k];
        }
#pragma unroll
        for (int g = 0; g < DP / 8; ++g)
#pragma unroll
          for (int k = 0; k < 4; ++k) w[4 * g + k] = r < p.rows && 8 * g < a.c.dim ? w[4 * g + k] ^ flip : 0u;
        if (S != KV_NONE) {
          float big = 0.0f;
#pragma unroll
          for (int k = 0; k < DP / 2; ++k)
            big = fmaxf(big, fmaxf(fabsf(half_bits_to_float<T>(w[k] & 0xFFFFu)), fabsf(half_bits_to_float<T>(w[k] >> 16))));
          const Pow2 f = fp16_shift(big);
          qmul = fmaxf(qmul * f.inverse, 1.1754943508222875e-38f);  // not 0, whatever the row's size
#pragma unroll
          for (int k = 0; k < DP / 2; ++k)
            w[k] = pack_half(half_bits_to_float<T>(w[k] & 0xFFFFu) * f.factor, half_bits_to_float<T>(w[k] >> 16) * f.factor);
        }
#pragma unroll
        for (int g = 0; g < DP / 8; ++g)
          *reinterpret_cast<uint4 *>(q0 + tile_at(row0 + lane, g)) = make_uint4(w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]);
        fence_async_proxy();
        tc5::fence_before_sync();
        warp_arrive(&bar.qfull[t]);
      }
      // From here on a thread works for rows 8 i + g of the warp's 32.
      // ref: the base-2 logarithm that weights are relative to; far below everything before the row has seen a key
      // (the first one then moves it).
      float qm[4], ref[4];
      F2 sum2[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qm[i] = __shfl_sync(0xFFFFFFFFu, qmul, 8 * i + g4);
        ref[i] = -3e38f;
        sum2[i] = pack2(0.0f, 0.0f);
      }
      const int steps = mine.p.steps, key0 = mine.p.key0, all_lo = mine.p.all_lo, all_hi = mine.p.all_hi;
      __syncwarp();
      for (int j = 0; j < steps; ++j) {
        const uint32_t n = step + j;
        const KeySlot &sl = slots[n % kSlots];
        if (!warp_wait(&bar.sfull[t], ssteps & 1, polls)) return false;
        tc5::fence_after_sync();
        Raw raw[2];
        ask(ts, raw[0]);
        // The slot after the scores, which a warp that had no rows for a while cannot be early for.
        if (!warp_wait(&bar.slot[n % kSlots], (n / kSlots) & 1, polls)) return false;
        const int p0 = key0 + j * kKeys;
        const bool whole = p0 >= all_lo && p0 + kKeys <= all_hi &&
                           ((sl.valid[0] & ~sl.dead[0]) & (sl.valid[1] & ~sl.dead[1]) & (sl.valid[2] & ~sl.dead[2]) &
                            (sl.valid[3] & ~sl.dead[3])) == 0xFFFFFFFFu;
        // The largest lift of the unit, seen or not: a score this far above the reference may have to move it.
        const float lift = S == KV_NONE ? 0.0f : lift_of(max(max(sl.top[0], sl.top[1]), max(sl.top[2], sl.top[3])));
        auto step_half = [&](const int half) {
          // With the reference as it is. It moves when a row's largest product has risen by more than 2**8 (or from
          // nothing), by whole powers of two, so that what it scales stays exact; the half is then computed again.
          uint32_t pw[2][kHalf / 4];
          F2 part2[4];
          if (half) ask(ts + kHalf, raw[half]);  // (asked for before the first half's arithmetic it came out slower)
          arrived(raw[half]);
          while (true) {
            Rows x;
            rows_of(raw[half], x);
            if (!whole) {
              int lo[4], hi[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                visible(a, mine.p.s, min(mine.it.tile * kRows + t * kTile + row0 + 8 * i + g4, mine.p.rows - 1) / a.group, lo[i], hi[i]);
                lo[i] -= p0 + kHalf * half;
                hi[i] -= p0 + kHalf * half;
              }
              mask_rows(x, sl.valid + 2 * half, sl.dead + 2 * half, t4, lo, hi);
            }
            float m[4];
            weights<S, kBf16>(x, sl.k + kHalf * half, sl.v + kHalf * half, t4, qm, ref, pw, part2, m);
            bool any = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) any |= m[i] * qm[i] > ref[i] + (kHeadroom - lift);
            if (!__any_sync(0xFFFFFFFFu, any)) break;
            // Where the unit's lifts lie close together the largest score and lift will do; else every key by itself.
            const bool narrow = S == KV_NONE || max(max(sl.top[0], sl.top[1]), max(sl.top[2], sl.top[3])) <=
                                                    min(min(sl.low[0], sl.low[1]), min(sl.low[2], sl.low[3])) + kNarrow;
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] = m[i] * qm[i] + lift;
            if (!narrow) highest(a, mine, sl, half, t, p0, whole, ts, qm, m);
            if (lift > (float)kMostLift) mine.odd = true;
            float keep[4];
            any = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              m[i] = fmaxf(m[i], __shfl_xor_sync(0xFFFFFFFFu, m[i], 1));
              m[i] = fmaxf(m[i], __shfl_xor_sync(0xFFFFFFFFu, m[i], 2));
              const float next = m[i] > ref[i] + kHeadroom ? ceilf(m[i]) - kBelow : ref[i];
              any |= next != ref[i];
              keep[i] = S == KV_NONE ? exp2_fast(ref[i] - next) : exp2_wide(ref[i] - next);
              ref[i] = next;
              sum2[i] = mul2(sum2[i], pack2(keep[i], keep[i]));
            }
            if (!__any_sync(0xFFFFFFFFu, any)) break;
            // The outputs so far: the products of the half before, which this half's scores did not wait for.
            if (j > 0 || half) {
              if (!warp_wait(&bar.pvdone[t], (half ^ 1) & 1, polls)) return false;
              tc5::fence_after_sync();
              rescale<DP>(keep, to);
            }
            ask(ts + kHalf * half, raw[half]);
            arrived(raw[half]);
          }
          tc5::tmem_st_pairs64(ts + kHalf * half, pw[0]);
          tc5::tmem_st_pairs64(ts + (16u << 16) + kHalf * half, pw[1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum2[i] = add2(sum2[i], part2[i]);
          tc5::tmem_wait_st();
          tc5::fence_before_sync();
          warp_arrive(&bar.pfull[t][half]);
          return true;
        };
        if (!step_half(0) || !step_half(1)) return false;
        ++ssteps;
      }
      // The item's part is done.
      if (!warp_wait_sleep(&bar.ofull[t], items++ & 1, polls)) return false;
      tc5::fence_after_sync();
      __syncwarp();
      if (S == KV_NONE ? __any_sync(0xFFFFFFFFu, left_out) : (int)mine.odd) {
        float live[4];  // the reference; NaN for a row whose sum is NaN, which it stays
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float s0, s1;
          unpack2(sum2[i], s0, s1);
          s0 += s1;
          s0 += __shfl_xor_sync(0xFFFFFFFFu, s0, 1);
          s0 += __shfl_xor_sync(0xFFFFFFFFu, s0, 2);
          live[i] = s0 != s0 ? s0 : ref[i];
        }
        add_odd<T, S, DP>(a, mine, q0, t, to, make_float4(qm[0], qm[1], qm[2], qm[3]), make_float4(live[0], live[1], live[2], live[3]));
      }
      const Part p = mine.p;
      const Item it = mine.it;
      const int first = it.tile * kRows + t * kTile + row0;
      const bool done = it.at == 0 && it.n == it.units;
      float *part = parts + (size_t)(2 * blockIdx.x + (it.at > 0 ? 0 : 1)) * partial_floats(kRows, DP);
      const int prow = t * kTile + row0 + g4;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        float sum[2], inv[2];
        int64_t out_row[2];
        bool real[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float s1;
          unpack2(h ? sum2[2 + i] : sum2[i], sum[i], s1);
          const float last = h ? ref[2 + i] : ref[i];
          sum[i] += s1;
          sum[i] += __shfl_xor_sync(0xFFFFFFFFu, sum[i], 1);
          sum[i] += __shfl_xor_sync(0xFFFFFFFFu, sum[i], 2);
          inv[i] = sum[i] == 0.0f ? 0.0f : 1.0f / sum[i];
          const int r = first + 16 * h + 8 * i + g4;
          real[i] = r < p.rows;
          out_row[i] = (p.s.q0 + min(r, p.rows - 1) / a.group) * a.heads + it.head * a.group + r % a.group;
          if (t4 == 0) {
            if (!done) {
              part[prow + 16 * h + 8 * i] = sum[i] == 0.0f ? -INFINITY : last;
              part[kRows + prow + 16 * h + 8 * i] = sum[i];
            } else if (a.lse && real[i]) {
              a.lse[out_row[i]] = sum[i] == 0.0f ? -INFINITY : (last + log2f(sum[i])) * 0.69314718055994531f;
            }
          }
        }
#pragma unroll 1
        for (int q = 0; q < DP / 32; ++q) {
          uint32_t o[16];
          tc5::tmem_ld_frag32(to + (h ? 16u << 16 : 0u) + 32 * q, o);
          tc5::tmem_wait_ld_frag(o);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int d = 32 * q + 8 * k + 2 * t4;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float v0 = u2f(o[4 * k + 2 * i]), v1 = u2f(o[4 * k + 2 * i + 1]);
              if (!done) {
                *reinterpret_cast<float2 *>(part + 2 * kRows + (prow + 16 * h + 8 * i) * DP + d) = make_float2(v0, v1);
              } else if (real[i] && d < a.c.dim) {
                *reinterpret_cast<uint32_t *>(static_cast<T *>(a.out) + out_row[i] * a.c.dim + d) =
                    sum[i] == 0.0f ? 0u : pack16<T>(v0 * inv[i], v1 * inv[i]);
              }
            }
          }
        }
      }
      tc5::fence_before_sync();
    }
    step += (uint32_t)mine.p.steps;
    Item it = mine.it;
    if (it.left == 0) return true;
    W::next(a, it);
    put(mine, it, part_of(a, it));
  }
}

template <typename T, int S, int DP>
__global__ void __launch_bounds__((S == KV_PACKED ? kPackedThreads : kThreads), 1) chunk_kernel(const __grid_constant__ Args a, float *parts, Stretch *stretches, int *status, int most, int polls,
                                                                 const unsigned char *packed, int max_units) {
  constexpr bool kPacked = S == KV_PACKED;
  constexpr int kFullArrivals = kPacked ? 1 : 4, kFeeders = kPacked ? 1 : kProducerWarps;
  constexpr bool kBf16 = S == KV_NONE && Same<T, __nv_bfloat16>::value;
  extern __shared__ unsigned char raw[];
  __shared__ KeySlot slots[kSlots];
  __shared__ Stash stash[kSoftmaxWarps + (kPacked ? 0 : kProducerWarps)];
  __shared__ __align__(8) Barriers bar;
  __shared__ Item first;
  __shared__ uint32_t tmem_base;
  __shared__ int failed, left_out;  // left_out: a producer of unquantized units has met values that the products leave out
  unsigned char *smem = raw + (1024 - (smem_addr(raw) & 1023)) % 1024;  // the swizzle is of address bits
  unsigned char *qs = smem, *ks = qs + 2 * Shape<DP>::kOperand, *vs = ks + 2 * Shape<DP>::kOperand;
  const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (warp == kSoftmaxWarps) {
    const Stretch mine = W::stretch(a, blockIdx.x, most);
    if (lane == 0) {
      first = mine.first;
      stretches[blockIdx.x] = mine;
      failed = 0;
      left_out = 0;
    }
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.kfull[i], kFullArrivals);
      mbar_init(&bar.vfull[i], kFullArrivals);
      mbar_init(&bar.kempty[i], 1);
      mbar_init(&bar.vempty[i], 1);
      mbar_init(&bar.qfull[i], 4);
      mbar_init(&bar.pfull[i][0], 4);
      mbar_init(&bar.pfull[i][1], 4);
      mbar_init(&bar.sfull[i], 1);
      mbar_init(&bar.pvdone[i], 1);
      mbar_init(&bar.ofull[i], 1);
    }
    for (int i = 0; i < kSlots; ++i) mbar_init(&bar.slot[i], kFullArrivals);
    mbar_init(&bar.drain, 1);
    fence_barrier_init();
  }
  if (warp == 1) tc5::tmem_alloc(&tmem_base, 512);
  tc5::fence_before_sync();
  __syncthreads();
  tc5::fence_after_sync();
  let_next_start();
  if (kPacked) wait_for_previous();
  const Item it = first;
  const uint32_t tmem = uniform(tmem_base);
  if (it.n > 0) {
    bool ok = true;
    if (warp < kSoftmaxWarps) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(softmax_regs(kPacked)));
      put(stash[warp], it, part_of(a, it));
      ok = softmax<T, S, DP>(a, qs, slots, stash[warp], tmem, bar, polls, parts, left_out);
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(other_regs(kPacked)));
      if (warp < kSoftmaxWarps + kFeeders) {
        if constexpr (kPacked) {
          if (lane == 0) ok = fetch<DP>(a, it, packed, max_units, ks, vs, slots, bar, polls);
        } else {
          put(stash[warp], it, part_of(a, it));
          ok = produce<T, S, DP>(a, ks, vs, slots, stash[warp], bar, polls, left_out);
          cp_async_wait_all();
        }
      } else if (warp == kSoftmaxWarps + kFeeders) {
        bool issued = false;
        ok = multiply<kBf16, DP>(a, it, smem_addr(qs), smem_addr(ks), smem_addr(vs), tmem, bar, polls, issued);
        if (issued) {
          // No MMA may be in flight when the block's shared memory and TMEM go.
          if (tc5::elect_one()) tc5::mma_commit(&bar.drain);
          __syncwarp();
          mbar_wait_sleep(&bar.drain, 0);
        }
      }
      __syncwarp();
    }
    if (!ok) failed = 1;
  }
  tc5::fence_before_sync();
  __syncthreads();
  tc5::fence_after_sync();
  if (warp == 1) tc5::tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0) status[blockIdx.x] = failed;
}

// ---------------------------------------------------------------- packing
// Lays units out as operands: a block one unit of a sequence's key / value head, a warp one of the jobs that the
// producers would do for every row tile again. Bound by the memory it writes: 16384 keys of 8 heads of 128 in 25 us,
// 4.0 TB/s.
template <int S, int DP>
__global__ void __launch_bounds__(256) pack_kernel(Args a, unsigned char *packed, int max_units) {
  constexpr int kRowBytes = S == KV_MXFP4 ? DP / 2 : DP, kCpr = kRowBytes / 16, kOut = S == KV_MXFP4 ? 4 : 2;
  const KvCache &c = a.c;
  const int unit = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
  const int side = threadIdx.x >> 7, quarter = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  let_next_start();
  const Seq s = sequence(a, b);
  if (s.n == 0) return;
  // Every unit that a row tile visits; the first one also where there are no keys.
  int lo, hi, unused;
  visible(a, s, 0, lo, hi);
  lo = min(lo, hi);
  visible(a, s, s.n - 1, unused, hi);
  if (unit * kKeys >= max(hi, 1) || (unit + 1) * kKeys <= lo) return;
  unsigned char *to = packed + ((int64_t)(b * c.heads + head) * max_units + unit) * Packed<DP>::kBytes;
  const int at = unit * kKeys + 32 * quarter + lane;
  int page = -1;
  if (at < hi) {
    const int pg = a.table[(int64_t)b * a.table_stride + (at >> c.page_shift)];
    page = pg < c.pages ? pg : -1;
  }
  auto row_at = [&](int pg, int in) -> int64_t {
    return (((int64_t)pg * c.heads + head) << c.page_shift) + ((at - lane + in) & (c.page_size - 1));
  };
  const uint32_t vw = page >= 0 ? scale_word<S, DP>(c, c.vs, row_at(page, lane)) : 0u;
  uint32_t word = vw;
  if (side == 0) {
    word = page >= 0 ? scale_word<S, DP>(c, c.ks, row_at(page, lane)) : 0u;
    put_keys<S, DP>(c, *reinterpret_cast<KeySlot *>(to + Packed<DP>::kSlot), quarter, page >= 0 ? row_at(page, lane) : -1, word,
                    vw);
  }
  // A key with a NaN value scale has NaN codes, which would be 0 * NaN for every row: they count as 0.
  const uint32_t dead = S == KV_FP8_ROW && side ? __ballot_sync(0xFFFFFFFFu, (vw & 0x7FFFFFFFu) > kInf) : 0u;
  const unsigned char *codes = side ? c.v : c.k;
  to += side * Shape<DP>::kOperand;
  uint4 buf[kCpr];
  // Lane and step i: chunk n % kCpr of key n / kCpr for n = 32 i + lane.
#pragma unroll
  for (int i = 0; i < kCpr; ++i) {
    const int key = (32 * i + lane) / kCpr, ch = lane % kCpr, pg = __shfl_sync(0xFFFFFFFFu, page, key);
    buf[i] = make_uint4(0, 0, 0, 0);
    if (pg >= 0 && 16 * ch < c.row_bytes) buf[i] = load_once(codes + row_at(pg, key) * c.row_bytes + 16 * ch);
  }
#pragma unroll
  for (int i = 0; i < kCpr; ++i) {
    const int key = (32 * i + lane) / kCpr, ch = lane % kCpr;
    const uint32_t w[4] = {buf[i].x, buf[i].y, buf[i].z, buf[i].w};
    uint32_t mul = 0u;
    if (S == KV_MXFP4) {
      const uint32_t sw = __shfl_sync(0xFFFFFFFFu, word, key);
      mul = group_mul((sw >> (8 * ch)) & 0xFFu, biggest<DP>(sw));
    }
#pragma unroll
    for (int g = 0; g < kOut; ++g) {
      uint32_t h[4];
      granule<S>(w, g, mul, h);
      if (S == KV_FP8_ROW && ((dead >> key) & 1u)) h[0] = h[1] = h[2] = h[3] = 0u;
      *reinterpret_cast<uint4 *>(to + tile_at(32 * quarter + key, ch * kOut + g)) = make_uint4(h[0], h[1], h[2], h[3]);
    }
  }
}

template <typename T, int S, int DP>
int launch(const Args &a, float *parts, Stretch *stretches, int *status, int most, cudaStream_t s, const unsigned char *packed = nullptr,
           int max_units = 0) {
  auto kern = chunk_kernel<T, S, DP>;
  static std::atomic<uint64_t> ready[2];  // devices whose shared-memory limit is raised
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return set_error(std::string("tc_paged_attention: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  if (dev >= 128 || !((ready[dev >> 6].load(std::memory_order_relaxed) >> (dev & 63)) & 1)) {
    // The warps share out the registers that the block is launched with: with fewer their first request would not end.
    constexpr int kBlockThreads = S == KV_PACKED ? kPackedThreads : kThreads;
    constexpr int kShares = 32 * kSoftmaxWarps * softmax_regs(S == KV_PACKED) + (kBlockThreads - 32 * kSoftmaxWarps) * other_regs(S == KV_PACKED);
    cudaFuncAttributes built;
    e = cudaFuncGetAttributes(&built, kern);
    if (e == cudaSuccess && built.numRegs * kBlockThreads < kShares)
      return set_error("tc_paged_attention: the chunk kernel was built with too few registers a thread"), TC_CUDA_ERROR;
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP>::kSmem);
    if (e != cudaSuccess) return set_error(std::string("tc_paged_attention: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
    if (dev < 128) ready[dev >> 6].fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(most);
  cfg.blockDim = dim3((S == KV_PACKED ? kPackedThreads : kThreads));
  cfg.dynamicSmemBytes = Shape<DP>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // over packed units: starts as pack_kernel ends
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = S == KV_PACKED ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, kern, a, parts, stretches, status, most, wait_polls(), packed, max_units);
  if (e != cudaSuccess) return set_error(std::string("tc_paged_attention: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  count_launch();
  return TC_OK;
}

template <int S>
int launch_scheme(const Args &a, float *parts, Stretch *stretches, int *status, int most, cudaStream_t s,
                  const unsigned char *packed = nullptr, int max_units = 0) {
  const bool bf16 = a.c.dtype == TC_BF16;
  if (a.c.dim <= 64)
    return bf16 ? launch<__nv_bfloat16, S, 64>(a, parts, stretches, status, most, s, packed, max_units) : launch<__half, S, 64>(a, parts, stretches, status, most, s, packed, max_units);
  return bf16 ? launch<__nv_bfloat16, S, 128>(a, parts, stretches, status, most, s, packed, max_units) : launch<__half, S, 128>(a, parts, stretches, status, most, s, packed, max_units);
}

// Packs the call's units, then runs the kernel over them.
template <int S>
int launch_packed(const Args &a, float *parts, Stretch *stretches, int *status, int most, unsigned char *packed, int max_units,
                  cudaStream_t s) {
  const dim3 grid((unsigned)max_units, (unsigned)a.c.heads, (unsigned)a.batch);
  if (a.c.dim <= 64) pack_kernel<S, 64><<<grid, 256, 0, s>>>(a, packed, max_units);
  else pack_kernel<S, 128><<<grid, 256, 0, s>>>(a, packed, max_units);
  count_launch();
  return launch_scheme<KV_PACKED>(a, parts, stretches, status, most, s, packed, max_units);
}

}  // namespace chunk
}  // namespace attn
}  // namespace tc
