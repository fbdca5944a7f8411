// Attention of new tokens over a paged cache: the call's arguments and what the kernels share.
#pragma once

#include "tc_mma16.cuh"
#include "tc_serve.cuh"

namespace tc {
namespace attn {

struct Args {
  KvCache c;
  const void *q;                  // [total_q][heads][dim] with token and head strides (elements)
  int64_t q_tok, q_head, total_q;
  int heads, group;               // query heads, and query heads that share a key / value head
  const int *table;               // [batch][max_pages], row stride table_stride
  int64_t table_stride;
  int max_pages;
  const int *lens;                // context of each sequence, its new tokens included
  const int *cu;                  // [batch + 1] first new token of each sequence, or nullptr: one each
  int batch, max_q;
  float scale;                    // of the scores, times log2(e): the kernels work in powers of two
  int causal, window;             // window 0: unlimited
  void *out;                      // [total_q][heads][dim]
  float *lse;                     // [total_q][heads] or nullptr
};

// New tokens [q0, q0 + n) and context length of a sequence, clamped to what the tensors hold. Of more than max_q new
// tokens (`all`) the first ones count, at their own positions.
struct Seq {
  int64_t q0;
  int n, len, all;
};
__device__ __forceinline__ Seq sequence(const Args &a, int b) {
  Seq s;
  const int total = (int)a.total_q;  // below 2**31
  const int lo = min(max(a.cu ? a.cu[b] : b, 0), total), hi = min(max(a.cu ? a.cu[b + 1] : b + 1, lo), total);
  s.q0 = lo;
  s.all = hi - lo;
  s.n = min(s.all, a.max_q);
  s.len = min(max(a.lens[b], 0), a.max_pages << a.c.page_shift);  // at most 2**30
  return s;
}

// Keys [lo, hi) that new token i of the sequence sees: it sits at position len - all + i, after the
// sequence's earlier context, and sees itself and what comes before it, at most `window` keys. A
// position below 0 (more new tokens than context) sees none.
__device__ __forceinline__ void visible(const Args &a, const Seq &s, int i, int &lo, int &hi) {
  const int at = s.len - s.all + i;
  hi = a.causal ? max(at + 1, 0) : s.len;
  // (Far before the first key the difference may wrap round, to an empty range as well.)
  lo = a.window > 0 ? max((int)((uint32_t)at + 1u - (uint32_t)a.window), 0) : 0;
}

// ---------------------------------------------------------------- work split
// The tensor-core kernels cut the call into items, one per (sequence, key / value head, tile of kRows query
// rows), and an item into units of kKeys keys. A query row is a (new token, head of the group) pair, tokens
// outermost, so the heads that share keys share their reads. All units form one line, sequences outermost,
// then heads, then row tiles; each of the blocks that run takes an equal stretch of it, whatever the lengths.
// An item that lies inside one block's stretch is finished there. The others leave partial results (the
// running maximum and sum of each row and its unnormalised output, fp32), at most two a block: slot
// 2 c for the stretch's first item when it began before the stretch, 2 c + 1 for its last when it goes
// on after it; the join kernel merges them in block order, so results do not depend on timing.
struct Item {
  int b, head, tile;  // sequence, key / value head, row tile
  int units;          // of the item, at least 1 (an item without keys still writes its rows)
  int at, n;          // the stretch's part: units [at, at + n)
  int64_t left;       // units of the stretch after this part
};

// What a block leaves for the join: where its stretch starts and in which item (n 0: it has none).
struct Stretch {
  Item first;
  int64_t start;
};

template <int kRows, int kKeys>
struct Work {
  // Keys [lo, hi) that any row of the tile sees, lo rounded down to a whole unit.
  static __device__ __forceinline__ void keys(const Args &a, const Seq &s, int tile, int &lo, int &hi) {
    const int first = tile * kRows / a.group;
    const int last = min((tile + 1) * kRows - 1, s.n * a.group - 1) / a.group;
    int unused;
    visible(a, s, first, lo, unused);
    visible(a, s, last, unused, hi);
    lo = min(lo, hi) / kKeys * kKeys;
  }
  static __device__ __forceinline__ int tiles(const Args &a, const Seq &s) {
    return (int)(((int64_t)s.n * a.group + kRows - 1) / kRows);
  }
  static __device__ __forceinline__ int units(const Args &a, const Seq &s, int tile) {
    int lo, hi;
    keys(a, s, tile, lo, hi);
    return max((hi - lo + kKeys - 1) / kKeys, 1);
  }
  // Units of one head of a sequence, by a whole warp; every lane gets the sum.
  static __device__ __forceinline__ int64_t head_units(const Args &a, const Seq &s) {
    const int n = tiles(a, s);
    int64_t sum = 0;
    for (int t = threadIdx.x & 31; t < n; t += 32) sum += units(a, s, t);
    for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, m);
    return sum;
  }
  // Calls visit(b, units of one head) for every sequence in order, by a whole warp, until it returns false.
  template <typename F>
  static __device__ __forceinline__ void scan(const Args &a, F visit) {
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      Seq s{0, 0, 0, 0};
      int one = 0;
      if (b0 + lane < a.batch) {
        s = sequence(a, b0 + lane);
        const int n = tiles(a, s);
        one = n == 0 ? 0 : n == 1 ? units(a, s, 0) : -1;
      }
      for (int i = 0; i < 32 && b0 + i < a.batch; ++i) {
        int64_t u = __shfl_sync(0xFFFFFFFFu, one, i);
        if (u < 0) {
          Seq t;
          t.q0 = __shfl_sync(0xFFFFFFFFu, s.q0, i);
          t.n = __shfl_sync(0xFFFFFFFFu, s.n, i);
          t.len = __shfl_sync(0xFFFFFFFFu, s.len, i);
          t.all = __shfl_sync(0xFFFFFFFFu, s.all, i);
          u = head_units(a, t);
        }
        if (!visit(b0 + i, u)) return;
      }
    }
  }
  // Units of the whole call, by a whole warp.
  static __device__ __forceinline__ int64_t total(const Args &a) {
    int64_t sum = 0;
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      Seq s{0, 0, 0, 0};
      int n = 0;
      if (b0 + lane < a.batch) {
        s = sequence(a, b0 + lane);
        n = tiles(a, s);
      }
      if (n == 1) sum += units(a, s, 0);
      uint32_t more = __ballot_sync(0xFFFFFFFFu, n > 1);
      while (more) {
        const int i = __ffs(more) - 1;
        more &= more - 1;
        Seq t;
        t.q0 = 0;
        t.n = __shfl_sync(0xFFFFFFFFu, s.n, i);
        t.len = __shfl_sync(0xFFFFFFFFu, s.len, i);
        t.all = __shfl_sync(0xFFFFFFFFu, s.all, i);
        const int nt = tiles(a, t);
        for (int k = lane; k < nt; k += 32) sum += units(a, t, k);
      }
    }
    for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, m);
    return sum * a.c.heads;
  }
  // The item that unit u of the line lies in, with at = u's place in it (n and left are not set).
  static __device__ __forceinline__ Item find(const Args &a, int64_t u) {
    Item it{0, 0, 0, 1, 0, 0, 0};
    int64_t per = 0;
    scan(a, [&](int b, int64_t n) {
      it.b = b;
      per = n;
      if (u < n * a.c.heads) return false;
      u -= n * a.c.heads;
      return true;
    });
    it.head = (int)(u / per);
    u -= it.head * per;
    const Seq s = sequence(a, it.b);
    const int nt = tiles(a, s), lane = threadIdx.x & 31;
    for (int t0 = 0; t0 < nt; t0 += 32) {
      const int mine = t0 + lane < nt ? units(a, s, t0 + lane) : 0;
      int64_t upto = mine;
      for (int m = 1; m < 32; m <<= 1) {
        const int64_t o = __shfl_up_sync(0xFFFFFFFFu, upto, m);
        if (lane >= m) upto += o;
      }
      const uint32_t past = __ballot_sync(0xFFFFFFFFu, u < upto);
      if (past) {
        const int i = __ffs(past) - 1;
        it.tile = t0 + i;
        it.units = __shfl_sync(0xFFFFFFFFu, mine, i);
        it.at = (int)(u - (__shfl_sync(0xFFFFFFFFu, upto, i) - it.units));
        return it;
      }
      u -= __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    return it;
  }
  // The next item of the line (any thread by itself); only called while units are left.
  static __device__ __forceinline__ void next(const Args &a, Item &it) {
    Seq s = sequence(a, it.b);
    if (++it.tile >= tiles(a, s)) {
      it.tile = 0;
      if (++it.head >= a.c.heads) {
        it.head = 0;
        do s = sequence(a, ++it.b);
        while (s.n == 0);
      }
    }
    it.units = units(a, s, it.tile);
    it.at = 0;
    it.n = (int)min((int64_t)it.units, it.left);
    it.left -= it.n;
  }
  // The stretch of block c of `most`, by a whole warp.
  static __device__ __forceinline__ Stretch stretch(const Args &a, int c, int most) {
    const int64_t sum = total(a);
    const int n = blocks(sum, most);
    Stretch s{{0, 0, 0, 0, 0, 0, 0}, sum};
    if (c < n) {
      const int64_t u0 = start(sum, c, n), u1 = start(sum, c + 1, n);
      s.first = find(a, u0);
      s.first.n = (int)min((int64_t)(s.first.units - s.first.at), u1 - u0);
      s.first.left = u1 - u0 - s.first.n;
      s.start = u0;
    }
    return s;
  }
  // Blocks that share `total` units, at most `most`.
  static __device__ __forceinline__ int blocks(int64_t total, int most) { return (int)min(total, (int64_t)most); }
  static __device__ __forceinline__ int64_t start(int64_t total, int c, int n) { return total * c / n; }
};

// Weights are kept relative to a row's reference: P = exp2(x - ref), and over quantized caches P * value scale is
// what the products take in fp16. With lift = floor(log2(value scale)), the reference follows the largest x + lift of
// the keys that the row sees, kBelow under it, and moves when one comes kHeadroom above it: products stay below
// 2**15, and those within 2**20 of a row's largest keep fp16's 11 bits whatever the scales of other keys are. lift is
// held at kLeastLift, so that P stays below 2**(kHeadroom - kLeastLift), with room for the sum of 2**19 such keys. A
// value scale above 2**kMostLift, or one that is not a number, stays out of the fp16 products, its values being added in
// fp32; it counts as kOddLift, where neither P times its values nor the products of ordinary scales leave their range.
// Parts whose references differ meet with weights down to 2**-149 (exp2_wide): what one loses had less than
// 2**(kMostLift - kLeastLift - 149) = 2**-19 of the other's weight.
constexpr float kBelow = 6.0f, kHeadroom = 14.0f;
constexpr int kLeastLift = -94, kMostLift = 36, kOddLift = -20;
// Lifts this close under the largest may count as the largest: the reference moves less often, and 16 of the 20 binades
// remain.
constexpr int kNarrow = 4;
// A row of zeros has the scale 1, which says nothing of other rows: no reference follows it.
constexpr uint32_t kOneScale = 0x3F800000u;
// The bits of four codes that make them other than zeros (of either sign).
template <int S>
__device__ __forceinline__ uint32_t nonzero_codes(uint32_t w) {
  return S == KV_FP8_ROW ? w & 0x7F7F7F7Fu : w;
}
// For the exponent field of a scale.
__device__ __forceinline__ float lift_of(int field) { return (float)max(field - 127, kLeastLift); }
// A value scale (its bits) that the fp16 products do not take: beyond 2**kMostLift, infinite, NaN or negative.
__device__ __forceinline__ bool odd_scale(uint32_t bits) { return bits > (uint32_t)(127 + kMostLift) << 23; }

// One partial result: kRows maxima (base-2 logarithms), kRows sums, then the outputs as the kernel holds them:
// [dim][kRows] of the split kernel (kRows 8 or 16), [kRows][dim] of the chunk kernel.
__host__ __device__ constexpr size_t partial_floats(int rows, int dim) { return (size_t)rows * (dim + 2); }

// Element d of a cached row, in fp32.
template <typename T>
__device__ __forceinline__ float cached(const KvCache &c, const unsigned char *codes, const unsigned char *scales, int d) {
  if (c.scheme == KV_NONE) return Io<T>::get(reinterpret_cast<const T *>(codes)[d]);
  if (c.scheme == KV_MXFP4) return __fmul_rn(decode_e2m1((codes[d >> 1] >> (4 * (d & 1))) & 15u), pow2_value(scales[d >> 5]));
  const float s = *reinterpret_cast<const float *>(scales);
  return __fmul_rn(c.scheme == KV_FP8_ROW ? decode_e4m3(codes[d]) : (float)(signed char)codes[d], s);
}

// Either half of a word is an element whose exponent is all ones.
template <typename T>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
  const uint32_t m = Same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u;
  return (w & m) == m || ((w >> 16) & m) == m;
}

// Whether the products leave a row's values out: those under an odd scale, and values without scales that are not
// finite, where rows differ in what they see. S: the scheme where it is known.
template <typename T, int S>
__device__ __forceinline__ bool odd_values(const KvCache &c, int64_t row) {
  if (S == KV_NONE) {
    const uint32_t *v = reinterpret_cast<const uint32_t *>(c.v + row * c.row_bytes);
    bool odd = false;
    for (int d = 0; d < c.row_bytes / 4; ++d) odd |= not_finite2<T>(v[d]);
    return odd;
  }
  if (c.scheme != KV_MXFP4) return odd_scale(*reinterpret_cast<const uint32_t *>(c.vs + row * 4));
  uint32_t big = 0u;
  for (int q = 0; q < c.scale_bytes; ++q) big = max(big, (uint32_t)c.vs[row * c.scale_bytes + q]);
  return odd_scale(f2u(pow2_value(big) * (1.0f / (1 << kGroupShift))));
}

// A warp a (new token, query head): lanes over the head's elements, one key at a time, with the running
// maximum and sum of the softmax. Every type, scheme and head size; all arithmetic in fp32.
template <typename T>
__device__ __noinline__ void plain_rows(const Args &a, int64_t warp, int64_t warps) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = a.total_q * a.heads;
  for (int64_t r = warp; r < rows; r += warps) {
    const int64_t token = r / a.heads;
    const int head = (int)(r % a.heads);
    // The last sequence whose first token is not after this one (idle sequences share their start with
    // the next one).
    int b = 0;
    if (a.batch == 0) {
      b = -1;
    } else if (a.cu) {
      int hi = a.batch;
      while (b + 1 < hi) {
        const int mid = (b + hi) >> 1;
        if (a.cu[mid] <= token) b = mid;
        else hi = mid;
      }
    } else {
      b = (int)token;
    }
    const Seq s = b < 0 ? Seq{0, 0, 0, 0} : sequence(a, b);
    if (token < s.q0 || token >= s.q0 + s.n) {
      for (int d = lane; d < a.c.dim; d += 32) static_cast<T *>(a.out)[r * a.c.dim + d] = Io<T>::put(0.0f);
      if (a.lse && lane == 0) a.lse[r] = -INFINITY;
      continue;
    }
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

// Lets the kernel queued behind this one start (it waits for this one's end before it reads results), and that
// wait. Without the launch attribute both do nothing.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Merges the partial results of the items that several blocks share. One block for each border between two
// stretches and up to 64 rows of the item; it acts if the border is the first inside its item. A row's maxima and
// sums are read side by side into shared memory (as many parts at a time as it holds). 64 rows a block keep the
// chunk kernel's join to one wave of blocks; where few items are cut into many parts, 16 rows a block have more
// loads in flight (427 rows of one head over 13476 keys: 133 us a call with 64, 70 with 16). The split kernel's
// items have 8 or 16. Where `status` is given and a block of the kernel before gave up a wait (which takes a fault
// elsewhere, or a test), everything is computed again by the plain rows. Four blocks an SM, so that one wave takes the
// split kernel's, and arguments that the call of the plain rows reads where they are: copied for it by every block they
// cost 2 us and more (64 sequences of 8192 keys 144 us a call, 138 so; 20 of 1612 27.0 and 25.1).
constexpr int kJoinThreads = 256;

// Zeros (and -Inf) for the tokens that no sequence covers, by one warp a block: the ones before the first sequence and
// after the last by all of them, those beyond max_q of a sequence by one. Nobody else writes there, so this needs no wait.
template <typename T>
__device__ __forceinline__ void fill_tokens(const Args &a, int64_t lo, int64_t hi, int64_t part, int64_t parts) {
  const int64_t rows = (hi - lo) * a.heads, words = rows * a.c.dim * (int64_t)sizeof(T) / 16;  // head_dim is a multiple of 16
  uint4 *out = reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + lo * a.heads * a.c.dim);
  for (int64_t k = part * 32 + (threadIdx.x & 31); k < words; k += parts * 32) out[k] = make_uint4(0, 0, 0, 0);
  if (a.lse)
    for (int64_t k = part * 32 + (threadIdx.x & 31); k < rows; k += parts * 32) a.lse[lo * a.heads + k] = -INFINITY;
}
template <typename T>
__device__ __forceinline__ void fill_uncovered(const Args &a) {
  const int64_t block = blockIdx.x, blocks = gridDim.x;
  const int64_t first = a.cu[0], last = a.cu[a.batch];
  for (int64_t b0 = block * 32; b0 < a.batch; b0 += blocks * 32) {
    const int64_t b = b0 + (threadIdx.x & 31);
    int64_t lo = 0, hi = 0;
    if (b < a.batch) {
      lo = min(max((int64_t)a.cu[b], (int64_t)0) + a.max_q, a.total_q);
      hi = min((int64_t)a.cu[b + 1], a.total_q);
    }
    for (uint32_t some = __ballot_sync(0xFFFFFFFFu, lo < hi); some; some &= some - 1)
      fill_tokens<T>(a, __shfl_sync(0xFFFFFFFFu, lo, __ffs(some) - 1), __shfl_sync(0xFFFFFFFFu, hi, __ffs(some) - 1), 0, 1);
  }
  if (first > 0) fill_tokens<T>(a, 0, min(first, a.total_q), block, blocks);
  if (last < a.total_q) fill_tokens<T>(a, max(last, (int64_t)0), a.total_q, block, blocks);
}

template <typename T, int kRows, int kJoinRows>
__global__ void __launch_bounds__(kJoinThreads, 4) join_kernel(const __grid_constant__ Args a, const float *parts, const Stretch *stretches, int dim_pad, int most, const int *status) {
  constexpr int kJoinParts = 2048 / kJoinRows;
  __shared__ Item item;
  __shared__ int from, upto;
  __shared__ float part_top[kJoinParts][kJoinRows], part_sum[kJoinParts][kJoinRows];
  __shared__ float top[kJoinRows], sum[kJoinRows], keep[kJoinRows];
  const int c = blockIdx.x + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.y == 0 && warp == 1 && a.cu) fill_uncovered<T>(a);  // beside what the first warp looks up
  wait_for_previous();
  if (status) {
    int bad = 0;
    for (int i = threadIdx.x; i < most; i += kJoinThreads) bad |= status[i];
    if (__syncthreads_or(bad)) {
      const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
      plain_rows<T>(a, block * (kJoinThreads / 32) + warp, (int64_t)gridDim.x * gridDim.y * (kJoinThreads / 32));
      return;
    }
  }
  if (warp == 0) {
    int end = 0;
    if (c < most) {
      const Stretch mine = stretches[c], before = stretches[c - 1];
      const int64_t begin = mine.start - mine.first.at;
      if (mine.first.n > 0 && mine.first.at > 0 && before.start <= begin) {
        // The blocks from here on whose stretch starts inside the item.
        end = c + 1;
        while (true) {
          const int k = end + lane;
          const bool in = k < most && stretches[k].first.n > 0 && stretches[k].start < begin + mine.first.units;
          const int n = __popc(__ballot_sync(0xFFFFFFFFu, in));
          end += n;
          if (n < 32) break;
        }
        if (lane == 0) {
          item = mine.first;
          from = c - 1;
        }
      }
    }
    if (lane == 0) upto = end;
  }
  __syncthreads();
  if (upto == 0) return;
  const Seq s = sequence(a, item.b);
  const int row0 = blockIdx.y * kJoinRows, first = item.tile * kRows + row0, rows = s.n * a.group;
  if (first >= rows) return;
  const size_t size = partial_floats(kRows, dim_pad);
  // The first block left it in its last slot, the others in their first.
  auto slot = [&](int k) { return parts + (size_t)(2 * k + (k == from ? 1 : 0)) * size + row0; };
  if (threadIdx.x < kJoinRows) {
    top[threadIdx.x] = -INFINITY;
    sum[threadIdx.x] = 0.0f;
  }
  // Outputs of a thread, four at a time: rows of every kLanesD-th dim, or dims of a row of every kStep-th four.
  constexpr bool kByRow = kRows > 16;
  constexpr int kQuads = kJoinRows / 4, kLanesD = kJoinThreads / kQuads;
  const int quad = threadIdx.x % kQuads, d0 = threadIdx.x / kQuads;
  constexpr int kFours = kByRow ? kJoinRows * (128 / 4) / kJoinThreads : (256 + kLanesD - 1) / kLanesD;
  const int per_row = dim_pad / 4;
  float4 acc[kFours];
#pragma unroll
  for (int i = 0; i < kFours; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int k0 = from; k0 < upto; k0 += kJoinParts) {
    const int n = min(kJoinParts, upto - k0);
    __syncthreads();
    for (int i = threadIdx.x; i < n * kJoinRows; i += kJoinThreads) {
      part_top[i / kJoinRows][i % kJoinRows] = slot(k0 + i / kJoinRows)[i % kJoinRows];
      part_sum[i / kJoinRows][i % kJoinRows] = slot(k0 + i / kJoinRows)[kRows + i % kJoinRows];
    }
    __syncthreads();
    for (int r = warp; r < kJoinRows; r += kJoinThreads / 32) {
      const float old = top[r];
      float m = old;
      for (int k = lane; k < n; k += 32) m = fmaxf(m, part_top[k][r]);
      for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, x));
      float l = 0.0f;
      for (int k = lane; k < n; k += 32) {
        const float w = part_top[k][r] == -INFINITY ? 0.0f : exp2_wide(part_top[k][r] - m);
        // A part that saw no key has no weight; one whose scores were all NaN has a NaN sum that stays.
        l += part_sum[k][r] == 0.0f ? 0.0f : w == 0.0f && part_sum[k][r] == part_sum[k][r] ? 0.0f : part_sum[k][r] * (part_sum[k][r] == part_sum[k][r] ? w : 1.0f);
        part_top[k][r] = w;
      }
      for (int x = 16; x; x >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, x);
      if (lane == 0) {
        const float f = old == -INFINITY ? 0.0f : exp2_wide(old - m);
        keep[r] = f;
        sum[r] = sum[r] * f + l;
        top[r] = m;
      }
    }
    __syncthreads();
    if constexpr (kByRow) {
      // A part's outputs of the block's rows lie together: all of a thread's are asked for before the first is used.
      const int fours = kJoinRows * per_row / kJoinThreads;
#pragma unroll
      for (int i = 0; i < kFours; ++i) {
        const float f = keep[min((threadIdx.x + i * kJoinThreads) / per_row, kJoinRows - 1)];
        acc[i].x *= f, acc[i].y *= f, acc[i].z *= f, acc[i].w *= f;
      }
      constexpr int kSide = 8 / kFours;  // parts side by side
      for (int k = 0; k < n; k += kSide) {
        float4 o[kSide][kFours];
#pragma unroll
        for (int u = 0; u < kSide; ++u) {
          const float4 *from4 = reinterpret_cast<const float4 *>(slot(k0 + min(k + u, n - 1)) - row0 + 2 * kRows + (size_t)row0 * dim_pad) + threadIdx.x;
#pragma unroll
          for (int i = 0; i < kFours; ++i) o[u][i] = from4[(i < fours ? i : 0) * kJoinThreads];
        }
#pragma unroll
        for (int u = 0; u < kSide; ++u) {
          if (k + u >= n) break;
#pragma unroll
          for (int i = 0; i < kFours; ++i) {
            const float w = part_top[k + u][min((threadIdx.x + i * kJoinThreads) / per_row, kJoinRows - 1)];
            const float4 v = o[u][i];
            if (w != 0.0f) acc[i].x += v.x * w, acc[i].y += v.y * w, acc[i].z += v.z * w, acc[i].w += v.w * w;
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kFours; ++i) {
        const int d = d0 + i * kLanesD;
        if (d >= a.c.dim) break;
        float4 v = acc[i];
        v.x *= keep[4 * quad], v.y *= keep[4 * quad + 1], v.z *= keep[4 * quad + 2], v.w *= keep[4 * quad + 3];
#pragma unroll 8
        for (int k = 0; k < n; ++k) {
          const float4 o = *reinterpret_cast<const float4 *>(slot(k0 + k) + (size_t)(2 + d) * kRows + 4 * quad);
          const float *w = &part_top[k][4 * quad];
          if (w[0] != 0.0f) v.x += o.x * w[0];
          if (w[1] != 0.0f) v.y += o.y * w[1];
          if (w[2] != 0.0f) v.z += o.z * w[2];
          if (w[3] != 0.0f) v.w += o.w * w[3];
        }
        acc[i] = v;
      }
    }
  }
  auto out_row = [&](int row) { return (s.q0 + row / a.group) * a.heads + item.head * a.group + row % a.group; };
  for (int in = threadIdx.x; a.lse && in < kJoinRows && first + in < rows; in += kJoinThreads)
    a.lse[out_row(first + in)] = sum[in] == 0.0f ? -INFINITY : (top[in] + log2f(sum[in])) * 0.69314718055994531f;
  if constexpr (kByRow) {
#pragma unroll
    for (int i = 0; i < kFours; ++i) {
      const int four = threadIdx.x + i * kJoinThreads, row = four / per_row, d = 4 * (four % per_row);
      if (row >= kJoinRows || first + row >= rows) break;
      if (d >= a.c.dim) continue;
      const float l = sum[row], inv = l == 0.0f ? 0.0f : 1.0f / l;
      *reinterpret_cast<uint2 *>(static_cast<T *>(a.out) + out_row(first + row) * a.c.dim + d) =
          make_uint2(pack16<T>(acc[i].x * inv, acc[i].y * inv), pack16<T>(acc[i].z * inv, acc[i].w * inv));
    }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int in = 4 * quad + r, row = first + in;
      if (row >= rows) continue;
      const float l = sum[in], inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t out = out_row(row);
#pragma unroll
      for (int i = 0; i < kFours; ++i) {
        const int d = d0 + i * kLanesD;
        if (d >= a.c.dim) break;
        const float v = r == 0 ? acc[i].x : r == 1 ? acc[i].y : r == 2 ? acc[i].z : acc[i].w;
        static_cast<T *>(a.out)[out * a.c.dim + d] = Io<T>::put(v * inv);
      }
    }
  }
}

// Queues the join behind the kernel before it, to start as that one ends.
template <typename T, int kRows, int kJoinRows = kRows>
inline int launch_join(const Args &a, const float *parts, const Stretch *stretches, int most, const int *status, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(most > 1 ? most - 1 : 1, kRows / kJoinRows);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const int pad = a.c.dim <= 64 ? 64 : a.c.dim <= 128 ? 128 : 256;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, join_kernel<T, kRows, kJoinRows>, a, parts, stretches, pad, most, status);
  if (e != cudaSuccess) return set_error(std::string("tc_paged_attention: ") + cudaGetErrorString(e)), TC_CUDA_ERROR;
  count_launch();
  return TC_OK;
}

// The width of a head in the kernels' tiles and partial results.
inline int split_width(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

}  // namespace attn
}  // namespace tc
