// The next tokens from their logits l [rows][vocab] and a random number u a row:
//   w_i = exp((l_i - max l) / T), those below 2**-126 count as 0
//   K = the top_k largest; of those, in descending order, the fewest whose weights reach top_p of all of K's; of those the
//   ones with w_i >= min_p. The token is the first i in index order at which the sum of the weights that are left exceeds u
//   times their total. T = 0: the largest logit. Descending order: by weight, among equal weights by logit, then by index.
// Every filter keeps a prefix of that order, so what is kept is a weight, all tokens above it, and the first m of its equals.
//
// A row is cut into stretches, one a block of a cluster, which hold their weights in shared memory: the logits are read once.
// The weight at the cut is found by its bits, nine at a time: histograms of counts (top_k) or masses (top_p) that the cluster adds
// up through distributed shared memory. Equal high bits mean an equal exponent, so a bin's mass is a sum of 24-bit integers, exact
// in two 32-bit words; totals are fp64 sums, of single weights, in a fixed order (sums of four in fp32 first, 6 us less below, moved borders
// by up to 1.2e-7 of the total). Nothing depends on timing. Where top_k leaves few tokens (kList with the rest
// of the last one's bin), one block sorts them and finishes alone.
//
// 256 rows of 150001 fp32 logits: 114 us without filters, 151 with top_k and top_p, 226 with top_p alone (16000 tokens
// kept of a row), where reading them takes 24; one row of 131072 in bf16 12.3, 15.3 and 27 us. A block's time there is 2 to 4 us for the
// logits, 5 for weights and histogram, 2 a meeting of the cluster (1 of them the barrier), 1 to 2 a further pass over the weights. The large
// case keeps 54% of issue slots busy with two blocks an SM, as many as 64 registers and the weights' room allow: instructions
// bound it (28 a logit for weight and histogram), then the meetings, which the other block covers in part.
#pragma once

#include <cooperative_groups.h>

#include <cfloat>

#include "tc_mma16.cuh"
#include "tc_serve.cuh"

namespace tc {
namespace sample {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 512, kMaxBlocks = 8;
constexpr int kList = 512;  // tokens that one block finishes alone
constexpr int kWarpChunks = 8, kChunks = kWarps * kWarpChunks;  // a stretch is cut into runs of a warp, these into chunks
static_assert(kBins == kThreads, "a thread a bin");

struct Args {
  const void *logits;
  int64_t rows, vocab, stride;
  const float *uniform;
  const float *temperature, *top_p, *min_p;  // one a row, or nullptr
  const int32_t *top_k;
  float all_temperature, all_top_p, all_min_p;  // where there is no array
  int32_t all_top_k;
  int64_t *tokens;
  float *logprobs;
  int blocks;     // of a cluster
  int part;       // positions of a block's stretch, a multiple of 128, at most 2**20
};

struct Shared {
  uint2 hist[2][kBins];               // by turns (others may still read the last one): lower and upper parts, or counts
  double slots[2][kMaxBlocks][3];     // by turns: what each block of the cluster has sent
  double part[kWarps];
  uint32_t tops[kWarps];
  uint32_t peak[kChunks];             // of each chunk, the largest weight's bits
  double mass[kChunks];
  int ties[kChunks];
  double found[2];                    // of a histogram's scan
  uint64_t shares[kMaxBlocks];        // what each block has in the bin that was found
  uint64_t list[kList];               // the first block's: logits of the cluster and where they stand, largest first
  int listed, mine, base;
  int bin;
};

// The warp's number, said in a way that lets the compiler know that its lanes agree on it.
__device__ __forceinline__ int warp_number() { return __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0); }

__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = f2u(__fadd_rn(v, 0.0f));  // both zeros are equal
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// max(a, b), NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A weight in fp64, by its bits: two whole-number operations, where the conversion instruction runs at an eighth of their rate. None (+0) becomes
// 2**-127, which a sum that holds the largest weight, 1, does not notice.
__device__ __forceinline__ double wide(uint32_t u) { return __hiloint2double((int)((u >> 3) + 0x38000000u), (int)(u << 29)); }

// w(l) = 2**y, y = (l - max) log2(e) / T. The difference of two fp32 numbers is exact in fp64 (to 2**-53 where one is 2**29 times the
// other); one FMA multiplies it and adds 3 * 2**28, whose last place is 2**-23, so the low word of the sum is y in units of 2**-23: a whole number
// and a fraction f without a conversion. 2**f is a polynomial of degree 6 in f - 1/2, fitted to the least relative error
// (2e-9) by Remez's exchange, 1 at f = 0 and in fp32 monotone over all 2**23 fractions: larger logits never weigh less. A
// weight is off by 1.3e-7 at most, 3e-8 in the mean, which tokens that equal a 64-bit formula's need: with a hardware exponential
// (2e-7) of a rounded argument (1e-6 at y = 20) one row of some thousands fell on the neighbour.
struct Weight {
  double top, c;
  float least;  // smaller logits have no weight
  __device__ __forceinline__ double sum(float l) const { return fma((double)l - top, c, 805306368.0); }
  __device__ __forceinline__ void set(float largest, float temperature) {
    top = (double)largest;
    c = 1.4426950408889634 / (double)fmaxf(temperature, 7.888609e-31f);  // 2**-100
    const double far = top - 126.0 / c;
    least = far > -FLT_MAX ? (float)far : -FLT_MAX;  // -Inf weighs nothing at any temperature
    if (((double)least - top) * c < -126.0) least = nextafterf(least, INFINITY);
  }
  __device__ __forceinline__ float operator()(float l) const {
    const uint32_t y = (uint32_t)__double2loint(sum(l));
    const float g = __fsub_rn(u2f((y & 0x7FFFFFu) | 0x3F800000u), 1.5f);
    float q = 2.1702255e-4f;
    q = __fmaf_rn(q, g, 1.8950364e-3f);
    q = __fmaf_rn(q, g, 1.3602598e-2f);
    q = __fmaf_rn(q, g, 7.8493506e-2f);
    q = __fmaf_rn(q, g, 3.3973154e-1f);
    q = __fmaf_rn(q, g, 9.8025817e-1f);
    q = __fmaf_rn(q, g, 1.4142135f);
    return l >= least ? u2f(f2u(q) + (y & 0xFF800000u)) : 0.0f;
  }
  // The same to 2e-10, in fp64, for rows without top-k and top-p: those keep up to all of their tokens, hundreds of thousands of borders, which a
  // 16-bit type's few distinct logits (each with its own error) would shift together; no step needs such a weight's bits. 2**g, g the
  // distance to the nearest whole number, is 1 + g p(g), p of degree 6 through (2**g - 1) / g at Chebyshev's nodes (error 1.1e-10): 1 at
  // the largest logit, so that a bound of 1 keeps it.
  __device__ __forceinline__ double precise(float l) const {
    const double y = ((double)l - top) * c, t = y + 6755399441055744.0;  // 1.5 * 2**52: the whole number in the low word
    const double g = y - (t - 6755399441055744.0);
    double q = 1.529732318378528e-05;
    q = fma(q, g, 0.00015461444698744708);
    q = fma(q, g, 0.0013333502388099057);
    q = fma(q, g, 0.009618056678519811);
    q = fma(q, g, 0.05550410883908015);
    q = fma(q, g, 0.24022650922288794);
    q = fma(q, g, 0.6931471805599454);
    q = fma(q, g, 1.0);
    const double w = __hiloint2double(__double2hiint(q) + (__double2loint(t) << 20), __double2loint(q));
    return l >= least ? w : 0.0;
  }
  // log(w), in fp64.
  __device__ __forceinline__ double log(float l) const { return ((double)l - top) * c * 0.6931471805599453; }
};

// A block's stretch of a row. Positions count from a 16-byte boundary at or before the row's begin, so that vectors are aligned for
// every row; positions outside the row read as -Inf.
template <typename T>
struct Stretch {
  const T *p;      // this block's position 0
  int first, end;  // its positions inside the row
  // Four logits from position i on, i a multiple of 4.
  __device__ __forceinline__ float4 load(int i) const {
    float v[4];
    if (i >= first && i + 4 <= end) {
      if constexpr (sizeof(T) == 4) return *reinterpret_cast<const float4 *>(p + i);
      const uint2 w = *reinterpret_cast<const uint2 *>(p + i);
      const uint32_t u[2] = {w.x, w.y};
#pragma unroll
      for (int k = 0; k < 2; ++k) v[2 * k] = half_bits_to_float<Half>(u[k] & 0xFFFFu), v[2 * k + 1] = half_bits_to_float<Half>(u[k] >> 16);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = i + k >= first && i + k < end ? Io<T>::get(p[i + k]) : -INFINITY;
    }
    return make_float4(v[0], v[1], v[2], v[3]);
  }
  __device__ __forceinline__ float at(int i) const { return Io<T>::get(p[i]); }

 private:
  template <typename U, bool B>
  struct Or { using type = U; };
  template <typename U>
  struct Or<U, true> { using type = __half; };
  using Half = typename Or<T, sizeof(T) == 4>::type;  // fp32 never gets there
};

// HELD: weights stand in shared memory; otherwise (rows beyond what a cluster holds) they are computed again by every pass. A warp takes
// a run of positions in chunks of `span`, each lane 4 neighbouring ones of every 128, in all passes alike: no barrier between them.
template <typename T, bool HELD>
struct Row {
  Stretch<T> z;
  Weight w;
  Shared &sh;
  float *held;
  int n, run, span;  // positions of the stretch, of a warp and of a chunk, multiples of 128
  int blocks, rank, turn, hist_turn;
  bool exact;     // whether cut() added masses last
  bool infinite;  // the row's largest logit is: its equals share everything, as logits of 0 beside -Inf
  cg::cluster_group cluster;

  __device__ __forceinline__ Row(Shared &s, float *h)
      : sh(s), held(h), turn(0), hist_turn(0), exact(false), infinite(false), cluster(cg::this_cluster()) {}

  static __device__ __forceinline__ float finite(float l) { return l == INFINITY ? 0.0f : -INFINITY; }
  __device__ __forceinline__ float4 weigh(float4 l) const {
    if (infinite) l = make_float4(finite(l.x), finite(l.y), finite(l.z), finite(l.w));
    return make_float4(w(l.x), w(l.y), w(l.z), w(l.w));
  }
  __device__ __forceinline__ float4 four(int i) const {
    return HELD ? *reinterpret_cast<const float4 *>(held + i) : weigh(z.load(i));
  }
  // f(position, the bits of four weights) for the chunks of this warp whose largest weight is `from` at least.
  template <typename F>
  __device__ __forceinline__ void each(uint32_t from, F f) const {
    chunks([&](int c, int at, int end) {
      if (sh.peak[c] >= from)
        steps(at, end, [&](int i) {
          const float4 q = four(i);
          f(i, make_uint4(f2u(q.x), f2u(q.y), f2u(q.z), f2u(q.w)));
        });
    });
  }
  // f(chunk, its first position, its end) for this warp's chunks, empty ones among them.
  template <typename F>
  __device__ __forceinline__ void chunks(F f) const {
    const int warp = warp_number(), end = min((warp + 1) * run, n);
#pragma unroll 1
    for (int c = 0; c < kWarpChunks; ++c) {
      const int at = warp * run + c * span;
      f(warp * kWarpChunks + c, at, min(at + span, end));
    }
  }
  // f(this lane's position) for 128 positions after the other; four times 128, what a chunk has where it is whole, without a loop.
  template <typename F>
  __device__ __forceinline__ void steps(int at, int end, F f) const {
    const int mine = (threadIdx.x & 31) * 4;
    for (; at + 512 <= end; at += 512)
#pragma unroll
      for (int k = 0; k < 4; ++k) f(at + k * 128 + mine);
#pragma unroll 1
    for (; at < end; at += 128) f(at + mine);
  }
  __device__ __forceinline__ int begin_of(int c) const { return c / kWarpChunks * run + c % kWarpChunks * span; }
  __device__ __forceinline__ int end_of(int c) const { return min(begin_of(c) + span, min((c / kWarpChunks + 1) * run, n)); }

  // The cluster's barrier: what its threads wrote before is seen by those that read after. A warp's lanes come together for it.
  static __device__ __forceinline__ void meet() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  // Another block's word (both of them where MASS) at an address of this one's shared memory.
  template <bool MASS>
  static __device__ __forceinline__ uint2 look(uint32_t here, int block) {
    uint2 v = make_uint2(0u, 0u);
    if (MASS)
      asm volatile("{\n.reg .u32 a;\nmapa.shared::cluster.u32 a, %2, %3;\nld.shared::cluster.v2.u32 {%0, %1}, [a];\n}"
                   : "=r"(v.x), "=r"(v.y)
                   : "r"(here), "r"(block)
                   : "memory");
    else
      asm volatile("{\n.reg .u32 a;\nmapa.shared::cluster.u32 a, %1, %2;\nld.shared::cluster.u32 %0, [a];\n}" : "=r"(v.x) : "r"(here), "r"(block) : "memory");
    return v;
  }
  // Up to three numbers from each block to all of them, to be read after the cluster's next barrier. Two turns apart the slots are
  // used again, and between them lies a barrier that a block reaches only after reading.
  using Slot = const double (*)[3];
  __device__ __forceinline__ Slot tell(double v, double x = 0.0, double y = 0.0) {
    double (*to)[3] = sh.slots[turn];
    if ((int)threadIdx.x < blocks) {
      double *there = cluster.map_shared_rank(&to[rank][0], threadIdx.x);
      there[0] = v, there[1] = x, there[2] = y;
    }
    turn ^= 1;
    return to;
  }
  // Sums in every thread of the block, in a fixed order: over a warp's lanes, then the warps' sums over 16 lanes of each warp.
  __device__ __forceinline__ double block_sum(double v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh.part[threadIdx.x & (kWarps - 1)];
#pragma unroll
    for (int m = kWarps / 2; m; m >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
    return v;
  }
  __device__ __forceinline__ double all_of(Slot slots) const {
    const int lane = threadIdx.x & (kMaxBlocks - 1);
    double v = lane < blocks ? slots[lane][0] : 0.0;
#pragma unroll
    for (int m = kMaxBlocks / 2; m; m >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
    return v;
  }
  // The largest of a key a thread: in every thread of the block, or of the cluster.
  __device__ __forceinline__ uint32_t block_max(uint32_t v) {
    v = warp_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.tops[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_max(sh.tops[threadIdx.x & (kWarps - 1)]);
  }
  __device__ __forceinline__ uint32_t largest_told(Slot all, int which) const {
    const int lane = threadIdx.x & (kMaxBlocks - 1);
    return warp_max(lane < blocks ? (uint32_t)all[lane][which] : 0u);
  }
  __device__ __forceinline__ uint32_t cluster_max(uint32_t v) {
    Slot all = tell((double)block_max(v));
    meet();
    return largest_told(all, 0);
  }

  // Adds a weight's bits to its bin: its count, or its 24-bit significand in parts of 12 bits (a stretch has at most 2**20
  // positions, so neither sum passes 32 bits).
  template <bool MASS>
  __device__ __forceinline__ void add(int bin, uint32_t u, bool yes) const {
    if (!yes) return;
    uint2 *to = &sh.hist[hist_turn][bin];
    if (MASS) {
      atomicAdd(&to->x, u & 0xFFFu);
      atomicAdd(&to->y, ((u >> 12) & 0x7FFu) | 0x800u);
    } else {
      atomicAdd(&to->x, 1u);
    }
  }
  // The first bin at which counts or masses of the cluster, on top of `over`, reach want(), kBins where none does (then, with
  // `last`, the last one that is not empty). over: what is before it; own: what is in it; exponent(bin): of the bin's weights. The
  // next histogram, which every block has read, is cleared.
  template <bool MASS, typename Q, typename X>
  __device__ __forceinline__ int reach(Q want, double &over, double &own, bool last, X exponent) {
    meet();
    const int bin = threadIdx.x, lane = bin & 31, warp = warp_number();
    const double need = want();
    double v;
    // All of them asked for before the first is used, and without a branch between them: a look at another block's shared memory
    // takes some 700 cycles.
    uint2 part[kMaxBlocks];
    const uint32_t here = smem_addr(&sh.hist[hist_turn][bin]);
#pragma unroll
    for (int b = 0; b < kMaxBlocks; ++b) part[b] = look<MASS>(here, min(b, blocks - 1));
    uint64_t sum = 0;
#pragma unroll
    for (int b = 0; b < kMaxBlocks; ++b) sum += b < blocks ? part[b].x + (MASS ? (uint64_t)part[b].y << 12 : 0) : 0;
    v = (double)sum;
    if (MASS) v *= __longlong_as_double((long long)(1023 + exponent(bin) - 23) << 52);
    hist_turn ^= 1;
    sh.hist[hist_turn][bin] = make_uint2(0u, 0u);
    double s = v;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const double o = __shfl_up_sync(0xFFFFFFFFu, s, m);
      if (lane >= m) s += o;
    }
    if (lane == 31) sh.part[warp] = s;
    if (bin == 0) sh.bin = kBins;
    __syncthreads();
    double base = sh.part[lane & (kWarps - 1)];  // the warps' totals, added up over 16 lanes
#pragma unroll
    for (int m = 1; m < kWarps; m <<= 1) {
      const double o = __shfl_up_sync(0xFFFFFFFFu, base, m);
      if ((lane & (kWarps - 1)) >= m) base += o;
    }
    const double all = over + __shfl_sync(0xFFFFFFFFu, base, kWarps - 1);
    base = __shfl_sync(0xFFFFFFFFu, base, max(warp - 1, 0));
    base = warp ? over + base : over;
    if (v > 0.0 && base + s >= need) atomicMin(&sh.bin, bin);
    __syncthreads();
    if (last && sh.bin == kBins) {  // the sums' last bits
      __syncthreads();
      if (bin == 0) sh.bin = -1;
      __syncthreads();
      if (v > 0.0) atomicMax(&sh.bin, bin);
      __syncthreads();
    }
    const int b = sh.bin;
    if (bin == b) {
      sh.found[0] = base + (s - v), sh.found[1] = v;
#pragma unroll
      for (int i = 0; i < kMaxBlocks; ++i) sh.shares[i] = part[i].x + (MASS ? (uint64_t)part[i].y << 12 : 0);
    }
    __syncthreads();
    over = b < kBins ? sh.found[0] : all;
    own = b < kBins ? sh.found[1] : 0.0;
    return b;
  }

  // Bins of 32 an octave below 1: weights of one bin share their exponent.
  static constexpr uint32_t kTop = 0x3F800000u >> 18;
  static constexpr int kWindows = (int)(kTop + kBins - 1 - (0x00800000u >> 18)) / kBins + 1;
  static __device__ __forceinline__ int bin_of(uint32_t u, int window) { return (int)(kTop - (u >> 18)) - window * kBins; }

  // The weight (its bits) at which counts or masses in descending order reach want(); over: those above it, equals: how many
  // have it. Weights below `from` do not count. false where all of them stay below. The first window's histogram is
  // there already where `filled`.
  template <bool MASS, typename Q>
  __device__ bool cut(Q want, uint32_t from, bool filled, uint32_t &weight, double &over, double &equals) {
    over = 0.0;
    double own;
    int window = 0, b = kBins;
    for (; window < kWindows; ++window) {
      if (window || !filled) {
        const uint32_t below = (uint32_t)max((int)kTop + 1 - (window + 1) * kBins, 0) << 18;  // the window's least
        each(max(from, below), [&](int, uint4 q) {
          const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int bin = bin_of(u[k], window);
            add<MASS>(bin, u[k], (unsigned)bin < (unsigned)kBins && u[k] >= from);
          }
        });
      }
      b = reach<MASS>(want, over, own, false, [&](int bin) { return (int)((kTop - bin - window * kBins) >> 5) - 127; });
      if (b < kBins) break;
    }
    if (b == kBins) return false;
    uint32_t high = kTop - (uint32_t)(b + window * kBins);
    const int exponent = (int)(high >> 5) - 127;
    exact = MASS;
#pragma unroll 1
    for (int shift = 9; shift >= 0; shift -= 9) {
      if (MASS) {
        // Two significands are 2**24 at least: a smaller sum is one token's, and says which weight it has.
        const double units = own * __longlong_as_double((long long)(1023 - exponent + 23) << 52);
        if (units < 16777216.0) {
          weight = (uint32_t)(exponent + 127) << 23 | ((uint32_t)units & 0x7FFFFFu);
          equals = 1.0;
          return true;
        }
      }
      each(high << (shift + 9), [&](int, uint4 q) {
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
        bool hit = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) hit |= u[k] - (high << (shift + 9)) < 1u << (shift + 9);
        if (__any_sync(0xFFFFFFFFu, hit))
#pragma unroll
          for (int k = 0; k < 4; ++k)
            add<MASS>(kBins - 1 - (int)((u[k] >> shift) & (kBins - 1)), u[k], u[k] >> (shift + 9) == high && u[k] >= from);
      });
      b = reach<MASS>(want, over, own, true, [&](int) { return exponent; });
      high = (high << 9) | (uint32_t)(kBins - 1 - b);
    }
    weight = high;
    equals = MASS ? rint(own / (double)u2f(high)) : own;
    return true;
  }

  // How many tokens at the weight that cut() found the blocks before this one have.
  __device__ __forceinline__ double equals_before(uint32_t weight) const {
    const double one = exact ? (double)((weight & 0x7FFFFFu) | 0x800000u) : 1.0;
    double n = 0.0;
    for (int i = 0; i < rank; ++i) n += rint((double)sh.shares[i] / one);
    return n;
  }

  // Whether one value of T alone has this weight: a logit computed from it, or a neighbour of that, has it, and the next ones on
  // both sides do not (weights are monotone).
  __device__ bool one_logit(uint32_t weight) const {
    if (infinite) return true;
    const float guess = (float)(w.top + log2((double)u2f(weight)) / w.c);
    int at;  // T's values in their order, as whole numbers
    if constexpr (sizeof(T) == 4) {
      at = (int)(key_of(guess) ^ 0x80000000u);
    } else {
      const T t = Io<T>::put(guess);
      const int bits = *reinterpret_cast<const unsigned short *>(&t);
      at = bits & 0x8000 ? 0x7FFF - bits : bits;
    }
    auto weight_at = [&](int k) {
      float l;
      if constexpr (sizeof(T) == 4) {
        const uint32_t key = (uint32_t)k ^ 0x80000000u;
        l = u2f((key >> 31) ? key & 0x7FFFFFFFu : ~key);
      } else {
        const unsigned short bits = (unsigned short)(k < 0 ? 0x7FFF - k : k);
        l = Io<T>::get(*reinterpret_cast<const T *>(&bits));
      }
      return f2u(w(l));
    };
    int have = 0, edges = 0;
#pragma unroll 1
    for (int k = -3; k <= 3; ++k) {
      const bool same = weight_at(at + k) == weight;
      have += same;
      edges += same && (k == -3 || k == 3);
    }
    return have == 1 && edges == 0;
  }

  // Where the `want` largest weights, with the rest of the last one's bin, are kList at most: they stand in the first block's list
  // then, logits and places as one number, in no order. Otherwise nothing is kept, and the counts are taken again.
  __device__ bool gather(double want, int64_t origin) {
    double over = 0.0, own;
    const int b = reach<false>([&] { return want; }, over, own, false, [](int) { return 0; });
    if (over + own > (double)kList || b == kBins) return false;
    uint64_t *local = reinterpret_cast<uint64_t *>(sh.hist[hist_turn]);  // clear, and as long as the list
    static_assert(sizeof(sh.hist[0]) == kList * sizeof(uint64_t), "a list's room");
    const uint32_t from = (kTop - (uint32_t)b) << 18;
    each(from, [&](int i, uint4 q) {
      const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (u[k] >= from) local[atomicAdd(&sh.mine, 1)] = (uint64_t)key_of(z.at(i + k)) << 32 | (0xFFFFFFFFu - (uint32_t)(origin + i + k));
    });
    __syncthreads();
    const int mine = sh.mine;
    if (threadIdx.x == 0) sh.base = atomicAdd(cluster.map_shared_rank(&sh.listed, 0), mine);
    __syncthreads();
    if ((int)threadIdx.x < mine) cluster.map_shared_rank(sh.list, 0)[sh.base + threadIdx.x] = local[threadIdx.x];
    meet();
    return true;
  }

  // The first block: the rest of the definition for the tokens of its list. Descending order by a bitonic sort, a thread a token.
  template <typename A>
  __device__ void finish(int64_t k, float p, float bound, double uniform, A answer) {
    const int n = sh.listed, t = threadIdx.x;
    int size = 32;
    while (size < n) size *= 2;
    uint64_t mine = t < n ? sh.list[t] : 0ull;
    for (int width = 2; width <= size; width *= 2)
      for (int step = width / 2; step; step /= 2) {
        uint64_t other;
        if (step >= 32) {
          __syncthreads();
          sh.list[t] = mine;
          __syncthreads();
          other = sh.list[t ^ step];
        } else {
          other = __shfl_xor_sync(0xFFFFFFFFu, mine, step);
        }
        const bool larger = ((t & step) == 0) == ((t & width) == 0 || width == size);
        mine = (other > mine) == larger ? other : mine;
      }
    const uint32_t key = (uint32_t)(mine >> 32), place = (uint32_t)mine;  // places count from the end
    float logit = u2f((key >> 31) ? key & 0x7FFFFFFFu : ~key);
    if (infinite) logit = finite(logit);
    const float weight = t < n && t < k ? w(logit) : 0.0f;
    // Sums of the weights up to each, over the block.
    auto scan = [&](double v, double &all) {
      const int lane = t & 31, warp = warp_number();
      double x = v;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const double o = __shfl_up_sync(0xFFFFFFFFu, x, m);
        if (lane >= m) x += o;
      }
      __syncthreads();
      if (lane == 31) sh.part[warp] = x;
      __syncthreads();
      double before = 0.0;
      all = 0.0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const double o = sh.part[i];
        before = i < warp ? before + o : before;
        all += o;
      }
      return before + x;
    };
    double all, total;
    const double upto = scan((double)weight, all);
    const bool keep = weight > 0.0f && !(weight < bound) && (t == 0 || !(p < 1.0f) || upto - (double)weight < (double)p * all);
    scan(keep ? (double)weight : 0.0, total);
    // In index order: of each kept token, the sum up to it.
    const int kept = __syncthreads_count(keep);
    sh.list[t] = (uint64_t)f2u(weight) << 32 | place;
    __syncthreads();
    const double aim = fmax(uniform * total, 0.0);
    uint32_t hit = 0u, last = 0u;  // the first token that passes the aim, and the last one of all, as a place
    if (keep) {
      double s = 0.0;
      for (int i = 0; i < kept; ++i) {
        const uint64_t o = sh.list[i];
        if ((uint32_t)o >= place) s += (double)u2f((uint32_t)(o >> 32));
      }
      if (s > aim) hit = place;
      last = 0xFFFFFFFFu - place;
    }
    hit = block_max(hit);
    last = block_max(last);
    const uint32_t found = hit ? hit : 0xFFFFFFFFu - last;
    if (keep && place == found) answer((int64_t)(0xFFFFFFFFu - place), (float)((infinite ? 0.0 : w.log(logit)) - log(total)));
  }

  // Of the tokens of a weight the first `want` are kept, larger logits first: the logit at which they end, and how many of
  // that logit's tokens stay.
  __device__ void cut_logits(uint32_t weight, int64_t want, float &logit, int64_t &quota) {
    double over = 0.0, own = 0.0;
    uint32_t high = 0;
#pragma unroll 1
    for (int shift = 27; shift >= 0; shift -= 9) {  // 5, 9, 9 and 9 bits
      each(weight, [&](int i, uint4 q) {
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (u[k] == weight) {
            const uint32_t key = key_of(z.at(i + k));
            add<false>(kBins - 1 - (int)((key >> shift) & (kBins - 1)), 0u, shift == 27 || key >> (shift + 9) == high);
          }
      });
      const int b = reach<false>([&] { return (double)want; }, over, own, true, [](int) { return 0; });
      high = (high << 9) | (uint32_t)(kBins - 1 - b);
    }
    logit = u2f((high >> 31) ? high & 0x7FFFFFFFu : ~high);
    quota = want - (int64_t)over;
  }

  // This thread's part of the weights above one.
  __device__ __forceinline__ double mass_above(uint32_t weight) {
    double s = 0.0;
    each(weight + 1, [&](int, uint4 q) {
      const uint32_t u[4] = {q.x, q.y, q.z, q.w};
      double t[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) t[k] = wide(u[k] > weight ? u[k] : 0u);
      s += (t[0] + t[1]) + (t[2] + t[3]);
    });
    return s;
  }

  // Weights in the logits' place, the chunks' largest, this thread's part of their sum, and the histogram that the first
  // filter begins with: of counts, or of masses.
  template <bool MASS>
  __device__ __forceinline__ double prepare() {
    const int lane = threadIdx.x & 31;
    double sum = 0.0;
    chunks([&](int c, int at, int end) {
      uint32_t top = 0u;
      steps(at, end, [&](int i) {
        float4 q;
        if (HELD) {
          q = *reinterpret_cast<const float4 *>(held + i);
          q = make_float4(w(q.x), w(q.y), w(q.z), w(q.w));
          *reinterpret_cast<float4 *>(held + i) = q;
        } else {
          q = four(i);
        }
        const uint32_t u[4] = {f2u(q.x), f2u(q.y), f2u(q.z), f2u(q.w)};
        sum += (wide(u[0]) + wide(u[1])) + (wide(u[2]) + wide(u[3]));
        top = max(max(max(u[0], u[1]), max(u[2], u[3])), top);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int b = bin_of(u[k], 0);
          add<MASS>(b, u[k], b < kBins);
        }
      });
      top = warp_max(top);
      if (lane == 0) sh.peak[c] = top;
    });
    __syncwarp();
    return sum;
  }

  // No filter but a bound of the weights: logits stay, and the chunks' sums are of precise weights.
  __device__ __forceinline__ float4 logits(int i) const {
    float4 l = HELD ? *reinterpret_cast<const float4 *>(held + i) : z.load(i);
    if (!HELD && infinite) l = make_float4(finite(l.x), finite(l.y), finite(l.z), finite(l.w));
    return l;
  }
  static __device__ __forceinline__ double bounded(double w, float bound) { return w < (double)bound ? 0.0 : w; }
  __device__ __forceinline__ void sum_all(float bound) {
    const int lane = threadIdx.x & 31;
    chunks([&](int c, int at, int end) {
      double sum = 0.0;
      steps(at, end, [&](int i) {
        const float4 l = logits(i);
        auto kept = [&](float v) { return bounded(w.precise(v), bound); };
        sum += (kept(l.x) + kept(l.y)) + (kept(l.z) + kept(l.w));
      });
#pragma unroll
      for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
      if (lane == 0) sh.mass[c] = sum, sh.ties[c] = 0;
    });
  }
};

template <typename T, bool HELD>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(Args a) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  __shared__ Shared shared;
  Row<T, HELD> row(shared, reinterpret_cast<float *>(dynamic));
  const int lane = threadIdx.x & 31, warp = warp_number();
  const int blocks = row.blocks = a.blocks, rank = row.rank = (int)row.cluster.block_rank();
  const int64_t r = blockIdx.x / blocks;
  int64_t origin;  // of position i the token is origin + i
  {
    const T *p = static_cast<const T *>(a.logits) + r * a.stride;
    const int64_t skip = (int64_t)((uintptr_t)p % 16 / sizeof(T)), lo = (int64_t)a.part * rank, end = skip + a.vocab - lo;
    row.z.p = p - skip + lo;
    row.z.first = rank ? 0 : (int)skip;
    row.z.end = (int)max(min((int64_t)a.part, end), (int64_t)0);
    row.n = (row.z.end + 127) / 128 * 128;
    // Chunks of 512 positions (their sums' reduction over the warp then costs little), longer ones where those are too many.
    const int each = (row.n / 128 + kWarps - 1) / kWarps;
    row.run = each * 128;
    row.span = max(4, (each + kWarpChunks - 1) / kWarpChunks) * 128;
    origin = lo - skip;
  }
  const Stretch<T> &z = row.z;
  const int n = row.n;
  float *held = row.held;
  shared.hist[0][threadIdx.x] = make_uint2(0u, 0u);  // added to after cluster_max's barriers
  if (threadIdx.x == 0) shared.listed = shared.mine = 0;
  auto started = row.cluster.barrier_arrive();

  // The logits, once, and the largest. fp32 goes to shared memory without a detour, all of a thread's at once.
  float top = -INFINITY;
  auto largest = [&](float4 v) { top = max_nan(top, max_nan(max_nan(v.x, v.y), max_nan(v.z, v.w))); };
  const int run_begin = warp * row.run, run_end = min(run_begin + row.run, n);
  if constexpr (HELD && sizeof(T) == 4) {
    row.steps(run_begin, run_end, [&](int i) {
      if (i >= z.first && i + 4 <= z.end) cp_async16(held + i, z.p + i);
      else *reinterpret_cast<float4 *>(held + i) = z.load(i);
    });
    cp_async_wait_all();
    row.steps(run_begin, run_end, [&](int i) { largest(*reinterpret_cast<const float4 *>(held + i)); });
  } else {
    row.steps(run_begin, run_end, [&](int i) {
      const float4 v = z.load(i);
      if (HELD) *reinterpret_cast<float4 *>(held + i) = v;
      largest(v);
    });
  }
  row.cluster.barrier_wait(static_cast<decltype(started) &&>(started));  // blocks that have not begun have no shared memory to write to
  {
    // NaN above Inf above every number.
    const uint32_t t = row.cluster_max(top != top ? 0xFFFFFFFFu : key_of(top));
    top = t == 0xFFFFFFFFu ? u2f(kQNaN) : u2f((t >> 31) ? t & 0x7FFFFFFFu : ~t);
  }
  const float heat = a.temperature ? a.temperature[r] : a.all_temperature;
  auto answer = [&](int64_t token, float logprob) {
    a.tokens[r] = token;
    if (a.logprobs) a.logprobs[r] = logprob;
  };
  if (!(top > -INFINITY)) {
    if (rank == 0 && threadIdx.x == 0) answer(-1, top);
  } else if (!(heat > 0.0f)) {
    uint32_t at = 0u;  // the first index, from the end
    row.steps(run_begin, run_end, [&](int i) {
      const float4 v = HELD ? *reinterpret_cast<const float4 *>(held + i) : z.load(i);
      const int k = v.x == top ? 0 : v.y == top ? 1 : v.z == top ? 2 : v.w == top ? 3 : -1;
      if (k >= 0 && !at) at = 0xFFFFFFFFu - (uint32_t)(origin + i + k);
    });
    at = row.cluster_max(at);
    if (rank == 0 && threadIdx.x == 0) answer((int64_t)(0xFFFFFFFFu - at), 0.0f);
  } else {
    row.infinite = top == INFINITY;
    row.w.set(row.infinite ? 0.0f : top, heat);
    if (HELD && row.infinite)
      row.steps(run_begin, run_end, [&](int i) {
        for (int e = i; e < i + 4; ++e) held[e] = Row<T, HELD>::finite(held[e]);
      });
    const int64_t k = a.top_k ? a.top_k[r] : a.all_top_k;
    const float p = a.top_p ? a.top_p[r] : a.all_top_p, low = a.min_p ? a.min_p[r] : a.all_min_p;
    const bool by_count = k > 0 && k < a.vocab, by_mass = p < 1.0f;
    const float bound = low > 1.0f ? 1.0f : low;  // NaN bounds nothing
    // Kept: weights above `cut`, and of the tokens at it the first m.
    uint32_t cut = 0u;
    double sum = 0.0;
    const bool bare = !by_count && !by_mass;
    if (by_count) sum = row.template prepare<false>();
    else if (by_mass) sum = row.template prepare<true>();
    else row.sum_all(bound);
    bool counted = by_count;  // whether the histogram of counts still stands
    if (by_count && k <= kList) {
      if (row.gather((double)k, origin)) {
        if (rank == 0) row.finish(k, p, bound, (double)a.uniform[r], answer);
        return;
      }
      counted = false;
    }
    double m = 0.0, equals = 0.0, over;
    if (by_count && row.template cut<false>([&] { return (double)k; }, 1u, counted, cut, over, equals)) m = (double)k - over;
    if (by_mass) {
      if (by_count) sum = row.mass_above(cut);
      const auto all = row.tell(row.block_sum(sum));
      double aim = 0.0;
      bool summed = false;
      auto want = [&] {  // after the next barrier
        if (!summed) aim = (double)p * (row.all_of(all) + m * (double)u2f(cut)), summed = true;
        return aim;
      };
      uint32_t c;
      double e;
      if (row.template cut<true>(want, max(cut, 1u), !by_count, c, over, e)) {
        const double need = fmin(fmax(ceil((aim - over) / (double)u2f(c)), 1.0), e);
        m = c == cut ? fmin(need, m) : need;
        cut = c, equals = e;
      }
    }
    if (m > 0.0 && (u2f(cut) < bound || m == equals)) {  // none or all of the equals
      if (!(u2f(cut) < bound)) cut -= 1;
      m = 0.0;
    }
    if (bound > u2f(cut)) cut = max(cut, f2u(bound) - 1);
    // Some of the equals, in the order of their logits: those above `tie`, and of those that have it the first `quota`. Equal
    // weights mostly come of equal logits.
    const bool some = m > 0.0;
    bool alike = true;
    float tie = 0.0f;
    int64_t left = 0;  // ties that this block may keep
    if (some) {
      int64_t quota = (int64_t)m;
      double others = row.equals_before(cut);
      alike = row.one_logit(cut);
      if (!alike) {
        row.cut_logits(cut, (int64_t)m, tie, quota);
        double mine = 0.0;
        row.each(cut, [&](int i, uint4 q) {
          const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (u[e] == cut && z.at(i + e) == tie) mine += 1.0;
        });
        const auto all = row.tell(row.block_sum(mine));
        row.meet();
        others = 0.0;
        for (int i = 0; i < rank; ++i) others += all[i][0];
      }
      left = max(quota - (int64_t)others, (int64_t)0);
    }
    auto equal = [&](int i, uint32_t u, bool &above) {  // a tie, or one whose logit is above it
      if (u != cut || alike) return u == cut;
      const float l = z.at(i);
      above = l > tie;
      return l == tie;
    };

    // Masses and ties by chunks.
    if (!bare) row.chunks([&](int c, int at, int end) {
      double s = 0.0;
      int e = 0;
      const uint32_t peak = shared.peak[c];
      if (!some && peak > cut) {
        row.steps(at, end, [&](int i) {
          const float4 q = row.four(i);
          auto kept = [&](float v) { return f2u(v) > cut ? wide(f2u(v)) : 0.0; };  // 0 says that nothing is kept
          s += (kept(q.x) + kept(q.y)) + (kept(q.z) + kept(q.w));
        });
      } else if (some && alike && peak >= cut) {
        row.steps(at, end, [&](int i) {
          const float4 q = row.four(i);
          auto kept = [&](float v) { return e += f2u(v) == cut, f2u(v) > cut ? wide(f2u(v)) : 0.0; };
          s += (kept(q.x) + kept(q.y)) + (kept(q.z) + kept(q.w));
        });
        e = (int)__reduce_add_sync(0xFFFFFFFFu, e);
      } else if (some && peak >= cut) {
        for (; at < end; at += 128) {
          const int i = at + lane * 4;
          const float4 q = row.four(i);
          const float v[4] = {q.x, q.y, q.z, q.w};
          double t[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            bool keep = f2u(v[x]) > cut;
            if (!keep) e += equal(i + x, f2u(v[x]), keep);
            t[x] = keep ? wide(f2u(v[x])) : 0.0;
          }
          s += (t[0] + t[1]) + (t[2] + t[3]);
        }
        e = (int)__reduce_add_sync(0xFFFFFFFFu, e);
      }
      if (peak > cut || (some && peak == cut)) {
#pragma unroll
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
      }
      if (lane == 0) shared.mass[c] = s, shared.ties[c] = e;
    });
    __syncthreads();
    // Chunks in order, four a lane of the first warp: ties that are left, and the mass before each.
    constexpr int kLane = kChunks / 32;
    double before = 0.0;
    if (warp == 0) {
      double own = 0.0;
      if (some) {
        int64_t mine = 0;
#pragma unroll
        for (int c = 0; c < kLane; ++c) mine += shared.ties[lane * kLane + c];
        int64_t upto = mine;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const int64_t o = __shfl_up_sync(0xFFFFFFFFu, upto, x);
          if (lane >= x) upto += o;
        }
        int64_t room = max(left - (upto - mine), (int64_t)0);
#pragma unroll
        for (int c = 0; c < kLane; ++c) {
          const int64_t take = min((int64_t)shared.ties[lane * kLane + c], room);
          shared.ties[lane * kLane + c] = (int)take;
          room -= take;
          shared.mass[lane * kLane + c] += (double)take * (double)u2f(cut);
        }
      }
#pragma unroll
      for (int c = 0; c < kLane; ++c) own += shared.mass[lane * kLane + c];
      before = own;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const double o = __shfl_up_sync(0xFFFFFFFFu, before, x);
        if (lane >= x) before += o;
      }
      const double all = __shfl_sync(0xFFFFFFFFu, before, 31);
      before -= own;
      if (lane == 0) shared.found[0] = all;
    }
    __syncthreads();
    const auto all = row.tell(shared.found[0]);
    row.meet();
    if (warp) return;
    // The block whose stretch the aim falls in; behind all of them (u = 1, or the last bits of the sums) the last one that
    // keeps anything.
    const double total = row.all_of(all), aim = fmax((double)a.uniform[r] * total, 0.0);
    int owner = -1;
    double start = 0.0, at = 0.0;
    for (int i = 0; i < blocks; ++i) {
      if (all[i][0] > 0.0) owner = i, start = at;
      at += all[i][0];
      if (all[i][0] > 0.0 && at > aim) break;
    }
    if (rank == owner) {
      // Its chunk, likewise.
      const double rest = aim - start;
      int chunk = -1;
      double s = before, chunk_start = 0.0;
#pragma unroll
      for (int c = 0; c < kLane; ++c) {
        const double v = shared.mass[lane * kLane + c];
        if (v > 0.0 && (chunk < 0 || chunk_start + shared.mass[chunk] <= rest)) chunk = lane * kLane + c, chunk_start = s;
        s += v;
      }
      const unsigned hit = __ballot_sync(0xFFFFFFFFu, chunk >= 0 && chunk_start + shared.mass[max(chunk, 0)] > rest);
      const unsigned any = __ballot_sync(0xFFFFFFFFu, chunk >= 0);
      const int source = hit ? __ffs(hit) - 1 : 31 - __clz(any);
      chunk = __shfl_sync(0xFFFFFFFFu, chunk, source);
      double need = rest - __shfl_sync(0xFFFFFFFFu, chunk_start, source);
      int room = shared.ties[chunk], found = -1, kept = -1;
      // Its tokens, 32 at a time.
      for (int i0 = row.begin_of(chunk); found < 0 && i0 < row.end_of(chunk); i0 += 32) {
        const int i = i0 + lane;
        const float4 q = bare ? row.logits(i & ~3) : row.four(i & ~3);
        const float v = (i & 2) ? ((i & 1) ? q.w : q.z) : (i & 1) ? q.y : q.x;
        double x = bare ? Row<T, HELD>::bounded(row.w.precise(v), bound) : (double)v;
        bool keep = bare ? x > 0.0 : f2u(v) > cut, mine = false;
        if (some && !keep) mine = equal(i, f2u(v), keep);
        const unsigned same = __ballot_sync(0xFFFFFFFFu, mine);
        if (mine) keep = __popc(same & ((1u << lane) - 1u)) < room;
        room = max(room - __popc(same), 0);
        const unsigned mask = __ballot_sync(0xFFFFFFFFu, keep);
        if (!keep) x = 0.0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const double o = __shfl_up_sync(0xFFFFFFFFu, x, d);
          if (lane >= d) x += o;
        }
        const unsigned over_it = __ballot_sync(0xFFFFFFFFu, x > need) & mask;
        if (mask) kept = i0 + 31 - __clz(mask);
        if (over_it) found = i0 + __ffs(over_it) - 1;
        need -= __shfl_sync(0xFFFFFFFFu, x, 31);
      }
      if (found < 0) found = kept;
      if (lane == 0) answer(origin + found, (float)((row.infinite ? 0.0 : row.w.log(z.at(found))) - log(total)));
    }
  }
  // The last barrier before this line comes after every block's last look at another one's shared memory, except where blocks tell
  // each other numbers: those are written before it.
}

}  // namespace sample
}  // namespace tc
