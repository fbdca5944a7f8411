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
// in two 32-bit words; totals are fp64 sums in a fixed order. Nothing depends on timing.
#pragma once

#include <cooperative_groups.h>

#include <cfloat>

#include "tc_mma16.cuh"
#include "tc_serve.cuh"

namespace tc {
namespace sample {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 512, kChunks = 256, kMaxBlocks = 16;
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
  int64_t part;   // positions of a block's stretch, a multiple of 8
};

struct Shared {
  uint32_t hist[2][2][kBins];         // by turns (others may still read the last one): lower and upper parts, or counts
  double slots[2][kMaxBlocks];        // by turns: what each block of the cluster has sent
  double part[kWarps];
  double mass[kChunks];
  int ties[kChunks];
  double found[3];                    // of a histogram's scan
  int bin;
};

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
  // log(w), in fp64.
  __device__ __forceinline__ double log(float l) const { return ((double)l - top) * c * 0.6931471805599453; }
};

// A block's stretch of a row. Positions count from a 16-byte boundary at or before the row's begin (`skip` elements before it), so that
// vectors are aligned for every row; positions outside the row read as -Inf.
template <typename T>
struct Stretch {
  const T *base;  // position 0
  int64_t lo, hi;        // this block's positions
  int64_t first, end;    // the row's
  static constexpr int kVec = 16 / sizeof(T);
  // kVec logits from position lo + i.
  __device__ __forceinline__ void load(int64_t i, float (&v)[kVec]) const {
    const int64_t p = lo + i;
    if (p >= first && p + kVec <= end) {
      const uint4 w = *reinterpret_cast<const uint4 *>(base + p);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) {
          v[k] = u2f(u[k]);
        } else if constexpr (Same<T, __nv_bfloat16>::value) {
          v[2 * k] = u2f(u[k] << 16), v[2 * k + 1] = u2f(u[k] & 0xFFFF0000u);
        } else {
          v[2 * k] = __half2float(__ushort_as_half((unsigned short)(u[k] & 0xFFFFu)));
          v[2 * k + 1] = __half2float(__ushort_as_half((unsigned short)(u[k] >> 16)));
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < kVec; ++k) v[k] = p + k >= first && p + k < end ? Io<T>::get(base[p + k]) : -INFINITY;
    }
  }
  __device__ __forceinline__ float at(int64_t i) const { return Io<T>::get(base[lo + i]); }
};

// HELD: weights stand in shared memory; otherwise (rows beyond what a cluster holds) they are computed again by every pass.
template <typename T, bool HELD>
struct Row {
  Stretch<T> z;
  Weight w;
  Shared &sh;
  float *held;
  int64_t n;      // positions, a multiple of 8
  int blocks, rank, turn, hist_turn;
  bool infinite;  // the row's largest logit is: its equals share everything, as logits of 0 beside -Inf
  cg::cluster_group cluster;

  __device__ __forceinline__ Row(Shared &s, float *h) : sh(s), held(h), turn(0), hist_turn(0), infinite(false), cluster(cg::this_cluster()) {}

  // f(position, four weights) for the block's positions.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if (HELD) {
      for (int i = threadIdx.x * 4; i < (int)n; i += kThreads * 4) f((int64_t)i, *reinterpret_cast<const float4 *>(held + i));
    } else {
      for (int64_t i = (int64_t)threadIdx.x * 8; i < n; i += kThreads * 8) {
        float4 a, b;
        weights8(i, a, b);
        f(i, a);
        f(i + 4, b);
      }
    }
  }
  __device__ __forceinline__ void logits8(int64_t i, float (&v)[8]) const {
    constexpr int kVec = Stretch<T>::kVec;
#pragma unroll
    for (int k = 0; k < 8; k += kVec) {
      float x[kVec];
      z.load(i + k, x);
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[k + e] = x[e];
    }
  }
  static __device__ __forceinline__ void finite8(float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = v[k] == INFINITY ? 0.0f : -INFINITY;
  }
  __device__ __forceinline__ void weights8(int64_t i, float4 &a, float4 &b) const {
    float v[8];
    logits8(i, v);
    if (infinite) finite8(v);
    a = make_float4(w(v[0]), w(v[1]), w(v[2]), w(v[3]));
    b = make_float4(w(v[4]), w(v[5]), w(v[6]), w(v[7]));
  }
  __device__ __forceinline__ float4 four(int64_t i) const {
    if (HELD) return *reinterpret_cast<const float4 *>(held + i);
    float4 a, b;
    weights8(i & ~(int64_t)7, a, b);
    return (i & 4) ? b : a;
  }

  // A number from each block, to all of them: slots() after it. Two meetings apart the slots are used again, and between
  // them lies a barrier that a block reaches only after reading.
  __device__ __forceinline__ const double *tell(double v) {
    double *to = sh.slots[turn];
    if ((int)threadIdx.x < blocks) cluster.map_shared_rank(to, threadIdx.x)[rank] = v;
    cluster.sync();
    turn ^= 1;
    return to;
  }
  // Sum over the block's threads, in every one of them.
  __device__ __forceinline__ double block_sum(double v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) v += sh.part[i];
    return v;
  }
  __device__ __forceinline__ double cluster_sum(double v) {
    const double *all = tell(block_sum(v));
    v = 0.0;
    for (int i = 0; i < blocks; ++i) v += all[i];
    return v;
  }
  __device__ __forceinline__ double cluster_max(double v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v = fmax(v, __shfl_xor_sync(0xFFFFFFFFu, v, m));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh.part[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) v = fmax(v, sh.part[i]);
    const double *all = tell(v);
    v = all[0];
    for (int i = 1; i < blocks; ++i) v = fmax(v, all[i]);
    return v;
  }

  __device__ __forceinline__ void clear() {
    sh.hist[hist_turn][0][threadIdx.x] = 0u;
    sh.hist[hist_turn][1][threadIdx.x] = 0u;
    __syncthreads();
  }
  // Adds a weight's bits to its bin: its count, or its 24-bit significand in parts of 12 bits (a stretch has at most 2**20
  // positions, so neither sum passes 32 bits).
  template <bool MASS>
  __device__ __forceinline__ void add(int bin, uint32_t u) {
    uint32_t (*h)[kBins] = sh.hist[hist_turn];
    if (MASS) {
      atomicAdd(&h[0][bin], u & 0xFFFu);
      atomicAdd(&h[1][bin], ((u >> 12) & 0x7FFu) | 0x800u);
    } else {
      atomicAdd(&h[0][bin], 1u);
    }
  }
  // The first bin at which counts or masses of the cluster, on top of `over`, reach `want`, kBins where none does (then, with
  // `last`, the last one that is not empty). over: what is before it. c: its own count; exponent(bin): of the bin's weights.
  template <bool MASS, typename X>
  __device__ __forceinline__ int reach(double want, double &over, double &own, bool last, X exponent) {
    cluster.sync();
    const int bin = threadIdx.x, lane = bin & 31, warp = bin >> 5;
    double v = 0.0;
    {
      uint64_t lo = 0, hi = 0;
      for (int b = 0; b < blocks; ++b) {
        lo += *cluster.map_shared_rank(&sh.hist[hist_turn][0][bin], b);
        if (MASS) hi += *cluster.map_shared_rank(&sh.hist[hist_turn][1][bin], b);
      }
      v = (double)(lo + (hi << 12));
      if (MASS) v = scalbn(v, exponent(bin) - 23);
    }
    hist_turn ^= 1;
    double s = v;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const double o = __shfl_up_sync(0xFFFFFFFFu, s, m);
      if (lane >= m) s += o;
    }
    if (lane == 31) sh.part[warp] = s;
    if (bin == 0) sh.bin = kBins;
    __syncthreads();
    double base = over;
    for (int i = 0; i < warp; ++i) base += sh.part[i];
    double all = base;
    for (int i = warp; i < kWarps; ++i) all += sh.part[i];
    if (v > 0.0 && base + s >= want) atomicMin(&sh.bin, bin);
    __syncthreads();
    if (last && sh.bin == kBins) {  // the sums' last bits
      __syncthreads();
      if (bin == 0) sh.bin = -1;
      __syncthreads();
      if (v > 0.0) atomicMax(&sh.bin, bin);
      __syncthreads();
    }
    const int b = sh.bin;
    if (bin == b) sh.found[0] = base + (s - v), sh.found[1] = v;
    if (bin == 0) sh.found[2] = all;
    __syncthreads();
    over = b < kBins ? sh.found[0] : sh.found[2];
    own = b < kBins ? sh.found[1] : 0.0;
    return b;
  }

  // Bins of 32 an octave below 1: weights of one bin share their exponent.
  static constexpr uint32_t kTop = 0x3F800000u >> 18;
  static constexpr int kWindows = (int)(kTop + kBins - 1 - (0x00800000u >> 18)) / kBins + 1;
  static __device__ __forceinline__ int bin_of(uint32_t u, int window) { return (int)(kTop - (u >> 18)) - window * kBins; }

  template <bool MASS>
  __device__ __forceinline__ void fill(int window, uint32_t from) {
    clear();
    each([&](int64_t, float4 q) {
      const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t u = f2u(v[k]);
        const int b = bin_of(u, window);
        if (b >= 0 && b < kBins && u >= from) add<MASS>(b, u);
      }
    });
  }

  // The weight (its bits) at which counts or masses in descending order reach `want`; over: those above it, equals: how many
  // have it. Weights below `from` do not count. false where all of them stay below. The first window's histogram is
  // there already where `filled`.
  template <bool MASS>
  __device__ bool cut(double want, uint32_t from, bool filled, uint32_t &weight, double &over, double &equals) {
    over = 0.0;
    double own;
    int window = 0, b = kBins;
    for (; window < kWindows; ++window) {
      if (window || !filled) fill<MASS>(window, from);
      b = reach<MASS>(want, over, own, false, [&](int bin) { return (int)((kTop - bin - window * kBins) >> 5) - 127; });
      if (b < kBins) break;
    }
    if (b == kBins) return false;
    uint32_t high = kTop - (uint32_t)(b + window * kBins);
    const int exponent = (int)(high >> 5) - 127;
#pragma unroll 1
    for (int shift = 9; shift >= 0; shift -= 9) {
      clear();
      each([&](int64_t, float4 q) {
        const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t u = f2u(v[k]);
          if (u >> (shift + 9) == high && u >= from) add<MASS>(kBins - 1 - (int)((u >> shift) & (kBins - 1)), u);
        }
      });
      b = reach<MASS>(want, over, own, true, [&](int) { return exponent; });
      high = (high << 9) | (uint32_t)(kBins - 1 - b);
    }
    weight = high;
    equals = MASS ? rint(own / (double)u2f(high)) : own;
    return true;
  }

  // Of the `equals` tokens of a weight the first `want` are kept, larger logits first: the logit at which they end, and
  // how many of that logit's tokens stay.
  __device__ void cut_logits(uint32_t weight, int64_t want, float &logit, int64_t &quota) {
    double over = 0.0, own = 0.0;
    uint32_t high = 0;
#pragma unroll 1
    for (int shift = 27; shift >= 0; shift -= 9) {  // 5, 9, 9 and 9 bits
      clear();
      each([&](int64_t i, float4 q) {
        const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (f2u(v[k]) == weight) {
            const uint32_t key = key_of(z.at(i + k));
            if (shift == 27 || key >> (shift + 9) == high) add<false>(kBins - 1 - (int)((key >> shift) & (kBins - 1)), 0u);
          }
      });
      const int b = reach<false>((double)want, over, own, true, [](int) { return 0; });
      high = (high << 9) | (uint32_t)(kBins - 1 - b);
    }
    logit = u2f((high >> 31) ? high & 0x7FFFFFFFu : ~high);
    quota = want - (int64_t)over;
  }

  __device__ __forceinline__ double mass_above(uint32_t weight) {
    double s = 0.0;
    each([&](int64_t, float4 q) {
      const float v[4] = {q.x, q.y, q.z, q.w};
      float t = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) t = __fadd_rn(t, f2u(v[k]) > weight ? v[k] : 0.0f);
      s += (double)t;
    });
    return cluster_sum(s);
  }
};

template <typename T, bool HELD>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(Args a) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  __shared__ Shared shared;
  Row<T, HELD> row(shared, reinterpret_cast<float *>(dynamic));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = row.blocks = a.blocks, rank = row.rank = (int)row.cluster.block_rank();
  const int64_t r = blockIdx.x / blocks;
  {
    const T *p = static_cast<const T *>(a.logits) + r * a.stride;
    const int64_t skip = (int64_t)((uintptr_t)p % 16 / sizeof(T));
    row.z.base = p - skip;
    row.z.first = skip, row.z.end = skip + a.vocab;
    row.z.lo = min(a.part * rank, (row.z.end + 7) / 8 * 8);
    row.z.hi = min(row.z.lo + a.part, (row.z.end + 7) / 8 * 8);
    row.n = row.z.hi - row.z.lo;
  }
  const Stretch<T> &z = row.z;
  const int64_t n = row.n;
  float *held = row.held;
  const int64_t origin = z.lo - z.first;  // of position i the token is origin + i

  // The logits, once, and the largest.
  float top = -INFINITY;
  for (int64_t i = (int64_t)threadIdx.x * 8; i < n; i += kThreads * 8) {
    float v[8];
    row.logits8(i, v);
    if (HELD) {
      *reinterpret_cast<float4 *>(held + i) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4 *>(held + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max_nan(top, v[k]);
  }
  {
    // NaN above Inf above every number.
    const double t = row.cluster_max(top != top ? DBL_MAX : top == INFINITY ? (double)FLT_MAX * 2.0 : top == -INFINITY ? -DBL_MAX : (double)top);
    top = t == DBL_MAX ? u2f(kQNaN) : t > (double)FLT_MAX ? INFINITY : t == -DBL_MAX ? -INFINITY : (float)t;
  }
  const float heat = a.temperature ? a.temperature[r] : a.all_temperature;
  auto answer = [&](int64_t token, float logprob) {
    a.tokens[r] = token;
    if (a.logprobs) a.logprobs[r] = logprob;
  };
  if (!(top > -INFINITY)) {
    if (rank == 0 && threadIdx.x == 0) answer(-1, top);
  } else if (!(heat > 0.0f)) {
    double at = -DBL_MAX;  // the negated first index
    for (int64_t i = (int64_t)threadIdx.x * 8; i < n && at == -DBL_MAX; i += kThreads * 8) {
      float v[8];
      if (HELD) {
        const float4 x = *reinterpret_cast<const float4 *>(held + i), y = *reinterpret_cast<const float4 *>(held + i + 4);
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
      } else {
        row.logits8(i, v);
      }
#pragma unroll
      for (int k = 7; k >= 0; --k)
        if (v[k] == top) at = -(double)(origin + i + k);
    }
    at = row.cluster_max(at);
    if (rank == 0 && threadIdx.x == 0) answer((int64_t)-at, 0.0f);
  } else {
    row.infinite = top == INFINITY;
    row.w.set(row.infinite ? 0.0f : top, heat);
    const Weight w = row.w;
    if (HELD && row.infinite)
      for (int64_t i = threadIdx.x * 4; i < n; i += kThreads * 4)
        for (int64_t e = i; e < i + 4; ++e) held[e] = held[e] == INFINITY ? 0.0f : -INFINITY;
    const int64_t k = a.top_k ? a.top_k[r] : a.all_top_k;
    const float p = a.top_p ? a.top_p[r] : a.all_top_p, low = a.min_p ? a.min_p[r] : a.all_min_p;
    const bool by_count = k > 0 && k < a.vocab, by_mass = p < 1.0f;
    // Weights in the logits' place, their sum, and the histogram that the first filter begins with.
    row.clear();
    double sum = 0.0;
    for (int64_t i = (int64_t)threadIdx.x * 4; i < n; i += kThreads * 4) {
      float4 q;
      if (HELD) {
        q = *reinterpret_cast<const float4 *>(held + i);
        q = make_float4(w(q.x), w(q.y), w(q.z), w(q.w));
        *reinterpret_cast<float4 *>(held + i) = q;
      } else {
        q = row.four(i);
      }
      sum += (double)__fadd_rn(__fadd_rn(q.x, q.y), __fadd_rn(q.z, q.w));
      if (by_count || by_mass) {
        const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t u = f2u(v[e]);
          const int b = Row<T, HELD>::bin_of(u, 0);
          if (b < kBins) by_count ? row.template add<false>(b, u) : row.template add<true>(b, u);
        }
      }
    }
    // Kept: weights above `cut`, and of the tokens at it the first m.
    uint32_t cut = 0;
    double m = 0.0, equals = 0.0, over;
    if (by_count && row.template cut<false>((double)k, 1u, true, cut, over, equals)) m = (double)k - over;
    if (by_mass) {
      if (!by_count) sum = row.cluster_sum(sum);
      else sum = row.mass_above(cut) + m * (double)u2f(cut);
      uint32_t c;
      double e;
      if (row.template cut<true>((double)p * sum, max(cut, 1u), !by_count, c, over, e)) {
        const double need = fmin(fmax(ceil(((double)p * sum - over) / (double)u2f(c)), 1.0), e);
        m = c == cut ? fmin(need, m) : need;
        cut = c, equals = e;
      }
    }
    const float bound = low > 1.0f ? 1.0f : low;  // NaN bounds nothing
    if (m > 0.0 && (u2f(cut) < bound || m == equals)) {  // none or all of the equals
      if (!(u2f(cut) < bound)) cut -= 1;
      m = 0.0;
    }
    if (bound > u2f(cut)) cut = max(cut, f2u(bound) - 1);
    // Some of the equals: the logit at which they end.
    const bool some = m > 0.0;
    float tie = 0.0f;
    int64_t quota = 0;
    if (some) row.cut_logits(cut, (int64_t)m, tie, quota);
    auto equal = [&](int64_t i, float v, bool &above) {  // the tie's own, or one whose logit is above it
      if (f2u(v) != cut) return false;
      const float l = z.at(i);
      above = l > tie;
      return l == tie;
    };

    // Masses and ties by chunks of consecutive positions, a warp a chunk.
    const int64_t span = ((n + kChunks - 1) / kChunks + 127) / 128 * 128;
    double ties = 0.0;
    for (int c = warp; c < kChunks; c += kWarps) {
      double s = 0.0;
      int e = 0;
      for (int64_t i = c * span + lane * 4; i < min((c + 1) * span, n); i += 128) {
        const float4 q = row.four(i);
        const float v[4] = {q.x, q.y, q.z, q.w};
        float t = 0.0f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          bool keep = f2u(v[x]) > cut;
          if (some && !keep) e += equal(i + x, v[x], keep);
          t = __fadd_rn(t, keep ? v[x] : 0.0f);
        }
        s += (double)t;
      }
#pragma unroll
      for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
      if (some) e = (int)__reduce_add_sync(0xFFFFFFFFu, e);
      if (lane == 0) shared.mass[c] = s, shared.ties[c] = e, ties += e;
    }
    int64_t left = 0;  // ties that this block may keep
    if (some) {
      const double *all = row.tell(row.block_sum(ties));
      left = quota;
      for (int i = 0; i < rank; ++i) left -= (int64_t)all[i];
      left = max(left, (int64_t)0);
    }
    __syncthreads();
    // Chunks in order, eight a lane of the first warp: ties that are left, and the mass before each.
    constexpr int kLane = kChunks / 32;
    double own = 0.0, before = 0.0;
    if (warp == 0) {
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
        own += shared.mass[lane * kLane + c];
      }
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
    const double *all = row.tell(shared.found[0]);
    // The block whose stretch the aim falls in; behind all of them (u = 1, or the last bits of the sums) the last one that
    // keeps anything.
    double total = 0.0;
    for (int i = 0; i < blocks; ++i) total += all[i];
    const double aim = fmax((double)a.uniform[r] * total, 0.0);
    int owner = -1;
    double start = 0.0, at = 0.0;
    for (int i = 0; i < blocks; ++i) {
      if (all[i] > 0.0) owner = i, start = at;
      at += all[i];
      if (all[i] > 0.0 && at > aim) break;
    }
    if (rank == owner && warp == 0) {
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
      int64_t room = shared.ties[chunk], found = -1, kept = -1;
      // Its tokens, 32 at a time.
      for (int64_t i0 = chunk * span; found < 0 && i0 < min((chunk + 1) * span, n); i0 += 32) {
        const int64_t i = i0 + lane;
        const bool real = i < n;
        float4 q = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (real) q = row.four(i & ~(int64_t)3);
        const float v = real ? ((i & 2) ? ((i & 1) ? q.w : q.z) : (i & 1) ? q.y : q.x) : 0.0f;
        bool keep = f2u(v) > cut, mine = false;
        if (some && !keep) mine = equal(i, v, keep);
        const unsigned same = __ballot_sync(0xFFFFFFFFu, mine);
        if (mine) keep = __popc(same & ((1u << lane) - 1u)) < room;
        room = max(room - __popc(same), (int64_t)0);
        const unsigned mask = __ballot_sync(0xFFFFFFFFu, keep);
        double x = keep ? (double)v : 0.0;
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
      if (lane == 0) answer(origin + found, (float)((row.infinite ? 0.0 : w.log(z.at(found))) - log(total)));
    }
  }
  row.cluster.sync();  // the other blocks may still read this one's shared memory
}

}  // namespace sample
}  // namespace tc
