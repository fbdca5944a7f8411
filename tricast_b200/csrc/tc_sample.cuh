// The next tokens from their logits l [rows][vocab] and a random number u a row:
//   w_i = exp((l_i - max l) / T), those below 2**-126 count as 0
//   K = the top_k largest (ties to the lower index); of those, in descending order, the fewest whose weights reach
//   top_p of all of K's; of those the ones with w_i >= min_p. The token is the first i in index order at which the sum
//   of the weights that are left exceeds u times their total. T = 0: the largest logit.
// Every filter keeps a prefix of the descending order, so what is kept is a value v, all logits above it and the first m
// that equal it.
//
// A row is cut into stretches, one a block of a cluster; blocks exchange what they find through distributed shared memory. The
// value v is found without sorting: counts of the logits in an interval by bins, then the bin (top_k) or the few bins around the
// estimate (top_p, whose masses are then summed exactly) that hold it are the next interval, until one value is left.
// Counts are integers, masses are summed in fp64 in a fixed order: results do not depend on timing.
#pragma once

#include <cooperative_groups.h>

#include <cfloat>

#include "tc_serve.cuh"

namespace tc {
namespace sample {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32, kBinBits = 10, kBins = 1 << kBinBits, kChunks = 256;

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
};

// What blocks exchange at one of their meetings.
struct Found {
  double s0, s1;
  float f[4];
  int64_t n;
};

struct Shared {
  Found mine[2];  // by turns: the other one may still be read
  struct {
    double s0[kWarps], s1[kWarps];
    float f[4][kWarps];
    int64_t n[kWarps];
  } part;
  uint32_t hist[kBins];   // this block's counts
  uint32_t total[kBins];  // the cluster's
  double mass[kChunks];
  int ties[kChunks];
  int bin;
  uint32_t before;
};

// Order-preserving bits of a float that is not NaN.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = f2u(__fadd_rn(v, 0.0f));  // both zeros are equal
  return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return u2f((k >> 31) ? k & 0x7FFFFFFFu : ~k); }

// Weights. With c = log2(e) / T in two floats, y = (l - max) c is split into a whole number and a fraction f in [-1/2, 1/2] that is
// good to 2**-26; 2**f is a polynomial of degree 6 fitted to the least relative error (2e-9) by Remez's exchange. A weight
// is within 1.4 ulp, 3e-8 in the mean: tokens are compared with a 64-bit formula's, which a hardware exponential (2e-7) with a rounded
// argument (1e-6 at y = 20) would miss in one row of some thousands.
struct Weight {
  float top, ch, cl;
  __device__ __forceinline__ void set(float max_logit, float temperature) {
    const double c = 1.4426950408889634 / (double)fmaxf(temperature, 7.888609e-31f);  // 2**-100
    top = max_logit;
    ch = (float)c;
    cl = (float)(c - (double)ch);
  }
  // y = hi + lo
  __device__ __forceinline__ float argument(float l, float &lo) const {
    const float x = __fsub_rn(l, top);
    // What the subtraction lost (0 for most 16-bit logits).
    const float bv = __fsub_rn(x, l), av = __fsub_rn(x, bv);
    const float xe = __fadd_rn(__fsub_rn(-top, bv), __fsub_rn(l, av));
    const float hi = __fmul_rn(x, ch);
    lo = __fmaf_rn(x, ch, -hi);
    lo = __fmaf_rn(x, cl, lo);
    lo = __fmaf_rn(xe, ch, lo);
    return hi;
  }
  __device__ __forceinline__ float operator()(float l) const {
    float lo;
    const float hi = argument(l, lo);
    const float t = __fadd_rn(hi, 12582912.0f);
    const float f = __fadd_rn(__fsub_rn(hi, __fsub_rn(t, 12582912.0f)), lo);
    float q = 1.5345695e-4f;
    q = __fmaf_rn(q, f, 1.3400063e-3f);
    q = __fmaf_rn(q, f, 9.6184904e-3f);
    q = __fmaf_rn(q, f, 5.5503286e-2f);
    q = __fmaf_rn(q, f, 2.4022647e-1f);
    q = __fmaf_rn(q, f, 6.9314721e-1f);
    q = __fmaf_rn(q, f, 1.0f);
    const float w = u2f(f2u(q) + ((f2u(t) - 0x4B400000u) << 23));
    // -Inf has no weight at any temperature, equals of an infinite maximum have 1, and whatever is NaN here 0.
    return l == top ? 1.0f : l > -INFINITY && hi >= -126.0f ? w : 0.0f;
  }
};

// A block's stretch of a row: n logits from `first` on.
template <typename T>
struct Stretch {
  const T *p;
  int64_t first, n;
  __device__ __forceinline__ float operator[](int64_t i) const { return Io<T>::get(p[i]); }
};

struct Bins {  // of the interval [lo, hi], the largest values in bin 0
  float lo, hi, scale, half;
  uint32_t khi;
  int shift;  // < 0: by values, else by bits
  __device__ __forceinline__ void by_value(float l, float h) {
    lo = l, hi = h, shift = -1;
    half = h - l > FLT_MAX ? 0.5f : 1.0f;
    const float d = h * half - l * half;
    scale = d > 0.0f ? fminf((float)kBins / d, FLT_MAX) : 0.0f;
  }
  __device__ __forceinline__ void by_bits(float l, float h) {
    lo = l, hi = h, khi = key_of(h), half = 1.0f, scale = 0.0f;
    const uint32_t range = khi - key_of(l);
    shift = max(0, 32 - __clz(range) - kBinBits);
  }
  __device__ __forceinline__ bool has(float v) const { return v >= lo && v <= hi; }
  __device__ __forceinline__ int operator()(float v) const {
    if (shift >= 0) return min((int)((khi - key_of(v)) >> shift), kBins - 1);
    return (int)fminf((hi * half - v * half) * scale, (float)(kBins - 1));
  }
  // The bin of the interval's least value.
  __device__ __forceinline__ int last() const { return (*this)(lo); }
  // A value near the middle of a bin, for estimates.
  __device__ __forceinline__ float middle(int b) const {
    if (shift >= 0) return of_key(khi - min(khi - key_of(lo), ((uint32_t)b << shift) + ((1u << shift) >> 1)));
    return scale > 0.0f ? fmaxf(lo, (hi * half - ((float)b + 0.5f) / scale) / half) : hi;
  }
};

template <typename T>
struct Row {
  Stretch<T> z;
  Weight w;
  Shared *sh;
  cg::cluster_group cluster;
  int turn;

  __device__ __forceinline__ Row(const Stretch<T> &s, Shared *shared) : z(s), sh(shared), cluster(cg::this_cluster()), turn(0) {}

  // Sums of s0, s1 and n, minima of f[0], f[1] and maxima of f[2], f[3] over the cluster's threads, in a fixed order;
  // before: s0 and n of the blocks before this one.
  __device__ Found meet(Found v, Found *before = nullptr) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto add = [](Found &a, const Found &b) {
      a.s0 += b.s0, a.s1 += b.s1, a.n += b.n;
      a.f[0] = fminf(a.f[0], b.f[0]), a.f[1] = fminf(a.f[1], b.f[1]);
      a.f[2] = fmaxf(a.f[2], b.f[2]), a.f[3] = fmaxf(a.f[3], b.f[3]);
    };
#pragma unroll
    for (int m = 16; m; m >>= 1) {
      Found o;
      o.s0 = __shfl_xor_sync(0xFFFFFFFFu, v.s0, m), o.s1 = __shfl_xor_sync(0xFFFFFFFFu, v.s1, m);
      o.n = __shfl_xor_sync(0xFFFFFFFFu, v.n, m);
#pragma unroll
      for (int k = 0; k < 4; ++k) o.f[k] = __shfl_xor_sync(0xFFFFFFFFu, v.f[k], m);
      add(v, o);
    }
    __syncthreads();  // the buffers of an earlier use are read
    if (lane == 0) {
      sh->part.s0[warp] = v.s0, sh->part.s1[warp] = v.s1, sh->part.n[warp] = v.n;
#pragma unroll
      for (int k = 0; k < 4; ++k) sh->part.f[k][warp] = v.f[k];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < kWarps; ++i) {
        Found o{sh->part.s0[i], sh->part.s1[i], {sh->part.f[0][i], sh->part.f[1][i], sh->part.f[2][i], sh->part.f[3][i]}, sh->part.n[i]};
        add(v, o);
      }
      sh->mine[turn] = v;
    }
    cluster.sync();
    const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    Found all = *cluster.map_shared_rank(&sh->mine[turn], 0);
    if (before) *before = Found{0.0, 0.0, {}, 0};
    if (before && rank > 0) *before = all;
    for (int i = 1; i < blocks; ++i) {
      add(all, *cluster.map_shared_rank(&sh->mine[turn], i));
      if (before && i + 1 <= rank) *before = all;
    }
    turn ^= 1;
    return all;
  }
  static __device__ __forceinline__ Found nothing() {
    return Found{0.0, 0.0, {INFINITY, INFINITY, -INFINITY, -INFINITY}, 0};
  }

  // Counts of the interval's logits by bins, of the whole cluster, in sh->total.
  __device__ void count(const Bins &bins) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh->hist[i] = 0u;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < z.n; i += kThreads) {
      const float v = z[i];
      if (bins.has(v)) atomicAdd(&sh->hist[bins(v)], 1u);
    }
    cluster.sync();
    const int blocks = (int)cluster.num_blocks();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      uint32_t n = 0;
      for (int b = 0; b < blocks; ++b) n += *cluster.map_shared_rank(&sh->hist[i], b);
      sh->total[i] = n;
    }
    cluster.sync();  // before anyone clears the counts again
  }

  // v and m such that the logits above v and the first m that equal it are the `want` largest of those from `least` on; false
  // where there are not more than that many.
  __device__ bool largest(int64_t want, float least, float &value, int64_t &m) {
    Bins bins;
    bins.by_value(least, w.top);
    int64_t above = 0;
    for (;;) {
      count(bins);
      if (threadIdx.x == 0) {
        int64_t sum = above;
        int b = 0;
        for (; b < kBins; ++b) {
          if (sum + sh->total[b] >= want) break;
          sum += sh->total[b];
        }
        sh->bin = b;
        sh->before = (uint32_t)(sum - above);
      }
      __syncthreads();
      const int b = sh->bin;
      above += sh->before;
      if (b == kBins) return false;
      Found f = nothing();
      for (int64_t i = threadIdx.x; i < z.n; i += kThreads) {
        const float v = z[i];
        if (bins.has(v) && bins(v) == b) f.f[0] = fminf(f.f[0], v), f.f[2] = fmaxf(f.f[2], v);
      }
      f = meet(f);
      if (f.f[0] == f.f[2]) {
        value = f.f[0];
        m = want - above;
        return true;
      }
      bins.by_bits(f.f[0], f.f[2]);
    }
  }

  // Sum of the weights above a value; n: logits that equal it.
  __device__ Found above(float value) {
    Found f = nothing();
    for (int64_t i = threadIdx.x; i < z.n; i += kThreads) {
      const float v = z[i];
      if (v > value) f.s0 += (double)w(v);
      f.n += v == value;
    }
    return meet(f);
  }

  // v and m such that the logits above v and the first m that equal it are the fewest whose weights reach `target`, which
  // those from `least` on do.
  __device__ void heaviest(double target, float least, float &value, int64_t &m) {
    Bins bins;
    bins.by_value(least, w.top);
    double over = 0.0;  // the weights above the interval
    // Rounds end: bins by bits put the interval's ends into different bins, of which no part below holds both; from the fourth
    // round on the interval is halved, so 32 more are the most.
    for (int round = 0;; ++round) {
      count(bins);
      // The bin that the target should fall in.
      if (threadIdx.x == 0) {
        double sum = over;
        int b = 0, last = 0;
        for (; b < kBins; ++b) {
          if (!sh->total[b]) continue;
          last = b;
          sum += (double)sh->total[b] * (double)w(bins.middle(b));
          if (sum >= target) break;
        }
        sh->bin = round >= 4 ? bins.last() / 2 : b < kBins ? b : last;
      }
      __syncthreads();
      const int side = round < 4 && bins.last() > 2;  // bins beside the estimate that still count as it
      const int lo = sh->bin - side, hi = sh->bin + side;
      double s0 = 0.0, s1 = 0.0;
      float lo0 = INFINITY, lo1 = INFINITY, lo2 = INFINITY, hi0 = -INFINITY, hi1 = -INFINITY, hi2 = -INFINITY;
      int64_t n0 = 0, n1 = 0, n2 = 0;
      for (int64_t i = threadIdx.x; i < z.n; i += kThreads) {
        const float v = z[i];
        if (!bins.has(v)) continue;
        const int b = bins(v);
        if (b < lo) s0 += (double)w(v), lo0 = fminf(lo0, v), hi0 = fmaxf(hi0, v), ++n0;
        else if (b <= hi) s1 += (double)w(v), lo1 = fminf(lo1, v), hi1 = fmaxf(hi1, v), ++n1;
        else lo2 = fminf(lo2, v), hi2 = fmaxf(hi2, v), ++n2;
      }
      const Found x = meet(Found{s0, s1, {lo0, lo1, hi0, hi1}, n0 + (n1 << 32)});
      const Found y = meet(Found{0.0, 0.0, {lo2, INFINITY, hi2, -INFINITY}, n2});
      const int64_t c0 = x.n & 0xFFFFFFFFll, c1 = x.n >> 32, c2 = y.n;
      float from, to;
      int64_t c;
      // The sums' last bits may leave the target behind all of them: the last part that has logits takes it.
      if (c0 && (over + x.s0 >= target || !(c1 + c2))) from = x.f[0], to = x.f[2], c = c0;
      else if (c1 && (over + x.s0 + x.s1 >= target || !c2)) over += x.s0, from = x.f[1], to = x.f[3], c = c1;
      else over += x.s0 + x.s1, from = y.f[0], to = y.f[2], c = c2;
      if (from == to) {
        const double need = ceil((target - over) / (double)w(from));
        value = from;
        m = need < 1.0 ? 1 : need < (double)c ? (int64_t)need : c;
        return;
      }
      bins.by_bits(from, to);
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(Args a) {
  __shared__ Shared shared;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), blocks = (int)cluster.num_blocks();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r = blockIdx.x / blocks;
  const int64_t part = (a.vocab + blocks - 1) / blocks, first = min(part * rank, a.vocab);
  Stretch<T> z{static_cast<const T *>(a.logits) + r * a.stride + first, first, min(part, a.vocab - first)};
  Row<T> row(z, &shared);
  Found f = Row<T>::nothing();
  for (int64_t i = threadIdx.x; i < z.n; i += kThreads) {
    const float v = z[i];
    f.f[2] = fmaxf(f.f[2], v);
    f.n += v != v;
  }
  f = row.meet(f);
  const float top = f.f[2];
  const float heat = a.temperature ? a.temperature[r] : a.all_temperature;
  auto answer = [&](int64_t token, float logprob) {
    a.tokens[r] = token;
    if (a.logprobs) a.logprobs[r] = logprob;
  };
  if (f.n || top == -INFINITY) {
    if (rank == 0 && threadIdx.x == 0) answer(-1, f.n ? u2f(kQNaN) : -INFINITY);
  } else if (!(heat > 0.0f)) {
    Found g = Row<T>::nothing();
    int64_t at = INT64_MAX;
    for (int64_t i = threadIdx.x; i < z.n && at == INT64_MAX; i += kThreads)
      if (z[i] == top) at = first + i;
    // An index as two floats that order like it: whole parts of 2**20.
    if (at != INT64_MAX) g.f[0] = (float)(at >> 20);
    g = row.meet(g);
    Found h = Row<T>::nothing();
    if (at != INT64_MAX && (float)(at >> 20) == g.f[0]) h.f[0] = (float)(at & 0xFFFFF);
    h = row.meet(h);
    if (rank == 0 && threadIdx.x == 0) answer(((int64_t)g.f[0] << 20) + (int64_t)h.f[0], 0.0f);
  } else {
    row.w.set(top, heat);
    const int64_t k = a.top_k ? a.top_k[r] : a.all_top_k;
    const float p = a.top_p ? a.top_p[r] : a.all_top_p, low = a.min_p ? a.min_p[r] : a.all_min_p;
    const float least_weight = low > 1.0f ? 1.0f : low;  // NaN bounds nothing
    // Everything that has a weight lies above this (88 > 126 log 2).
    const double reach = (double)top - 88.0 * (double)fmaxf(heat, 7.888609e-31f);
    const float least = top == INFINITY ? top : reach > -FLT_MAX ? (float)reach : -FLT_MAX;
    float value = -INFINITY;
    int64_t m = 0;
    if (k > 0 && k < a.vocab) row.largest(k, least, value, m);
    if (p < 1.0f) {
      const Found g = row.above(value);
      const double mass = g.s0 + (m ? (double)m * (double)row.w(value) : 0.0);
      float v;
      int64_t n;
      row.heaviest((double)p * mass, fmaxf(least, value), v, n);
      m = v == value && m ? min(m, n) : n;
      value = v;
    }
    if (m && row.w(value) < least_weight) m = 0;
    auto weight = [&](float v) {
      const float u = v > value ? row.w(v) : 0.0f;
      return u < least_weight ? 0.0f : u;
    };
    // Weights and ties by chunks of consecutive logits, a warp a chunk.
    const int64_t span = ((z.n + kChunks - 1) / kChunks + 31) / 32 * 32;
    const double tie = m ? (double)row.w(value) : 0.0;
    Found g = Row<T>::nothing();
    for (int c = warp; c < kChunks; c += kWarps) {
      double s = 0.0;
      int n = 0;
      for (int64_t i = c * span + lane; i < min((c + 1) * span, z.n); i += 32) {
        const float v = z[i];
        s += (double)weight(v);
        n += m && v == value;
      }
#pragma unroll
      for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, x), n += __shfl_xor_sync(0xFFFFFFFFu, n, x);
      if (lane == 0) {
        shared.mass[c] = s, shared.ties[c] = n;
        g.n += n;
      }
    }
    Found before;
    row.meet(g, &before);
    const int64_t quota = max(m - before.n, (int64_t)0);  // ties that this block may keep
    double own = 0.0;
    if (threadIdx.x == 0) {
      int64_t left = quota;
      for (int c = 0; c < kChunks; ++c) {
        const int64_t n = min((int64_t)shared.ties[c], left);
        left -= n;
        own += shared.mass[c] += (double)n * tie;
      }
    }
    Found mass = Row<T>::nothing();
    mass.s0 = own;
    mass = row.meet(mass, &before);
    const double total = mass.s0, aim = fmax((double)a.uniform[r] * total, 0.0);
    // The block whose stretch the aim falls in; behind all of them (u = 1, or the last bits of the sums) the last one that
    // keeps anything.
    Found last = Row<T>::nothing();
    if (own > 0.0) last.f[2] = (float)rank;
    last = row.meet(last);
    if (threadIdx.x == 0)
      shared.bin = own > 0.0 && before.s0 <= aim && (before.s0 + own > aim || (float)rank == last.f[2]);
    __syncthreads();
    if (shared.bin && warp == 0) {
      // Its chunk, likewise.
      double rest = aim - before.s0;
      int chunk = -1;
      int64_t left = quota, chunk_left = 0;
      double chunk_rest = 0.0;
      for (int c = 0; c < kChunks; ++c) {
        const double s = shared.mass[c];
        if (s > 0.0) chunk = c, chunk_left = left, chunk_rest = rest;
        if (s > rest) break;
        rest -= s;
        left -= min((int64_t)shared.ties[c], left);
      }
      // Its logits, 32 at a time.
      int64_t found = -1, kept = -1;
      for (int64_t i0 = chunk * span; found < 0 && i0 < min((chunk + 1) * span, z.n); i0 += 32) {
        const int64_t i = i0 + lane;
        const bool real = i < min((chunk + 1) * span, z.n);
        const float v = real ? z[i] : -INFINITY;
        double s = (double)weight(v);
        const unsigned equal = __ballot_sync(0xFFFFFFFFu, real && m && v == value);
        if ((equal >> lane & 1u) && __popc(equal & ((1u << lane) - 1u)) < chunk_left) s = tie;
        chunk_left -= min((int64_t)__popc(equal), chunk_left);
        const unsigned some = __ballot_sync(0xFFFFFFFFu, s > 0.0);
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const double o = __shfl_up_sync(0xFFFFFFFFu, s, x);
          if (lane >= x) s += o;
        }
        const unsigned hit = __ballot_sync(0xFFFFFFFFu, s > chunk_rest) & some;
        if (some) kept = i0 + 31 - __clz(some);
        if (hit) found = i0 + __ffs(hit) - 1;
        chunk_rest -= __shfl_sync(0xFFFFFFFFu, s, 31);
      }
      if (found < 0) found = kept;
      if (lane == 0) {
        float lo;
        const float hi = row.w.argument(z[found], lo);
        const double x = z[found] == top ? 0.0 : ((double)hi + (double)lo) * 0.6931471805599453;
        answer(first + found, (float)(x - log(total)));
      }
    }
  }
  cluster.sync();  // the other blocks may still read this one's findings
}

}  // namespace sample
}  // namespace tc
