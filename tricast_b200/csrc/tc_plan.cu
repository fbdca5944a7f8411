// Page plans of a batch: which pages its new tokens take, the slot, sequence and position of every one, and the
// pages of ended sequences back on the stack of free ones.
//   used_i = ceil(len_i / P), n_i = the new tokens that fit, need_i = min(ceil((len_i + n_i) / P), max_pages) - used_i
//   page (i, used_i + j) = free[taken + need_0 + .. + need_(i-1) + j],   slot = page * P + position % P
// All of it is latency: 64 sequences with a token each 3 us, 157 with 33001 tokens 4.8 us, 2048 whose pages go back before 131072
// tokens take them 16 us (four kernels).
#include <string>

#include "tc_common.cuh"

namespace tc {
namespace plan {

constexpr int kThreads = 1024;

struct Args {
  const int32_t *lens, *fresh;  // tokens that a sequence has, and new ones
  int32_t *table;
  int64_t table_stride;
  const int32_t *free_pages;
  int64_t num_free;
  const int32_t *taken;
  int64_t tokens;
  int32_t batch, width, shift;  // rows and columns of the table, logarithm of the page size
  int32_t *out_lens, *cu, *sequence, *positions, *out_taken, *missing;
  int64_t *slots;
  int64_t *first;  // workspace: of each sequence, where its first new page stands in free_pages
};

__device__ __forceinline__ int64_t warp_prefix(int64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int64_t o = __shfl_up_sync(0xFFFFFFFFu, v, m);
    if (lane >= m) v += o;
  }
  return v;
}

// Exclusive prefix sums of two values a thread over the block, and their totals in every thread.
struct Two {
  int64_t a, b;
};
__device__ __forceinline__ Two block_prefix(Two v, Two (&part)[32], Two &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const Two s{warp_prefix(v.a), warp_prefix(v.b)};
  if (lane == 31) part[warp] = s;
  __syncthreads();
  const Two w = lane < warps ? part[lane] : Two{0, 0}, t{warp_prefix(w.a), warp_prefix(w.b)};
  total = Two{__shfl_sync(0xFFFFFFFFu, t.a, 31), __shfl_sync(0xFFFFFFFFu, t.b, 31)};
  const Two before{__shfl_sync(0xFFFFFFFFu, t.a - w.a, warp), __shfl_sync(0xFFFFFFFFu, t.b - w.b, warp)};
  __syncthreads();
  return Two{before.a + s.a - v.a, before.b + s.b - v.b};
}

__device__ __forceinline__ int64_t taken_at_start(const Args &a) {
  const int64_t t = *a.taken;
  return t < 0 ? 0 : t < a.num_free ? t : a.num_free;
}

// A sequence's new tokens: its length stays a number of 32 bits.
__device__ __forceinline__ int64_t wanted(const Args &a, int64_t i, int64_t len) {
  return min((int64_t)max(a.fresh[i], 0), (int64_t)INT32_MAX - len);
}

// A sequence's pages before its new tokens, and the new ones: its table's room bounds both.
__device__ __forceinline__ int64_t used_pages(const Args &a, int64_t len) { return (len + (1ll << a.shift) - 1) >> a.shift; }
__device__ __forceinline__ int64_t new_pages(const Args &a, int64_t len, int64_t n) {
  const int64_t used = used_pages(a, len);
  return min(used_pages(a, len + n) - used, max(a.width - used, (int64_t)0));
}

__global__ void __launch_bounds__(kThreads) scan_kernel(Args a) {
  __shared__ Two part[32];
  int64_t tokens = 0, pages = taken_at_start(a), beyond = 0;
  for (int64_t at = 0; at < a.batch; at += kThreads) {
    const int64_t i = at + threadIdx.x;
    const bool real = i < a.batch;
    const int64_t len = real ? max(a.lens[i], 0) : 0, want = real ? wanted(a, i, len) : 0;
    Two total;
    const int64_t start = min(tokens + block_prefix(Two{want, 0}, part, total).a, a.tokens);
    tokens += total.a;
    const int64_t n = min(want, a.tokens - start);
    const int64_t need = real ? new_pages(a, len, n) : 0, lacking = used_pages(a, len + n) - used_pages(a, len) - need;
    const int64_t first = pages + block_prefix(Two{need, lacking}, part, total).a;
    pages += total.a;
    beyond += total.b;
    if (real) {
      a.cu[i] = (int32_t)start;
      a.out_lens[i] = (int32_t)(len + n);
      a.first[i] = first;
      if (i == a.batch - 1) a.cu[a.batch] = (int32_t)(start + n);
    }
  }
  if (threadIdx.x == 0) {
    const int64_t out = min(pages, a.num_free);
    *a.out_taken = (int32_t)out;
    *a.missing = (int32_t)min(pages - out + beyond, (int64_t)INT32_MAX);
  }
}

// What a new token of sequence i gets: its slot, where its page is one of the row's or a new one.
__device__ __forceinline__ int64_t slot_of(const Args &a, int i, int64_t len, int64_t first, int64_t p) {
  const int64_t column = p >> a.shift, used = used_pages(a, len), at = first + column - used;
  int32_t page = -1;
  if (column < used && column < a.width) page = a.table[i * a.table_stride + column];
  else if (column < a.width && at < a.num_free) page = a.free_pages[at];
  return page < 0 ? -1 : ((int64_t)page << a.shift) + (p & ((1ll << a.shift) - 1));
}
__device__ __forceinline__ void fill_row(const Args &a, int64_t i, int64_t len, int64_t n, int64_t first) {
  const int64_t used = used_pages(a, len), need = new_pages(a, len, n);
  for (int64_t j = threadIdx.x & 31; j < need; j += 32) {
    const int64_t at = first + j;
    a.table[i * a.table_stride + used + j] = at < a.num_free ? a.free_pages[at] : -1;
  }
}
__device__ __forceinline__ void no_token(const Args &a, int64_t t) { a.slots[t] = -1, a.sequence[t] = -1, a.positions[t] = -1; }

// Many sequences, after scan_kernel: tokens by threads, which look their sequence up, new table entries by warps.
__global__ void __launch_bounds__(256) fill_kernel(Args a) {
  const int64_t thread = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, threads = (int64_t)gridDim.x * blockDim.x;
  const int64_t real = a.cu[a.batch];
  for (int64_t t = thread; t < a.tokens; t += threads) {
    if (t >= real) {
      no_token(a, t);
      continue;
    }
    int lo = 0, hi = a.batch - 1;  // the first sequence whose end is behind t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid + 1] > t) hi = mid;
      else lo = mid + 1;
    }
    const int64_t len = max(a.lens[lo], 0), p = len + t - a.cu[lo];
    a.slots[t] = slot_of(a, lo, len, a.first[lo], p);
    a.sequence[t] = lo;
    a.positions[t] = (int32_t)p;
  }
  for (int64_t i = thread >> 5; i < a.batch; i += threads >> 5)
    fill_row(a, i, max(a.lens[i], 0), a.cu[i + 1] - a.cu[i], a.first[i]);
}

// Up to kThreads sequences in one kernel: every block adds the lengths up itself (a thread a sequence: some 2 us, which a kernel of its own
// and the launch after it would cost too), keeps the sums in shared memory and fills its share of the tokens and rows.
__global__ void __launch_bounds__(kThreads) plan_kernel(Args a) {
  __shared__ Two part[32];
  __shared__ int32_t start[kThreads + 1], length[kThreads];
  __shared__ int64_t first[kThreads];
  const int i = threadIdx.x, width = blockDim.x;
  const bool real = i < a.batch;
  const int64_t len = real ? max(a.lens[i], 0) : 0, want = real ? wanted(a, i, len) : 0, taken = taken_at_start(a);
  Two total;
  const int64_t at = min(block_prefix(Two{want, 0}, part, total).a, a.tokens), n = min(want, a.tokens - at);
  const int64_t need = real ? new_pages(a, len, n) : 0, lacking = used_pages(a, len + n) - used_pages(a, len) - need;
  first[i] = taken + block_prefix(Two{need, lacking}, part, total).a;
  start[i] = (int32_t)at, length[i] = (int32_t)len;
  if (i == width - 1) start[width] = (int32_t)(at + n);
  if (blockIdx.x == 0) {
    if (real) a.cu[i] = (int32_t)at, a.out_lens[i] = (int32_t)(len + n);
    if (i == 0) {
      const int64_t out = min(taken + total.a, a.num_free);
      *a.out_taken = (int32_t)out;
      *a.missing = (int32_t)min(taken + total.a - out + total.b, (int64_t)INT32_MAX);
    }
  }
  __syncthreads();
  const int32_t end = start[width];  // behind the batch's sequences every start is the end
  if (blockIdx.x == 0 && i == 0) a.cu[a.batch] = end;
  const int64_t threads = (int64_t)gridDim.x * width, thread = (int64_t)blockIdx.x * width + i;
  for (int64_t t = thread; t < a.tokens; t += threads) {
    if (t >= end) {
      no_token(a, t);
      continue;
    }
    int lo = 0;  // the last sequence that begins at t or before: an empty one begins where the next one does
    for (int step = width / 2; step; step >>= 1)
      if (start[lo + step] <= t) lo += step;
    const int64_t l = length[lo], p = l + t - start[lo];
    a.slots[t] = slot_of(a, lo, l, first[lo], p);
    a.sequence[t] = lo;
    a.positions[t] = (int32_t)p;
  }
  for (int64_t row = thread >> 5; row < a.batch; row += threads >> 5)
    fill_row(a, row, length[row], start[row + 1] - start[row], first[row]);
}

struct Release {
  int32_t *table;
  int64_t table_stride;
  const unsigned char *ended;
  int32_t batch, width;
  int32_t *free_pages;
  int64_t num_free;
  const int32_t *taken;
  int32_t *out_taken;
  int32_t *counts;  // workspace: pages of each ended sequence
};

__device__ __forceinline__ int warp_sum(int v) { return __reduce_add_sync(0xFFFFFFFFu, v); }

__global__ void __launch_bounds__(256) count_kernel(Release a) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * 8;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < a.batch; i += warps) {
    int n = 0;
    if (a.ended[i])
      for (int64_t c = lane; c < a.width; c += 32) n += a.table[i * a.table_stride + c] >= 0;
    n = warp_sum(n);
    if (lane == 0) a.counts[i] = n;
  }
}

// A warp a sequence; every block adds the counts before its eight sequences, and all of them.
__global__ void __launch_bounds__(256) push_kernel(Release a) {
  __shared__ int64_t part[2][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row0 = (int64_t)blockIdx.x * 8;
  int64_t before = 0, all = 0;
  for (int64_t i = threadIdx.x; i < a.batch; i += 256) {
    const int64_t n = a.counts[i];
    all += n;
    if (i < row0) before += n;
  }
#pragma unroll
  for (int m = 16; m; m >>= 1) before += __shfl_xor_sync(0xFFFFFFFFu, before, m), all += __shfl_xor_sync(0xFFFFFFFFu, all, m);
  if (lane == 0) part[0][warp] = before, part[1][warp] = all;
  __syncthreads();
  before = all = 0;
  for (int w = 0; w < 8; ++w) before += part[0][w], all += part[1][w];
  int64_t base = *a.taken;
  base = (base < a.num_free ? base : a.num_free) - all;  // below 0 where pages come back that were not taken: those are dropped
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.out_taken = (int32_t)(base < 0 ? 0 : base);
  const int64_t i = row0 + warp;
  if (i >= a.batch || !a.ended[i]) return;
  for (int64_t r = row0; r < i; ++r) before += a.counts[r];
  int64_t at = base + before;
  for (int64_t c0 = 0; c0 < a.width; c0 += 32) {
    const int64_t c = c0 + lane;
    const int32_t page = c < a.width ? a.table[i * a.table_stride + c] : -1;
    const unsigned held = __ballot_sync(0xFFFFFFFFu, page >= 0);
    const int64_t to = at + __popc(held & ((1u << lane) - 1u));
    if (page >= 0 && to >= 0) a.free_pages[to] = page;
    if (c < a.width) a.table[i * a.table_stride + c] = -1;
    at += __popc(held);
  }
}

}  // namespace plan
}  // namespace tc

using namespace tc;

static int plan_status(const char *what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(std::string(what) + ": " + cudaGetErrorString(e)), TC_CUDA_ERROR;
  count_launch();
  return TC_OK;
}

extern "C" size_t tc_plan_pages_workspace(int32_t batch) { return batch > plan::kThreads ? (size_t)batch * sizeof(int64_t) : 0; }

extern "C" int tc_plan_pages(const int32_t *seq_lens, const int32_t *new_lens, int32_t batch, int32_t *block_table,
                             int64_t table_stride, int32_t max_pages, const int32_t *free_pages, int64_t num_free,
                             const int32_t *taken, int32_t page_size, int64_t tokens, int32_t *out_lens, int32_t *cu_q,
                             int64_t *slots, int32_t *sequence, int32_t *positions, int32_t *out_taken, int32_t *missing,
                             void *workspace, size_t workspace_bytes, tc_stream stream) {
  auto bad = [](const char *m) { return set_error(std::string("tc_plan_pages: ") + m), (int)TC_INVALID_ARGUMENT; };
  if (batch < 0 || max_pages < 0 || tokens < 0 || num_free < 0) return bad("negative size");
  if (tokens > 0x7FFFFFFFll || num_free > 0x7FFFFFFFll) return bad("more than 2**31 - 1 tokens or pages");
  if (page_size < 1 || page_size > (1 << 20) || (page_size & (page_size - 1))) return bad("page_size must be a power of two");
  if (max_pages > (1 << 30) / page_size) return bad("contexts hold at most 2**30 tokens");
  if (batch > 1 && table_stride < max_pages) return bad("table_stride must be at least max_pages");
  if ((batch && (!seq_lens || !new_lens || !out_lens)) || (batch && max_pages && !block_table) || (num_free && !free_pages) ||
      !taken || !cu_q || !out_taken || !missing || (tokens && (!slots || !sequence || !positions)))
    return bad("null pointer");
  if (batch > plan::kThreads && (!workspace || workspace_bytes < tc_plan_pages_workspace(batch)))
    return set_error("tc_plan_pages: workspace too small"), TC_WORKSPACE_TOO_SMALL;
  plan::Args a{seq_lens, new_lens, block_table, table_stride, free_pages, num_free, taken, tokens, batch, max_pages, 0,
               out_lens, cu_q, sequence, positions, out_taken, missing, slots, static_cast<int64_t *>(workspace)};
  while ((1 << a.shift) < page_size) ++a.shift;
  cudaStream_t s = (cudaStream_t)stream;
  if (batch <= plan::kThreads) {
    int threads = 256;  // a power of two, for the search
    while (threads < batch) threads *= 2;
    const int64_t work = tokens > (int64_t)batch * 32 ? tokens : (int64_t)batch * 32, blocks = (work + threads - 1) / threads;
    const int64_t most = (int64_t)sm_count() * (1024 / threads);
    plan::plan_kernel<<<(unsigned)(blocks < 1 ? 1 : blocks < most ? blocks : most), threads, 0, s>>>(a);
    return plan_status("tc_plan_pages");
  }
  plan::scan_kernel<<<1, plan::kThreads, 0, s>>>(a);
  if (const int st = plan_status("tc_plan_pages")) return st;
  const int64_t work = tokens > (int64_t)batch * 32 ? tokens : (int64_t)batch * 32;
  const int64_t blocks = (work + 255) / 256, most = (int64_t)sm_count() * 8;
  plan::fill_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, s>>>(a);
  return plan_status("tc_plan_pages");
}

extern "C" size_t tc_release_pages_workspace(int32_t batch) { return batch > 0 ? (size_t)batch * sizeof(int32_t) : 0; }

extern "C" int tc_release_pages(int32_t *block_table, int64_t table_stride, int32_t max_pages, const uint8_t *ended, int32_t batch,
                                int32_t *free_pages, int64_t num_free, const int32_t *taken, int32_t *out_taken, void *workspace,
                                size_t workspace_bytes, tc_stream stream) {
  auto bad = [](const char *m) { return set_error(std::string("tc_release_pages: ") + m), (int)TC_INVALID_ARGUMENT; };
  if (batch < 0 || max_pages < 0 || num_free < 0 || num_free > 0x7FFFFFFFll) return bad("sizes out of range");
  if (batch > 1 && table_stride < max_pages) return bad("table_stride must be at least max_pages");
  if ((batch && !ended) || (batch && max_pages && !block_table) || (num_free && !free_pages) || !taken || !out_taken)
    return bad("null pointer");
  if (batch && (!workspace || workspace_bytes < tc_release_pages_workspace(batch)))
    return set_error("tc_release_pages: workspace too small"), TC_WORKSPACE_TOO_SMALL;
  plan::Release a{block_table, table_stride, ended, batch, max_pages, free_pages, num_free, taken, out_taken,
                  static_cast<int32_t *>(workspace)};
  cudaStream_t s = (cudaStream_t)stream;
  const int64_t blocks = ((int64_t)batch + 7) / 8, most = (int64_t)sm_count() * 8;
  if (blocks) {
    plan::count_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, s>>>(a);
    if (const int st = plan_status("tc_release_pages")) return st;
  }
  plan::push_kernel<<<(unsigned)(blocks ? blocks : 1), 256, 0, s>>>(a);
  return plan_status("tc_release_pages");
}
