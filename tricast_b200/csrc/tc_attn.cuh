// Attention of new tokens over a paged cache: the call's arguments and what the kernels share.
#pragma once

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

// New tokens [q0, q0 + n) and context length of a sequence, clamped to what the tensors hold.
struct Seq {
  int64_t q0;
  int n, len;
};
__device__ __forceinline__ Seq sequence(const Args &a, int b) {
  Seq s;
  int64_t lo = a.cu ? a.cu[b] : b, hi = a.cu ? a.cu[b + 1] : b + 1;
  lo = min(max(lo, (int64_t)0), a.total_q);
  hi = min(max(hi, lo), a.total_q);
  s.q0 = lo;
  s.n = (int)min(hi - lo, (int64_t)a.max_q);
  const int64_t held = (int64_t)a.max_pages << a.c.page_shift;
  s.len = (int)min((int64_t)max(a.lens[b], 0), held);
  return s;
}

// Keys [lo, hi) that new token i of the sequence sees: it sits at position len - n + i, after the
// sequence's earlier context, and sees itself and what comes before it, at most `window` keys. A
// position below 0 (more new tokens than context) sees none.
__device__ __forceinline__ void visible(const Args &a, const Seq &s, int i, int &lo, int &hi) {
  const int at = s.len - s.n + i;
  hi = a.causal ? max(at + 1, 0) : s.len;
  lo = a.window > 0 ? max(at + 1 - a.window, 0) : 0;
}

}  // namespace attn
}  // namespace tc
