// What the attention kernels share: the problem, and which keys a query sees.
#pragma once

#include "internal.h"

namespace mg {

// Tensors are (batch, tokens, heads, dim), C-contiguous; statistics of rows are (batch, heads, tokens).
struct Attention {
  int B, TQ, TK, HQ, HK, D;
  int group;  // query heads that share a key head
  int causal, window;
  int longest, mean;      // keys in use of the item with most, and of all about
  float scale, cap, bend;  // cap 0: scores as they are; bend: scale / cap, or float's largest (infinity times a product of zero is no number)
  double scale64, cap64;  // the same for double precision
  const int32_t *lengths, *prefix, *starts, *ends;
  const void *slopes;  // float, double for double precision
};

// Keys [lo, hi) are visible to a query that stands at `place` among them.  Every mask is one interval for each row: what is causal
// ends it, a window or a document begins it, a prefix moves its end.
struct Span {
  int lo, hi, place;
};

__device__ __forceinline__ Span span_of(const Attention &p, int b, int i) {
  const int n = p.lengths ? min(max(p.lengths[b], 0), p.longest) : p.TK;
  Span s{0, n, i + n - p.TQ};
  if (p.starts) {
    if (s.place < 0 || s.place >= n) return Span{0, 0, s.place};
    const long long at = (long long)b * p.TK + s.place;
    s.lo = max(p.starts[at], 0);
    s.hi = min(p.ends[at], n);
  }
  const int first = s.lo, last = s.hi;
  if (p.causal) s.hi = min(s.hi, s.place + 1);
  if (p.window) {
    s.lo = max(s.lo, s.place - p.window + 1);
    if (!p.causal) s.hi = min(s.hi, s.place + p.window);
  }
  if (p.prefix) s.hi = max(s.hi, first + min(max(p.prefix[b], 0), last - first));
  if (s.hi <= s.lo) s.lo = s.hi = 0;
  return s;
}

// How many keys a window lets some neighbouring rows see between them, at most: beyond 2^31 for the largest window both ways.
__host__ __device__ constexpr unsigned window_of_rows(int window, int causal, int rows) {
  return (causal ? 1u : 2u) * (unsigned)window + (unsigned)rows;
}

}  // namespace mg
