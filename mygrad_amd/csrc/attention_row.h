// One row of an attention by one wavefront, keys over its lanes: any type, head dimension up to 256 and mask.  What the row does not see never
// enters its sums.
#pragma once

#include "attention_rows.h"

namespace mg {

constexpr int kMaxDim = 256;
constexpr double kLog2e64 = 1.44269504088896340736;
constexpr int kParts = kMaxDim / 64;  // values of a row that a lane holds

template <typename C>
__device__ __forceinline__ C wave_sum(C v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

template <typename C>
__device__ __forceinline__ C wave_max(C v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = max(v, __shfl_xor(v, m));
  return v;
}

// The score behind cap and bias; `through`: its derivative by the plain product.
template <typename C>
__device__ __forceinline__ C score(const Attention &p, C dot, C slope, int distance, C &through) {
  const bool wide = sizeof(C) == 8;
  const C scale = wide ? (C)p.scale64 : (C)p.scale, cap = wide ? (C)p.cap64 : (C)p.cap;
  C s = dot * scale;
  through = scale;
  if (cap > 0) {
    const C bent = tanh(s / cap);
    s = cap * bent;
    through *= 1 - bent * bent;
  }
  return s - slope * (C)(distance < 0 ? -distance : distance);
}

template <typename T, typename C>
__device__ __forceinline__ C dot_row(const C *row, const T *other, int D) {
  C sum = 0;
  for (int d = 0; d < D; ++d) sum += row[d] * (C)other[d];
  return sum;
}

// What the lanes of a wavefront wrote to LDS is there for all of them.
__device__ __forceinline__ void wave_sees() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Row i of head h of batch item b; `mine`: LDS of this wavefront for the row's D values.
template <typename T, typename C>
__device__ __forceinline__ void attend_row(const Attention &p, int b, int h, int i, C *mine, const T *__restrict__ q, const T *__restrict__ k,
                                           const T *__restrict__ v, T *__restrict__ out, _Float16 *__restrict__ rest, C *__restrict__ lse) {
  const int lane = threadIdx.x & 63;
  const long long step = (long long)p.HK * p.D, head = ((long long)b * p.TK * p.HK + h / p.group) * p.D;
  const long long at = (((long long)b * p.TQ + i) * p.HQ + h) * p.D;
  const C slope = p.slopes ? ((const C *)p.slopes)[h] : C(0);
  wave_sees();
  for (int d = lane; d < p.D; d += 64) mine[d] = (C)q[at + d];
  wave_sees();
  const Span span = span_of(p, b, i);
  C top = -INFINITY, total = 0, sum[kParts] = {};
  for (int j0 = span.lo; j0 < span.hi; j0 += 64) {
    const int j = j0 + lane, count = min(64, span.hi - j0);
    C s = -INFINITY, through;
    if (lane < count) s = score<C>(p, dot_row<T, C>(mine, k + head + j * step, p.D), slope, span.place - j, through);
    const C now = max(top, wave_max(s)), base = now == -INFINITY ? C(0) : now;
    const C back = exp(top - base);
    const C e = lane < count ? exp(s - base) : C(0);
    total = total * back + wave_sum(e);
    top = now;
#pragma unroll
    for (int c = 0; c < kParts; ++c) sum[c] *= back;
    for (int n = 0; n < count; ++n) {
      const C weight = __shfl(e, n);
      const T *row = v + head + (j0 + n) * step;
#pragma unroll
      for (int c = 0; c < kParts; ++c)
        if (lane + 64 * c < p.D) sum[c] += weight * (C)row[lane + 64 * c];
    }
  }
  const bool none = total == 0;
#pragma unroll
  for (int c = 0; c < kParts; ++c)
    if (lane + 64 * c < p.D) {
      const C value = none ? C(0) : sum[c] / total;
      out[at + lane + 64 * c] = (T)value;
      if (rest) rest[at + lane + 64 * c] = (_Float16)((value - (C)(T)value) * (C)kRest);
    }
  if (lse && lane == 0) lse[((long long)b * p.HQ + h) * p.TQ + i] = none ? (C)INFINITY : top * (C)kLog2e64 + log2(total);  // no weight on any key
}

// Row i of dq; `mine`: LDS of this wavefront for twice D values.
template <typename T, typename C>
__device__ __forceinline__ void dq_row(const Attention &p, int b, int h, int i, C *mine, const T *__restrict__ q, const T *__restrict__ k,
                                       const T *__restrict__ v, const T *__restrict__ grad, const C *__restrict__ lse, const C *__restrict__ delta,
                                       T *__restrict__ dq) {
  const int lane = threadIdx.x & 63;
  const long long step = (long long)p.HK * p.D, head = ((long long)b * p.TK * p.HK + h / p.group) * p.D;
  const long long at = (((long long)b * p.TQ + i) * p.HQ + h) * p.D, stat = ((long long)b * p.HQ + h) * p.TQ + i;
  const C slope = p.slopes ? ((const C *)p.slopes)[h] : C(0);
  wave_sees();
  for (int d = lane; d < p.D; d += 64) mine[d] = (C)q[at + d], mine[p.D + d] = (C)grad[at + d];
  wave_sees();
  const Span span = span_of(p, b, i);
  const C norm = lse[stat], mean = delta[stat];
  C sum[kParts] = {};
  for (int j0 = span.lo; j0 < span.hi; j0 += 64) {
    const int j = j0 + lane, count = min(64, span.hi - j0);
    C ds = 0;
    if (lane < count) {
      C through;
      const C s = score<C>(p, dot_row<T, C>(mine, k + head + j * step, p.D), slope, span.place - j, through);
      ds = exp2(s * (C)kLog2e64 - norm) * (dot_row<T, C>(mine + p.D, v + head + j * step, p.D) - mean) * through;
    }
    for (int n = 0; n < count; ++n) {
      const C weight = __shfl(ds, n);
      const T *row = k + head + (j0 + n) * step;
#pragma unroll
      for (int c = 0; c < kParts; ++c)
        if (lane + 64 * c < p.D) sum[c] += weight * (C)row[lane + 64 * c];
    }
  }
#pragma unroll
  for (int c = 0; c < kParts; ++c)
    if (lane + 64 * c < p.D) dq[at + lane + 64 * c] = (T)sum[c];
}

// Row j of dk and dv: queries over the lanes, the heads that share the key one after the other; `mine` as for dq_row.
template <typename T, typename C>
__device__ __forceinline__ void dkv_row(const Attention &p, int b, int hk, int j, C *mine, const T *__restrict__ q, const T *__restrict__ k,
                                        const T *__restrict__ v, const T *__restrict__ grad, const C *__restrict__ lse, const C *__restrict__ delta,
                                        T *__restrict__ dk, T *__restrict__ dv) {
  const int lane = threadIdx.x & 63;
  const long long at = (((long long)b * p.TK + j) * p.HK + hk) * p.D, step = (long long)p.HQ * p.D;
  wave_sees();
  for (int d = lane; d < p.D; d += 64) mine[d] = (C)k[at + d], mine[p.D + d] = (C)v[at + d];
  wave_sees();
  C sum_k[kParts] = {}, sum_v[kParts] = {};
  for (int h = hk * p.group; h < (hk + 1) * p.group; ++h) {
    const long long head = ((long long)b * p.TQ * p.HQ + h) * p.D, stats = ((long long)b * p.HQ + h) * p.TQ;
    const C slope = p.slopes ? ((const C *)p.slopes)[h] : C(0);
    for (int i0 = 0; i0 < p.TQ; i0 += 64) {
      const int i = i0 + lane;
      C weight = 0, ds = 0;
      bool sees = false;
      if (i < p.TQ) {
        const Span span = span_of(p, b, i);
        sees = j >= span.lo && j < span.hi;
        if (sees) {
          C through;
          const C s = score<C>(p, dot_row<T, C>(mine, q + head + i * step, p.D), slope, span.place - j, through);
          weight = exp2(s * (C)kLog2e64 - lse[stats + i]);
          ds = weight * (dot_row<T, C>(mine + p.D, grad + head + i * step, p.D) - delta[stats + i]) * through;
        }
      }
      for (unsigned long long left = __ballot(sees); left; left &= left - 1) {
        const int n = __ffsll(left) - 1;
        const C of_v = __shfl(weight, n), of_k = __shfl(ds, n);
        const T *qr = q + head + (i0 + n) * step, *gr = grad + head + (i0 + n) * step;
#pragma unroll
        for (int c = 0; c < kParts; ++c)
          if (lane + 64 * c < p.D) {
            sum_k[c] += of_k * (C)qr[lane + 64 * c];
            sum_v[c] += of_v * (C)gr[lane + 64 * c];
          }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < kParts; ++c)
    if (lane + 64 * c < p.D) dk[at + lane + 64 * c] = (T)sum_k[c], dv[at + lane + 64 * c] = (T)sum_v[c];
}

// ---- which rows to compute once more -------------------------------------------------------------------------------------------
// A row of a result that is no number has to be computed again by the functions above only if what it does not see may have made it one.  It need
// not where what it sees does, whatever stands elsewhere:
//   out: the sum of the row's weights is no number (scores of unseen keys never enter it; where rows share pieces in LDS: and q_i or a key is none);
//        else, where a value that it sees is no number or infinite, that value is what the row has there (weights are not zero);
//   dq:  lse_i or D_i of the row is none, which makes each of its dS_ij none (a row that sees nothing has no dS);
//   dk, dv: the same of a query that sees the key, for all of dk and for dv where that query's grad is none (all of it where lse_i is).
// So an upstream gradient that overflowed, or operands that are no numbers throughout, cost a step what numbers do.
template <typename C>
__device__ __forceinline__ bool no_number(C v) { return !(fabs(v) < INFINITY); }

__device__ __forceinline__ bool dq_stands(const Span &span, float lse, float delta) { return span.hi > span.lo && (lse != lse || no_number(delta)); }

// Whether row i of an attention, whose weights' sum is no number, stands; the same in every lane.  An infinity may give weights of zero: those are
// computed again.
template <typename T>
__device__ __forceinline__ bool out_stands(const Attention &p, int b, int h, int i, const T *__restrict__ q, const T *__restrict__ k) {
  if (!shares_pieces(p, sizeof(T))) return true;
  const int lane = threadIdx.x & 63;
  const Span span = span_of(p, b, i);
  if (span.hi <= span.lo) return false;
  const T *row = q + (((long long)b * p.TQ + i) * p.HQ + h) * p.D, *keys = k + ((long long)b * p.TK * p.HK + h / p.group) * p.D;
  auto none = [&](const T *from) {
    bool none = false;
    for (int d = lane; d < p.D; d += 64) none |= from[d] != from[d];
    return none;
  };
  if (__any(none(row))) return true;
  for (int j = span.lo; j < span.hi; ++j)
    if (__any(none(keys + (long long)j * p.HK * p.D))) return true;
  return false;
}

// The rows of a head's values among [lo, hi) that hold one that is no number, in no order; a block's four wavefronts find them together, eight
// rows at a time each (2048 of 64 values: 40 us).
struct OddValues {
  static constexpr int kMost = 256;
  int count, rows[kMost];  // more than kMost: they are not all here

  template <typename T>
  __device__ __forceinline__ void find(const Attention &p, int b, int hk, int lo, int hi, const T *__restrict__ v) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long step = (long long)p.HK * p.D;
    const T *head = v + ((long long)b * p.TK * p.HK + hk) * p.D;
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    for (int j0 = lo < hi ? lo + 8 * wave : hi; j0 < hi; j0 += 32) {
      bool odd[8] = {};
#pragma unroll
      for (int c = 0; c < kParts; ++c)
        if (64 * c < p.D) {
          T values[8];
#pragma unroll
          for (int n = 0; n < 8; ++n) values[n] = lane + 64 * c < p.D && j0 + n < hi ? head[(j0 + n) * step + lane + 64 * c] : T(0);
#pragma unroll
          for (int n = 0; n < 8; ++n) odd[n] |= no_number((float)values[n]);
        }
#pragma unroll
      for (int n = 0; n < 8; ++n)
        if (__any(odd[n]) && lane == 0) {
          const int at = atomicAdd(&count, 1);
          if (at < kMost) rows[at] = j0 + n;
        }
    }
    __syncthreads();
  }
};

// Puts into row i of `out` what the values that it sees make of those that are no number there; false if they do not explain all of them.
template <typename T>
__device__ __forceinline__ bool out_settled(const Attention &p, int b, int h, int i, const OddValues &odd, const T *__restrict__ v, T *__restrict__ out,
                                            _Float16 *__restrict__ rest) {
  const int lane = threadIdx.x & 63;
  const long long at = (((long long)b * p.TQ + i) * p.HQ + h) * p.D, step = (long long)p.HK * p.D;
  const T *head = v + ((long long)b * p.TK * p.HK + h / p.group) * p.D;
  const Span span = span_of(p, b, i);
  const bool listed = odd.count <= OddValues::kMost;
  unsigned open = 0, up = 0, down = 0;  // bit c: value lane + 64 c is no number, with an infinity among what makes it, or one of the other sign
#pragma unroll
  for (int c = 0; c < kParts; ++c)
    if (lane + 64 * c < p.D && no_number((float)out[at + lane + 64 * c])) open |= 1u << c;
  const unsigned all = open;
  const int last = listed ? odd.count : span.hi - span.lo;
  for (int n = 0; n < last && __any(open & ~(up & down)); ++n) {
    const int j = listed ? odd.rows[n] : span.lo + n;
    if (j < span.lo || j >= span.hi) continue;
#pragma unroll
    for (int c = 0; c < kParts; ++c)
      if (open >> c & 1) {
        const float value = (float)head[j * step + lane + 64 * c];
        if (no_number(value) && !(value < 0)) up |= 1u << c;
        if (no_number(value) && !(value > 0)) down |= 1u << c;
      }
  }
  if (__any(all & ~(up | down))) return false;
#pragma unroll
  for (int c = 0; c < kParts; ++c)
    if (all >> c & 1) {
      const float value = (up & down) >> c & 1 ? NAN : up >> c & 1 ? INFINITY : -INFINITY;
      out[at + lane + 64 * c] = (T)value;
      if (rest) rest[at + lane + 64 * c] = (_Float16)NAN;
    }
  return true;
}

// Whether row j of dk (`of_k`: it holds one that is no number) and dv (bit c of `of_v`: value lane + 64 c is none) stands; the same in every lane.
template <typename T>
__device__ __forceinline__ bool dkv_stands(const Attention &p, int b, int hk, int j, bool of_k, unsigned of_v, const T *__restrict__ grad,
                                           const float *__restrict__ lse, const float *__restrict__ delta) {
  const int lane = threadIdx.x & 63;
  for (int h = hk * p.group; h < (hk + 1) * p.group; ++h) {
    const long long head = ((long long)b * p.TQ * p.HQ + h) * p.D, step = (long long)p.HQ * p.D, stats = ((long long)b * p.HQ + h) * p.TQ;
    for (int i0 = 0; i0 < p.TQ; i0 += 64) {
      const int i = i0 + lane;
      bool all = false, some = false;
      if (i < p.TQ) {
        const Span span = span_of(p, b, i);
        if (j >= span.lo && j < span.hi) all = lse[stats + i] != lse[stats + i], some = no_number(delta[stats + i]);
      }
      if (__any(all)) return true;
      for (unsigned long long left = __ballot(some); left; left &= left - 1) {
        of_k = false;
        const T *row = grad + head + (i0 + __ffsll(left) - 1) * step;
#pragma unroll
        for (int c = 0; c < kParts; ++c)
          if ((of_v >> c & 1) && no_number((float)row[lane + 64 * c])) of_v &= ~(1u << c);
        if (!__any(of_v)) return true;
      }
    }
  }
  return !of_k && !__any(of_v);
}

// The rows that lanes c and 32 + c of a wavefront mark, as bits.
__device__ __forceinline__ unsigned marks_of(bool mark) {
  const unsigned long long all = __ballot(mark);
  return (unsigned)all | (unsigned)(all >> 32);
}

// f(row) for the rows marked in `words`, shared out among four wavefronts.
template <int WORDS, typename F>
__device__ __forceinline__ void each_marked(const unsigned *words, F f) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int turn = 0;
  for (int w = 0; w < WORDS; ++w)
    for (unsigned left = __builtin_amdgcn_readfirstlane(words[w]); left; left &= left - 1, ++turn)
      if ((turn & 3) == wave) f(32 * w + __ffs(left) - 1);
}

}  // namespace mg
