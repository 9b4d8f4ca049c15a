// Attention of float16 and float32 on the matrix cores: tiles of queries against tiles of keys, one pass with the running maximum
// and sum of the softmax, nothing of the scores in memory.
//
// The tiles' products multiply what a row does not see by weights of zero, which an infinity or a NaN there turns into NaN.  So rows
// whose results hold one that is no number are computed once more, a row at a time, unless what they see explains it (attention_row.h).
#include "attention_tiles.h"

#include "attention_row.h"

#include <algorithm>

namespace mg {

namespace {

constexpr int kBlockRows = 128;  // queries of a block: 32 for each of its four wavefronts

// The forward pass: 4 D operations for each query and key, on the matrix cores with the softmax's exponentials beside them.  Four wavefronts of 32
// queries share the tiles of keys and values, the next ones on their way while these are multiplied; 64 keys in two buffers are 64 KB at 128
// values of float16, so two blocks share a compute unit and one's products run while the other takes exponentials (with half of the unit's
// queries gone, as at the end of a causal launch, three fifths of the rate are left).  Float32's products take eight times as long: 32 keys do.
// 2 x 4096 tokens, 16 heads of 128, float16: 382 us (1080 TFLOP/s of three products, as weights come in two parts; a large product reaches 1168), causal
// 220 (940), with a cap 480 (860); of 64: 227 (910).  2 x 2048, 8 heads of 128, float32: 324 (106; a large product 154).
template <typename T, int DP, int KEYS, bool BENT>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2)
attention_tiles_kernel(Attention p, Deal deal, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, T *__restrict__ out,
                       _Float16 *__restrict__ rest, float *__restrict__ lse) {
  typedef TileOf<T, DP, KEYS> Tile;
  typedef typename Fragment<T>::V V;
  constexpr int kSteps = DP / 16, kParts = DP / 32;
  __shared__ __attribute__((aligned(1024))) char tiles[4 * Tile::kBytes];
  __shared__ int edges[2][4];
  __shared__ unsigned bad[2][4];  // rows with one that is no number, and those whose weights' sum is none
  const unsigned lds = (unsigned)(unsigned long long)(MG_LDS char *)tiles;
  const Dealt at = dealt(deal, blockIdx.x);
  const int b = at.pair / p.HK, hk = at.pair % p.HK, hq = hk * p.group + at.head;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
  const int tile = tile_of_rank<false>(p, b, deal.tiles - 1 - at.tile, deal.tiles, kBlockRows), i = tile * kBlockRows + wave * 32 + c;
  const bool in = i < p.TQ;
  const Span span = in ? span_of(p, b, i) : Span{0, 0, 0};
  const Reach reach = reach_of(span, in);
  if (lane == 0) edges[0][wave] = reach.lo, edges[1][wave] = reach.hi;

  V rows[kSteps];
  const T *row = q + (((long long)b * p.TQ + (in ? i : 0)) * p.HQ + hq) * p.D;
#pragma unroll
  for (int n = 0; n < kSteps; ++n) rows[n] = fragment_of(row, 16 * n + 8 * h, p.D, in);

  __syncthreads();
  const int lo = __builtin_amdgcn_readfirstlane(min(min(edges[0][0], edges[0][1]), min(edges[0][2], edges[0][3])));
  const int hi = __builtin_amdgcn_readfirstlane(max(max(edges[1][0], edges[1][1]), max(edges[1][2], edges[1][3])));
  const int count = hi > lo ? (hi - lo + KEYS - 1) / KEYS : 0;
  const unsigned stride = (unsigned)(p.HK * p.D) * (unsigned)sizeof(T);
  const typename Tile::template Loader<256> load(stride, (unsigned)p.D * (unsigned)sizeof(T));
  const long long head = (((long long)b * p.TK + lo) * p.HK + hk) * p.D * (long long)sizeof(T);
  const char *kb = (const char *)k + head, *vb = (const char *)v + head;
  auto stage = [&](int t) {
    const long long from = (long long)t * KEYS * stride;
    const int last = hi - lo - t * KEYS;
    const unsigned to = lds + (unsigned)(t & 1) * (2 * Tile::kBytes);
    load(kb + from, last, to);
    load(vb + from, last, to + Tile::kBytes);
  };

  Running<T, DP, KEYS / 32, BENT> run;
  run.begin();
  const typename Tile::Place place = Tile::place(lane);
  const Scores how = scores_of(p, hq);
  if (count) stage(0);
  all_landed();
  for (int t = 0; t < count; ++t) {
    if (t + 1 < count) stage(t + 1);
    const int key0 = lo + t * KEYS;
    if (key0 < reach.hi && key0 + KEYS > reach.lo) {
      const unsigned keys = lds + (unsigned)(t & 1) * (2 * Tile::kBytes);
      run.take(p, how, keys, keys + Tile::kBytes, rows, span, key0, key0 >= reach.all_lo && key0 + KEYS <= reach.all_hi, place, h);
    }
    all_landed();
#pragma unroll
    for (int n = 0; n < kParts; ++n) asm volatile("" : "+v"(run.sums[n]));  // one set of registers, whichever way a round went
  }

  const float total = sum_halves(run.total);
  const float by = total > 0 ? 1.0f / total : total == 0 ? 0.0f : NAN;
  bool odd = false;
  if (in) {
    const long long to = (((long long)b * p.TQ + i) * p.HQ + hq) * p.D;
#pragma unroll
    for (int n = 0; n < kParts; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int d = 32 * n + row_of(r, h);
        if (d >= p.D) continue;
        const f32x4 value = four_of(run.sums[n], r) * by;
        odd |= put_four(out + to + d, value);
        if constexpr (sizeof(T) == 2)
          if (rest) put_four(rest + to + d, (value - __builtin_convertvector(__builtin_convertvector(value, f16x4), f32x4)) * kRest);
      }
    if (lse && h == 0) lse[((long long)b * p.HQ + hq) * p.TQ + i] = total == 0 ? INFINITY : run.top + __builtin_log2f(total) - kLift;
  }
  const unsigned marks = marks_of(odd), none = marks_of(odd && total != total);
  if (lane == 0) bad[0][wave] = marks, bad[1][wave] = none;
  all_landed();  // what is stored, too: other wavefronts may write it again
  OddValues &values = *(OddValues *)(tiles + 4 * kMaxDim * sizeof(float));  // behind what rows need
  static_assert(4 * kMaxDim * sizeof(float) + sizeof values <= sizeof tiles, "no room for them");
  if ((bad[0][0] & ~bad[1][0]) | (bad[0][1] & ~bad[1][1]) | (bad[0][2] & ~bad[1][2]) | (bad[0][3] & ~bad[1][3])) values.find(p, b, hk, lo, hi, v);
  each_marked<4>(bad[0], [&](int n) {
    const int again = tile * kBlockRows + n;
    if (bad[1][n >> 5] >> (n & 31) & 1 ? !out_stands(p, b, hq, again, q, k) : !out_settled(p, b, hq, again, values, v, out, rest))
      attend_row<T, float>(p, b, hq, again, (float *)tiles + wave * kMaxDim, q, k, v, out, rest, lse);
  });
}

// ---- gradient ----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float sum16(float v) {
#pragma unroll
  for (int m = 8; m; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

// Sixteen lanes a row, eight values each at a time.  Bound by reading out, what it left over and grad: 100 MB in 20 us, 5 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) attention_stats_kernel(Attention p, Stats stats, const T *__restrict__ out, const _Float16 *__restrict__ rest,
                                                              const float *__restrict__ lse, const T *__restrict__ grad) {
  const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
  const int bh = blockIdx.x / stats.chunks, chunk = blockIdx.x % stats.chunks, b = bh / p.HQ, h = bh % p.HQ;
  for (int n = group; n < stats.rows; n += 16) {
    const int i = chunk * stats.rows + n;
    float dot = 0;
    if (i < p.TQ) {
      const long long at = (((long long)b * p.TQ + i) * p.HQ + h) * p.D;
      for (int d = lane * 8; d < p.D; d += 128) {
        const f32x8 g = __builtin_convertvector(fragment_of(grad + at, d, p.D, true), f32x8);
        f32x8 o = __builtin_convertvector(fragment_of(out + at, d, p.D, true), f32x8);
        if (rest) o += __builtin_convertvector(fragment_of(rest + at, d, p.D, true), f32x8) * (1.0f / kRest);
#pragma unroll
        for (int j = 0; j < 8; ++j) dot += g[j] * o[j];
      }
    }
    dot = sum16(dot);
    if (i < p.TQ && lane == 0) {
      const long long at = (long long)bh * p.TQ + i;
      stats.level[at] = lse[at] - (sizeof(T) == 2 ? kShift : 0.0f);
      stats.delta[at] = dot;
    }
  }
  if (h != 0 || threadIdx.x >= 64) return;
  Reach r{0x7fffffff, 0, 0, 0x7fffffff};
  for (int n = threadIdx.x; n < stats.rows; n += 64) {
    const int i = chunk * stats.rows + n;
    const bool in = i < p.TQ;
    const Span s = in ? span_of(p, b, i) : Span{0, 0, 0};
    if (in) stats.lo[(long long)b * p.TQ + i] = s.lo, stats.hi[(long long)b * p.TQ + i] = s.hi;
    if (s.hi > s.lo) r.lo = min(r.lo, s.lo), r.hi = max(r.hi, s.hi);
    r.all_lo = max(r.all_lo, s.lo), r.all_hi = min(r.all_hi, s.hi);  // a chunk with rows beyond the last query is never whole
  }
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    r.lo = min(r.lo, __shfl_xor(r.lo, m)), r.hi = max(r.hi, __shfl_xor(r.hi, m));
    r.all_lo = max(r.all_lo, __shfl_xor(r.all_lo, m)), r.all_hi = min(r.all_hi, __shfl_xor(r.all_hi, m));
  }
  if (threadIdx.x == 0) stats.reach[(long long)b * stats.chunks + chunk] = r;
}

// dq^T = K^T dS^T: as the forward pass, with the queries' rows of grad beside those of q; S and dP are formed again here and by the keys'
// kernel, two of seven products more than one kernel would need, which would have to add to dq or to dk and dv across blocks, in no order.
// Bound by the matrix cores: 2 x 4096 tokens, 16 heads of 128, float16: 500 us (1100 TFLOP/s of four products, dS in two counted), causal 276;
// float32, 2 x 2048, 8 heads of 128: 455 (113 of 154).
template <typename T, int DP, int KEYS, bool BENT>
__global__ void __launch_bounds__(256, DP > (sizeof(T) == 4 ? 64 : 128) ? 1 : 2)
attention_dq_kernel(Attention p, Deal deal, Stats stats, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                    const T *__restrict__ grad, const float *__restrict__ lse, T *__restrict__ dq) {
  typedef TileOf<T, DP, KEYS> Tile;
  typedef typename Fragment<T>::V V;
  constexpr int kSteps = DP / 16, kParts = DP / 32, kSubs = KEYS / 32;
  __shared__ __attribute__((aligned(1024))) char tiles[4 * Tile::kBytes];
  __shared__ int edges[2][4];
  __shared__ unsigned bad[4];
  const unsigned lds = (unsigned)(unsigned long long)(MG_LDS char *)tiles;
  const Dealt at = dealt(deal, blockIdx.x);
  const int b = at.pair / p.HK, hk = at.pair % p.HK, hq = hk * p.group + at.head;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
  const int tile = tile_of_rank<false>(p, b, deal.tiles - 1 - at.tile, deal.tiles, kBlockRows), i = tile * kBlockRows + wave * 32 + c;
  const bool in = i < p.TQ;
  const Span span = in ? span_of(p, b, i) : Span{0, 0, 0};
  const Reach reach = reach_of(span, in);
  if (lane == 0) edges[0][wave] = reach.lo, edges[1][wave] = reach.hi;

  V rows[kSteps], grads[kSteps];
  const long long row = (((long long)b * p.TQ + (in ? i : 0)) * p.HQ + hq) * p.D;
#pragma unroll
  for (int n = 0; n < kSteps; ++n) {
    rows[n] = fragment_of(q + row, 16 * n + 8 * h, p.D, in);
    grads[n] = fragment_of(grad + row, 16 * n + 8 * h, p.D, in);
  }
  const long long stat = ((long long)b * p.HQ + hq) * p.TQ + (in ? i : 0);
  const float own_level = in ? stats.level[stat] : INFINITY, delta = in ? stats.delta[stat] : 0.0f;
  const bool stands = dq_stands(span, own_level, delta);

  __syncthreads();
  const int lo = __builtin_amdgcn_readfirstlane(min(min(edges[0][0], edges[0][1]), min(edges[0][2], edges[0][3])));
  const int hi = __builtin_amdgcn_readfirstlane(max(max(edges[1][0], edges[1][1]), max(edges[1][2], edges[1][3])));
  const int count = hi > lo ? (hi - lo + KEYS - 1) / KEYS : 0;
  const unsigned stride = (unsigned)(p.HK * p.D) * (unsigned)sizeof(T);
  const typename Tile::template Loader<256> load(stride, (unsigned)p.D * (unsigned)sizeof(T));
  const long long head = (((long long)b * p.TK + lo) * p.HK + hk) * p.D * (long long)sizeof(T);
  const char *kb = (const char *)k + head, *vb = (const char *)v + head;
  auto stage = [&](int t) {
    const long long from = (long long)t * KEYS * stride;
    const int last = hi - lo - t * KEYS;
    const unsigned to = lds + (unsigned)(t & 1) * (2 * Tile::kBytes);
    load(kb + from, last, to);
    load(vb + from, last, to + Tile::kBytes);
  };

  Pulled<T, DP, KEYS, BENT> run;
  run.begin();
  const typename Tile::Place place = Tile::place(lane);
  const Scores how = scores_of(p, hq);
  if (count) stage(0);
  all_landed();
  for (int t = 0; t < count; ++t) {
    if (t + 1 < count) stage(t + 1);
    const unsigned keys = lds + (unsigned)(t & 1) * (2 * Tile::kBytes);  // and values behind them
#pragma unroll BENT ? 1 : kSubs
    for (int n = 0; n < kSubs; ++n) {
      const int from = lo + t * KEYS + 32 * n;
      if (from < reach.hi && from + 32 > reach.lo)
        run.take(p, how, keys, n, rows, grads, own_level, delta, span, from, from >= reach.all_lo && from + 32 <= reach.all_hi, place, h);
    }
    all_landed();
  }

  const float by = run.by(p);
  bool odd = false;
  if (in) {
#pragma unroll
    for (int n = 0; n < kParts; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int d = 32 * n + row_of(r, h);
        if (d < p.D) odd |= put_four(dq + row + d, four_of(run.sums[n], r) * by);
      }
  }
  const unsigned marks = marks_of(odd && !stands);
  if (lane == 0) bad[wave] = marks;
  all_landed();  // what is stored, too: other wavefronts may write it again
  each_marked<4>(bad, [&](int n) {
    dq_row<T, float>(p, b, hq, tile * kBlockRows + n, (float *)tiles + wave * 2 * kMaxDim, q, k, v, grad, lse, stats.delta, dq);
  });
}

// dv^T = grad^T P and dk^T = q^T dS: a block keeps 128 keys, 32 for each wavefront in its lanes' columns, and goes through the chunks of queries
// that see any of them, head by head of those that share the keys.  Where there are few blocks they are cut: each of `cuts` takes an equal share
// of the chunks and leaves its sums in float32, which attention_dkv_join_kernel adds up in order.
// Bound by the matrix cores: 2 x 4096 tokens, 16 heads of 128, float16: 775 us (1065 TFLOP/s of six products, P and dS in two counted), causal 425;
// float32, 2 x 2048, 8 heads of 128: 582 (118 of 154).  Documents end at different times, which leaves units idle: 8192 tokens of five of them, 16
// heads of 128, take 275 us where even work would take 200; cut in two they would leave 134 MB of sums to be joined in 80 us.
// With VALUES the keys' values lie in LDS instead of registers: at 128 values of float16 a head the two results and k take 160 of a lane's 256,
// and with v's 32 as well the scores would not fit.
template <typename T, int DP, int ROWS, bool VALUES, bool BENT>
__global__ void __launch_bounds__(256, DP > (sizeof(T) == 4 ? 64 : 128) ? 1 : 2)
attention_dkv_kernel(Attention p, Deal deal, Stats stats, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                     const T *__restrict__ grad, const float *__restrict__ lse, T *__restrict__ dk, T *__restrict__ dv, int cuts,
                     float *__restrict__ parts) {
  typedef TileOf<T, DP, ROWS> Tile;
  typedef typename Fragment<T>::V V;
  constexpr int kSteps = DP / 16, kParts = DP / 32, kSubs = ROWS / 32;
  constexpr int kBuffer = 2 * Tile::kBytes + 4 * 256;  // rows of q and grad; level, delta, lo, hi of each
  typedef TileOf<T, DP, kBlockRows> Whole;
  __shared__ __attribute__((aligned(1024))) char tiles[2 * kBuffer + (VALUES ? Whole::kBytes : 0)];
  __shared__ unsigned bad[2][4];  // rows with one that is no number in dk or dv, and in dk
  const unsigned lds = (unsigned)(unsigned long long)(MG_LDS char *)tiles;
  const Dealt at = dealt(deal, blockIdx.x);  // its head is the cut
  const int b = at.pair / p.HK, hk = at.pair % p.HK;
  const int tile = tile_of_rank<true>(p, b, deal.tiles - 1 - at.tile, deal.tiles, kBlockRows);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
  const int block0 = tile * kBlockRows, key0 = block0 + wave * 32, j = key0 + c;
  const bool in = j < p.TK;

  V rows[kSteps], values[VALUES ? 1 : kSteps];
  const long long row = (((long long)b * p.TK + (in ? j : 0)) * p.HK + hk) * p.D;
#pragma unroll
  for (int n = 0; n < kSteps; ++n) {
    rows[n] = fragment_of(k + row, 16 * n + 8 * h, p.D, in);
    if constexpr (!VALUES) values[n] = fragment_of(v + row, 16 * n + 8 * h, p.D, in);
  }
  Unit unit;
  const int n_keys = p.lengths ? min(max(p.lengths[b], 0), p.longest) : p.TK;

  f32x16 sum_k[kParts], sum_v[kParts];
#pragma unroll
  for (int n = 0; n < kParts; ++n) sum_k[n] = sum_v[n] = zeros();
  const typename Tile::Place place = Tile::place(lane);
  const unsigned stride = (unsigned)(p.HQ * p.D) * (unsigned)sizeof(T);
  const typename Tile::template Loader<256> load(stride, (unsigned)p.D * (unsigned)sizeof(T));
  const Reach *reaches = stats.reach + (long long)b * stats.chunks;
  // of chunks base .. base + 63, those with a query that sees a key of the block
  auto seeing = [&](int base) -> unsigned long long {
    bool sees = false;
    if (base + lane < stats.chunks) {
      const Reach r = reaches[base + lane];
      sees = r.lo < block0 + kBlockRows && r.hi > block0;
    }
    return __ballot(sees);
  };
  int of_head = 0;
  for (int base = 0; base < stats.chunks; base += 64) of_head += __popcll(seeing(base));
  const long long every = (long long)of_head * p.group;
  const int from = (int)(every * at.head / cuts), count = (int)(every * (at.head + 1) / cuts) - from;
  int head = hk * p.group, base = 0;
  unsigned long long left = 0;
  if (count) {
    head += from / of_head;
    left = seeing(0);
    for (int skip = from % of_head; skip > 0;) {
      const int here = __popcll(left);
      if (here <= skip) {
        skip -= here;
        left = seeing(base += 64);
      } else {
        for (; skip > 0; --skip) left &= left - 1;
      }
    }
  }
  auto find = [&] {  // the next chunk, of this head or a later one; only where there is one
    while (!left) {
      base += 64;
      if (base >= stats.chunks) base = 0, ++head;
      left = seeing(base);
    }
  };
  auto stage = [&](int chunk, unsigned to) {
    const int first = chunk * ROWS;
    const long long from = (((long long)b * p.TQ + first) * p.HQ + head) * p.D * (long long)sizeof(T);
    load((const char *)q + from, p.TQ - first, to);
    load((const char *)grad + from, p.TQ - first, to + Tile::kBytes);
    const long long stat = ((long long)b * p.HQ + head) * p.TQ + first, span = (long long)b * p.TQ + first;
    const char *from_stats = wave == 0 ? (const char *)(stats.level + stat) : wave == 1 ? (const char *)(stats.delta + stat)
                           : wave == 2 ? (const char *)(stats.lo + span) : (const char *)(stats.hi + span);
    const __amdgpu_buffer_rsrc_t buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(from_stats), 0, 0x7fffffff, 0x00020000);
    typedef MG_LDS void *LdsPointer;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (LdsPointer)(unsigned long long)(to + 2 * Tile::kBytes + (unsigned)wave * 256u), 4,
                                             (int)(lane < ROWS && first + lane < p.TQ ? (unsigned)lane * 4u : kBeyond), 0, 0, 0);
  };

  const unsigned whole_values = lds + 2 * kBuffer;
  if constexpr (VALUES) {
    const unsigned key_stride = (unsigned)(p.HK * p.D) * (unsigned)sizeof(T);
    const typename Whole::template Loader<256> load_values(key_stride, (unsigned)p.D * (unsigned)sizeof(T));
    load_values((const char *)(v + (((long long)b * p.TK + block0) * p.HK + hk) * p.D), p.TK - block0, whole_values);
  }
  unsigned side = 0;
  int chunk = 0, hq = 0;
  if (count) {
    find();
    chunk = base + __ffsll(left) - 1, hq = head;
    stage(chunk, lds);
  }
  all_landed();
  if constexpr (VALUES)
    if (p.D % 8 && h == 0)  // the second half of a row's last piece came from behind the row, and from behind the rows of grad there, too
      *(MG_LDS unsigned long long *)(unsigned long long)(whole_values + (unsigned)(wave * 32 + c) * Whole::kRowBytes +
                                                         (unsigned)((p.D / 8) ^ Whole::turn(c)) * 16u + 8u) = 0;
  for (int n = 0; n < count; ++n) {
    const int first = chunk * ROWS, this_hq = hq;
    const Reach reach = reaches[chunk];
    if (n + 1 < count) {
      left &= left - 1;
      find();
      chunk = base + __ffsll(left) - 1, hq = head;
      stage(chunk, lds + (side ^ 1) * kBuffer);
    }
    const unsigned queries = lds + side * kBuffer, levels = queries + 2 * Tile::kBytes;  // grads between them
    if (reach.lo < key0 + 32 && reach.hi > key0) {
      const Scores how = scores_of(p, this_hq);
      const bool whole = key0 >= reach.all_lo && key0 + 32 <= reach.all_hi;
#pragma unroll 1
      for (int n = 0; n < kSubs; ++n) {
        f32x16 s = zeros(), dp = zeros();
#pragma unroll
        for (int m = 0; m < kSteps; ++m) {
          s = Fragment<T>::mma(Tile::along(queries, place, n, m), rows[m], s);
          const V value = VALUES ? Tile::along(whole_values + (unsigned)(wave * 32) * Tile::kRowBytes, place, 0, m) : values[VALUES ? 0 : m];
          dp = Fragment<T>::mma(Tile::along(queries, place, n, m, Tile::kBytes), value, dp);
        }
        const unsigned stats_at = levels + (unsigned)(32 * n + 4 * h) * 4u;  // registers r .. r + 3 are rows r * 2 and on
        auto stat = [&](int which, int r) { return *(MG_LDS const f32x4 *)(unsigned long long)(stats_at + (unsigned)(which * 256 + r * 8)); };
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const f32x4 delta = stat(1, r);
#pragma unroll
          for (int m = 0; m < 4; ++m) dp[r + m] -= delta[m];
        }
        gradients_of<T, false, BENT>(p, s, dp, how, (float)(first + 32 * n + 4 * h + n_keys - p.TQ - j), [&](int r) { return stat(0, r); });
        if (!whole) {
#pragma unroll
          for (int r = 0; r < 16; r += 4) {
            typedef int s32x4 __attribute__((ext_vector_type(4)));
            const s32x4 los = __builtin_bit_cast(s32x4, stat(2, r)), his = __builtin_bit_cast(s32x4, stat(3, r));
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const bool sees = j >= los[m] && j < his[m];
              s[r + m] = sees ? s[r + m] : 0.0f;
              dp[r + m] = sees ? dp[r + m] : 0.0f;
            }
          }
        }
        V weights[2], back[2], more[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) weights[m] = rows_of<T>(s, m, more[m]);
#pragma unroll
        for (int part = 0; part < kParts; ++part)
#pragma unroll
          for (int m = 0; m < 2; ++m) sum_v[part] = mma_of_two<T>(Tile::across(queries, place, part, 2 * n + m, Tile::kBytes), weights[m], more[m], sum_v[part]);
        in_units<T>(unit, dp, sum_k);
#pragma unroll
        for (int m = 0; m < 2; ++m) back[m] = rows_of<T>(dp, m, more[m]);
#pragma unroll
        for (int part = 0; part < kParts; ++part)
#pragma unroll
          for (int m = 0; m < 2; ++m) sum_k[part] = mma_of_two<T>(Tile::across(queries, place, part, 2 * n + m), back[m], more[m], sum_k[part]);
      }
    }
    all_landed();
    side ^= 1;
  }

  const float lift = sizeof(T) == 2 ? 0x1p-14f : 1.0f, by = sizeof(T) == 2 ? p.scale / unit.by * lift : p.scale;  // 2^-kShift
  bool odd_k = false, odd_v = false;
  if (in) {
#pragma unroll
    for (int n = 0; n < kParts; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int d = 32 * n + row_of(r, h);
        if (d >= p.D) continue;
        if (cuts == 1) {
          odd_k |= put_four(dk + row + d, four_of(sum_k[n], r) * by);
          odd_v |= put_four(dv + row + d, four_of(sum_v[n], r) * lift);
        } else {
          const long long all = (long long)p.B * p.TK * p.HK * p.D;
          put_four(parts + at.head * all + row + d, four_of(sum_k[n], r) * by);
          put_four(parts + (cuts + at.head) * all + row + d, four_of(sum_v[n], r) * lift);
        }
      }
  }
  if (cuts > 1) return;
  const unsigned marks_k = marks_of(odd_k), marks = marks_k | marks_of(odd_v);
  unsigned *which = (unsigned *)(tiles + 4 * 2 * kMaxDim * sizeof(float));  // a bit for each value of dv that is no number, behind what rows need
  static_assert(4 * 2 * kMaxDim * sizeof(float) + kBlockRows * kParts * sizeof(unsigned) <= sizeof tiles, "marks do not fit");
  if (marks) {
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
      unsigned bits = 0;
#pragma unroll
      for (int r = 0; r < 16; ++r) bits |= no_number(sum_v[n][r] * lift) && 32 * n + row_of(r, h) < p.D ? 1u << row_of(r, h) : 0u;
      bits |= __shfl_xor(bits, 32);
      if (h == 0) which[(wave * 32 + c) * kParts + n] = bits;
    }
  }
  if (lane == 0) bad[0][wave] = marks, bad[1][wave] = marks_k;
  all_landed();  // what is stored, too: other wavefronts may write it again
  each_marked<4>(bad[0], [&](int n) {
    unsigned of_v = 0;
    for (int m = lane >> 5; m < kParts; m += 2) of_v |= (which[n * kParts + m] >> (lane & 31) & 1) << (m >> 1);
    if (!dkv_stands(p, b, hk, block0 + n, bad[1][n >> 5] >> (n & 31) & 1, of_v, grad, lse, stats.delta))
      dkv_row<T, float>(p, b, hk, block0 + n, (float *)tiles + wave * 2 * kMaxDim, q, k, v, grad, lse, stats.delta, dk, dv);
  });
}

constexpr int kJoinKeys = 16;

// Adds the cuts' sums in their order, four values a thread; a block takes sixteen keys of one head.  Bound by reading them: 4 x 2048 keys, 4 heads
// of 128 in four cuts, 134 MB and 17 written, 29 us (5.2 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) attention_dkv_join_kernel(Attention p, Stats stats, int tiles, int cuts, const float *__restrict__ parts,
                                                                 const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                                                                 const T *__restrict__ grad, const float *__restrict__ lse, T *__restrict__ dk,
                                                                 T *__restrict__ dv) {
  __shared__ unsigned bad[2], which[kJoinKeys][kMaxDim / 32];  // rows as in attention_dkv_kernel, and a bit for each value of dv
  __shared__ float mine[4][2 * kMaxDim];
  if (threadIdx.x < 2) bad[threadIdx.x] = 0;
  if (threadIdx.x < kJoinKeys * (kMaxDim / 32)) which[0][threadIdx.x] = 0;
  __syncthreads();
  const int pair = blockIdx.x / tiles, tile = blockIdx.x % tiles, b = pair / p.HK, hk = pair % p.HK, of_row = p.D / 4;
  const long long all = (long long)p.B * p.TK * p.HK * p.D;
  for (int n = threadIdx.x; n < 2 * kJoinKeys * of_row; n += 256) {
    const int of_v = n / (kJoinKeys * of_row), rest = n - of_v * kJoinKeys * of_row, row = rest / of_row, j = tile * kJoinKeys + row, d = rest % of_row * 4;
    if (j >= p.TK) continue;
    const long long at = (((long long)b * p.TK + j) * p.HK + hk) * p.D + d;
    f32x4 sum{};
    for (int m = 0; m < cuts; ++m) sum += *(const f32x4 *)(parts + (of_v * cuts + m) * all + at);
    if (put_four((of_v ? dv : dk) + at, sum)) {
      atomicOr(&bad[0], 1u << row);
      if (!of_v) atomicOr(&bad[1], 1u << row);
#pragma unroll
      for (int m = 0; m < 4; ++m)
        if (of_v && no_number(sum[m])) atomicOr(&which[row][d >> 5], 1u << ((d & 31) + m));
    }
  }
  all_landed();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  each_marked<1>(bad, [&](int n) {
    unsigned of_v = 0;
#pragma unroll
    for (int c = 0; c < kParts; ++c) of_v |= (which[n][2 * c + (lane >> 5)] >> (lane & 31) & 1) << c;
    if (!dkv_stands(p, b, hk, tile * kJoinKeys + n, bad[1] >> n & 1, of_v, grad, lse, stats.delta))
      dkv_row<T, float>(p, b, hk, tile * kJoinKeys + n, mine[wave], q, k, v, grad, lse, stats.delta, dk, dv);
  });
}

// How many cuts the blocks of attention_dkv_kernel are made in: as many as make the estimate of the time least.  A block takes `chunk` for each
// chunk of queries it goes through, while two of them on a compute unit run beside each other in float16 (in float32 one keeps the matrix cores
// four fifths busy), and the first keys of a causal mask are seen by all queries, twice the mean.  Joining takes a launch and 16 bytes written
// and read for each value of k and cut.  Measured with the join at 4 x 2048 tokens, 16 heads over 4, causal, float16: 490 us in one piece, 297 in two, 258 in
// four; 4 x 75 tokens, 32 heads over 4: 64 in one, 45 in two, 35 in eight.
int cuts_of(const Attention &p, const Stats &stats, int size, int blocks) {
  const double at_once = (size == 2 ? 2.0 : 1.25) * runtime().props.multiProcessorCount, every = (double)p.group * stats.chunks;
  const double chunk = 1e-6 + stats.rows * 128.0 * ((p.D + 31) / 32 * 32) * 8 / (size == 2 ? 3.0e12 : 0.5e12);
  const double bytes = 16.0 * p.B * p.TK * p.HK * p.D;
  int best = 1;
  double least = 0;
  for (int cuts = 1; cuts <= 32 && cuts <= every; cuts *= 2) {
    const double turns = std::max(blocks * every * (p.causal ? 0.5 : 1.0) / at_once, every / cuts);
    const double time = turns * chunk + (cuts > 1 ? 5e-6 + cuts * bytes / 3e12 : 0.0);
    if (cuts == 1 || time < least) best = cuts, least = time;
  }
  return best;
}

template <typename T, int ROWS>
int backward_of(const Attention &p, const void *q, const void *k, const void *v, const void *out, const void *rest, const void *lse,
                const void *grad, void *dq, void *dk, void *dv) {
  Stats stats{};
  stats.rows = sizeof(T) == 2 && p.D > 96 ? 32 : ROWS, stats.chunks = (int)ceil_div(p.TQ, stats.rows);
  const size_t rows = (size_t)p.B * p.TQ, all = rows * p.HQ, chunks = (size_t)p.B * stats.chunks, keys = (size_t)p.B * p.TK * p.HK * p.D;
  const int key_tiles = (int)ceil_div(p.TK, kBlockRows), cuts = dk ? cuts_of(p, stats, sizeof(T), p.B * p.HK * key_tiles) : 1;
  const bool few = dq && few_take(p, sizeof(T));
  // sums of splits of dq and of cuts of dk and dv: one after the other
  const size_t sums = std::max(cuts > 1 ? 8 * cuts * keys : 0, few ? few_dq_bytes(p) : 0);
  void *space = nullptr;
  int rc = workspace(sums + sizeof(Reach) * chunks + 4 * (2 * all + 2 * rows), &space);
  if (rc) return rc;
  float *partial = (float *)space;  // whole pieces of 16 bytes: dim is a multiple of 4
  stats.reach = (Reach *)((char *)space + sums);
  stats.level = (float *)(stats.reach + chunks);
  stats.delta = stats.level + all;
  stats.lo = (int *)(stats.delta + all);
  stats.hi = stats.lo + rows;
  hipStream_t s = runtime().stream;
  const T *tq = (const T *)q, *tk = (const T *)k, *tv = (const T *)v, *tg = (const T *)grad;
  const float *tl = (const float *)lse;
  {
    ScopedTiming timed(TAG_ATTENTION_DELTA);
    attention_stats_kernel<T><<<dim3((unsigned)(p.B * p.HQ * stats.chunks)), dim3(256), 0, s>>>(p, stats, (const T *)out, (const _Float16 *)rest, tl, tg);
    MG_HIP(hipGetLastError());
  }
  if (few) {
    rc = dq_few(p, stats, sizeof(T) == 2 ? MG_F16 : MG_F32, q, k, v, grad, lse, dq, partial);
    if (rc) return rc;
  } else if (dq) {
    ScopedTiming timed(TAG_ATTENTION_DQ);
    const Deal deal = deal_of(p, p.group, (int)ceil_div(p.TQ, kBlockRows));
    with_shape<T>(p, [&](auto dim, auto bent) {
      attention_dq_kernel<T, dim, dim <= 128 ? ROWS : 32, bent><<<dim3((unsigned)(deal.pairs * deal.heads * deal.tiles)), dim3(256), 0, s>>>(
          p, deal, stats, tq, tk, tv, tg, tl, (T *)dq);
    });
    MG_HIP(hipGetLastError());
  }
  if (!dk) return MG_OK;
  {
    ScopedTiming timed(TAG_ATTENTION_DKV);
    const Deal deal = deal_of(p, cuts, key_tiles);
    with_shape<T>(p, [&](auto dim, auto bent) {
      constexpr bool wide = sizeof(T) == 2 && dim >= 128;
      attention_dkv_kernel<T, dim, wide ? 32 : ROWS, wide, bent><<<dim3((unsigned)(deal.pairs * deal.heads * deal.tiles)), dim3(256), 0, s>>>(
          p, deal, stats, tq, tk, tv, tg, tl, (T *)dk, (T *)dv, cuts, partial);
    });
    MG_HIP(hipGetLastError());
  }
  if (cuts == 1) return MG_OK;
  ScopedTiming timed(TAG_ATTENTION_JOIN);
  const int join_tiles = (int)ceil_div(p.TK, kJoinKeys);
  attention_dkv_join_kernel<T><<<dim3((unsigned)(p.B * p.HK * join_tiles)), dim3(256), 0, s>>>(p, stats, join_tiles, cuts, partial, tq, tk, tv, tg, tl, (T *)dk,
                                                                                               (T *)dv);
  MG_HIP(hipGetLastError());
  return MG_OK;
}

}  // namespace

// Head dimensions that are multiples of 4, up to 128 or, in float16, 256, in buffers that start on 16 bytes, rows of a tile within reach
// of 32 bits.  Of 256 values a block has a compute unit to itself: 2048 causal tokens, 8 heads over 2, float16, 69 us forward and 102 dq (both 32
// columns a block), 310 dk and dv and 44 to join them (3127, 3472 and 24976 us a row at a time).
bool tiles_take(const Attention &p, int size, uintptr_t ends) {
  return p.D <= (size == 2 ? 256 : 128) && p.D % 4 == 0 && ends % 16 == 0 && (long long)p.HQ * p.D * size * 128 < (1ll << 31) &&
         (long long)p.B * p.HQ * ceil_div(p.TQ, 32) < (1 << 24) && (long long)p.B * p.HK * ceil_div(p.TK, 32) < (1 << 24);
}

// Up to 32 queries one head would not fill a wavefront's columns.  And a few blocks of 128 queries, each on a compute unit of its own, are slower
// than four times as many of 32 columns whose keys four wavefronts share: in float16 while that leaves half the units idle, in float32, whose
// products take longer than the keys' way, up to a block a unit.  Forward and dq, microseconds on tiles and here: float16, 4096 causal tokens of two
// heads of 128 249 against 109, 2 x 769 of 4 of 64 49 against 27, 1024 of 16 of 128 83 against 62, and beyond the rule 4096 of 8 258 against 238;
// float32, 1500 causal tokens of 12 heads of 128 497 against 230, 4 x 1024 of 8 of 64, with no mask, 211 against 201, beyond it 4 x 2048 684 against 697.
bool few_take(const Attention &p, int size) {
  return p.TQ <= 32 || (size == 4 ? 1 : 2) * (long long)p.B * p.HQ * ceil_div(p.TQ, kBlockRows) <= runtime().props.multiProcessorCount;
}

int forward_tiles(const Attention &p, int dtype, const void *q, const void *k, const void *v, void *out, void *rest, void *lse) {
  ScopedTiming timed(TAG_ATTENTION);
  const Deal deal = deal_of(p, p.group, (int)ceil_div(p.TQ, kBlockRows));
  const dim3 grid((unsigned)(deal.pairs * deal.heads * deal.tiles));
  auto launch = [&](auto zero) {
    using T = decltype(zero);
    with_shape<T>(p, [&](auto dim, auto bent) {
      attention_tiles_kernel<T, dim, sizeof(T) == 2 && dim <= 128 ? 64 : 32, bent><<<grid, dim3(256), 0, runtime().stream>>>(
          p, deal, (const T *)q, (const T *)k, (const T *)v, (T *)out, (_Float16 *)rest, (float *)lse);
    });
  };
  dtype == MG_F16 ? launch(_Float16(0)) : launch(0.0f);
  MG_HIP(hipGetLastError());
  return MG_OK;
}

int backward_tiles(const Attention &p, int dtype, const void *q, const void *k, const void *v, const void *out, const void *rest, const void *lse,
                   const void *grad, void *dq, void *dk, void *dv) {
  return dtype == MG_F16 ? backward_of<_Float16, 64>(p, q, k, v, out, rest, lse, grad, dq, dk, dv)
                         : backward_of<float, 32>(p, q, k, v, out, rest, lse, grad, dq, dk, dv);
}

}  // namespace mg
