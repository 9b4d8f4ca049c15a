// Attention of few queries, or of few blocks of them: 32 queries x heads that share a key head make up the 32 columns of a block (a group of
// eight heads and four tokens, say), its four wavefronts take every fourth tile of 32 keys, each with a running softmax (or sums of a
// gradient) of its own over tiles that it brings into LDS for itself, without a barrier; they are joined through LDS at the end.  Where
// that makes few blocks still, the keys are split among blocks, which are joined by a second launch.
//
// With a step of generation over a cache this is bound by reading keys and values once: the sixteen products of a tile (128 values a head, float16)
// wait for its bytes even where most columns are empty.  32 histories of 4000 to 8000 tokens, 32 heads over 8 of 128 in float16 (787 MB): 154 us, 5.1
// TB/s (a stream that only reads reaches 6.25, a copy 5.2); one history of 131001 tokens with a cap (537 MB): 105 and 6 to join, 4.8 TB/s.  At 128 values a
// head a block holds 128 KB of tiles, one block a compute unit: four wavefronts with two tiles of 16 KB each (float32 one of twice that).
#include "attention_tiles.h"

#include "attention_row.h"

#include <algorithm>

namespace mg {

namespace {

constexpr int kMostSplits = 2048;

struct Split {
  int splits;   // blocks along the keys
  int columns;  // query heads of a key head times queries
  int panels;   // of 32 columns
};

// What a lane has to know of its column, and the block of its keys.  Column n of a pair of batch item and key head is query n / group, head
// n % group.  Panels with the last queries, which see most where the mask is causal, come first, of all pairs.
struct Panel {
  int part, pair, b, hk, first_column, columns;
  int i, hq;
  bool in;
  Span span;
  Reach reach;
  int first, last;  // tiles of 32 keys from reach.lo on
};

__device__ __forceinline__ Panel panel_of(const Attention &p, const Split &split, int c) {
  Panel at;
  at.part = blockIdx.x % split.splits;
  const int rest = blockIdx.x / split.splits, pairs = p.B * p.HK, panel = split.panels - 1 - rest / pairs;
  at.pair = rest % pairs;
  at.b = at.pair / p.HK, at.hk = at.pair % p.HK;
  at.first_column = panel * 32, at.columns = min(32, split.columns - panel * 32);
  const int column = at.first_column + c;
  at.i = column / p.group, at.hq = at.hk * p.group + column % p.group;
  at.in = c < at.columns;
  at.span = at.in ? span_of(p, at.b, at.i) : Span{0, 0, 0};
  at.reach = reach_of(at.span, at.in);
  const int tiles = at.reach.hi > at.reach.lo ? (at.reach.hi - at.reach.lo + 31) / 32 : 0;
  at.first = (int)((long long)tiles * at.part / split.splits), at.last = (int)((long long)tiles * (at.part + 1) / split.splits);
  return at;
}

// A wavefront's every fourth tile: brings keys and values into its own part of LDS, one tile ahead where there is room (STAGES 2), and calls
// f(the tile's place, its first key, whether all columns see all of it).
template <typename T, typename Tile, int STAGES, typename F>
__device__ __forceinline__ void each_tile(const Attention &p, const Panel &at, const void *k, const void *v, unsigned lds, int wave, F f) {
  const unsigned stride = (unsigned)(p.HK * p.D) * (unsigned)sizeof(T);
  const typename Tile::template Loader<64> load(stride, (unsigned)p.D * (unsigned)sizeof(T));
  const long long head = (((long long)at.b * p.TK + at.reach.lo) * p.HK + at.hk) * p.D * (long long)sizeof(T);
  const char *kb = (const char *)k + head, *vb = (const char *)v + head;
  auto stage = [&](int t, int side) {
    const long long from = (long long)t * 32 * stride;
    const unsigned to = lds + (unsigned)side * (2 * Tile::kBytes);
    load(kb + from, at.reach.hi - at.reach.lo - t * 32, to);
    load(vb + from, at.reach.hi - at.reach.lo - t * 32, to + Tile::kBytes);
  };
  int side = 0;
  if (at.first + wave < at.last) stage(at.first + wave, 0);
  for (int t = at.first + wave; t < at.last; t += 4) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const bool more = t + 4 < at.last;
    if (STAGES == 2 && more) stage(t + 4, side ^ 1);
    const int key0 = at.reach.lo + t * 32;
    f(lds + (unsigned)side * (2 * Tile::kBytes), key0, key0 >= at.reach.all_lo && key0 + 32 <= at.reach.all_hi);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (STAGES == 2)
      side ^= 1;
    else if (more)
      stage(t + 4, 0);
  }
}

// The four wavefronts' sums, times `by`, side by side in LDS: wavefront, column, value.
template <int DP>
struct Joined {
  static constexpr int kPitch = DP + 4, kBytes = 4 * 32 * kPitch * 4;

  static __device__ __forceinline__ void put(float *space, const f32x16 (&sums)[DP / 32], float by, int wave, int c, int h) {
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *(f32x4 *)(space + (wave * 32 + c) * kPitch + 32 * n + row_of(r, h)) = f32x4{sums[n][r], sums[n][r + 1], sums[n][r + 2], sums[n][r + 3]} * by;
  }

  static __device__ __forceinline__ f32x4 sum(const float *space, int column, int d) {
    f32x4 sum = *(const f32x4 *)(space + column * kPitch + d);
#pragma unroll
    for (int w = 1; w < 4; ++w) sum += *(const f32x4 *)(space + (w * 32 + column) * kPitch + d);
    return sum;
  }
};

// With one split the result itself; else sums at the block's own top, and that with the total.
template <typename T, int DP, int STAGES, bool BENT>
__global__ void __launch_bounds__(256) attention_few_kernel(Attention p, Split split, const T *__restrict__ q, const T *__restrict__ k,
                                                            const T *__restrict__ v, T *__restrict__ out, _Float16 *__restrict__ remains,
                                                            float *__restrict__ lse, float *__restrict__ sums, float2 *__restrict__ ends) {
  typedef TileOf<T, DP, 32> Tile;
  typedef typename Fragment<T>::V V;
  typedef Joined<DP> Join;
  constexpr int kSteps = DP / 16, kTiles = 4 * STAGES * 2 * Tile::kBytes;
  __shared__ __attribute__((aligned(1024))) char space[kTiles > Join::kBytes ? kTiles : Join::kBytes];
  __shared__ float tops[4][32], totals[4][32];
  __shared__ unsigned bad, numbers;  // columns with one that is no number, and those of them whose total is one
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
  const Panel at = panel_of(p, split, c);

  V rows[kSteps];
  const T *row = q + (((long long)at.b * p.TQ + (at.in ? at.i : 0)) * p.HQ + at.hq) * p.D;
#pragma unroll
  for (int n = 0; n < kSteps; ++n) rows[n] = fragment_of(row, 16 * n + 8 * h, p.D, at.in);
  const Scores how = scores_of(p, at.hq);

  Running<T, DP, 1, BENT> run;
  run.begin();
  const typename Tile::Place place = Tile::place(lane);
  const unsigned lds = (unsigned)(unsigned long long)(MG_LDS char *)space + (unsigned)wave * (STAGES * 2 * Tile::kBytes);
  each_tile<T, Tile, STAGES>(p, at, k, v, lds, wave, [&](unsigned keys, int key0, bool whole) {
    run.take(p, how, keys, keys + Tile::kBytes, rows, at.span, key0, whole, place, h);
  });

  const float total = sum_halves(run.total);
  if (h == 0) tops[wave][c] = run.top, totals[wave][c] = total;
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int n = 0; n < 4; ++n) top = __builtin_fmaxf(top, tops[n][c]);
  float *join = (float *)space;
  Join::put(join, run.sums, run.top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(run.top - top), wave, c, h);
  float all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w)  // without a top the total is 0, or no number where no score is one
    all += totals[w][c] * (tops[w][c] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(tops[w][c] - top));
  __syncthreads();
  const long long base = ((long long)at.pair * split.splits + at.part) * split.columns + at.first_column;
  if (split.splits > 1) {
    for (int n = threadIdx.x; n < at.columns * (DP / 4); n += 256) {
      const int column = n / (DP / 4), d = n % (DP / 4) * 4;
      if (d < p.D) *(f32x4 *)(sums + (base + column) * p.D + d) = Join::sum(join, column, d);
    }
    if ((int)threadIdx.x < at.columns) ends[base + c] = make_float2(top, all);
    return;
  }
  if (wave == 0 && h == 0) {
    tops[0][c] = all > 0 ? 1.0f / all : all == 0 ? 0.0f : NAN;
    if (lse && at.in) lse[((long long)at.b * p.HQ + at.hq) * p.TQ + at.i] = all == 0 ? INFINITY : top + __builtin_log2f(all) - kLift;
  }
  if (threadIdx.x == 0) bad = numbers = 0;
  __syncthreads();
  for (int n = threadIdx.x; n < at.columns * (DP / 4); n += 256) {
    const int column = n / (DP / 4), d = n % (DP / 4) * 4, all_columns = at.first_column + column;
    if (d >= p.D) continue;
    const float by = tops[0][column];
    const f32x4 value = Join::sum(join, column, d) * by;
    const long long to = (((long long)at.b * p.TQ + all_columns / p.group) * p.HQ + at.hk * p.group + all_columns % p.group) * p.D + d;
    if (put_four(out + to, value)) {
      atomicOr(&bad, 1u << column);
      if (by == by) atomicOr(&numbers, 1u << column);
    }
    if constexpr (sizeof(T) == 2) {
      if (remains) put_four(remains + to, (value - __builtin_convertvector(__builtin_convertvector(value, f16x4), f32x4)) * kRest);
    }
  }
  all_landed();  // what is stored, too: other wavefronts may write it again
  OddValues &values = *(OddValues *)(space + 4 * kMaxDim * sizeof(float));  // behind what rows need
  static_assert(4 * kMaxDim * sizeof(float) + sizeof values <= sizeof space, "no room for them");
  if (numbers) values.find(p, at.b, at.hk, at.reach.lo, at.reach.hi, v);
  each_marked<1>(&bad, [&](int n) {
    const int column = at.first_column + n, hq = at.hk * p.group + column % p.group, i = column / p.group;
    if (numbers >> n & 1 ? !out_settled(p, at.b, hq, i, values, v, out, remains) : !out_stands(p, at.b, hq, i, q, k))
      attend_row<T, float>(p, at.b, hq, i, (float *)space + wave * kMaxDim, q, k, v, out, remains, lse);
  });
}

// A block per row of the result: the splits' sums at a common top, in their order.  A row that comes out as no number is computed once more, unless
// what it sees explains it, so that what it does not see leaves no mark (products with weights of zero do, where that is no number).
template <typename T, int PARTS>
__global__ void __launch_bounds__(256) attention_join_kernel(Attention p, Split split, const float *__restrict__ sums, const float2 *__restrict__ ends,
                                                             const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                                                             T *__restrict__ out, _Float16 *__restrict__ rest, float *__restrict__ lse) {
  __shared__ float parts[4][64 * PARTS], totals[4], mine[kMaxDim], weights[kMostSplits];
  __shared__ int odd[4];
  __shared__ OddValues values;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int hq = blockIdx.x % p.HQ, i = blockIdx.x / p.HQ % p.TQ, b = blockIdx.x / p.HQ / p.TQ;
  const long long first = ((long long)b * p.HK + hq / p.group) * split.splits * split.columns + i * p.group + hq % p.group;
  float top = -INFINITY;
  for (int n = lane; n < split.splits; n += 64) top = __builtin_fmaxf(top, ends[first + (long long)n * split.columns].x);
  top = wave_max(top);
  float total = 0, sum[PARTS] = {};
  for (int n = threadIdx.x; n < split.splits; n += 256) {
    const float2 end = ends[first + (long long)n * split.columns];
    weights[n] = end.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(end.x - top);
    total += end.y * weights[n];
  }
  total = wave_sum(total);
  __syncthreads();
  const float *from = sums + first * p.D;
  const long long step = (long long)split.columns * p.D;
  int at[PARTS];  // values that the row does not have repeat its first
#pragma unroll
  for (int m = 0; m < PARTS; ++m) at[m] = lane + 64 * m < p.D ? lane + 64 * m : 0;
#pragma unroll 8
  for (int n = wave; n < split.splits; n += 4) {
    const float by = weights[n];
#pragma unroll
    for (int m = 0; m < PARTS; ++m) sum[m] += from[n * step + at[m]] * by;
  }
#pragma unroll
  for (int m = 0; m < PARTS; ++m) parts[wave][lane + 64 * m] = sum[m];
  if (lane == 0) totals[wave] = total;
  __syncthreads();
  total = totals[0] + totals[1] + totals[2] + totals[3];
  const long long to = (((long long)b * p.TQ + i) * p.HQ + hq) * p.D;
  bool bad = !(total < INFINITY);
  if ((int)threadIdx.x < p.D) {
    const int d = threadIdx.x;
    const float value = total == 0 ? 0.0f : (parts[0][d] + parts[1][d] + parts[2][d] + parts[3][d]) / total;
    const T near = (T)value;
    out[to + d] = near;
    if (rest) rest[to + d] = (_Float16)((value - (float)near) * kRest);
    bad |= no_number(value);
  }
  if (lse && threadIdx.x == 0) lse[((long long)b * p.HQ + hq) * p.TQ + i] = total == 0 ? INFINITY : top + __builtin_log2f(total) - kLift;
  bad = __any(bad);
  if (lane == 0) odd[wave] = bad;
  all_landed();  // what is stored, too: it may be written again
  if (!(odd[0] | odd[1] | odd[2] | odd[3])) return;
  if (total == total) {
    const Span span = span_of(p, b, i);
    values.find(p, b, hq / p.group, span.lo, span.hi, v);
  }
  if (wave == 0 && (total == total ? !out_settled(p, b, hq, i, values, v, out, rest) : !out_stands(p, b, hq, i, q, k)))
    attend_row<T, float>(p, b, hq, i, mine, q, k, v, out, rest, lse);
}

// dq of a panel's columns; with one split the result itself.  Up to 64 values a head two blocks share a compute unit: 77 us for
// 4 x 1024 tokens behind a prefix, 8 heads of 64 in float32, where registers for one block alone made it 94.
template <typename T, int DP, int STAGES, bool BENT>
__global__ void __launch_bounds__(256, DP <= 64 ? 2 : 1) attention_few_dq_kernel(Attention p, Split split, Stats stats, const T *__restrict__ q, const T *__restrict__ k,
                                                               const T *__restrict__ v, const T *__restrict__ grad, const float *__restrict__ lse,
                                                               T *__restrict__ dq, float *__restrict__ sums) {
  typedef TileOf<T, DP, 32> Tile;
  typedef typename Fragment<T>::V V;
  typedef Joined<DP> Join;
  constexpr int kSteps = DP / 16, kTiles = 4 * STAGES * 2 * Tile::kBytes;
  __shared__ __attribute__((aligned(1024))) char space[kTiles > Join::kBytes ? kTiles : Join::kBytes];
  __shared__ unsigned bad;  // columns to be computed again
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
  const Panel at = panel_of(p, split, c);

  V rows[kSteps], grads[kSteps];
  const long long row = (((long long)at.b * p.TQ + (at.in ? at.i : 0)) * p.HQ + at.hq) * p.D;
#pragma unroll
  for (int n = 0; n < kSteps; ++n) {
    rows[n] = fragment_of(q + row, 16 * n + 8 * h, p.D, at.in);
    grads[n] = fragment_of(grad + row, 16 * n + 8 * h, p.D, at.in);
  }
  const long long stat = ((long long)at.b * p.HQ + at.hq) * p.TQ + (at.in ? at.i : 0);
  const float level = at.in ? stats.level[stat] : INFINITY, delta = at.in ? stats.delta[stat] : 0.0f;
  const unsigned stand = marks_of(dq_stands(at.span, level, delta));
  const Scores how = scores_of(p, at.hq);

  Pulled<T, DP, 32, BENT> run;
  run.begin();
  const typename Tile::Place place = Tile::place(lane);
  const unsigned lds = (unsigned)(unsigned long long)(MG_LDS char *)space + (unsigned)wave * (STAGES * 2 * Tile::kBytes);
  each_tile<T, Tile, STAGES>(p, at, k, v, lds, wave, [&](unsigned keys, int key0, bool whole) {
    run.take(p, how, keys, 0, rows, grads, level, delta, at.span, key0, whole, place, h);
  });

  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  float *join = (float *)space;
  Join::put(join, run.sums, run.by(p), wave, c, h);
  __syncthreads();
  const long long base = ((long long)at.pair * split.splits + at.part) * split.columns + at.first_column;
  for (int n = threadIdx.x; n < at.columns * (DP / 4); n += 256) {
    const int column = n / (DP / 4), d = n % (DP / 4) * 4, all_columns = at.first_column + column;
    if (d >= p.D) continue;
    const f32x4 value = Join::sum(join, column, d);
    if (split.splits > 1)
      *(f32x4 *)(sums + (base + column) * p.D + d) = value;
    else if (put_four(dq + (((long long)at.b * p.TQ + all_columns / p.group) * p.HQ + at.hk * p.group + all_columns % p.group) * p.D + d, value) &&
             !(stand >> column & 1))
      atomicOr(&bad, 1u << column);
  }
  if (split.splits > 1) return;
  all_landed();  // what is stored, too: other wavefronts may write it again
  each_marked<1>(&bad, [&](int n) {
    const int column = at.first_column + n;
    dq_row<T, float>(p, at.b, at.hk * p.group + column % p.group, column / p.group, (float *)space + wave * 2 * kMaxDim, q, k, v, grad, lse, stats.delta, dq);
  });
}

// A wavefront per row of dq.
template <typename T, int PARTS>
__global__ void __launch_bounds__(256) attention_dq_join_kernel(Attention p, Split split, Stats stats, const float *__restrict__ sums,
                                                                const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                                                                const T *__restrict__ grad, const float *__restrict__ lse, T *__restrict__ dq) {
  __shared__ float mine[4][2 * kMaxDim];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long at_row = (long long)blockIdx.x * 4 + wave;
  if (at_row >= (long long)p.B * p.TQ * p.HQ) return;
  const int hq = (int)(at_row % p.HQ), i = (int)(at_row / p.HQ % p.TQ), b = (int)(at_row / p.HQ / p.TQ);
  const long long first = ((long long)b * p.HK + hq / p.group) * split.splits * split.columns + i * p.group + hq % p.group;
  const float *from = sums + first * p.D;
  const long long step = (long long)split.columns * p.D;
  float sum[PARTS] = {};
  int at[PARTS];  // values that the row does not have repeat its first
#pragma unroll
  for (int m = 0; m < PARTS; ++m) at[m] = lane + 64 * m < p.D ? lane + 64 * m : 0;
#pragma unroll 8
  for (int n = 0; n < split.splits; ++n)
#pragma unroll
    for (int m = 0; m < PARTS; ++m) sum[m] += from[n * step + at[m]];
  bool odd = false;
#pragma unroll
  for (int m = 0; m < PARTS; ++m)
    if (lane + 64 * m < p.D) dq[at_row * p.D + lane + 64 * m] = (T)sum[m], odd |= !(__builtin_fabsf(sum[m]) < INFINITY);
  const long long stat = ((long long)b * p.HQ + hq) * p.TQ + i;
  if (__any(odd) && !dq_stands(span_of(p, b, i), stats.level[stat], stats.delta[stat])) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    dq_row<T, float>(p, b, hq, i, mine[wave], q, k, v, grad, lse, stats.delta, dq);
  }
}

// f(values of a row that a lane of 64 holds)
template <typename F>
void with_parts(const Attention &p, F f) {
  if (p.D <= 64)
    f(std::integral_constant<int, 1>{});
  else if (p.D <= 128)
    f(std::integral_constant<int, 2>{});
  else
    f(std::integral_constant<int, 4>{});
}

// Tiles ahead of four wavefronts: as many as there is room for.
template <typename T>
constexpr int stages_of(int dim) { return sizeof(T) == 2 && dim <= 128 ? 2 : 1; }

// Keys are split until there is a block for each compute unit, and no further: at 128 values a head, where this was measured, a block takes a unit's
// LDS to itself, so the next one's first tiles wait for its last (at 64 two blocks would fit a unit).  One history of 131001 tokens, 32 heads over 8
// of 128, float16: 110 us with the join, 140 in eight times as many blocks; 32 of 4000 to 8000 tokens 156 in one piece, 170.  Where lengths differ, for as
// many times more as the longest has the mean.  Pieces are 128 keys (a tile for each wavefront) or more; with more queries a join takes as long as 512.
Split split_of(const Attention &p) {
  const bool single = p.TQ <= 32;
  Split split;
  split.columns = p.TQ * p.group;
  split.panels = (int)ceil_div(split.columns, 32);
  const long long pairs = (long long)p.B * p.HK * split.panels, blocks = (long long)runtime().props.multiProcessorCount * std::max(1, p.longest / std::max(p.mean, 1));
  split.splits = (int)std::min<int64_t>({kMostSplits, std::max<int64_t>(1, blocks / pairs), std::max<int64_t>(1, ceil_div(p.longest, single ? 128 : 512))});
  return split;
}

template <typename T>
int few_of(const Attention &p, const void *q, const void *k, const void *v, void *out, void *rest, void *lse) {
  const Split split = split_of(p);
  const size_t rows = split.splits > 1 ? (size_t)p.B * p.HK * split.splits * split.columns : 0;
  void *space = nullptr;
  const int rc = workspace(rows * (sizeof(float2) + p.D * sizeof(float)), &space);
  if (rc) return rc;
  float *sums = (float *)space;  // D is a multiple of 4: what follows is aligned
  float2 *ends = (float2 *)(sums + rows * p.D);
  {
    ScopedTiming timed(TAG_ATTENTION);
    const dim3 grid((unsigned)(p.B * p.HK * split.panels * split.splits));
    with_shape<T>(p, [&](auto dim, auto bent) {
      attention_few_kernel<T, dim, stages_of<T>(dim), bent><<<grid, dim3(256), 0, runtime().stream>>>(
          p, split, (const T *)q, (const T *)k, (const T *)v, (T *)out, (_Float16 *)rest, (float *)lse, sums, ends);
    });
    MG_HIP(hipGetLastError());
  }
  if (split.splits == 1) return MG_OK;
  ScopedTiming timed(TAG_ATTENTION_JOIN);
  with_parts(p, [&](auto parts) {
    attention_join_kernel<T, parts><<<dim3((unsigned)(p.B * p.TQ * p.HQ)), dim3(256), 0, runtime().stream>>>(
        p, split, sums, ends, (const T *)q, (const T *)k, (const T *)v, (T *)out, (_Float16 *)rest, (float *)lse);
  });
  MG_HIP(hipGetLastError());
  return MG_OK;
}

template <typename T>
int few_dq_of(const Attention &p, const Stats &stats, const void *q, const void *k, const void *v, const void *grad, const void *lse, void *dq, float *sums) {
  const Split split = split_of(p);
  {
    ScopedTiming timed(TAG_ATTENTION_DQ);
    const dim3 grid((unsigned)(p.B * p.HK * split.panels * split.splits));
    with_shape<T>(p, [&](auto dim, auto bent) {
      attention_few_dq_kernel<T, dim, stages_of<T>(dim), bent><<<grid, dim3(256), 0, runtime().stream>>>(
          p, split, stats, (const T *)q, (const T *)k, (const T *)v, (const T *)grad, (const float *)lse, (T *)dq, sums);
    });
    MG_HIP(hipGetLastError());
  }
  if (split.splits == 1) return MG_OK;
  ScopedTiming timed(TAG_ATTENTION_JOIN);
  with_parts(p, [&](auto parts) {
    attention_dq_join_kernel<T, parts><<<dim3((unsigned)ceil_div((int64_t)p.B * p.TQ * p.HQ, 4)), dim3(256), 0, runtime().stream>>>(
        p, split, stats, sums, (const T *)q, (const T *)k, (const T *)v, (const T *)grad, (const float *)lse, (T *)dq);
  });
  MG_HIP(hipGetLastError());
  return MG_OK;
}

}  // namespace

int forward_few(const Attention &p, int dtype, const void *q, const void *k, const void *v, void *out, void *rest, void *lse) {
  return dtype == MG_F16 ? few_of<_Float16>(p, q, k, v, out, rest, lse) : few_of<float>(p, q, k, v, out, rest, lse);
}

size_t few_dq_bytes(const Attention &p) {
  const Split split = split_of(p);
  return split.splits > 1 ? (size_t)p.B * p.HK * split.splits * split.columns * p.D * sizeof(float) : 0;
}

int dq_few(const Attention &p, const Stats &stats, int dtype, const void *q, const void *k, const void *v, const void *grad, const void *lse, void *dq,
           float *sums) {
  return dtype == MG_F16 ? few_dq_of<_Float16>(p, stats, q, k, v, grad, lse, dq, sums) : few_dq_of<float>(p, stats, q, k, v, grad, lse, dq, sums);
}

}  // namespace mg
