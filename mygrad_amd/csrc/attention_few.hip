// Attention of few queries over many keys: the tokens of a step of generation over a cache.
//
// Bound by reading keys and values once: 32 queries x heads that share a key head make up the 32 columns of a wavefront (a group of eight
// heads and four tokens, say), so the sixteen products of a tile of 32 keys wait for the tile's bytes even where most columns are empty.
// Each wavefront keeps a running softmax of its own over tiles that it brings into LDS for itself, without a barrier; the four of a block
// are joined through LDS, blocks that split one sequence's keys by a second launch.
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

// Column n of a panel is query n / group, head n % group.
template <typename T, int DP, int STAGES, bool BENT>
__global__ void __launch_bounds__(256) attention_few_kernel(Attention p, Split split, const T *__restrict__ q, const T *__restrict__ k,
                                                            const T *__restrict__ v, float *__restrict__ sums, float2 *__restrict__ ends) {
  typedef TileOf<T, DP, 32> Tile;
  typedef typename Fragment<T>::V V;
  constexpr int kSteps = DP / 16, kPitch = DP + 4;
  constexpr int kTiles = 4 * STAGES * 2 * Tile::kBytes, kJoin = 4 * 32 * kPitch * 4;
  __shared__ __attribute__((aligned(1024))) char space[kTiles > kJoin ? kTiles : kJoin];
  __shared__ float tops[4][32], totals[4][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
  const int part = blockIdx.x % split.splits, rest = blockIdx.x / split.splits, panel = rest % split.panels, pair = rest / split.panels;
  const int b = pair / p.HK, hk = pair % p.HK;
  const int column = panel * 32 + c, i = column / p.group, hq = hk * p.group + column % p.group;
  const bool in = column < split.columns;
  const Span span = in ? span_of(p, b, i) : Span{0, 0, 0};
  const Reach reach = reach_of(span, in);

  V rows[kSteps];
  const T *row = q + (((long long)b * p.TQ + (in ? i : 0)) * p.HQ + hq) * p.D;
#pragma unroll
  for (int n = 0; n < kSteps; ++n) rows[n] = fragment_of(row, 16 * n + 8 * h, p.D, in);
  const Scores how = scores_of(p, hq);

  const int tiles = reach.hi > reach.lo ? (reach.hi - reach.lo + 31) / 32 : 0;
  const int first = (int)((long long)tiles * part / split.splits), last = (int)((long long)tiles * (part + 1) / split.splits);
  const unsigned stride = (unsigned)(p.HK * p.D) * (unsigned)sizeof(T);
  const typename Tile::template Loader<64> load(stride, (unsigned)p.D * (unsigned)sizeof(T));
  const long long head = (((long long)b * p.TK + reach.lo) * p.HK + hk) * p.D * (long long)sizeof(T);
  const char *kb = (const char *)k + head, *vb = (const char *)v + head;
  const unsigned lds = (unsigned)(unsigned long long)(MG_LDS char *)space + (unsigned)wave * (STAGES * 2 * Tile::kBytes);
  auto stage = [&](int t, int side) {
    const long long from = (long long)t * 32 * stride;
    const unsigned to = lds + (unsigned)side * (2 * Tile::kBytes);
    load(kb + from, stride, reach.hi - reach.lo - t * 32, to);
    load(vb + from, stride, reach.hi - reach.lo - t * 32, to + Tile::kBytes);
  };

  Running<T, DP, 1, BENT> run;
  run.begin();
  const typename Tile::Place place = Tile::place(lane);
  int side = 0;
  if (first + wave < last) stage(first + wave, 0);
  for (int t = first + wave; t < last; t += 4) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const bool more = t + 4 < last;
    if (STAGES == 2 && more) stage(t + 4, side ^ 1);
    const int key0 = reach.lo + t * 32;
    const unsigned keys = lds + (unsigned)side * (2 * Tile::kBytes);
    run.take(p, how, keys, keys + Tile::kBytes, rows, span, key0, key0 >= reach.all_lo && key0 + 32 <= reach.all_hi, place, h);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (STAGES == 2)
      side ^= 1;
    else if (more)
      stage(t + 4, 0);
  }

  // the block's four: sums at a common top, one after the other's space
  const float total = sum_halves(run.total);
  if (h == 0) tops[wave][c] = run.top, totals[wave][c] = total;
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int n = 0; n < 4; ++n) top = __builtin_fmaxf(top, tops[n][c]);
  const float by = run.top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(run.top - top);
  float *join = (float *)space;
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *(f32x4 *)(join + (wave * 32 + c) * kPitch + 32 * n + row_of(r, h)) =
          f32x4{run.sums[n][r], run.sums[n][r + 1], run.sums[n][r + 2], run.sums[n][r + 3]} * by;
  __syncthreads();
  const int columns = min(32, split.columns - panel * 32);
  const long long base = ((long long)pair * split.splits + part) * split.columns + panel * 32;
  for (int n = threadIdx.x; n < columns * (DP / 4); n += 256) {
    const int column = n / (DP / 4), d = n % (DP / 4) * 4;
    if (d >= p.D) continue;
    f32x4 sum = *(const f32x4 *)(join + column * kPitch + d);
#pragma unroll
    for (int w = 1; w < 4; ++w) sum += *(const f32x4 *)(join + (w * 32 + column) * kPitch + d);
    *(f32x4 *)(sums + (base + column) * p.D + d) = sum;
  }
  if ((int)threadIdx.x < columns) {
    float all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (tops[w][c] != -INFINITY) all += totals[w][c] * __builtin_amdgcn_exp2f(tops[w][c] - top);
    ends[base + c] = make_float2(top, all);
  }
}

// A block per row of the result: the splits' sums at a common top, in their order.  A row that comes out as no number is computed once more, so
// that what it does not see leaves no mark (products with weights of zero do, where that is no number).
template <typename T>
__global__ void __launch_bounds__(256) attention_join_kernel(Attention p, Split split, const float *__restrict__ sums, const float2 *__restrict__ ends,
                                                             const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                                                             T *__restrict__ out, _Float16 *__restrict__ rest, float *__restrict__ lse) {
  __shared__ float parts[4][128], totals[4], mine[kMaxDim], weights[kMostSplits];
  __shared__ int odd[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int hq = blockIdx.x % p.HQ, i = blockIdx.x / p.HQ % p.TQ, b = blockIdx.x / p.HQ / p.TQ;
  const long long first = ((long long)b * p.HK + hq / p.group) * split.splits * split.columns + i * p.group + hq % p.group;
  float top = -INFINITY;
  for (int n = lane; n < split.splits; n += 64) top = __builtin_fmaxf(top, ends[first + (long long)n * split.columns].x);
  top = wave_max(top);
  float total = 0, sum0 = 0, sum1 = 0;
  for (int n = threadIdx.x; n < split.splits; n += 256) {
    const float2 end = ends[first + (long long)n * split.columns];
    weights[n] = end.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(end.x - top);
    total += end.y * weights[n];
  }
  total = wave_sum(total);
  __syncthreads();
  const float *from = sums + first * p.D + (lane < p.D ? lane : 0);
  const long long step = (long long)split.columns * p.D;
  const int second = lane + 64 < p.D ? 64 : 0;
#pragma unroll 8
  for (int n = wave; n < split.splits; n += 4) {
    const float by = weights[n];
    sum0 += from[n * step] * by;
    sum1 += from[n * step + second] * by;
  }
  parts[wave][lane] = sum0, parts[wave][lane + 64] = sum1;
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
    bad |= !(__builtin_fabsf(value) < INFINITY);
  }
  if (lse && threadIdx.x == 0) lse[((long long)b * p.HQ + hq) * p.TQ + i] = total == 0 ? INFINITY : top + __builtin_log2f(total) - kLift;
  bad = __any(bad);
  if (lane == 0) odd[wave] = bad;
  all_landed();  // what is stored, too: it may be written again
  if (wave == 0 && (odd[0] | odd[1] | odd[2] | odd[3])) attend_row<T, float>(p, b, hq, i, mine, q, k, v, out, rest, lse);
}

template <typename T>
int few_of(const Attention &p, const void *q, const void *k, const void *v, void *out, void *rest, void *lse) {
  constexpr int kStages = sizeof(T) == 2 ? 2 : 1;  // as many as four wavefronts have room for at 128 values a head
  Split split;
  split.columns = p.TQ * p.group;
  split.panels = (int)ceil_div(split.columns, 32);
  // A block for each 128 keys (a tile for each wavefront) while there are fewer than fill the device eight times over: a batch of ragged lengths
  // evens out over that many.
  const int pairs = p.B * p.HK * split.panels, most = std::min(kMostSplits, std::max(1, 8 * runtime().props.multiProcessorCount / pairs));
  split.splits = (int)std::min<int64_t>(most, std::max<int64_t>(1, ceil_div(p.longest, 128)));
  const size_t rows = (size_t)p.B * p.HK * split.splits * split.columns;
  void *space = nullptr;
  const int rc = workspace(rows * (sizeof(float2) + p.D * sizeof(float)), &space);
  if (rc) return rc;
  float *sums = (float *)space;  // D is a multiple of 8: what follows is aligned
  float2 *ends = (float2 *)(sums + rows * p.D);
  {
    ScopedTiming timed(TAG_ATTENTION);
    const dim3 grid((unsigned)(p.B * p.HK * split.panels * split.splits));
    with_shape(p, [&](auto dim, auto bent) {
      attention_few_kernel<T, dim, kStages, bent><<<grid, dim3(256), 0, runtime().stream>>>(p, split, (const T *)q, (const T *)k, (const T *)v, sums, ends);
    });
    MG_HIP(hipGetLastError());
  }
  ScopedTiming timed(TAG_ATTENTION_JOIN);
  attention_join_kernel<T><<<dim3((unsigned)(p.B * p.TQ * p.HQ)), dim3(256), 0, runtime().stream>>>(
      p, split, sums, ends, (const T *)q, (const T *)k, (const T *)v, (T *)out, (_Float16 *)rest, (float *)lse);
  MG_HIP(hipGetLastError());
  return MG_OK;
}

}  // namespace

int forward_few(const Attention &p, int dtype, const void *q, const void *k, const void *v, void *out, void *rest, void *lse) {
  return dtype == MG_F16 ? few_of<_Float16>(p, q, k, v, out, rest, lse) : few_of<float>(p, q, k, v, out, rest, lse);
}

}  // namespace mg
