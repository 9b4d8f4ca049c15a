// Attention of float16 and float32 on the matrix cores: tiles of queries against tiles of keys, one pass with the running maximum
// and sum of the softmax, nothing of the scores in memory.
#include "attention_tiles.h"

#include "attention_rows.h"

namespace mg {

namespace {

constexpr int kBlockRows = 128;  // queries of a block: 32 for each of its four wavefronts

// Weights are kept as 2^kLift times exp2(score - top): in float16 they are whole down to 2^-29 of the row's largest then.  `top` follows the
// row's maximum only when that has grown by more than kSlack, so the sums are seldom scaled; 2^(kLift + kSlack) stays below 65504.
constexpr float kLift = 7.0f, kSlack = 8.0f;

// S^T = K Q^T has a query in each lane's column, so a row's maximum and sum are taken within a lane (and its partner in the other half),
// and the weights are the right operand of out^T = V^T P^T as they lie.
template <typename T, int DP, int KEYS>
__global__ void __launch_bounds__(256, 2) attention_tiles_kernel(Attention p, Deal deal, const T *__restrict__ q, const T *__restrict__ k,
                                                                 const T *__restrict__ v, T *__restrict__ out, _Float16 *__restrict__ rest,
                                                                 float *__restrict__ lse, int *__restrict__ redo) {
  typedef TileOf<T, DP, KEYS> Tile;
  typedef typename Fragment<T>::V V;
  constexpr int kSteps = DP / 16, kParts = DP / 32, kSubs = KEYS / 32;
  __shared__ __attribute__((aligned(1024))) char tiles[4 * Tile::kBytes];
  __shared__ int edges[2][4];
  __shared__ int bad[4];
  const unsigned lds = (unsigned)(unsigned long long)(MG_LDS char *)tiles;
  const Dealt at = dealt(deal, blockIdx.x);
  const int b = at.pair / p.HK, hk = at.pair % p.HK, hq = hk * p.group + at.head;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, c = lane & 31;
  const int i = at.tile * kBlockRows + wave * 32 + c;
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
  const unsigned stride = (unsigned)(p.HK * p.D) * (unsigned)sizeof(T), dim = (unsigned)p.D * (unsigned)sizeof(T);
  const long long head = (((long long)b * p.TK + lo) * p.HK + hk) * p.D * (long long)sizeof(T);
  const char *kb = (const char *)k + head, *vb = (const char *)v + head;
  auto stage = [&](int t) {
    const long long from = (long long)t * KEYS * stride;
    const int last = hi - lo - t * KEYS;
    const unsigned to = lds + (unsigned)(t & 1) * (2 * Tile::kBytes);
    Tile::load(kb + from, stride, 0, last, dim, to);
    Tile::load(vb + from, stride, 0, last, dim, to + Tile::kBytes);
  };

  f32x16 sums[kParts];
#pragma unroll
  for (int n = 0; n < kParts; ++n) sums[n] = zeros();
  float top = -INFINITY, total = 0;
  const float bend = p.cap > 0 ? p.scale / p.cap : 0.0f, factor = (p.cap > 0 ? p.cap : p.scale) * kLog2e;
  const float slope = p.slopes ? p.slopes[hq] * kLog2e : 0.0f;

  if (count) stage(0);
  all_landed();
  for (int t = 0; t < count; ++t) {
    if (t + 1 < count) stage(t + 1);
    const int key0 = lo + t * KEYS;
    if (key0 < reach.hi && key0 + KEYS > reach.lo) {
      const unsigned keys = lds + (unsigned)(t & 1) * (2 * Tile::kBytes), values = keys + Tile::kBytes;
      f32x16 s[kSubs];
#pragma unroll
      for (int n = 0; n < kSubs; ++n) s[n] = zeros();
#pragma unroll
      for (int m = 0; m < kSteps; ++m)
#pragma unroll
        for (int n = 0; n < kSubs; ++n) s[n] = Fragment<T>::mma(Tile::along(keys, 32 * n + c, m, h), rows[m], s[n]);

      if (p.cap > 0) {
#pragma unroll
        for (int n = 0; n < kSubs; ++n) {
          s[n] *= bend;
          tanh_of_all(s[n]);
        }
      }
#pragma unroll
      for (int n = 0; n < kSubs; ++n) s[n] *= factor;
      if (p.slopes) {
        const float away = (float)(span.place - key0 - 4 * h);
#pragma unroll
        for (int n = 0; n < kSubs; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[n][r] -= slope * __builtin_fabsf(away - (float)(32 * n + row_of(r, 0)));
      }
      if (key0 < reach.all_lo || key0 + KEYS > reach.all_hi) {
        const unsigned seen = (unsigned)(span.hi - span.lo);
        const int from = key0 + 4 * h - span.lo;
#pragma unroll
        for (int n = 0; n < kSubs; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[n][r] = (unsigned)(from + 32 * n + row_of(r, 0)) < seen ? s[n][r] : -INFINITY;
      }
      float most = s[0][0];
#pragma unroll
      for (int n = 0; n < kSubs; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) most = __builtin_fmaxf(most, s[n][r]);
      most = larger_half(most);
      if (__any(most > top + kSlack)) {  // also the first keys that a row sees
        const float now = __builtin_fmaxf(top, most), back = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - now);
        top = now;
        total *= back;
#pragma unroll
        for (int n = 0; n < kParts; ++n) sums[n] *= back;
      }
      const float base = top == -INFINITY ? 0.0f : top - kLift;
#pragma unroll
      for (int n = 0; n < kSubs; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[n][r] = __builtin_amdgcn_exp2f(s[n][r] - base);
          total += s[n][r];
        }
#pragma unroll
      for (int m = 0; m < 2 * kSubs; ++m) {
        const V weights = rows_of<T>(s[m >> 1], m & 1);
#pragma unroll
        for (int n = 0; n < kParts; ++n) sums[n] = Fragment<T>::mma(Tile::across(values, n, m, lane), weights, sums[n]);
      }
    }
    all_landed();
  }

  total = sum_halves(total);
  const float by = total > 0 ? 1.0f / total : total == 0 ? 0.0f : NAN;
  bool odd = !(__builtin_fabsf(by) < INFINITY);
  if (in) {
    const long long to = (((long long)b * p.TQ + i) * p.HQ + hq) * p.D;
#pragma unroll
    for (int n = 0; n < kParts; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int d = 32 * n + row_of(r, h);
        if (d >= p.D) continue;
        f32x4 value;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          value[j] = sums[n][r + j] * by;
          odd |= !(__builtin_fabsf(value[j]) < INFINITY);
        }
        if constexpr (sizeof(T) == 2) {
          const f16x4 near = __builtin_convertvector(value, f16x4);
          *reinterpret_cast<f16x4 *>(out + to + d) = near;
          if (rest) *reinterpret_cast<f16x4 *>(rest + to + d) = __builtin_convertvector((value - __builtin_convertvector(near, f32x4)) * kRest, f16x4);
        } else {
          *reinterpret_cast<f32x4 *>(out + to + d) = value;
        }
      }
    if (lse && h == 0) lse[((long long)b * p.HQ + hq) * p.TQ + i] = total == 0 ? INFINITY : (top + __builtin_log2f(total) - kLift) * kLn2;
  }
  odd = __any(in && odd);
  if (lane == 0) bad[wave] = odd;
  __syncthreads();
  if (threadIdx.x == 0) redo[((long long)b * p.HQ + hq) * deal.tiles + at.tile] = bad[0] | bad[1] | bad[2] | bad[3];
}

template <typename T, int DP, int KEYS>
void launch_forward(const Attention &p, const void *q, const void *k, const void *v, void *out, void *rest, void *lse, int *redo) {
  const Deal deal{p.B * p.HK, p.group, (int)ceil_div(p.TQ, kBlockRows)};
  const unsigned blocks = (unsigned)(deal.pairs * deal.heads * deal.tiles);
  attention_tiles_kernel<T, DP, KEYS><<<dim3(blocks), dim3(256), 0, runtime().stream>>>(p, deal, (const T *)q, (const T *)k, (const T *)v, (T *)out,
                                                                                        (_Float16 *)rest, (float *)lse, redo);
}

}  // namespace

// Head dimensions up to 128 in whole pieces of 16 bytes, from buffers that start on one, rows of a tile within reach of 32 bits.
bool tiles_take(const Attention &p, int size, uintptr_t ends) {
  return p.D <= 128 && p.D * size % 16 == 0 && ends % 16 == 0 && (long long)p.HQ * p.D * size * 128 < (1ll << 31) &&
         (long long)p.B * p.HQ * ceil_div(p.TQ, 32) < (1 << 24) && (long long)p.B * p.HK * ceil_div(p.TK, 32) < (1 << 24);
}

int forward_tiles(const Attention &p, int dtype, const void *q, const void *k, const void *v, void *out, void *rest, void *lse) {
  void *space = nullptr;
  const int rc = workspace((size_t)p.B * p.HQ * ceil_div(p.TQ, kBlockRows) * sizeof(int), &space);
  if (rc) return rc;
  int *redo = (int *)space;
  {
    ScopedTiming timed(TAG_ATTENTION);
    const int parts = (p.D + 31) / 32;
    if (dtype == MG_F16) {
      if (parts == 1) launch_forward<_Float16, 32, 64>(p, q, k, v, out, rest, lse, redo);
      if (parts == 2) launch_forward<_Float16, 64, 64>(p, q, k, v, out, rest, lse, redo);
      if (parts == 3) launch_forward<_Float16, 96, 64>(p, q, k, v, out, rest, lse, redo);
      if (parts == 4) launch_forward<_Float16, 128, 64>(p, q, k, v, out, rest, lse, redo);
    } else {
      if (parts == 1) launch_forward<float, 32, 32>(p, q, k, v, out, rest, lse, redo);
      if (parts == 2) launch_forward<float, 64, 32>(p, q, k, v, out, rest, lse, redo);
      if (parts == 3) launch_forward<float, 96, 32>(p, q, k, v, out, rest, lse, redo);
      if (parts == 4) launch_forward<float, 128, 32>(p, q, k, v, out, rest, lse, redo);
    }
    MG_HIP(hipGetLastError());
  }
  return forward_rows_again(p, dtype, q, k, v, out, rest, lse, redo, kBlockRows);
}

}  // namespace mg
