// A norm for each head with rotary positions in the same pass, and its gradient, for gfx950.
//
//   r = 1 / sqrt(mean(x^2) + eps)     z = w * x * r       (over the D values of one head of one token)
//   y_a = z_a cos - z_b sin,  y_b = z_b cos + z_a sin     for the P pairs (a, b) = (p, p + P), or (2p, 2p + 1) interleaved
//   u = the same turn backwards of grad                   dw = sum u x r       dx = r (w u - x r^2 mean(w u x))
//
// cos and sin of pair p lie in a table, at the row that the token's position along the pair's axis names.
// Bandwidth-bound: x is read once forward, x and grad once backward; the table's rows are shared by a token's heads.
#include "internal.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace mg {

namespace {

constexpr int kMaxDim = 1024;

struct HeadNorm {
  long long rows;  // tokens * heads
  int heads, D, pairs, axes, table_rows, interleaved, norm, weight_heads;  // weight_heads: 0 no weight, 1 shared, else one for each head
  double eps;
  const int32_t *positions;  // (tokens, axes)
  const uint8_t *axis_of;    // (pairs)
};

template <typename C>
__device__ __forceinline__ C wave_sum(C v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

// The place of a pair's first value and how far off the second one is.
__device__ __forceinline__ int first_of(const HeadNorm &p, int pair) { return p.interleaved ? 2 * pair : pair; }
__device__ __forceinline__ int apart(const HeadNorm &p) { return p.interleaved ? 1 : p.pairs; }

template <typename C>
__device__ __forceinline__ void turn_of(const HeadNorm &p, const C *table, long long token, int pair, C &cos, C &sin) {
  const int row = p.positions[token * p.axes + p.axis_of[pair]];
  const C *at = table + 2 * ((long long)min(max(row, 0), p.table_rows - 1) * p.pairs + pair);
  cos = at[0], sin = at[1];
}

// A wavefront per row.
template <typename T, typename C>
__global__ void __launch_bounds__(256) head_norm_kernel(HeadNorm p, const T *__restrict__ x, const T *__restrict__ w, const C *__restrict__ table,
                                                        T *__restrict__ y) {
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  const long long token = row / p.heads;
  const int head = (int)(row - token * p.heads);
  const T *xr = x + row * p.D, *wr = w + (p.weight_heads > 1 ? (long long)head * p.D : 0);
  T *yr = y + row * p.D;
  C r = 1;
  if (p.norm) {
    C sum = 0;
    for (int d = lane; d < p.D; d += 64) sum += (C)xr[d] * (C)xr[d];
    r = 1 / sqrt(wave_sum(sum) / p.D + (C)p.eps);
  }
  auto z = [&](int d) { return (C)xr[d] * r * (p.weight_heads ? (C)wr[d] : C(1)); };
  for (int n = lane; n < p.pairs; n += 64) {
    C cos, sin;
    turn_of<C>(p, table, token, n, cos, sin);
    const int a = first_of(p, n), b = a + apart(p);
    const C za = z(a), zb = z(b);
    yr[a] = (T)(za * cos - zb * sin);
    yr[b] = (T)(zb * cos + za * sin);
  }
  for (int d = 2 * p.pairs + lane; d < p.D; d += 64) yr[d] = (T)z(d);
}

// A wavefront per row, for dx.
template <typename T, typename C>
__global__ void __launch_bounds__(256) head_norm_dx_kernel(HeadNorm p, const T *__restrict__ x, const T *__restrict__ w, const C *__restrict__ table,
                                                           const T *__restrict__ grad, T *__restrict__ dx) {
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  const long long token = row / p.heads;
  const int head = (int)(row - token * p.heads);
  const T *xr = x + row * p.D, *gr = grad + row * p.D, *wr = w + (p.weight_heads > 1 ? (long long)head * p.D : 0);
  T *out = dx + row * p.D;
  auto weight = [&](int d) { return p.weight_heads ? (C)wr[d] : C(1); };
  C squares = 0, mix = 0;
  auto add = [&](int d, C u) {
    const C value = (C)xr[d];
    squares += value * value;
    mix += value * weight(d) * u;
  };
  for (int n = lane; n < p.pairs; n += 64) {
    C cos, sin;
    turn_of<C>(p, table, token, n, cos, sin);
    const int a = first_of(p, n), b = a + apart(p);
    const C ga = (C)gr[a], gb = (C)gr[b];
    add(a, ga * cos + gb * sin);
    add(b, gb * cos - ga * sin);
  }
  for (int d = 2 * p.pairs + lane; d < p.D; d += 64) add(d, (C)gr[d]);
  C r = 1, m = 0;
  if (p.norm) {
    r = 1 / sqrt(wave_sum(squares) / p.D + (C)p.eps);
    m = r * r * (wave_sum(mix) / p.D);
  }
  auto put = [&](int d, C u) { out[d] = (T)(p.norm ? r * (weight(d) * u - (C)xr[d] * m) : weight(d) * u); };  // without a norm x has no part in it
  for (int n = lane; n < p.pairs; n += 64) {
    C cos, sin;
    turn_of<C>(p, table, token, n, cos, sin);
    const int a = first_of(p, n), b = a + apart(p);
    const C ga = (C)gr[a], gb = (C)gr[b];
    put(a, ga * cos + gb * sin);
    put(b, gb * cos - ga * sin);
  }
  for (int d = 2 * p.pairs + lane; d < p.D; d += 64) put(d, (C)gr[d]);
}

// Sums of u x r over the rows of one head (or of all) that block `blockIdx.y` takes, in double; a block's wavefronts go through them
// in turn and are added in their order.
template <typename T, typename C>
__global__ void __launch_bounds__(256) head_norm_dw_kernel(HeadNorm p, long long per_block, const T *__restrict__ x, const C *__restrict__ table,
                                                           const T *__restrict__ grad, double *__restrict__ parts) {
  __shared__ double sums[4][kMaxDim];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, head = blockIdx.x;
  const bool each = p.weight_heads > 1;
  const long long count = each ? p.rows / p.heads : p.rows;
  const long long from = blockIdx.y * per_block, to = min(count, from + per_block);
  for (int d = lane; d < p.D; d += 64) sums[wave][d] = 0;
  for (long long n = from + wave; n < to; n += 4) {
    const long long row = each ? n * p.heads + head : n, token = row / p.heads;
    const T *xr = x + row * p.D, *gr = grad + row * p.D;
    C r = 1;
    if (p.norm) {
      C squares = 0;
      for (int d = lane; d < p.D; d += 64) squares += (C)xr[d] * (C)xr[d];
      r = 1 / sqrt(wave_sum(squares) / p.D + (C)p.eps);
    }
    for (int q = lane; q < p.pairs; q += 64) {
      C cos, sin;
      turn_of<C>(p, table, token, q, cos, sin);
      const int a = first_of(p, q), b = a + apart(p);
      const C ga = (C)gr[a], gb = (C)gr[b];
      sums[wave][a] += (double)((ga * cos + gb * sin) * (C)xr[a] * r);
      sums[wave][b] += (double)((gb * cos - ga * sin) * (C)xr[b] * r);
    }
    for (int d = 2 * p.pairs + lane; d < p.D; d += 64) sums[wave][d] += (double)((C)gr[d] * (C)xr[d] * r);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.D; d += 256)
    parts[((long long)blockIdx.y * gridDim.x + head) * p.D + d] = sums[0][d] + sums[1][d] + sums[2][d] + sums[3][d];
}

// A wavefront per value: its lanes take the parts in turn and are added as a tree.
template <typename T>
__global__ void __launch_bounds__(256) head_norm_dw_join_kernel(int values, int parts, const double *__restrict__ from, T *__restrict__ dw) {
  const int lane = threadIdx.x & 63, n = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= values) return;
  double sum = 0;
#pragma unroll 8  // as many loads on their way: 2048 parts take 10 us, 13 one by one
  for (int part = lane; part < parts; part += 64) sum += from[(long long)part * values + n];
  sum = wave_sum(sum);
  if (lane == 0) dw[n] = (T)sum;
}

// What the lanes of a wavefront wrote to LDS is there for all of them.
__device__ __forceinline__ void wave_sees() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---- rows in whole pieces ----------------------------------------------------------------------------------------------------
// A lane holds V neighbouring values (16 bytes where the head dimension allows) of a row and LANES = 2^k lanes a row; the wavefront keeps to
// a token, whose cos and sin stay in registers, while it goes through the heads.  A value's partner in its pair lies in another lane or
// not, wherever sections and layout put it: rows are handed over through LDS, a wavefront's own.
// Bound by memory: float16, 16384 tokens of 32 heads of 128 values (134 MB a tensor), 58 us forward (4.6 TB/s; a copy reaches 5.2) and 99 back with dw
// (4.1); float32, 14256 tokens of 16 heads of 72 (66 MB), 31 and 55 (4.2 and 3.6).  A wavefront per row took 1681 and 618 us for both passes.
// NEAR: a lane's values turn with neighbours, a whole piece of them (halves of a row that are whole pieces); it then needs one place.
template <typename T, typename C, int V, bool NEAR>
struct Pieces {
  typedef T Held __attribute__((ext_vector_type(V)));
  typedef C Wide __attribute__((ext_vector_type(V)));
  Wide cos, sin;  // sin with the sign that the partner's value takes
  int partner[NEAR ? 1 : V];

  static __device__ __forceinline__ int pair_of(const HeadNorm &p, int d) {
    return d >= 2 * p.pairs ? -1 : p.interleaved ? d / 2 : d < p.pairs ? d : d - p.pairs;
  }

  // What each of the lane's values turns with; those without a pair with a zero at `nothing` (an infinity times their sine of 0 would be no number).
  __device__ __forceinline__ void find(const HeadNorm &p, int d0, int nothing) {
#pragma unroll
    for (int n = 0; n < (NEAR ? 1 : V); ++n) {
      const int d = d0 + n;
      const bool first = p.interleaved ? d % 2 == 0 : d < p.pairs;
      partner[n] = pair_of(p, d) < 0 ? nothing : first ? d + apart(p) : d - apart(p);
    }
#pragma unroll
    for (int n = 0; n < V; ++n) cos[n] = 1, sin[n] = 0;
  }

  __device__ __forceinline__ void turn_at(const HeadNorm &p, const C *table, long long token, int d0) {
    if (NEAR && p.axes == 1) {  // a run of the table's row
      const int pair = pair_of(p, d0);
      if (pair < 0) return;
      typedef C Both __attribute__((ext_vector_type(2)));
      const int row = min(max(p.positions[token], 0), p.table_rows - 1);
      const Both *at = reinterpret_cast<const Both *>(table) + ((long long)row * p.pairs + pair);
      const C sign = partner[0] > d0 ? -1 : 1;
#pragma unroll
      for (int n = 0; n < V; ++n) {
        const Both both = at[n];
        cos[n] = both[0], sin[n] = both[1] * sign;
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < V; ++n) {
      const int d = d0 + n, pair = pair_of(p, d);
      if (pair < 0) continue;
      C c, s;
      turn_of<C>(p, table, token, pair, c, s);
      cos[n] = c, sin[n] = partner[NEAR ? 0 : n] > d0 + (NEAR ? 0 : n) ? -s : s;
    }
  }
};

// The sum over each run of `lanes` lanes, a power of two: sixteen are added by moves within a row of lanes, more through LDS.
template <int CONTROL>
__device__ __forceinline__ float moved(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CONTROL, 0xf, 0xf, true));
}
template <int CONTROL>
__device__ __forceinline__ double moved(double v) {
  typedef int Two __attribute__((ext_vector_type(2)));
  Two q = __builtin_bit_cast(Two, v);
  q[0] = __builtin_amdgcn_mov_dpp(q[0], CONTROL, 0xf, 0xf, true), q[1] = __builtin_amdgcn_mov_dpp(q[1], CONTROL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, q);
}
template <typename C>
__device__ __forceinline__ C sum_of_lanes(C v, int lanes) {
  if (lanes > 1) v += moved<0xb1>(v);   // lanes 1 0 3 2 of four
  if (lanes > 2) v += moved<0x4e>(v);   // 2 3 0 1
  if (lanes > 4) v += moved<0x141>(v);  // eight from behind
  if (lanes > 8) v += moved<0x140>(v);  // sixteen from behind
  if (lanes > 16) v += __shfl_xor(v, 16);
  if (lanes > 32) v += __shfl_xor(v, 32);
  return v;
}

// Four wavefronts a SIMD: two registers more in the gradient would leave three, 156 us for a step instead of 144 (float16, 16384 tokens of 32 heads of 128).
template <typename T, typename C, int V, bool BACK, bool NEAR>
__global__ void __launch_bounds__(256, 4) head_norm_pieces_kernel(HeadNorm p, int lanes, const T *__restrict__ x, const T *__restrict__ w,
                                                               const C *__restrict__ table, const T *__restrict__ grad, T *__restrict__ out,
                                                               double *__restrict__ parts) {
  // Rounds whose values are on their way together: forward and in float16 two take 55 us where one takes 61; backward (108 against 98) and in
  // float32 (2 x 7128 tokens of 16 heads of 72: 37 against 31) the registers for two cost more waves than they gain.
  constexpr int kAtOnce = !BACK && sizeof(T) == 2 ? 2 : 1;
  typedef Pieces<T, C, V, NEAR> P;
  typedef typename P::Held Held;
  typedef typename P::Wide Wide;
  typedef std::conditional_t<(kAtOnce > 1), Held, Wide> Kept;
  __shared__ __attribute__((aligned(64))) char space[(4 * 64 + 4) * V * sizeof(double)];  // rows of four wavefronts, or sums; a zero for each of them
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & (lanes - 1), g = lane / lanes, groups = 64 / lanes;
  const int d0 = l * V;
  const bool in = d0 < p.D, each = p.weight_heads > 1;
  C *row = (C *)space + wave * 64 * V + g * lanes * V;
  C *nothing = (C *)(space + 4 * 64 * V * sizeof(double)) + wave * V;
  if (lane < V) nothing[lane] = 0;
  P piece;
  piece.find(p, in ? d0 : 0, (int)(nothing - row));
  // The groups take heads of one token side by side, of several tokens where these have few.  With weights for each head and their gradient
  // wanted, a group keeps to one head.
  const bool keep = BACK && parts && each;
  const int side = keep ? 1 : min(groups, p.heads), tokens_at_once = keep ? 1 : groups / side;
  const int all_rounds = (p.heads + side - 1) / side, share = (all_rounds + gridDim.y - 1) / gridDim.y;  // blockIdx.y takes a share of the heads
  const int first_head = keep ? blockIdx.y * groups + g : g % side + blockIdx.y * share * side;
  const int rounds = keep ? 1 : min(share, all_rounds - (int)blockIdx.y * share);
  const bool mine = in && (keep || g / side < tokens_at_once);
  const long long tokens = p.rows / p.heads, stride = (long long)gridDim.x * 4 * tokens_at_once;

  Wide weight;
#pragma unroll
  for (int n = 0; n < V; ++n) weight[n] = 1;
  if (p.weight_heads == 1 && in) weight = __builtin_convertvector(*reinterpret_cast<const Held *>(w + d0), Wide);
  double sums[BACK ? V : 1] = {};
  for (long long first = ((long long)blockIdx.x * 4 + wave) * tokens_at_once; first < tokens; first += stride) {
    const long long token = first + (keep ? 0 : g / side);
    const bool here = mine && token < tokens;
    if (here && p.pairs) piece.turn_at(p, table, token, d0);
    for (int round = 0; round < rounds; round += kAtOnce) {
      Kept values[kAtOnce] = {}, others[BACK ? kAtOnce : 1] = {};
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int head = first_head + (round + u) * side;
        if (here && head < p.heads && round + u < rounds) {
          const long long at = (token * p.heads + head) * p.D + d0;
          values[u] = __builtin_convertvector(*reinterpret_cast<const Held *>(x + at), Kept);
          if constexpr (BACK) others[u] = __builtin_convertvector(*reinterpret_cast<const Held *>(grad + at), Kept);
          if (each && kAtOnce == 1) weight = __builtin_convertvector(*reinterpret_cast<const Held *>(w + (long long)head * p.D + d0), Wide);
        }
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int head = first_head + (round + u) * side;
        const bool take = here && head < p.heads && round + u < rounds;
        const long long at = (token * p.heads + head) * p.D + d0;
        const Wide value = __builtin_convertvector(values[u], Wide), other = __builtin_convertvector(others[BACK ? u : 0], Wide);
        if (each && kAtOnce > 1 && take) weight = __builtin_convertvector(*reinterpret_cast<const Held *>(w + (long long)head * p.D + d0), Wide);
        C squares = 0;
#pragma unroll
        for (int n = 0; n < V; ++n) squares += value[n] * value[n];
        C r = 1;
        if (p.norm) {
          squares = sum_of_lanes(squares, lanes);
          r = 1 / sqrt(squares / p.D + (C)p.eps);
        }
        Wide z = BACK ? other : value * r * weight;
        if (p.pairs) {
          wave_sees();
          *reinterpret_cast<Wide *>(row + l * V) = z;
          wave_sees();
          Wide there;
          if constexpr (NEAR) {
            there = *reinterpret_cast<const Wide *>(row + piece.partner[0]);
          } else {
#pragma unroll
            for (int n = 0; n < V; ++n) there[n] = row[piece.partner[n]];
          }
          z = z * piece.cos + there * (BACK ? -piece.sin : piece.sin);
        }
        if constexpr (BACK) {
          if (take && parts) {
#pragma unroll
            for (int n = 0; n < V; ++n) sums[n] += (double)(z[n] * value[n] * r);
          }
          z *= weight;
          if (p.norm) {  // without one x has no part in dx
            C mean = 0;
#pragma unroll
            for (int n = 0; n < V; ++n) mean += z[n] * value[n];
            mean = sum_of_lanes(mean, lanes) * (r * r / p.D);
            z = (z - value * mean) * r;
          }
        }
        if (take && out) *reinterpret_cast<Held *>(out + at) = __builtin_convertvector(z, Held);
      }
    }
  }
  if constexpr (BACK) {
    if (!parts) return;
    // the block's sums: of the groups that share a weight (all of them, but where each head has its own), then of its wavefronts
    if (!each) {
      for (int m = lanes; m < 64; m <<= 1)
#pragma unroll
        for (int n = 0; n < V; ++n) sums[n] += __shfl_xor(sums[n], m);
    }
    __syncthreads();
    double *all = (double *)space;
#pragma unroll
    for (int n = 0; n < V; ++n) all[(wave * 64 + lane) * V + n] = sums[n];
    __syncthreads();
    const int held = each ? 64 * V : lanes * V;
    for (int n = threadIdx.x; n < held; n += 256) {
      const int head = each ? blockIdx.y * groups + n / (lanes * V) : 0, d = n % (lanes * V);
      if (d >= p.D || head >= p.weight_heads) continue;
      const long long part = each ? (long long)blockIdx.x : (long long)blockIdx.y * gridDim.x + blockIdx.x;
      parts[(part * p.weight_heads + head) * p.D + d] = all[n] + all[64 * V + n] + all[128 * V + n] + all[192 * V + n];
    }
  }
}

// Values a lane holds: as many as 16 bytes have, fewer where rows start elsewhere or 64 lanes do not suffice the other way round; 0: no way.
int values_of(const HeadNorm &p, int size, uintptr_t ends) {
  for (int v = 16 / size; v >= 1; v /= 2)
    if (p.D % v == 0 && ends % (v * size) == 0) return p.D <= 64 * v ? v : 0;
  return 0;
}

struct Grid {
  int lanes, blocks, shares;  // blocks along the tokens and along the heads
};

// Blocks whose wavefronts go through all tokens, up to eight a compute unit; where tokens are few, several share a token's heads.  With weights
// for each head and their gradient a group keeps to a head, and blocks along the tokens are the fewer.
Grid grid_of(const HeadNorm &p, int values, bool keep) {
  Grid grid{1, 1, 1};
  while (grid.lanes * values < p.D) grid.lanes *= 2;
  const int cus = runtime().props.multiProcessorCount, groups = 64 / grid.lanes;
  const long long blocks = ceil_div(p.rows / p.heads, 4);
  grid.blocks = (int)std::min<long long>(blocks, 8 * cus);
  if (keep) {
    grid.shares = (int)ceil_div(p.heads, groups);
    grid.blocks = std::max(1, std::min(grid.blocks, (int)ceil_div(8 * cus, grid.shares)));
  } else if (groups < p.heads) {
    grid.shares = (int)std::min<long long>(ceil_div(p.heads, groups), ceil_div(8 * cus, blocks));
  }
  return grid;
}

template <typename T, typename C, bool BACK>
int launch_pieces(const HeadNorm &p, const Grid &shape, int values, const void *x, const void *w, const void *table, const void *grad, void *out,
                  double *parts) {
  const bool near = !p.interleaved && p.pairs % values == 0;
  const dim3 grid((unsigned)shape.blocks, (unsigned)shape.shares);
  auto run = [&](auto v) {
    auto kernel = near ? head_norm_pieces_kernel<T, C, v, BACK, true> : head_norm_pieces_kernel<T, C, v, BACK, false>;
    kernel<<<grid, dim3(256), 0, runtime().stream>>>(p, shape.lanes, (const T *)x, (const T *)w, (const C *)table, (const T *)grad, (T *)out, parts);
  };
  if (values == 1) run(std::integral_constant<int, 1>{});
  if (values == 2) run(std::integral_constant<int, 2>{});
  if constexpr (sizeof(T) <= 4)
    if (values == 4) run(std::integral_constant<int, 4>{});
  if constexpr (sizeof(T) == 2)
    if (values == 8) run(std::integral_constant<int, 8>{});
  MG_HIP(hipGetLastError());
  return MG_OK;
}

template <typename T, typename C>
int forward(const HeadNorm &p, const void *x, const void *w, const void *table, void *y) {
  ScopedTiming timed(TAG_HEAD_NORM);
  const int values = values_of(p, sizeof(T), (uintptr_t)x | (uintptr_t)y | (uintptr_t)w);
  if (values) return launch_pieces<T, C, false>(p, grid_of(p, values, false), values, x, w, table, nullptr, y, nullptr);
  head_norm_kernel<T, C><<<dim3((unsigned)ceil_div(p.rows, 4)), dim3(256), 0, runtime().stream>>>(p, (const T *)x, (const T *)w, (const C *)table, (T *)y);
  MG_HIP(hipGetLastError());
  return MG_OK;
}

template <typename T, typename C>
int backward(const HeadNorm &p, const void *x, const void *w, const void *table, const void *grad, void *dx, void *dw) {
  hipStream_t s = runtime().stream;
  const int values = values_of(p, sizeof(T), (uintptr_t)x | (uintptr_t)dx | (uintptr_t)w | (uintptr_t)grad);
  if (values) {  // both gradients in one pass
    const bool keep = dw && p.weight_heads > 1;
    const Grid grid = grid_of(p, values, keep);
    const int parts = keep ? grid.blocks : grid.blocks * grid.shares;
    void *sums = nullptr;
    if (dw) {
      const int rc = workspace((size_t)parts * p.weight_heads * p.D * sizeof(double), &sums);
      if (rc) return rc;
    }
    ScopedTiming timed(TAG_HEAD_NORM_BWD);
    const int rc = launch_pieces<T, C, true>(p, grid, values, x, w, table, grad, dx, (double *)sums);
    if (rc || !dw) return rc;
    head_norm_dw_join_kernel<T><<<dim3((unsigned)ceil_div(p.weight_heads * p.D, 4)), dim3(256), 0, s>>>(p.weight_heads * p.D, parts, (const double *)sums, (T *)dw);
    MG_HIP(hipGetLastError());
    return MG_OK;
  }
  if (dx) {
    ScopedTiming timed(TAG_HEAD_NORM_BWD);
    head_norm_dx_kernel<T, C><<<dim3((unsigned)ceil_div(p.rows, 4)), dim3(256), 0, s>>>(p, (const T *)x, (const T *)w, (const C *)table, (const T *)grad, (T *)dx);
    MG_HIP(hipGetLastError());
  }
  if (dw) {
    const int heads = p.weight_heads;
    const long long count = heads > 1 ? p.rows / p.heads : p.rows;
    const long long per_block = ceil_div(count, 256), parts = ceil_div(count, per_block);
    void *sums = nullptr;
    const int rc = workspace((size_t)parts * heads * p.D * sizeof(double), &sums);
    if (rc) return rc;
    ScopedTiming timed(TAG_HEAD_NORM_BWD);
    head_norm_dw_kernel<T, C><<<dim3((unsigned)heads, (unsigned)parts), dim3(256), 0, s>>>(p, per_block, (const T *)x, (const C *)table, (const T *)grad, (double *)sums);
    MG_HIP(hipGetLastError());
    head_norm_dw_join_kernel<T><<<dim3((unsigned)ceil_div(heads * p.D, 4)), dim3(256), 0, s>>>(heads * p.D, (int)parts, (const double *)sums, (T *)dw);
    MG_HIP(hipGetLastError());
  }
  return MG_OK;
}

int check(const mg_head_norm_desc *d, HeadNorm *p, const char *who) {
  if (!d) return fail(MG_ERR_BAD_ARG, "%s: null descriptor", who);
  if (d->dtype != MG_F32 && d->dtype != MG_F64 && d->dtype != MG_F16) return fail(MG_ERR_UNSUPPORTED, "%s: dtype %d", who, d->dtype);
  if (d->tokens < 0 || d->heads <= 0 || d->D <= 0 || d->pairs < 0 || 2 * d->pairs > d->D || d->eps < 0 || !std::isfinite(d->eps))
    return fail(MG_ERR_BAD_ARG, "%s: %lld tokens, %lld heads, dim %lld, %lld pairs, eps %g", who, (long long)d->tokens, (long long)d->heads,
                (long long)d->D, (long long)d->pairs, d->eps);
  if (d->D > kMaxDim || d->heads > 65535 || d->tokens >= (1ll << 40) / d->heads || ceil_div(d->tokens * d->heads, 4) >= (1 << 24))
    return fail(MG_ERR_UNSUPPORTED, "%s: %lld tokens, %lld heads, dim %lld (at most %d)", who, (long long)d->tokens, (long long)d->heads,
                (long long)d->D, kMaxDim);
  if (d->weight_heads != 0 && d->weight_heads != 1 && d->weight_heads != d->heads)
    return fail(MG_ERR_BAD_ARG, "%s: weights of %d heads for %lld", who, d->weight_heads, (long long)d->heads);
  if (d->pairs && (d->axes < 1 || d->axes > 255 || d->table_rows < 1 || d->table_rows >= (1 << 30) || !d->positions || !d->axis_of))
    return fail(MG_ERR_BAD_ARG, "%s: %d axes, a table of %lld rows, or no positions", who, d->axes, (long long)d->table_rows);
  p->rows = d->tokens * d->heads;
  p->heads = (int)d->heads, p->D = (int)d->D, p->pairs = (int)d->pairs, p->axes = d->axes, p->table_rows = (int)d->table_rows;
  p->interleaved = d->interleaved, p->norm = d->norm, p->weight_heads = d->weight_heads, p->eps = d->eps;
  p->positions = d->positions, p->axis_of = d->axis_of;
  return MG_OK;
}

}  // namespace

}  // namespace mg

using namespace mg;

extern "C" {

int mg_head_norm_fwd(const mg_head_norm_desc *desc, const void *x, const void *weight, const void *table, void *y) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  HeadNorm p{};
  const int rc = check(desc, &p, "mg_head_norm_fwd");
  if (rc) return rc;
  if (p.rows == 0) return MG_OK;
  if (!x || !y || (p.weight_heads && !weight) || (p.pairs && !table)) return fail(MG_ERR_BAD_ARG, "null pointer in mg_head_norm_fwd");
  if (desc->dtype == MG_F64) return forward<double, double>(p, x, weight, table, y);
  if (desc->dtype == MG_F32) return forward<float, float>(p, x, weight, table, y);
  return forward<_Float16, float>(p, x, weight, table, y);
}

int mg_head_norm_bwd(const mg_head_norm_desc *desc, const void *x, const void *weight, const void *table, const void *grad, void *dx, void *dweight) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  HeadNorm p{};
  const int rc = check(desc, &p, "mg_head_norm_bwd");
  if (rc) return rc;
  if (dweight && !p.weight_heads) return fail(MG_ERR_BAD_ARG, "mg_head_norm_bwd: a gradient of weights that there are none of");
  if (p.rows == 0) {
    const size_t size = desc->dtype == MG_F64 ? 8 : desc->dtype == MG_F32 ? 4 : 2;
    return dweight ? mg_memset_zero(dweight, (size_t)p.weight_heads * p.D * size) : MG_OK;
  }
  if (!x || !grad || (p.weight_heads && !weight) || (p.pairs && !table)) return fail(MG_ERR_BAD_ARG, "null pointer in mg_head_norm_bwd");
  if (desc->dtype == MG_F64) return backward<double, double>(p, x, weight, table, grad, dx, dweight);
  if (desc->dtype == MG_F32) return backward<float, float>(p, x, weight, table, grad, dx, dweight);
  return backward<_Float16, float>(p, x, weight, table, grad, dx, dweight);
}

}  // extern "C"
