// Layer norm and its gradient for gfx950.
//
//   mu = mean x     d = x - mu     r = 1 / sqrt(mean(d^2) + eps)     n = d r     y = w n + b     (over the D values of a row)
//   u = r w grad    dx = u - mean(u) - n r mean(u d)                 dw = sum grad n             db = sum grad   (over the rows)
//
// Behind a row's end threads go on with x = 0 and grad = 0.  There n may be infinite (in a row of equal values far from zero, whose r is that of
// eps alone), and grad n no number; u and d are numbers, and u d is 0.
//
// The mean is taken twice: x - mean is exact to a unit of itself where a row lies far from zero, so the mean of what is left, and the
// variance around it, are those of the row to single precision whatever its offset.  The forward pass keeps both parts and r, three
// numbers a row, so that the backward pass has one sum over a row to wait for instead of three.
//
// Bound by memory: a row stays in registers from its load to its result, and blocks keep to their columns, whose weights they load once
// and whose sums over rows they hold, while they go through the rows.
#include "row_device.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace mg {

namespace {

struct LayerNorm {
  long long rows;
  long long D;
  double eps;
};

template <typename C>
struct Moments {
  C shift, mean, r;  // x - shift - mean, times r
};

// Calls f with each of the block's values of a row, or of two side by side: a piece, the place of its first value and how many of its values are there.
constexpr int kLong = 512;  // threads that share a long row
template <typename T, typename F>
__device__ __forceinline__ void over_row(const LayerNorm &p, F f) {
  for (long long d = (long long)threadIdx.x * Piece<T>::V; d < p.D; d += kLong * Piece<T>::V) f(d, (int)min(p.D - d, (long long)Piece<T>::V));
}

// Of a row that the whole block goes through.
template <typename T, typename C>
__device__ __forceinline__ Moments<C> moments_of(const LayerNorm &p, const T *row, C *space) {
  typedef typename Piece<T>::Held Held;
  C sum[1] = {0};
  over_row<T>(p, [&](long long d, int count) {
    const Held v = Piece<T>::load(row + d, count, T(0));
#pragma unroll
    for (int n = 0; n < Piece<T>::V; ++n) sum[0] += (C)v[n];
  });
  block_add(sum, space);
  const C shift = sum[0] / (C)p.D;
  C both[2] = {0, 0};
  over_row<T>(p, [&](long long d, int count) {
    const Held v = Piece<T>::load(row + d, count, T(0));
#pragma unroll
    for (int n = 0; n < Piece<T>::V; ++n) {
      const C t = n < count ? (C)v[n] - shift : C(0);
      both[0] += t, both[1] += t * t;
    }
  });
  block_add(both, space);
  const C mean = both[0] / (C)p.D;
  return Moments<C>{shift, mean, 1 / sqrt(max(both[1] / (C)p.D - mean * mean, C(0)) + (C)p.eps)};
}

// ---- a block per row, which it goes through three times ------------------------------------------------------------------------
// Again from L2, mostly: rows of 40000 halves, 2^27 bytes of x, 79 us forward and 195 back (a copy of as many values 51; one value a thread at a time 226 and 367).
template <typename T, typename C>
__global__ void __launch_bounds__(kLong) layer_norm_kernel(LayerNorm p, const T *__restrict__ x, const T *__restrict__ w, const T *__restrict__ b,
                                                           T *__restrict__ y, Moments<C> *__restrict__ kept) {
  typedef typename Piece<T>::Held Held;
  __shared__ C space[32];
  const T *row = x + blockIdx.x * p.D;
  T *out = y + blockIdx.x * p.D;
  const Moments<C> m = moments_of(p, row, space);
  if (kept && threadIdx.x == 0) kept[blockIdx.x] = m;
  over_row<T>(p, [&](long long d, int count) {
    Held v = Piece<T>::load(row + d, count, T(0));
    const Held weight = w ? Piece<T>::load(w + d, count, T(0)) : Held{}, bias = b ? Piece<T>::load(b + d, count, T(0)) : Held{};
#pragma unroll
    for (int n = 0; n < Piece<T>::V; ++n) v[n] = (T)(((C)v[n] - m.shift - m.mean) * m.r * (w ? (C)weight[n] : C(1)) + (C)bias[n]);
    Piece<T>::store(out + d, count, v);
  });
}

template <typename T, typename C>
__global__ void __launch_bounds__(kLong) layer_norm_dx_kernel(LayerNorm p, const T *__restrict__ x, const T *__restrict__ w, const T *__restrict__ grad,
                                                              const Moments<C> *__restrict__ kept, T *__restrict__ dx) {
  typedef typename Piece<T>::Held Held;
  __shared__ C space[32];
  const T *row = x + blockIdx.x * p.D, *g = grad + blockIdx.x * p.D;
  const Moments<C> m = kept[blockIdx.x];
  C sums[2] = {0, 0};
  auto each = [&](long long d, int count, auto f) {  // u and x - mean; behind the row's end u is 0
    const Held xs = Piece<T>::load(row + d, count, T(0)), gs = Piece<T>::load(g + d, count, T(0));
    const Held weight = w ? Piece<T>::load(w + d, count, T(0)) : Held{};
#pragma unroll
    for (int n = 0; n < Piece<T>::V; ++n) f(n, (C)gs[n] * (w ? (C)weight[n] : C(1)) * m.r, (C)xs[n] - m.shift - m.mean);
  };
  over_row<T>(p, [&](long long d, int count) { each(d, count, [&](int, C u, C t) { sums[0] += u, sums[1] += u * t; }); });
  block_add(sums, space);
  const C first = sums[0] / (C)p.D, second = m.r * (sums[1] / (C)p.D);
  over_row<T>(p, [&](long long d, int count) {
    Held out;
    each(d, count, [&](int k, C u, C t) { out[k] = (T)(u - first - t * m.r * second); });
    Piece<T>::store(dx + blockIdx.x * p.D + d, count, out);
  });
}

// Sums over the rows of one share (blockIdx.y): a thread per piece of the columns.
template <typename T, typename C>
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(LayerNorm p, long long share, const T *__restrict__ x, const T *__restrict__ grad,
                                                                 const Moments<C> *__restrict__ kept, double *__restrict__ parts) {
  typedef typename Piece<T>::Held Held;
  constexpr int V = Piece<T>::V;
  const long long d = ((long long)blockIdx.x * 256 + threadIdx.x) * V, left = p.D - d;
  if (left <= 0) return;
  const long long from = blockIdx.y * share, to = min(p.rows, from + share);
  double dw[V] = {}, db[V] = {};
#pragma unroll 2
  for (long long row = from; row < to; ++row) {
    const Moments<C> m = kept[row];
    const Held xs = Piece<T>::load(x + row * p.D + d, left, T(0)), gs = Piece<T>::load(grad + row * p.D + d, left, T(0));
#pragma unroll
    for (int n = 0; n < V; ++n) dw[n] += (double)((C)gs[n] * (((C)xs[n] - m.shift - m.mean) * m.r)), db[n] += (double)(C)gs[n];
  }
#pragma unroll
  for (int n = 0; n < V; ++n)
    if (n < left) parts[(2ll * blockIdx.y) * p.D + d + n] = dw[n], parts[(2ll * blockIdx.y + 1) * p.D + d + n] = db[n];
}

// Adds the parts of dw and db (blockIdx.y): 64 columns a block, whose 16 wavefronts take a share of the parts each.
template <typename T, typename P>
__global__ void __launch_bounds__(1024) layer_norm_join_kernel(long long D, int parts, const P *__restrict__ from, T *__restrict__ dw, T *__restrict__ db) {
  __shared__ double space[16][64];
  T *const out = blockIdx.y ? db : dw;
  if (!out) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, share = (parts + 15) / 16;
  const long long d = (long long)blockIdx.x * 64 + lane;
  double sum = 0;
  if (d < D) {
#pragma unroll 8  // as many loads on their way
    for (int n = wave * share; n < min(parts, (wave + 1) * share); ++n) sum += (double)from[(2ll * n + blockIdx.y) * D + d];
  }
  space[wave][lane] = sum;
  __syncthreads();
  if (wave || d >= D) return;
  sum = 0;
#pragma unroll
  for (int n = 0; n < 16; ++n) sum += space[n][lane];
  out[d] = (T)sum;
}

// ---- rows in registers ------------------------------------------------------------------------------------------------------------
// A row's pieces go to a part of a wavefront or one (WAVES = 1: `lanes` threads, 256 / lanes rows at once), or to a whole block of 2, 4 or 16
// wavefronts, N pieces for each thread.
template <int WAVES>
constexpr int kThreads = WAVES == 1 ? 256 : WAVES * 64;

// The sums of two values over a row's threads.  Blocks hand them over in LDS in two places in turn: who is at the next sum has all
// others behind the one before.
template <int WAVES, typename C>
struct RowSums {
  C (*space)[2][WAVES];
  int turn = 0;
  __device__ __forceinline__ void add(C &a, C &b, int lanes) {
    a = lanes_add(a, WAVES == 1 ? lanes : 64), b = lanes_add(b, WAVES == 1 ? lanes : 64);
    if constexpr (WAVES > 1) {
      if ((threadIdx.x & 63) == 0) space[turn][0][threadIdx.x >> 6] = a, space[turn][1][threadIdx.x >> 6] = b;
      __syncthreads();
      a = b = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) a += space[turn][0][w], b += space[turn][1][w];
      turn ^= 1;
    }
  }
};

template <typename T, typename C, int WAVES, int N>
__global__ void __launch_bounds__(kThreads<WAVES>) layer_norm_rows_kernel(LayerNorm p, int lanes, const T *__restrict__ x, const T *__restrict__ w,
                                                                          const T *__restrict__ b, T *__restrict__ y, Moments<C> *__restrict__ kept) {
  typedef typename Piece<T>::Held Held;
  constexpr int V = Piece<T>::V;
  __shared__ C space[2][2][WAVES];
  RowSums<WAVES, C> rows{space};
  const int lane = WAVES == 1 ? threadIdx.x & (lanes - 1) : threadIdx.x, groups = WAVES == 1 ? 256 / lanes : 1;
  const int group = WAVES == 1 ? threadIdx.x / lanes : 0, step = (WAVES == 1 ? lanes : kThreads<WAVES>) * V, d0 = lane * V;
  Held weight[N], bias[N];
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const int d = d0 + u * step;
    if (w) weight[u] = Piece<T>::load(w + d, p.D - d, T(0));
    if (b) bias[u] = Piece<T>::load(b + d, p.D - d, T(0));
  }
  const C count = (C)p.D;
  for (long long row0 = (long long)blockIdx.x * groups; row0 < p.rows; row0 += (long long)gridDim.x * groups) {
    const long long row = row0 + group;
    const bool here = row < p.rows;  // all threads go through the sums
    const T *from = x + row * p.D;
    Held held[N];
    C v[N][V], sum = 0, other = 0;
#pragma unroll
    for (int u = 0; u < N; ++u) held[u] = Piece<T>::load(from + d0 + u * step, here ? p.D - d0 - u * step : 0, T(0));
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int n = 0; n < V; ++n) sum += v[u][n] = (C)held[u][n];
    rows.add(sum, other, lanes);
    const C shift = sum / count;
    sum = other = 0;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const long long left = p.D - d0 - u * step;
#pragma unroll
      for (int n = 0; n < V; ++n) v[u][n] -= shift;
      if (left < V) {
#pragma unroll
        for (int n = 0; n < V; ++n)
          if (n >= left) v[u][n] = 0;
      }
#pragma unroll
      for (int n = 0; n < V; ++n) sum += v[u][n], other += v[u][n] * v[u][n];
    }
    rows.add(sum, other, lanes);
    const C mean = sum / count, r = 1 / sqrt(max(other / count - mean * mean, C(0)) + (C)p.eps);
    if (!here) continue;
    if (kept && lane == 0) kept[row] = Moments<C>{shift, mean, r};
#pragma unroll
    for (int u = 0; u < N; ++u) {
      Held out;
#pragma unroll
      for (int n = 0; n < V; ++n) out[n] = (T)((v[u][n] - mean) * r * (w ? (C)weight[u][n] : C(1)) + (b ? (C)bias[u][n] : C(0)));
      const int d = d0 + u * step;
      Piece<T>::store(y + row * p.D + d, p.D - d, out);
    }
  }
}

// With one or two pieces the next row is on its way during a row's sums, which registers for four do not allow: 2^27 bytes of x, us with and
// without, 2048 pieces of float16 157 and 95, 512 pieces 85 and 91.
template <typename T, typename C, int WAVES, int N>
__global__ void __launch_bounds__(kThreads<WAVES>) layer_norm_rows_bwd_kernel(LayerNorm p, int lanes, const T *__restrict__ x, const T *__restrict__ w,
                                                                              const T *__restrict__ grad, const Moments<C> *__restrict__ kept,
                                                                              T *__restrict__ dx, C *__restrict__ parts) {
  typedef typename Piece<T>::Held Held;
  constexpr int V = Piece<T>::V;
  __shared__ C space[2][2][WAVES];
  RowSums<WAVES, C> rows{space};
  const int lane = WAVES == 1 ? threadIdx.x & (lanes - 1) : threadIdx.x, groups = WAVES == 1 ? 256 / lanes : 1;
  const int group = WAVES == 1 ? threadIdx.x / lanes : 0, step = (WAVES == 1 ? lanes : kThreads<WAVES>) * V, d0 = lane * V;
  constexpr bool AHEAD = N == 1 || (N == 2 && WAVES < 16), HELD = WAVES < 16 || N < 4;  // the next row is loaded early; the weight stays in registers
  Held weight[N];
  auto load_weight = [&] {
#pragma unroll
    for (int u = 0; u < N; ++u) weight[u] = w ? Piece<T>::load(w + d0 + u * step, p.D - d0 - u * step, T(0)) : Held{};
  };
  if (HELD) load_weight();
  C dw[N][V] = {}, db[N][V] = {};
  Held xs[N], gs[N];
  auto load = [&](long long row) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const long long left = row < p.rows ? p.D - d0 - u * step : 0;
      xs[u] = Piece<T>::load(x + row * p.D + d0 + u * step, left, T(0));
      gs[u] = Piece<T>::load(grad + row * p.D + d0 + u * step, left, T(0));
    }
  };
  const long long stride = (long long)gridDim.x * groups;
  if (AHEAD) load((long long)blockIdx.x * groups + group);
  for (long long row0 = (long long)blockIdx.x * groups; row0 < p.rows; row0 += stride) {
    const long long row = row0 + group;
    const bool here = row < p.rows;
    const Moments<C> m = here ? kept[row] : Moments<C>{0, 0, 0};
    C first = 0, second = 0;
    if constexpr (AHEAD) {
      C v[N][V], u_of[N][V];
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int n = 0; n < V; ++n) {
          const C g = (C)gs[u][n], d = (C)xs[u][n] - m.shift - m.mean, t = d * m.r;
          v[u][n] = t;
          u_of[u][n] = (w ? g * (C)weight[u][n] : g) * m.r;
          first += u_of[u][n], second += u_of[u][n] * d;
          dw[u][n] += g * t, db[u][n] += g;
        }
      load(row + stride);  // the next row is on its way during the sums
      if (dx) {
        rows.add(first, second, lanes);
        first /= (C)p.D, second = m.r * (second / (C)p.D);
#pragma unroll
        for (int u = 0; u < N; ++u) {
          Held out;
#pragma unroll
          for (int n = 0; n < V; ++n) out[n] = (T)(u_of[u][n] - first - v[u][n] * second);
          const int d = d0 + u * step;
          if (here) Piece<T>::store(dx + row * p.D + d, p.D - d, out);
        }
      }
    } else {
      load(row);
      if constexpr (!HELD) load_weight();
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int n = 0; n < V; ++n) {
          const C g = (C)gs[u][n], d = (C)xs[u][n] - m.shift - m.mean, ur = (w ? g * (C)weight[u][n] : g) * m.r;
          first += ur, second += ur * d;
          dw[u][n] += g * (d * m.r), db[u][n] += g;
        }
      if (dx) {
        rows.add(first, second, lanes);
        first /= (C)p.D, second = m.r * (second / (C)p.D);
#pragma unroll
        for (int u = 0; u < N; ++u) {
          Held out;
#pragma unroll
          for (int n = 0; n < V; ++n) {
            const C g = (C)gs[u][n], t = ((C)xs[u][n] - m.shift - m.mean) * m.r;
            out[n] = (T)((w ? g * (C)weight[u][n] : g) * m.r - first - t * second);
          }
          const int d = d0 + u * step;
          if (here) Piece<T>::store(dx + row * p.D + d, p.D - d, out);
        }
      }
    }
  }
  if (!parts) return;
  C *const to = parts + 2ll * blockIdx.x * p.D;
  if constexpr (WAVES == 1) {
    // groups of a wavefront, then the block's four in their order
    __shared__ C sums[4][64 * V];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        auto &mine = which ? db : dw;
        for (int k = lanes; k < 64; k <<= 1)
#pragma unroll
          for (int n = 0; n < V; ++n) mine[u][n] += __shfl_xor(mine[u][n], k);
        __syncthreads();
        if ((threadIdx.x & 63) < lanes)
#pragma unroll
          for (int n = 0; n < V; ++n) sums[threadIdx.x >> 6][d0 + n] = mine[u][n];
        __syncthreads();
        for (int d = threadIdx.x; d < lanes * V; d += 256)
          if (u * step + d < p.D) to[which * p.D + u * step + d] = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
      }
  } else {
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int n = 0; n < V; ++n) {
        const int d = d0 + u * step + n;
        if (d < p.D) to[d] = dw[u][n], to[p.D + d] = db[u][n];
      }
  }
}

// Threads and pieces for a row.  Two wavefronts with a piece each rather than one with two, which in float16 leaves three wavefronts a SIMD
// (800 values, 2^27 bytes of x: 104 us back, 135).  Longer rows do not stay in registers.
struct Shape {
  int waves, pieces, lanes;
};
template <typename T, bool BACK>
Shape shape_of(long long D) {
  const long long pieces = ceil_div(D, Piece<T>::V);
  Shape s{0, 0, 64};
  if (pieces <= 64) {
    s = Shape{1, 1, 1};
    while (s.lanes < pieces) s.lanes *= 2;
  } else if (pieces <= 256) {
    s = Shape{pieces <= 128 ? 2 : 4, 1, 64};
  } else if (pieces <= 512) {
    s = Shape{4, 2, 64};
  } else if (pieces <= 1024) {
    s = sizeof(T) == 2 ? Shape{16, 1, 64} : Shape{4, 4, 64};  // 85 us and 95 back in float16, 84 and 80 in float32
  } else if (pieces <= (BACK && sizeof(T) == 2 ? 2048 : 4096)) {  // four pieces' sums of float16 do not fit: 265 us back, 190 by the kernels for longer rows
    s = Shape{16, pieces <= 2048 ? 2 : 4, 64};
  }
  return s;
}

// Calls f with a Shape's numbers of wavefronts and pieces as constants.
template <typename T, bool BACK, typename F>
void with_shape(const Shape &s, F f) {
  typedef std::integral_constant<int, 1> One;
  typedef std::integral_constant<int, 2> Two;
  typedef std::integral_constant<int, 4> Four;
  typedef std::integral_constant<int, 16> Sixteen;
  if (s.waves == 1) f(One{}, One{});
  if (s.waves == 2) f(Two{}, One{});
  if (s.waves == 4 && s.pieces == 1) f(Four{}, One{});
  if (s.waves == 4 && s.pieces == 2) f(Four{}, Two{});
  if constexpr (sizeof(T) == 2) {
    if (s.waves == 16 && s.pieces == 1) f(Sixteen{}, One{});
  } else {
    if (s.waves == 4 && s.pieces == 4) f(Four{}, Four{});
  }
  if (s.waves == 16 && s.pieces == 2) f(Sixteen{}, Two{});
  if constexpr (!BACK || sizeof(T) > 2) {
    if (s.waves == 16 && s.pieces == 4) f(Sixteen{}, Four{});
  }
}

template <typename T, typename C>
int forward(const LayerNorm &p, const void *x, const void *w, const void *b, void *y, void *kept) {
  ScopedTiming timed(TAG_LAYER_NORM);
  hipStream_t s = runtime().stream;
  const Shape shape = shape_of<T, false>(p.D);
  if (shape.waves) {
    // eight blocks of 256 a compute unit, or as many threads in larger or smaller ones
    const long long most = (shape.waves == 1 ? 8 : 32 / shape.waves) * runtime().props.multiProcessorCount;
    const long long blocks = std::min<long long>(ceil_div(p.rows, shape.waves == 1 ? 256 / shape.lanes : 1), most);
    with_shape<T, false>(shape, [&](auto waves, auto pieces) {
      layer_norm_rows_kernel<T, C, waves, pieces><<<dim3((unsigned)blocks), dim3(kThreads<waves>), 0, s>>>(p, shape.lanes, (const T *)x, (const T *)w,
                                                                                                          (const T *)b, (T *)y, (Moments<C> *)kept);
    });
  } else {
    if (p.rows >= 1 << 23) return fail(MG_ERR_UNSUPPORTED, "mg_layer_norm_fwd: %lld rows of %lld values", p.rows, p.D);  // a block each
    layer_norm_kernel<T, C><<<dim3((unsigned)p.rows), dim3(kLong), 0, s>>>(p, (const T *)x, (const T *)w, (const T *)b, (T *)y, (Moments<C> *)kept);
  }
  MG_HIP(hipGetLastError());
  return MG_OK;
}

template <typename T, typename C>
int backward(const LayerNorm &p, const void *x, const void *w, const void *kept, const void *grad, void *dx, void *dw, void *db) {
  hipStream_t s = runtime().stream;
  const bool columns = dw || db;
  if (p.rows == 0) {  // sums of no rows
    if (!columns) return MG_OK;
    ScopedTiming timed(TAG_LAYER_NORM_BWD);
    layer_norm_join_kernel<T, double><<<dim3((unsigned)ceil_div(p.D, 64), 2), dim3(1024), 0, s>>>(p.D, 0, nullptr, (T *)dw, (T *)db);
    MG_HIP(hipGetLastError());
    return MG_OK;
  }
  const Shape shape = shape_of<T, true>(p.D);
  void *space = nullptr;
  if (shape.waves) {
    // Each block's sums are written once and read once: four blocks of 256 a compute unit (or as many threads) where a thread has one piece, two
    // where it has more, and more only where one would add up 256 rows or more.  256 pieces, us: four 85, two 96; 512 pieces 94 and 85.
    const int groups = shape.waves == 1 ? 256 / shape.lanes : 1, wavefronts = shape.pieces == 1 ? 16 : 8;
    const long long few = std::max(1, wavefronts / (shape.waves == 1 ? 4 : shape.waves)) * runtime().props.multiProcessorCount;
    const long long most = std::max<long long>(few, ceil_div(p.rows, 256ll * groups));
    const long long blocks = std::min<long long>(ceil_div(p.rows, groups), most);
    if (columns)
      if (const int rc = workspace((size_t)(2 * blocks * p.D) * sizeof(C), &space)) return rc;
    ScopedTiming timed(TAG_LAYER_NORM_BWD);
    with_shape<T, true>(shape, [&](auto waves, auto pieces) {
      layer_norm_rows_bwd_kernel<T, C, waves, pieces><<<dim3((unsigned)blocks), dim3(kThreads<waves>), 0, s>>>(
          p, shape.lanes, (const T *)x, (const T *)w, (const T *)grad, (const Moments<C> *)kept, (T *)dx, (C *)space);
    });
    MG_HIP(hipGetLastError());
    if (!columns) return MG_OK;
    layer_norm_join_kernel<T, C><<<dim3((unsigned)ceil_div(p.D, 64), 2), dim3(1024), 0, s>>>(p.D, (int)blocks, (const C *)space, (T *)dw, (T *)db);
    MG_HIP(hipGetLastError());
    return MG_OK;
  }
  if (p.rows >= 1 << 23) return fail(MG_ERR_UNSUPPORTED, "mg_layer_norm_bwd: %lld rows of %lld values", p.rows, p.D);
  const long long share = std::max<long long>(ceil_div(p.rows, 256), 16), shares = ceil_div(p.rows, share);
  if (columns)
    if (const int rc = workspace((size_t)(2 * shares * p.D) * sizeof(double), &space)) return rc;
  ScopedTiming timed(TAG_LAYER_NORM_BWD);
  if (dx) {
    layer_norm_dx_kernel<T, C><<<dim3((unsigned)p.rows), dim3(kLong), 0, s>>>(p, (const T *)x, (const T *)w, (const T *)grad, (const Moments<C> *)kept, (T *)dx);
    MG_HIP(hipGetLastError());
  }
  if (!columns) return MG_OK;
  layer_norm_columns_kernel<T, C><<<dim3((unsigned)ceil_div(p.D, 256 * Piece<T>::V), (unsigned)shares), dim3(256), 0, s>>>(p, share, (const T *)x, (const T *)grad,
                                                                                                          (const Moments<C> *)kept, (double *)space);
  MG_HIP(hipGetLastError());
  layer_norm_join_kernel<T, double><<<dim3((unsigned)ceil_div(p.D, 64), 2), dim3(1024), 0, s>>>(p.D, (int)shares, (const double *)space, (T *)dw, (T *)db);
  MG_HIP(hipGetLastError());
  return MG_OK;
}

int check(int dtype, int64_t rows, int64_t D, double eps, const char *who) {
  if (dtype != MG_F32 && dtype != MG_F64 && dtype != MG_F16) return fail(MG_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (rows < 0 || D <= 0 || !(eps >= 0) || !std::isfinite(eps))
    return fail(MG_ERR_BAD_ARG, "%s: %lld rows of %lld values, eps %g", who, (long long)rows, (long long)D, eps);
  if (rows > 0x7fffffff || D > 1 << 24) return fail(MG_ERR_UNSUPPORTED, "%s: %lld rows of %lld values", who, (long long)rows, (long long)D);
  return MG_OK;
}

}  // namespace

}  // namespace mg

using namespace mg;

extern "C" {

int mg_layer_norm_fwd(int dtype, int64_t rows, int64_t D, double eps, const void *x, const void *weight, const void *bias, void *y,
                      void *kept) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  const int rc = check(dtype, rows, D, eps, "mg_layer_norm_fwd");
  if (rc || rows == 0) return rc;
  if (!x || !y) return fail(MG_ERR_BAD_ARG, "null pointer in mg_layer_norm_fwd");
  const LayerNorm p{rows, D, eps};
  if (dtype == MG_F64) return forward<double, double>(p, x, weight, bias, y, kept);
  if (dtype == MG_F32) return forward<float, float>(p, x, weight, bias, y, kept);
  return forward<_Float16, float>(p, x, weight, bias, y, kept);
}

int mg_layer_norm_bwd(int dtype, int64_t rows, int64_t D, const void *x, const void *weight, const void *kept, const void *grad, void *dx,
                      void *dweight, void *dbias) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  const int rc = check(dtype, rows, D, 0, "mg_layer_norm_bwd");
  if (rc) return rc;
  if (!dx && !dweight && !dbias) return fail(MG_ERR_BAD_ARG, "mg_layer_norm_bwd: no gradient is wanted");
  if (rows && (!x || !grad || !kept)) return fail(MG_ERR_BAD_ARG, "null pointer in mg_layer_norm_bwd");
  const LayerNorm p{rows, D, 0};
  if (dtype == MG_F64) return backward<double, double>(p, x, weight, kept, grad, dx, dweight, dbias);
  if (dtype == MG_F32) return backward<float, float>(p, x, weight, kept, grad, dx, dweight, dbias);
  return backward<_Float16, float>(p, x, weight, kept, grad, dx, dweight, dbias);
}

}  // extern "C"
