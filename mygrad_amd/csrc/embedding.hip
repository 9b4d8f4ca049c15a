// Rows of a table by token, and the gradient of the table, for gfx950.
//
//   y[n] = scale W[ids[n]]  (zeros where ids[n] < 0)          dW[v] = scale * sum of grad[n] over the n with ids[n] = v, in their order
//
// Both are bound by memory.  The gradient sorts the tokens, so that the rows to be added lie in a run, whatever the text: a run is cut
// into chunks of a few rows that are summed side by side, what a cut went through is joined in order, and rows that no token names are
// filled with zeros by the same launch.  Nothing is added by atomics: the same bits every time.
#include "row_device.h"

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

namespace mg {

namespace {

struct Embedding {
  long long tokens;
  int rows;
  long long D;
  double scale;
};

// What values are scaled in: a single-precision product of a rounded scale would be rounded twice.
template <typename T>
using Scaled = std::conditional_t<sizeof(T) == 2, float, double>;

// Rows of D values go to `lanes` = 2^k threads of a block of 256, a piece each (or several in turn).
int lanes_of(long long pieces) {
  int lanes = 1;
  while (lanes < 256 && lanes < pieces) lanes *= 2;
  return lanes;
}

// A group of threads takes AT_ONCE tokens, whose rows are on their way together.
template <typename T, int AT_ONCE>
__global__ void __launch_bounds__(256) embedding_kernel(Embedding p, int lanes, const int32_t *__restrict__ ids, const T *__restrict__ weight,
                                                        T *__restrict__ out) {
  typedef typename Piece<T>::Held Held;
  constexpr int V = Piece<T>::V;
  const int lane = threadIdx.x & (lanes - 1), groups = 256 / lanes;
  const long long first = ((long long)blockIdx.x * groups + threadIdx.x / lanes) * AT_ONCE;
  int id[AT_ONCE];
#pragma unroll
  for (int u = 0; u < AT_ONCE; ++u) {
    id[u] = first + u < p.tokens ? ids[first + u] : -1;
    if (id[u] >= p.rows) id[u] = -1;
  }
  for (long long d = (long long)lane * V; d < p.D; d += (long long)lanes * V) {
    Held v[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) v[u] = id[u] < 0 ? Held{} : Piece<T>::load(weight + id[u] * p.D + d, p.D - d, T(0));
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      if (first + u >= p.tokens) break;
#pragma unroll
      for (int n = 0; n < V; ++n) v[u][n] = id[u] < 0 ? T(0) : (T)((Scaled<T>)v[u][n] * (Scaled<T>)p.scale);
      Piece<T>::store(out + (first + u) * p.D + d, p.D - d, v[u]);
    }
  }
}

// ---- tokens in order --------------------------------------------------------------------------------------------------------------
// A stable sort by digits of `bits` bits from the lowest on: a token's new place is the number of tokens with a lower digit, and of those
// before it with the same one.  A block of 16 wavefronts takes 1024 K tokens, K of them a lane, in 16 runs of 64 K; within a wavefront, lanes with the
// same digit find one another by a vote on each bit.  Tokens that are none (or beyond the table) sort behind all others, as `rows`; places
// behind the last token hold 2^32 - 1, whose digits are the largest: they stay last.
constexpr int kSorters = 16;
constexpr int kMostBits = 10;
constexpr int kMostInBlock = 16384;

// What the lanes of a wavefront wrote to LDS is there for all of them.
__device__ __forceinline__ void wave_sees() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

struct Digit {
  int shift, bits;
  __device__ __forceinline__ int of(unsigned key) const { return (int)(key >> shift) & ((1 << bits) - 1); }
};

// counts[w][d]: tokens of wavefront w with digit d; place[i]: how many of those stand before the lane's i-th.
template <int K>
__device__ __forceinline__ void count_digits(Digit digit, const unsigned (&key)[K], unsigned short *counts, int (&place)[K]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bins = 1 << digit.bits;
  unsigned short *own = counts + wave * bins;
  for (int d = lane; d < bins; d += 64) own[d] = 0;
  wave_sees();
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int d = digit.of(key[i]);
    unsigned long long alike = ~0ull;
    for (int b = 0; b < digit.bits; ++b) {
      const unsigned long long vote = __ballot(d >> b & 1);
      alike &= d >> b & 1 ? vote : ~vote;
    }
    const int before = __popcll(alike & ((1ull << lane) - 1)), old = own[d];
    place[i] = old + before;
    wave_sees();
    if (before == 0) own[d] = (unsigned short)(old + __popcll(alike));
    wave_sees();
  }
}

// counts[w][d] becomes the number of tokens with digit d in wavefronts before w; the number in all is returned to thread d.
__device__ __forceinline__ int over_wavefronts(int bins, unsigned short *counts) {
  int total = 0;
  if ((int)threadIdx.x < bins)
    for (int w = 0; w < kSorters; ++w) {
      const int here = counts[w * bins + threadIdx.x];
      counts[w * bins + threadIdx.x] = (unsigned short)total;
      total += here;
    }
  return total;
}

// The sum of the values of all threads before this one, of a block of 1024; `space` is 16 values of LDS.
__device__ __forceinline__ int sum_before(int value, int *space) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int sum = value;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int other = __shfl_up(sum, m);
    if (lane >= m) sum += other;
  }
  __syncthreads();
  if (lane == 63) space[wave] = sum;
  __syncthreads();
  for (int w = 0; w < wave; ++w) sum += space[w];
  return sum - value;
}

__device__ __forceinline__ unsigned key_of(const int32_t *ids, long long n, long long tokens, int rows) {
  if (n >= tokens) return 0xffffffffu;
  const int id = ids[n];
  return id < 0 || id >= rows ? (unsigned)rows : (unsigned)id;
}

// All digits of up to 1024 K tokens by one block.
template <int K>
__global__ void __launch_bounds__(1024) sort_block_kernel(int tokens, int rows, int bits, int passes, const int32_t *__restrict__ ids,
                                                          unsigned *__restrict__ keys, unsigned *__restrict__ order) {
  extern __shared__ __attribute__((aligned(16))) unsigned lds[];
  __shared__ int space[16], base[1 << kMostBits];
  unsigned *const held = lds;                                             // 1024 K values
  unsigned short *const counts = (unsigned short *)(lds + 1024 * K);  // kSorters << bits
  const int from = (threadIdx.x >> 6) * 64 * K + (threadIdx.x & 63), bins = 1 << bits;
  unsigned key[K], at[K];
  int place[K];
#pragma unroll
  for (int i = 0; i < K; ++i) at[i] = from + i * 64, key[i] = key_of(ids, at[i], tokens, rows);
  for (int pass = 0; pass < passes; ++pass) {
    const Digit digit{pass * bits, bits};
    count_digits(digit, key, counts, place);
    __syncthreads();
    const int total = over_wavefronts(bins, counts), before = sum_before(total, space);
    if ((int)threadIdx.x < bins) base[threadIdx.x] = before;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int d = digit.of(key[i]);
      place[i] += counts[(threadIdx.x >> 6) * bins + d] + base[d];
    }
    // keys, then what they came with, go to their places
#pragma unroll
    for (int i = 0; i < K; ++i) held[place[i]] = key[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i) key[i] = held[from + i * 64];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i) held[place[i]] = at[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i) at[i] = held[from + i * 64];
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < K; ++i)
    if (from + i * 64 < tokens) keys[from + i * 64] = key[i], order[from + i * 64] = at[i];
}

// More tokens than a block takes: for each digit the blocks count theirs, then each finds its places from all counts.
constexpr int kTileK = 4;
constexpr int kTile = 1024 * kTileK;

struct Tiles {
  long long tokens;
  int rows;
  Digit digit;
  const int32_t *ids;  // of the first digit; keys and order come after
  const unsigned *keys, *order;
};

__device__ __forceinline__ void load_tile(const Tiles &p, unsigned (&key)[kTileK]) {
  const long long from = (long long)blockIdx.x * kTile + (threadIdx.x >> 6) * 64 * kTileK + (threadIdx.x & 63);
#pragma unroll
  for (int i = 0; i < kTileK; ++i) {
    const long long n = from + i * 64;
    key[i] = p.ids ? key_of(p.ids, n, p.tokens, p.rows) : n < p.tokens ? p.keys[n] : 0xffffffffu;
  }
}

__global__ void __launch_bounds__(1024) sort_count_kernel(Tiles p, unsigned *__restrict__ totals) {
  __shared__ unsigned short counts[kSorters << kMostBits];
  unsigned key[kTileK];
  int place[kTileK];
  const int bins = 1 << p.digit.bits;
  load_tile(p, key);
  count_digits(p.digit, key, counts, place);
  __syncthreads();
  const int total = over_wavefronts(bins, counts);
  if ((int)threadIdx.x < bins) totals[(long long)blockIdx.x * bins + threadIdx.x] = total;
}

__global__ void __launch_bounds__(1024) sort_place_kernel(Tiles p, const unsigned *__restrict__ totals, unsigned *__restrict__ keys, unsigned *__restrict__ order) {
  __shared__ unsigned short counts[kSorters << kMostBits];
  __shared__ int space[16];
  __shared__ unsigned base[1 << kMostBits];
  unsigned key[kTileK];
  int place[kTileK];
  const int bins = 1 << p.digit.bits;
  load_tile(p, key);
  count_digits(p.digit, key, counts, place);
  __syncthreads();
  over_wavefronts(bins, counts);
  unsigned before = 0, all = 0;
  if ((int)threadIdx.x < bins) {
#pragma unroll 8
    for (unsigned tile = 0; tile < gridDim.x; ++tile) {
      const unsigned here = totals[(long long)tile * bins + threadIdx.x];
      all += here;
      before += tile < blockIdx.x ? here : 0;
    }
  }
  const int lower = sum_before((int)all, space);
  if ((int)threadIdx.x < bins) base[threadIdx.x] = lower + before;
  __syncthreads();
  const long long from = (long long)blockIdx.x * kTile + (threadIdx.x >> 6) * 64 * kTileK + (threadIdx.x & 63);
#pragma unroll
  for (int i = 0; i < kTileK; ++i) {
    const long long n = from + i * 64;
    if (n >= p.tokens) continue;
    const int d = p.digit.of(key[i]);
    const unsigned to = base[d] + counts[(threadIdx.x >> 6) * bins + d] + place[i];
    keys[to] = key[i], order[to] = p.ids ? (unsigned)n : p.order[n];
  }
}

// ---- rows by runs of tokens ---------------------------------------------------------------------------------------------------------
struct Runs {
  long long tokens;
  int rows;
  long long D;
  double scale;
  int lanes;          // threads for a row's pieces
  int chunk;          // tokens of a chunk
  long long chunks;
  int sum_blocks;     // blocks that add (times those along a row); the others fill
  int fill_rows;      // rows of the table for a block that fills
  const unsigned *keys, *order;
};

// A group of threads adds the rows of a chunk's tokens.  A run that lies in the chunk becomes a row of the table's gradient; of one that comes in from
// the chunk before it, the part here goes to parts[2 chunk], and of one that begins here and goes on, to parts[2 chunk + 1].
template <typename T, typename C>
__global__ void __launch_bounds__(256) embedding_runs_kernel(Runs p, const T *__restrict__ grad, T *__restrict__ dweight, C *__restrict__ parts) {
  typedef typename Piece<T>::Held Held;
  constexpr int V = Piece<T>::V, kAtOnce = 8;
  if ((int)blockIdx.x >= p.sum_blocks) {
    // which of 64 rows have tokens: a search by each lane
    if (blockIdx.y) return;
    const int lane = threadIdx.x & 63;
    const long long first = (long long)(blockIdx.x - p.sum_blocks) * p.fill_rows;
    for (long long row0 = first; row0 < min(first + p.fill_rows, (long long)p.rows); row0 += 64) {
      const long long row = row0 + lane;
      long long lo = 0, hi = p.tokens;
      while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if ((long long)p.keys[mid] < row) lo = mid + 1;
        else hi = mid;
      }
      const bool empty = row < p.rows && (lo == p.tokens || p.keys[lo] != (unsigned)row);
      unsigned long long left = __ballot(empty);
      const int wave = threadIdx.x >> 6;
      // a wavefront takes every fourth of the rows to be filled
      for (int nth = 0; left; ++nth) {
        const int n = __builtin_ctzll(left);
        left &= left - 1;
        if ((nth & 3) != wave) continue;
        T *to = dweight + (row0 + n) * p.D;
        for (long long d = (long long)lane * V; d < p.D; d += 64 * V) Piece<T>::store(to + d, p.D - d, Held{});
      }
    }
    return;
  }
  const int lane = threadIdx.x & (p.lanes - 1), groups = 256 / p.lanes;
  const long long c = (long long)blockIdx.x * groups + threadIdx.x / p.lanes, d = ((long long)blockIdx.y * p.lanes + lane) * V;
  if (c >= p.chunks || d >= p.D) return;
  const long long from = c * p.chunk, to = min(from + p.chunk, p.tokens), count = p.D - d;
  unsigned key = p.keys[from];
  bool came = from > 0 && p.keys[from - 1] == key;
  const unsigned next = to < p.tokens ? p.keys[to] : 0xffffffffu;
  C sum[V] = {};
  auto put = [&](bool goes) {
    if (key >= (unsigned)p.rows) return;
    if (came || goes) {
      C *part = parts + (2 * c + (came ? 0 : 1)) * p.D + d;
#pragma unroll
      for (int n = 0; n < V; ++n)
        if (n < count) part[n] = sum[n];
    } else {
      Held v;
#pragma unroll
      for (int n = 0; n < V; ++n) v[n] = (T)((Scaled<T>)sum[n] * (Scaled<T>)p.scale);
      Piece<T>::store(dweight + key * p.D + d, count, v);
    }
  };
  for (long long n0 = from; n0 < to; n0 += kAtOnce) {
    unsigned keys[kAtOnce];
    Held rows[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const long long n = min(n0 + u, to - 1);
      keys[u] = p.keys[n];
      rows[u] = keys[u] < (unsigned)p.rows ? Piece<T>::load(grad + p.order[n] * p.D + d, count, T(0)) : Held{};
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (n0 + u >= to) break;
      if (keys[u] != key) {
        put(false);
        key = keys[u], came = false;
#pragma unroll
        for (int n = 0; n < V; ++n) sum[n] = 0;
      }
#pragma unroll
      for (int n = 0; n < V; ++n) sum[n] += (C)rows[u][n];
    }
  }
  put(next == key);
}

// Runs that were cut: those that begin in chunk blockIdx.x and go on, 64 values of the row a block.  Its four wavefronts take a share of
// the chunks each and are added in their order.
template <typename T, typename C>
__global__ void __launch_bounds__(256) embedding_join_kernel(Runs p, const C *__restrict__ parts, T *__restrict__ dweight) {
  __shared__ C space[4][64];
  const long long c = blockIdx.x, to = (c + 1) * p.chunk;
  if (to >= p.tokens) return;
  const unsigned key = p.keys[to];
  if (key >= (unsigned)p.rows || p.keys[to - 1] != key) return;
  // begins here: it did not fill the chunk, or the one before ended with another token
  if (p.keys[c * p.chunk] == key && c > 0 && p.keys[c * p.chunk - 1] == key) return;
  long long lo = to, hi = p.tokens;  // the end of the run
  while (lo < hi) {
    const long long mid = (lo + hi) >> 1;
    if (p.keys[mid] <= key) lo = mid + 1;
    else hi = mid;
  }
  const long long more = (lo - to + p.chunk - 1) / p.chunk;  // chunks after this one
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long share = (more + 3) / 4, first = c + 1 + wave * share, end = min(first + share, c + 1 + more);
  for (long long d0 = (long long)blockIdx.y * 64; d0 < p.D; d0 += (long long)gridDim.y * 64) {
    const long long d = d0 + lane;
    C sum = 0;
    if (d < p.D) {
      if (wave == 0) sum = parts[(2 * c + 1) * p.D + d];
#pragma unroll 8
      for (long long n = first; n < end; ++n) sum += parts[2 * n * p.D + d];
    }
    __syncthreads();
    space[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && d < p.D)
      dweight[key * p.D + d] = (T)((Scaled<T>)(space[0][lane] + space[1][lane] + space[2][lane] + space[3][lane]) * (Scaled<T>)p.scale);
  }
}

int check(int dtype, int64_t tokens, int64_t rows, int64_t D, double scale, const char *who) {
  if (dtype != MG_F32 && dtype != MG_F64 && dtype != MG_F16) return fail(MG_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (tokens < 0 || rows < 0 || D < 0 || !(std::fabs(scale) <= 1e30))  // single precision holds it
    return fail(MG_ERR_BAD_ARG, "%s: %lld tokens, a table of %lld rows of %lld values, scale %g", who, (long long)tokens, (long long)rows, (long long)D,
                scale);
  if (tokens > 1 << 26 || rows > 1 << 29 || D > 1 << 24)  // what the grids hold
    return fail(MG_ERR_UNSUPPORTED, "%s: %lld tokens, a table of %lld rows of %lld values", who, (long long)tokens, (long long)rows, (long long)D);
  return MG_OK;
}

template <typename T>
int forward(const Embedding &p, const int32_t *ids, const void *weight, void *out) {
  ScopedTiming timed(TAG_EMBEDDING);
  const int lanes = lanes_of(ceil_div(p.D, Piece<T>::V)), groups = 256 / lanes;
  // several rows a group where that leaves eight blocks a compute unit
  const bool many = p.tokens >= 4ll * groups * 8 * runtime().props.multiProcessorCount;
  auto kernel = many ? embedding_kernel<T, 4> : embedding_kernel<T, 1>;
  kernel<<<dim3((unsigned)ceil_div(p.tokens, groups * (many ? 4 : 1))), dim3(256), 0, runtime().stream>>>(p, lanes, ids, (const T *)weight, (T *)out);
  MG_HIP(hipGetLastError());
  return MG_OK;
}

template <int K>
int sort_block(const Embedding &p, int bits, int passes, const int32_t *ids, unsigned *keys, unsigned *order) {
  const int lds = 1024 * K * 4 + (kSorters << bits) * 2;
  static const hipError_t allowed = hipFuncSetAttribute((const void *)sort_block_kernel<K>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                        1024 * K * 4 + (kSorters << kMostBits) * 2);
  MG_HIP(allowed);
  sort_block_kernel<K><<<dim3(1), dim3(1024), lds, runtime().stream>>>((int)p.tokens, p.rows, bits, passes, ids, keys, order);
  MG_HIP(hipGetLastError());
  return MG_OK;
}

// The tokens in order, and where each came from, in `keys` and `order`; `other` has room for both once more, `totals` for the counts.
int sort(const Embedding &p, const int32_t *ids, unsigned *keys, unsigned *order, unsigned *other, unsigned *totals, int bits, int passes) {
  if (p.tokens <= 1024) return sort_block<1>(p, bits, passes, ids, keys, order);
  if (p.tokens <= 4096) return sort_block<4>(p, bits, passes, ids, keys, order);
  if (p.tokens <= kMostInBlock) return sort_block<16>(p, bits, passes, ids, keys, order);
  const unsigned tiles = (unsigned)ceil_div(p.tokens, kTile);
  unsigned *from[2] = {nullptr, nullptr}, *to[2] = {keys, order}, *spare[2] = {other, other + p.tokens};
  if (passes % 2 == 0) std::swap(to, spare);  // the last digit's go to where they are wanted
  for (int pass = 0; pass < passes; ++pass) {
    const Tiles t{p.tokens, p.rows, Digit{pass * bits, bits}, pass ? nullptr : ids, from[0], from[1]};
    sort_count_kernel<<<dim3(tiles), dim3(1024), 0, runtime().stream>>>(t, totals);
    MG_HIP(hipGetLastError());
    sort_place_kernel<<<dim3(tiles), dim3(1024), 0, runtime().stream>>>(t, totals, to[0], to[1]);
    MG_HIP(hipGetLastError());
    from[0] = to[0], from[1] = to[1];
    std::swap(to, spare);
  }
  return MG_OK;
}

template <typename T, typename C>
int backward(const Embedding &p, const int32_t *ids, const void *grad, void *dweight) {
  if (p.tokens == 0) return mg_memset_zero(dweight, (size_t)p.rows * p.D * sizeof(T));
  int width = 1, passes = 1;
  while (width < 31 && (1ll << width) <= p.rows) ++width;  // digits of 0 to rows
  passes = (int)ceil_div(width, kMostBits);
  const int bits = (int)ceil_div(width, passes);

  constexpr int V = Piece<T>::V;
  Runs r{};
  r.tokens = p.tokens, r.rows = p.rows, r.D = p.D, r.scale = p.scale;
  const long long pieces = ceil_div(p.D, V);
  r.lanes = lanes_of(pieces);
  r.chunk = p.tokens <= 8192 ? 16 : 32;
  r.chunks = ceil_div(p.tokens, r.chunk);
  r.sum_blocks = (int)ceil_div(r.chunks, 256 / r.lanes);
  r.fill_rows = 64;

  const long long tiles = p.tokens > kMostInBlock ? ceil_div(p.tokens, kTile) : 0;
  const size_t parts = (size_t)(2 * r.chunks * p.D) * sizeof(C), places = (size_t)p.tokens * 4;
  char *space = nullptr;
  if (const int rc = workspace(parts + places * (tiles ? 4 : 2) + (size_t)(tiles << bits) * 4, (void **)&space)) return rc;
  unsigned *keys = (unsigned *)(space + parts), *order = keys + p.tokens, *other = order + p.tokens, *totals = other + 2 * p.tokens;
  hipStream_t s = runtime().stream;
  ScopedTiming timed(TAG_EMBEDDING_BWD);
  if (const int rc = sort(p, ids, keys, order, other, totals, bits, passes)) return rc;
  r.keys = keys, r.order = order;
  const unsigned along = (unsigned)ceil_div(pieces, r.lanes);
  embedding_runs_kernel<T, C><<<dim3((unsigned)(r.sum_blocks + ceil_div(p.rows, r.fill_rows)), along), dim3(256), 0, s>>>(r, (const T *)grad, (T *)dweight, (C *)space);
  MG_HIP(hipGetLastError());
  if (r.chunks > 1) {
    embedding_join_kernel<T, C><<<dim3((unsigned)(r.chunks - 1), (unsigned)std::min<long long>(ceil_div(p.D, 64), 65535)), dim3(256), 0, s>>>(r, (const C *)space, (T *)dweight);
    MG_HIP(hipGetLastError());
  }
  return MG_OK;
}

}  // namespace

}  // namespace mg

using namespace mg;

extern "C" {

int mg_embedding_fwd(int dtype, int64_t tokens, int64_t rows, int64_t D, double scale, const int32_t *ids, const void *weight, void *out) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  const int rc = check(dtype, tokens, rows, D, scale, "mg_embedding_fwd");
  if (rc || tokens == 0 || D == 0) return rc;
  if (!ids || !out || (rows && !weight)) return fail(MG_ERR_BAD_ARG, "null pointer in mg_embedding_fwd");
  const Embedding p{tokens, (int)rows, D, scale};
  if (dtype == MG_F64) return forward<double>(p, ids, weight, out);
  if (dtype == MG_F32) return forward<float>(p, ids, weight, out);
  return forward<_Float16>(p, ids, weight, out);
}

int mg_embedding_bwd(int dtype, int64_t tokens, int64_t rows, int64_t D, double scale, const int32_t *ids, const void *grad, void *dweight) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  const int rc = check(dtype, tokens, rows, D, scale, "mg_embedding_bwd");
  if (rc || rows == 0 || D == 0) return rc;
  if (!dweight || (tokens && (!ids || !grad))) return fail(MG_ERR_BAD_ARG, "null pointer in mg_embedding_bwd");
  const Embedding p{tokens, (int)rows, D, scale};
  if (dtype == MG_F64) return backward<double, double>(p, ids, grad, dweight);
  if (dtype == MG_F32) return backward<float, float>(p, ids, grad, dweight);
  return backward<_Float16, float>(p, ids, grad, dweight);
}

}  // extern "C"
