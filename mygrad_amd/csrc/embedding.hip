// Rows of a table by token, and the gradient of the table, for gfx950.
//
//   y[n] = scale W[ids[n]]  (zeros where ids[n] < 0)          dW[v] = scale * sum of grad[n] over the n with ids[n] = v
//
// Both are bound by memory.  The gradient sorts the tokens, so that the rows to be added lie in a run, whatever the text: the sorted list is cut
// into chunks of 16 to 256 tokens that are summed side by side, in the order of the tokens, and of a run that cuts go through the sums of chunks are joined in four
// shares.  Where the cuts lie hangs on all tokens of the call, and with it the last bits of a row.  Rows that no token names are zeros, which
// all rows are filled with first.  Nothing is added by atomics: the same call gives the same bits every time.
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

// A group of threads takes AT_ONCE tokens, whose rows are on their way together.  Where they are more than 40 MB they are stored past the last-level
// cache (PAST), which the table has a better use for.  The same table of 205 MB of halves each time, us alone, with a pass over the rows behind it, and with the
// gradient and passes over both, first as usual and then past it: rows of 16 MB 10.6, 21 and 95 either way, 32 MB 11, 24 and 109, 108; 48 MB 11.5, 24 and 126, 10.5, 24
// and 123; 56 MB 12.8, 26 and 136, 10.6, 26 and 133; 80 MB 17, 35 and 169, 14, 35 and 163; 128 MB 26, 51 and 225, 21, 51 and 220; 410 MB 85, 205 and 456, 64, 142 and 405.
template <typename T, int AT_ONCE, bool PAST>
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
      Piece<T>::template store<PAST>(out + (first + u) * p.D + d, p.D - d, v[u]);
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
  if ((int)threadIdx.x < bins) {
    int here[kSorters];
#pragma unroll
    for (int w = 0; w < kSorters; ++w) here[w] = counts[w * bins + threadIdx.x];
#pragma unroll
    for (int w = 0; w < kSorters; ++w) counts[w * bins + threadIdx.x] = (unsigned short)total, total += here[w];
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

// A block owns `own` rows of the table: it looks at all tokens, counts those of rows before its own, which is where its own tokens go, and puts
// these in order by itself.  One launch, no block waits for another.  Tokens are taken 16384 at a time: threads look at 16 neighbours
// each, what is the block's own goes into a queue in LDS as it stands, and wavefronts take a run of the queue each.
// All that waits for loads and for LDS, so the blocks behind them fill the gradient with zeros meanwhile.
// 16384 tokens of 50000 rows: 9 us (one block that sorts them by digits 46), 31 with 205 MB to fill, 6.6 TB/s.
constexpr int kLook = 16;
constexpr int kOwnMost = 1024;
constexpr int kOwnTile = 1024 * kLook;

struct Owners {
  int tokens, rows, own, owners;
  const int32_t *ids;
  unsigned *keys, *order;
  char *zeros;  // to be filled
  unsigned long long bytes;
};

// Zeros by the part'th of `parts` blocks of 1024.
__device__ __forceinline__ void fill_zeros(char *to, unsigned long long bytes, unsigned part, unsigned parts) {
  const unsigned long long before = min((16 - (unsigned long long)to % 16) % 16, bytes), whole = (bytes - before) / 16, after = before + whole * 16;
  uint4 *const at = reinterpret_cast<uint4 *>(to + before);
  for (unsigned long long n = (unsigned long long)part * 1024 + threadIdx.x; n < whole; n += parts * 1024ull) at[n] = uint4{0, 0, 0, 0};
  if (part == 0 && threadIdx.x < before) to[threadIdx.x] = 0;
  if (part == 0 && threadIdx.x < bytes - after) to[after + threadIdx.x] = 0;
}

__global__ void __launch_bounds__(1024) fill_kernel(char *to, unsigned long long bytes) { fill_zeros(to, bytes, blockIdx.x, gridDim.x); }

__global__ void __launch_bounds__(1024) order_kernel(Owners p) {
  if ((int)blockIdx.x >= p.owners) {
    fill_zeros(p.zeros, p.bytes, blockIdx.x - p.owners, gridDim.x - p.owners);
    return;
  }
  extern __shared__ __attribute__((aligned(16))) unsigned lds[];
  __shared__ int space[16], base[kOwnMost];
  unsigned *const queue = lds, *const counts = lds + kOwnTile;  // counts[w][d]: of wavefront w and row d
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, own = p.own;
  const int lo = blockIdx.x * own, hi = min(lo + own, p.rows);
  int bits = 1;
  while (1 << bits < own) ++bits;
  int less[1] = {0}, all = 0;  // tokens of rows before, and (thread d) of row lo + d
  if (p.tokens > kOwnTile) {
    if (t < own) base[t] = 0;
    __syncthreads();
    for (int n = t; n < p.tokens; n += 1024) {
      const int id = p.ids[n];
      less[0] += id >= 0 && id < lo;
      if (id >= lo && id < hi) atomicAdd(&base[id - lo], 1);
    }
    __syncthreads();
    if (t < own) all = base[t];
  }
  int places = 0;  // (thread d) where the next token of row lo + d goes
  for (int tile = 0; tile < p.tokens; tile += kOwnTile) {
    int id[kLook], mine = 0;
    const int from = tile + t * kLook;
    if (from + kLook <= p.tokens) {
      typedef int Quad __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
      for (int i = 0; i < kLook; i += 4) {
        const Quad four = *reinterpret_cast<const Quad *>(p.ids + from + i);
#pragma unroll
        for (int u = 0; u < 4; ++u) id[i + u] = four[u];
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLook; ++i) id[i] = from + i < p.tokens ? p.ids[from + i] : -1;
    }
#pragma unroll
    for (int i = 0; i < kLook; ++i) {
      if (p.tokens <= kOwnTile) less[0] += id[i] >= 0 && id[i] < lo;
      mine += id[i] >= lo && id[i] < hi;
    }
    int at = sum_before(mine, space);
    __shared__ int queued;
    if (t == 1023) queued = at + mine;
#pragma unroll
    for (int i = 0; i < kLook; ++i)
      if (id[i] >= lo && id[i] < hi) queue[at++] = (unsigned)(id[i] - lo) << 14 | (unsigned)(t * kLook + i);
    for (int n = t; n < kSorters * own; n += 1024) counts[n] = 0;
    __syncthreads();
    const int q = queued, rounds = (q + 1023) >> 10, begin = wave * 64 * rounds;
    for (int i = 0; i < rounds; ++i) {
      const int n = begin + i * 64 + lane;
      if (n < q) atomicAdd(&counts[wave * own + (queue[n] >> 14)], 1u);
    }
    __syncthreads();
    int total = 0;
    if (t < own) {
      int here[kSorters];
#pragma unroll
      for (int w = 0; w < kSorters; ++w) here[w] = counts[w * own + t];
#pragma unroll
      for (int w = 0; w < kSorters; ++w) counts[w * own + t] = total, total += here[w];
    }
    if (tile == 0) {
      if (p.tokens <= kOwnTile) all = total;
      block_add(less, space);
      places = less[0] + sum_before(all, space);
    }
    if (t < own) base[t] = places;
    places += total;
    __syncthreads();
    for (int i = 0; i < rounds; ++i) {
      const int n = begin + i * 64 + lane;
      const unsigned entry = n < q ? queue[n] : 0;
      const int d = entry >> 14;
      unsigned long long alike = __ballot(n < q);
      for (int b = 0; b < bits; ++b) {
        const unsigned long long vote = __ballot(d >> b & 1);
        alike &= d >> b & 1 ? vote : ~vote;
      }
      const int before = __popcll(alike & ((1ull << lane) - 1)), old = counts[wave * own + d];
      wave_sees();
      if (n < q) {
        if (before == 0) counts[wave * own + d] = old + __popcll(alike);
        p.keys[base[d] + old + before] = lo + d;
        p.order[base[d] + old + before] = tile + (entry & 16383);
      }
      wave_sees();
    }
    __syncthreads();
  }
  if (hi == p.rows) {  // tokens that are none come last
    __shared__ int end;
    if (t == own - 1) end = places;
    __syncthreads();
    for (int n = end + t; n < p.tokens; n += 1024) p.keys[n] = p.rows;
  }
}

// More tokens than a block takes: for each digit the blocks count theirs, then each finds its places from all counts.  These are read by every
// block, the square of the blocks' number in all, which shows from millions of tokens on (2048 blocks for 2^23 tokens, 4 KB of counts each).
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
constexpr int kAtOnce = 16;  // tokens whose rows are on their way together

struct Runs {
  long long tokens;
  int rows;
  long long D;
  double scale;
  int lanes;          // threads for a row's pieces
  long long chunks;
  int chunk;          // tokens of a chunk
  const unsigned *keys, *order;
};

// 16384 tokens of 50000 rows of 2048 halves: 28 us (67 MB read and 24 written, while what was filled leaves the caches for memory), and 9 for
// the join.  With eight rows on their way, and chunks of 32, it was half as much again.  Rows without tokens filled by this launch instead, from a
// bit for each that the ordering left: 9 + 57 us where the two take 31 + 35, and 8 + 19 where they take 20 + 8 (1999 tokens of 32003 x 771 floats).
//
// A group of threads adds the rows of a chunk's tokens.  A run that lies in the chunk becomes a row of the table's gradient; of one that comes in from
// the chunk before it, the part here goes to parts[2 chunk], and of one that begins here and goes on, to parts[2 chunk + 1].
template <typename T, typename C>
__global__ void __launch_bounds__(256) embedding_runs_kernel(Runs p, const T *__restrict__ grad, T *__restrict__ dweight, C *__restrict__ parts) {
  typedef typename Piece<T>::Held Held;
  constexpr int V = Piece<T>::V;
  const int lane = threadIdx.x & (p.lanes - 1), group = threadIdx.x / p.lanes, groups = 256 / p.lanes;
  const long long c = (long long)blockIdx.x * groups + group, d = ((long long)blockIdx.y * p.lanes + lane) * V;
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
  for (long long at = from; at < to; at += kAtOnce) {
    unsigned keys[kAtOnce], order[kAtOnce];
    Held rows[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const long long n = min(at + u, to - 1);
      keys[u] = p.keys[n], order[u] = p.order[n];
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      rows[u] = keys[u] < (unsigned)p.rows && at + u < to ? Piece<T>::load(grad + order[u] * p.D + d, count, T(0)) : Held{};
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (at + u >= to) break;
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

// Runs that were cut: those that begin in chunk blockIdx.x and go on, 256 values of the row a block.  Its four wavefronts take a
// share of a run's chunks each and are added in their order.
template <typename T, typename C>
__global__ void __launch_bounds__(256) embedding_join_kernel(Runs p, const C *__restrict__ parts, T *__restrict__ dweight) {
  constexpr int V = 4;
  typedef C Sums __attribute__((ext_vector_type(V), aligned(sizeof(C))));
  __shared__ Sums space[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long c = blockIdx.x, from = c * p.chunk, to = from + p.chunk;
  const unsigned key = p.keys[to], last = p.keys[to - 1], first_key = p.keys[from], came = p.keys[max(from - 1, 0ll)];
  if (key >= (unsigned)p.rows || last != key || (c > 0 && first_key == key && came == key)) return;
  long long more = 1;  // chunks after this one: 64 of them are looked at in each step
  for (;;) {
    const long long n = c + 1 + more + lane;
    const bool on = n < p.chunks && p.keys[n * p.chunk] == key && p.keys[n * p.chunk - 1] == key;
    const unsigned long long off = ~__ballot(on);
    if (off) {
      more += __builtin_ctzll(off);
      break;
    }
    more += 64;
  }
  const long long share = (more + 3) / 4, first = c + 1 + wave * share, end = min(first + share, c + 1 + more);
  for (long long d0 = (long long)blockIdx.y * 64 * V; d0 < p.D; d0 += (long long)gridDim.y * 64 * V) {
    const long long d = d0 + lane * V, count = p.D - d;
    auto load = [&](const C *at) {
      Sums v{};
      if (count >= V) return *reinterpret_cast<const Sums *>(at);
#pragma unroll
      for (int n = 0; n < V; ++n)
        if (n < count) v[n] = at[n];
      return v;
    };
    Sums sum{};
    if (count > 0) {
      if (wave == 0) sum = load(parts + (2 * c + 1) * p.D + d);
#pragma unroll 4
      for (long long n = first; n < end; ++n) sum += load(parts + 2 * n * p.D + d);
    }
    __syncthreads();
    space[wave][lane] = sum;
    __syncthreads();
    if (wave == 0) {
      sum = ((space[0][lane] + space[1][lane]) + space[2][lane]) + space[3][lane];
#pragma unroll
      for (int n = 0; n < V; ++n)
        if (n < count) dweight[key * p.D + d + n] = (T)((Scaled<T>)sum[n] * (Scaled<T>)p.scale);
    }
  }
}

int check(int dtype, int64_t tokens, int64_t rows, int64_t D, double scale, const char *who) {
  if (dtype != MG_F32 && dtype != MG_F64 && dtype != MG_F16) return fail(MG_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (tokens < 0 || rows < 0 || D < 0 || !(std::fabs(scale) <= 1e30))  // single precision holds it
    return fail(MG_ERR_BAD_ARG, "%s: %lld tokens, a table of %lld rows of %lld values, scale %g", who, (long long)tokens, (long long)rows, (long long)D,
                scale);
  if (tokens >= 1 << 26 || rows > 1 << 29 || D > 1 << 24)  // what the grids hold
    return fail(MG_ERR_UNSUPPORTED, "%s: %lld tokens, a table of %lld rows of %lld values", who, (long long)tokens, (long long)rows, (long long)D);
  return MG_OK;
}

template <typename T>
int forward(const Embedding &p, const int32_t *ids, const void *weight, void *out) {
  ScopedTiming timed(TAG_EMBEDDING);
  const int lanes = lanes_of(ceil_div(p.D, Piece<T>::V)), groups = 256 / lanes;
  // several rows a group where that leaves eight blocks a compute unit
  const bool many = p.tokens >= 4ll * groups * 8 * runtime().props.multiProcessorCount;
  const bool past = (double)p.tokens * p.D * sizeof(T) > 4e7;
  auto kernel = many ? past ? embedding_kernel<T, 4, true> : embedding_kernel<T, 4, false>
                     : past ? embedding_kernel<T, 1, true> : embedding_kernel<T, 1, false>;
  // A launch has fewer than 2^32 threads; rows that a block takes four of at a time reach that with 2^26 - 3 tokens.
  const long long at_once = groups * (many ? 4 : 1), most = ((1ll << 24) - 1) * at_once;
  for (long long at = 0; at < p.tokens; at += most) {
    Embedding part = p;
    part.tokens = std::min(p.tokens - at, most);
    kernel<<<dim3((unsigned)ceil_div(part.tokens, at_once)), dim3(256), 0, runtime().stream>>>(part, lanes, ids + at, (const T *)weight, (T *)out + at * p.D);
    MG_HIP(hipGetLastError());
  }
  return MG_OK;
}

// The tokens in order, and where each came from, in `keys` and `order`, and `zeros` filled: by blocks that own rows, or ...
int order_by_owners(const Embedding &p, const int32_t *ids, unsigned *keys, unsigned *order, void *zeros, size_t bytes) {
  const int own = std::max<int>(64, (int)ceil_div(ceil_div(p.rows, runtime().props.multiProcessorCount), 64) * 64);
  const int lds = (kOwnTile + kSorters * own) * 4;
  static const hipError_t allowed = hipFuncSetAttribute((const void *)order_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (kOwnTile + kSorters * kOwnMost) * 4);
  MG_HIP(allowed);
  const int owners = (int)ceil_div(p.rows, own), fillers = (int)std::min<long long>(ceil_div((long long)bytes, 16 * 1024 * 4), 4 * runtime().props.multiProcessorCount);
  order_kernel<<<dim3((unsigned)(owners + fillers)), dim3(1024), lds, runtime().stream>>>(
      Owners{(int)p.tokens, p.rows, own, owners, ids, keys, order, (char *)zeros, bytes});
  MG_HIP(hipGetLastError());
  return MG_OK;
}

int fill(void *to, size_t bytes) {
  const long long blocks = std::min<long long>(ceil_div((long long)bytes, 16 * 1024 * 4), 4 * runtime().props.multiProcessorCount);
  fill_kernel<<<dim3((unsigned)blocks), dim3(1024), 0, runtime().stream>>>((char *)to, bytes);
  MG_HIP(hipGetLastError());
  return MG_OK;
}

// ... by digits; `other` has room for keys and order once more, `totals` for the counts.
int order_by_digits(const Embedding &p, const int32_t *ids, unsigned *keys, unsigned *order, unsigned *other, unsigned *totals, int bits, int passes,
                    void *zeros, size_t bytes) {
  if (const int rc = fill(zeros, bytes)) return rc;
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
  int width = 1, passes = 1;
  while (width < 31 && (1ll << width) <= p.rows) ++width;  // digits of 0 to rows
  passes = (int)ceil_div(width, kMostBits);
  const int bits = (int)ceil_div(width, passes);

  const size_t bytes = (size_t)p.rows * p.D * sizeof(T);
  if (p.tokens == 0) {
    ScopedTiming timed(TAG_EMBEDDING_BWD);
    return fill(dweight, bytes);
  }
  constexpr int V = Piece<T>::V;
  Runs r{};
  r.tokens = p.tokens, r.rows = p.rows, r.D = p.D, r.scale = p.scale;
  const long long pieces = ceil_div(p.D, V);
  r.lanes = lanes_of(pieces);
  // One round of a thread's loads where there are threads for more; else up to 16, which leave fewer cuts to join.
  const long long rounds = std::max((p.tokens / kAtOnce * r.lanes) >> 18, p.tokens >> 17);
  r.chunk = kAtOnce * (int)std::min<long long>(std::max<long long>(rounds, 1), 16);
  r.chunks = ceil_div(p.tokens, r.chunk);

  // 50000 rows, us by owners and by digits: 16384 tokens 9 and 39, 65536 38 and 46, 131072 80 and 48.
  const bool owners = p.rows <= kOwnMost * runtime().props.multiProcessorCount && p.tokens <= 1 << 16;
  const long long tiles = owners ? 0 : ceil_div(p.tokens, kTile);
  const size_t parts = (size_t)(2 * r.chunks * p.D) * sizeof(C), places = (size_t)p.tokens * 4;
  char *space = nullptr;
  if (const int rc = workspace(parts + places * (owners ? 2 : 4) + (size_t)(tiles << bits) * 4, (void **)&space)) return rc;
  unsigned *keys = (unsigned *)(space + parts), *order = keys + p.tokens, *other = order + p.tokens, *totals = other + 2 * p.tokens;
  hipStream_t s = runtime().stream;
  ScopedTiming timed(TAG_EMBEDDING_BWD);
  if (const int rc = owners ? order_by_owners(p, ids, keys, order, dweight, bytes)
                              : order_by_digits(p, ids, keys, order, other, totals, bits, passes, dweight, bytes))
    return rc;
  r.keys = keys, r.order = order;
  const unsigned along = (unsigned)ceil_div(pieces, r.lanes);
  embedding_runs_kernel<T, C><<<dim3((unsigned)ceil_div(r.chunks, 256 / r.lanes), along), dim3(256), 0, s>>>(r, (const T *)grad, (T *)dweight, (C *)space);
  MG_HIP(hipGetLastError());
  if (r.chunks > 1) {
    embedding_join_kernel<T, C><<<dim3((unsigned)(r.chunks - 1), (unsigned)std::min<long long>(ceil_div(p.D, 256), 65535)), dim3(256), 0, s>>>(r, (const C *)space, (T *)dweight);
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
