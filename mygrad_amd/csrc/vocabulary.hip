// What a model's logits say of the tokens of a vocabulary, and its gradients, for gfx950.
//
//   m = max z     t = z - m     s = sum e^t     p = e^t / s     a = sum p t                               (over the V logits of a row)
//   log probability of token k: t_k - log s     entropy: log s - a     the likeliest tokens: the largest z, the lowest one among equals
//   dz_j = g (delta_jk - p_j) - h p_j (t_j - a)        with the gradients g of the log probability and h of the entropy
//
//   distillation: t = (z - m) / T, and q = softmax(y / T) of a teacher's logits y for K tokens c_k
//   loss = sum_k q_k (log q_k - log p_{c_k})           dz_j = g / T (p_j - sum of the q_k with c_k = j)
//
// A row whose logits are all minus infinity has no distribution: its log probabilities are minus infinity (a loss against it is infinite),
// its entropy 0 and its gradient zeros.  Infinity or NaN among the logits makes a row's results NaN.
#include "row_device.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace mg {

namespace {

constexpr int kMostTop = 128;     // likeliest tokens that are looked for
constexpr int kMostTaught = 256;  // a teacher's tokens for a row: a thread of a block each, or kTurns for each that shares a row otherwise
constexpr int kTurns = 4;

struct Vocabulary {
  long long rows;
  int V;
  int top;         // likeliest tokens wanted, or a teacher's
  double per;      // 1 / temperature
};

template <typename C>
__device__ __forceinline__ C infinity() {
  return sizeof(C) == 4 ? (C)__builtin_inff() : (C)__builtin_inf();
}

// What the backward pass needs of a row.
template <typename C>
struct Row {
  C m, s, a;  // the largest logit (0 in a row without any), the sum of exponentials, the mean of t (distillation: 1, or 0 without a teacher's token)
};

// The log probability of a token with logit z.
template <typename C>
__device__ __forceinline__ C log_probability(const Row<C> &row, C z, C per) {
  return row.s == 0 ? -infinity<C>() : (z - row.m) * per - log(row.s);
}

// Whole numbers in the order of the values, NaN last of all and both zeros alike.
__device__ __forceinline__ uint32_t order_of(float z) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, z + 0.0f);
  return z != z ? 0xffffffffu : bits >> 31 ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_of(double z) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, z + 0.0);
  return z != z ? ~0ull : bits >> 63 ? ~bits : bits | 1ull << 63;
}
__device__ __forceinline__ float value_of(uint32_t order) { return __builtin_bit_cast(float, order >> 31 ? order & 0x7fffffffu : ~order); }
__device__ __forceinline__ double value_of(uint64_t order) { return __builtin_bit_cast(double, order >> 63 ? order & ~(1ull << 63) : ~order); }

// The exponential of a number that is not positive.  For logits of float16 it is the instruction's own, of an argument rounded in single precision: off by
// |x| 2^-24 of itself.  A gradient is rounded to 11 bits after that.  The results of the sums are not, but there the terms weigh it: s is off by |a| 2^-24 of
// itself, where |a| is at most log V, which is what the rounding of t leaves of it, too.
template <typename T>
__device__ __forceinline__ float exponential(float x) {
  return sizeof(T) == 2 ? __builtin_amdgcn_exp2f(x * 1.4426950408889634f) : expf(x);
}
template <typename T>
__device__ __forceinline__ double exponential(double x) {
  return exp(x);
}

// LANES threads that share a row: eight, sixteen, a wavefront, or a block of 256.  All of them call; `space` is 16 values of LDS for a block.
template <int LANES, typename C>
__device__ __forceinline__ C group_max(C v, C *space) {
  v = lanes_max(v, min(LANES, 64));
  if (LANES <= 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) space[threadIdx.x >> 6] = v;
  __syncthreads();
  return max(max(space[0], space[1]), max(space[2], space[3]));
}
template <int LANES, typename C>
__device__ __forceinline__ C group_add(C v, C *space) {
  v = lanes_add(v, min(LANES, 64));
  if (LANES <= 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) space[threadIdx.x >> 6] = v;
  __syncthreads();
  return (space[0] + space[1]) + (space[2] + space[3]);
}

// ---- sums of a row in one pass --------------------------------------------------------------------------------------------------
constexpr int kAtOnce = 4;  // pieces that a thread has on their way together

// m: the largest logit so far (minus infinity: none); s = sum e^t and w = sum e^t t with t = (z - m) / T, none of them from a logit of minus infinity.
template <typename C>
struct Sums {
  C m, s, w;
};

// A t of minus infinity times its exponential of 0 is no number; this is.
template <typename C>
__device__ __forceinline__ C bounded(C t) {
  return max(t, (C)-1e30);
}
template <typename C>
__device__ __forceinline__ C base_of(C m) {
  return m == -infinity<C>() ? C(0) : m;
}

// t and e^t as the sums take them.  In single precision t is held at -104 and above (a NaN stays one), where the exponential is less than half of
// the smallest number, so zero.  A Cody-Waite reduction: with n = round(t log2 e), made by adding 1.5 2^23, and log2 e in two parts, 2^(t log2 e - n) is the
// instruction's, to a unit or two, and the result is that times 2^n: nine instructions where the library's function has thirteen.  1021 x 32003 logits with
// entropies and alternatives take 34 us so, 40 with that.
template <typename T>
__device__ __forceinline__ float term(float &t) {
  if constexpr (sizeof(T) == 2) {
    const float e = exponential<T>(t);
    t = bounded(t);
    return e;
  } else {
    constexpr float kMagic = 12582912.0f, kHigh = 1.44269504f, kLow = 1.925963033e-8f;  // log2 e in two parts
    t = __builtin_elementwise_maximum(t, -104.0f);
    const float shifted = __builtin_fmaf(t, kHigh, kMagic), n = shifted - kMagic;
    const float rest = __builtin_fmaf(t, kLow, __builtin_fmaf(t, kHigh, -n));
    return __builtin_ldexpf(__builtin_amdgcn_exp2f(rest), (int)n);
  }
}
template <typename T>
__device__ __forceinline__ double term(double &t) {
  const double e = exp(t);
  t = bounded(t);
  return e;
}

// As seen from a larger m.
template <typename T, bool MEAN, typename C>
__device__ __forceinline__ void move_to(Sums<C> &a, C m, C per) {
  const C step = bounded((a.m - base_of(m)) * per), c = exponential<T>(step);
  if (MEAN) a.w = c * (a.w + a.s * step);
  a.s *= c;
  a.m = m;
}

// Returns the largest of the pieces' values, NaN passed over.
template <typename T, bool MEAN, int PIECES, typename C>
__device__ __forceinline__ C add_pieces(Sums<C> &a, const typename Piece<T>::Held (&z)[kAtOnce], C per) {
  constexpr int V = Piece<T>::V;
  T most = z[0][0];  // a NaN is passed over: the sum shows it
#pragma unroll
  for (int u = 0; u < PIECES; ++u)
#pragma unroll
    for (int n = 0; n < V; ++n) most = sizeof(T) == 2 ? (T)__builtin_fmaxf16((_Float16)most, (_Float16)z[u][n]) : (T)max((C)most, (C)z[u][n]);
  move_to<T, MEAN>(a, max(a.m, (C)most), per);
  const C base = base_of(a.m);
  C s[kAtOnce] = {}, w[kAtOnce] = {};
#pragma unroll
  for (int n = 0; n < V; ++n)
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      C t = ((C)z[u][n] - base) * per;
      const C e = term<T>(t);
      s[u] += e;
      if (MEAN) w[u] += e * t;
    }
  a.s += (s[0] + s[1]) + (s[2] + s[3]);
  if (MEAN) a.w += (w[0] + w[1]) + (w[2] + w[3]);
  return (C)most;
}

// Of the first `pieces`, the same number for all threads that share a row: the others hold nothing.
template <typename T, bool MEAN, typename C>
__device__ __forceinline__ C add_pieces(Sums<C> &a, const typename Piece<T>::Held (&z)[kAtOnce], C per, long long pieces) {
  static_assert(kAtOnce == 4);
  if (pieces >= 4) return add_pieces<T, MEAN, 4>(a, z, per);
  if (pieces == 1) return add_pieces<T, MEAN, 1>(a, z, per);
  if (pieces == 2) return add_pieces<T, MEAN, 2>(a, z, per);
  return add_pieces<T, MEAN, 3>(a, z, per);
}

// Of all threads' sums.
template <int LANES, typename T, bool MEAN, typename C>
__device__ __forceinline__ Sums<C> join(Sums<C> a, C per, C *space) {
  move_to<T, MEAN>(a, lanes_max(a.m, min(LANES, 64)), per);
  a.s = lanes_add(a.s, min(LANES, 64));
  if (MEAN) a.w = lanes_add(a.w, min(LANES, 64));
  if (LANES <= 64) return a;
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) space[wave] = a.m, space[4 + wave] = a.s, space[8 + wave] = a.w;
  __syncthreads();
  Sums<C> all{max(max(space[0], space[1]), max(space[2], space[3])), 0, 0};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    Sums<C> one{space[w], space[4 + w], space[8 + w]};
    move_to<T, MEAN>(one, all.m, per);
    all.s += one.s, all.w += one.w;
  }
  return all;
}

template <typename C>
__device__ __forceinline__ Row<C> row_of(const Sums<C> &a) {
  return Row<C>{base_of(a.m), a.s, a.s == 0 ? C(0) : a.w / a.s};
}

// Pieces of a thread's from `at` on, LANES threads side by side.
template <int LANES, typename T>
__device__ __forceinline__ void load_pieces(typename Piece<T>::Held (&z)[kAtOnce], const T *row, long long at, long long end) {
  constexpr int V = Piece<T>::V;
#pragma unroll
  for (int u = 0; u < kAtOnce; ++u) {
    const long long d = at + (long long)u * LANES * V;
    z[u] = Piece<T>::load(row + d, end - d, (T)-__builtin_inff());
  }
}

// ---- the likeliest tokens ---------------------------------------------------------------------------------------------------------
// The threads' own maxima in a block's first step bound the k-th largest logit from below: k of them are as large as the k-th of them.  What is
// not below that bound is collected in LDS as the pass over the row goes on (k for each step, about) and ranked there at its end by comparing
// all with all.  Where that is more than there is room for (ties, mostly), or logits are NaN, a second pass begins with the bound by all values and
// drops all but the first k when the list is full; the last of those is the new bound.
// 8 rows of 50001 halves with 8 alternatives: 6.3 us and 4.4 for the join.  With each thread comparing its maximum with all others', and every logit's
// order with the bound's, 10.8 and 7.4.
template <typename C>
struct Candidate {  // in double precision; one number in single
  uint64_t value;
  int where;
  __device__ __forceinline__ Candidate() {}
  __device__ __forceinline__ Candidate(uint64_t order, int place) : value(order), where(place) {}
  __device__ __forceinline__ uint64_t order() const { return value; }
  __device__ __forceinline__ int place() const { return where; }
  __device__ __forceinline__ bool before(const Candidate &o) const { return value > o.value || (value == o.value && where < o.where); }
};
template <>
struct Candidate<float> {
  uint64_t key;  // the order of the value, then that of the place from behind
  __device__ __forceinline__ Candidate() {}
  __device__ __forceinline__ Candidate(uint32_t order, int place) : key((uint64_t)order << 32 | ~(uint32_t)place) {}
  __device__ __forceinline__ uint32_t order() const { return (uint32_t)(key >> 32); }
  __device__ __forceinline__ int place() const { return (int)~(uint32_t)key; }
  __device__ __forceinline__ bool before(const Candidate &o) const { return key > o.key; }
};

template <typename T, typename C>
struct Likeliest {
  static constexpr int kStep = 256 * Piece<T>::V;  // that a block may add before it looks at the count
  static constexpr int kRoom = 2 * kStep < 1024 ? 1024 : 2 * kStep;
  typedef Candidate<C> Found;
  typedef decltype(order_of(C(0))) Order;
  Found held[kRoom];
  Found first[kMostTop];
  Order most[256];
  int count;
  Found bound;  // what does not come before it, and is not it, is not wanted

  // The largest number of which no more than its highest bits are set that k of the values of a wavefront's lanes are not less than: two bits a step.
  template <int N>
  __device__ __forceinline__ static Order not_above(const Order (&v)[N], int k) {
    constexpr int BITS = 8 * sizeof(Order), LEAST = sizeof(C) == 4 ? 12 : 40;
    Order found = 0;
#pragma unroll
    for (int b = BITS - 2; b >= LEAST; b -= 2) {
      const Order one = (Order)1 << b;
      int n[3] = {};
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int i = 0; i < 3; ++i) n[i] += __popcll(__ballot(v[u] >= found + (i + 1) * one));
      found += one * ((n[0] >= k) + (n[1] >= k) + (n[2] >= k));
    }
    return found;
  }
  // Returns a bound by the k-th of the threads' largest values (0: a thread has none), or of those of four threads each where that are enough, by their
  // highest bits; all that float16 has are among these.  Fewer than k: all numbers are wanted.
  __device__ __forceinline__ C begin(Order own, int k) {
    most[threadIdx.x] = own;
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    Order four[4];  // each wavefront for itself
#pragma unroll
    for (int u = 0; u < 4; ++u) four[u] = most[(threadIdx.x & 63) + 64 * u];
    const Order one[1] = {max(max(four[0], four[1]), max(four[2], four[3]))};
    const Order found = max(k <= 32 ? not_above(one, k) : not_above(four, k), order_of(-infinity<C>()));
    if (threadIdx.x == 0) bound = Found(found, 0x7fffffff);
    return value_of(found);
  }
  __device__ __forceinline__ void add(const Found &f) {
    const int n = atomicAdd(&count, 1);
    if (n < kRoom) held[n] = f;
  }
  // What is not less than `least`, of the first `pieces`.  A NaN is passed over.
  __device__ __forceinline__ void add_pieces(const typename Piece<T>::Held (&z)[kAtOnce], C least, long long d, long long end, long long pieces) {
    constexpr int V = Piece<T>::V;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (u >= pieces) break;
      const long long at = d + u * kStep, left = end - at;
      int hits = 0;
#pragma unroll
      for (int n = 0; n < V; ++n) hits |= (C)z[u][n] >= least ? 1 << n : 0;
      if (left < V) hits &= left <= 0 ? 0 : (1 << left) - 1;
      if (hits == 0) continue;
      int n = atomicAdd(&count, __popc(hits));
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (hits >> i & 1) {
          if (n < kRoom) held[n] = Found(order_of((C)z[u][i]), (int)at + i);
          ++n;
        }
    }
  }
  // The first k of the list, in order, in `first`; returns how many there are.  All threads call.
  __device__ __forceinline__ int rank(int k) {
    __syncthreads();
    const int n = count;
    for (int i = threadIdx.x; i < n; i += 256) {
      const Found mine = held[i];
      int better = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) better += held[j].before(mine);
      if (better < k) first[better] = mine;
    }
    __syncthreads();
    return min(n, k);
  }
  // Room for another step.  All threads call.
  __device__ __forceinline__ void make_room(int k) {
    __syncthreads();
    const int now = count;
    __syncthreads();  // nobody adds before all have seen the same count
    if (now + kStep <= kRoom) return;
    const int left = rank(k);
    if ((int)threadIdx.x < left) held[threadIdx.x] = first[threadIdx.x];
    if (threadIdx.x == 0) count = left, bound = first[left - 1];
    __syncthreads();
  }
  __device__ __forceinline__ bool wants(const Found &f) const { return f.order() >= bound.order() && !bound.before(f); }
};

template <typename T, typename C>
__device__ __forceinline__ void collect(Likeliest<T, C> &list, const typename Piece<T>::Held &z, long long d, long long end, int k) {
  list.make_room(k);
#pragma unroll
  for (int n = 0; n < Piece<T>::V; ++n) {
    const Candidate<C> f(order_of((C)z[n]), (int)(d + n));
    if (d + n < end && list.wants(f)) list.add(f);
  }
}

// ---- log probabilities ----------------------------------------------------------------------------------------------------------
// What is made of a row's sums.
template <typename T, typename C>
struct Scores {
  static constexpr bool kTempered = false;  // the temperature is 1, which saves a product for each logit: 4096 x 50000 halves 209 us both passes, 213 with it
  const int32_t *ids;
  const T *logits;
  C *scores, *entropy;
  Row<C> *kept;

  template <int LANES>
  __device__ __forceinline__ void end(const Vocabulary &p, long long r, int lane, const Sums<C> &sums, C *) const {
    if (lane) return;
    const Row<C> row = row_of(sums);
    if (kept) kept[r] = row;
    if (scores) {
      const int id = ids[r];
      scores[r] = id < 0 || id >= p.V ? C(0) : log_probability<C>(row, (C)logits[r * p.V + id], 1);
    }
    if (entropy) entropy[r] = row.s == 0 ? C(0) : log(row.s) - row.a;
  }
};

// Or of those and a teacher's logits: a thread takes one of them, or up to four in turns.  q goes to memory for the backward
// pass: that of all entries of a token where it stands first, and -1 for those that have nothing to add.
template <typename T, typename Y, typename C>
struct Distillation {
  static constexpr bool kTempered = true;
  const int32_t *ids;
  const T *logits;
  const Y *teacher;
  C *loss;
  Row<C> *kept;
  C *shares;

  template <int LANES>
  __device__ __forceinline__ void end(const Vocabulary &p, long long r, int lane, const Sums<C> &sums, C *space) const {
    constexpr int TURNS = LANES < 256 ? kTurns : 1, MOST = TURNS * LANES;
    const C per = (C)p.per;
    Row<C> row = row_of(sums);
    int id[TURNS];
    C y[TURNS], z[TURNS], most = -infinity<C>();
#pragma unroll
    for (int n = 0; n < TURNS; ++n) {
      const int k = lane + n * LANES;
      id[n] = k < p.top ? ids[r * p.top + k] : -1;
      const bool there = id[n] >= 0 && id[n] < p.V;
      y[n] = there ? (C)teacher[r * p.top + k] : -infinity<C>();
      z[n] = there ? (C)logits[r * p.V + id[n]] : C(0);
      most = max(most, y[n]);
    }
    const C base = base_of(group_max<LANES>(most, space));
    C total = 0, f[TURNS];
#pragma unroll
    for (int n = 0; n < TURNS; ++n) {
      y[n] = (y[n] - base) * per;
      total += f[n] = exp(y[n]);
    }
    total = group_add<LANES>(total, space);
    C sum = 0;
#pragma unroll
    for (int n = 0; n < TURNS; ++n) {
      f[n] = total == 0 ? C(0) : f[n] / total;
      sum += f[n] == 0 ? C(0) : f[n] * ((y[n] - log(total)) - log_probability<C>(row, z[n], per));
    }
    sum = group_add<LANES>(sum, space);
    if (shares) {
      __shared__ __attribute__((aligned(16))) int tokens[256 / LANES][MOST];
      __shared__ C q[256 / LANES][MOST];
      const int group = threadIdx.x / LANES;
#pragma unroll
      for (int n = 0; n < TURNS; ++n) tokens[group][lane + n * LANES] = id[n] < p.V ? id[n] : -1, q[group][lane + n * LANES] = f[n];
      if (LANES <= 64) wave_sees();
      else __syncthreads();
#pragma unroll
      for (int n = 0; n < TURNS; ++n) {
        const int k = lane + n * LANES;
        if (k >= p.top) break;
        const int own = id[n] < p.V ? id[n] : -1;
        int alike = 0;  // seldom more than one
#pragma unroll 4
        for (int j = 0; j < p.top; j += 4) {
          typedef int Quad __attribute__((ext_vector_type(4)));
          const Quad four = *reinterpret_cast<const Quad *>(&tokens[group][j]);
          alike += (four[0] == own) + (four[1] == own) + (four[2] == own) + (four[3] == own);
        }
        C all = f[n];
        bool adds = own >= 0;
        if (adds && alike > 1) {
          all = 0;
          for (int j = 0; j < p.top; ++j)
            if (tokens[group][j] == own) all += q[group][j], adds = adds && j >= k;
        }
        shares[r * p.top + k] = adds ? all : C(-1);
      }
      if (LANES <= 64) wave_sees();
      else __syncthreads();
    }
    if (lane) return;
    loss[r] = sum;
    row.a = total == 0 ? C(0) : total / total;  // 1, or NaN
    if (kept) kept[r] = row;
  }
};

struct Top {
  int parts;      // of a row, each for a block
  int part;       // logits in one
  void *partial;  // sums of parts
  void *found;    // and their candidates: (rows, parts, top)
  void *scores;
  int32_t *ids;
};

// Eight or sixteen threads or a wavefront per row, or a block per part of a row.  Bound by memory, and in float16 nearly by the
// exponentials.
template <typename T, typename C, int LANES, bool MEAN, bool TOP, typename End>
__global__ void __launch_bounds__(256) row_kernel(Vocabulary p, Top w, const T *__restrict__ logits, End end) {
  constexpr int V = Piece<T>::V, kStep = LANES * V * kAtOnce;
  __shared__ C space[16];
  __shared__ std::conditional_t<TOP, Likeliest<T, C>, int> list;
  const int lane = threadIdx.x & (LANES - 1);
  constexpr bool SHARED = LANES < 256;  // rows share a block
  const long long units = SHARED ? (p.rows + 256 / LANES - 1) / (256 / LANES) : p.rows * w.parts;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const long long r = SHARED ? unit * (256 / LANES) + threadIdx.x / LANES : unit / w.parts;
    if (SHARED && r >= p.rows) return;
    const int part = SHARED ? 0 : (int)(unit - r * w.parts);
    const T *row = logits + r * p.V;
    const long long from = (long long)part * w.part, to = min(from + w.part, (long long)p.V);
    const C per = End::kTempered ? (C)p.per : C(1);
    Sums<C> sums{-infinity<C>(), 0, 0};
    typename Piece<T>::Held z[kAtOnce];
    if constexpr (TOP) {
      __syncthreads();  // the list of the unit before has been read
      C least;
      for (long long d0 = from; d0 < to; d0 += kStep) {
        const long long d = d0 + lane * V, pieces = (to - d0 + LANES * V - 1) / (LANES * V);
        load_pieces<LANES>(z, row, d, to);
        const C most = add_pieces<T, MEAN>(sums, z, per, pieces);
        if (d0 == from) least = list.begin(d < to ? order_of(most) : 0, p.top);
        if (most >= least) list.add_pieces(z, least, d, to, pieces);
      }
    } else {
      for (long long d0 = from; d0 < to; d0 += kStep) {
        load_pieces<LANES>(z, row, d0 + lane * V, to);
        add_pieces<T, MEAN>(sums, z, per, (to - d0 + LANES * V - 1) / (LANES * V));
      }
    }
    const C own = sums.m;
    sums = join<LANES, T, MEAN>(sums, per, space);
    const bool whole = SHARED || w.parts == 1;
    if (!whole && lane == 0) ((Sums<C> *)w.partial)[unit] = sums;
    if (!TOP && whole) end.template end<LANES>(p, r, lane, sums, space);
    if constexpr (TOP) {
      __syncthreads();
      const bool again = list.count > Likeliest<T, C>::kRoom || sums.s != sums.s;
      if (again) {
        __syncthreads();
        list.begin(from + lane * V < to ? order_of(own) : 0, p.top);
        for (long long d0 = from; d0 < to; d0 += kStep) {
          const long long d = d0 + lane * V;
          load_pieces<LANES>(z, row, d, to);
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u)
            if (d0 + u * LANES * V < to) collect<T, C>(list, z[u], d + u * LANES * V, to, p.top);
        }
      }
      const int found = list.rank(p.top);
      if ((int)threadIdx.x < p.top) {
        const bool there = (int)threadIdx.x < found;
        const Candidate<C> f = there ? list.first[threadIdx.x] : Candidate<C>(0, 0);
        const long long at = unit * p.top + threadIdx.x;
        if (w.parts == 1) {
          w.ids[at] = f.place();
          ((C *)w.scores)[at] = log_probability<C>(row_of(sums), (C)row[f.place()], 1);
        } else {
          ((Candidate<C> *)w.found)[at] = f;
        }
      }
      if (whole) end.template end<LANES>(p, r, lane ^ 192, sums, space);  // by a wavefront that has nothing else to wait for, mostly
      __syncthreads();
    }
  }
}

// Joins the parts of a row.
template <typename T, typename C, bool MEAN, bool TOP, typename End>
__global__ void __launch_bounds__(256) row_join_kernel(Vocabulary p, Top w, const T *__restrict__ logits, End end) {
  __shared__ C space[16];
  __shared__ std::conditional_t<TOP, Likeliest<T, C>, int> list;
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const C per = End::kTempered ? (C)p.per : C(1);
    const int all = w.parts * p.top;
    const Candidate<C> *found = (const Candidate<C> *)w.found + r * all;
    Candidate<C> mine(0, 0);
    if (TOP && (int)threadIdx.x < all) mine = found[threadIdx.x];  // on its way with the sums
    Sums<C> sums{-infinity<C>(), 0, 0};
    for (int n = threadIdx.x; n < w.parts; n += 256) {
      Sums<C> next = ((const Sums<C> *)w.partial)[r * w.parts + n];
      const C m = max(sums.m, next.m);
      move_to<T, MEAN>(sums, m, per);
      move_to<T, MEAN>(next, m, per);
      sums.s += next.s, sums.w += next.w;
    }
    sums = join<256, T, MEAN>(sums, per, space);
    if constexpr (!TOP) end.template end<256>(p, r, threadIdx.x, sums, space);
    if constexpr (TOP) {
      auto most = mine.order();
      for (int n = threadIdx.x + 256; n < all; n += 256) most = max(most, found[n].order());
      list.begin(most, p.top);
      for (int n0 = 0; n0 < all; n0 += 256) {
        list.make_room(p.top);
        if (n0 + (int)threadIdx.x < all) {
          const Candidate<C> f = n0 ? found[n0 + threadIdx.x] : mine;
          if (f.order() && list.wants(f)) list.add(f);
        }
      }
      list.rank(p.top);
      if ((int)threadIdx.x < p.top) {
        const int place = list.first[threadIdx.x].place();
        w.ids[r * p.top + threadIdx.x] = place;
        ((C *)w.scores)[r * p.top + threadIdx.x] = log_probability<C>(row_of(sums), (C)logits[r * p.V + place], 1);
      }
      end.template end<256>(p, r, threadIdx.x ^ 192, sums, space);
      __syncthreads();
    }
  }
}

// How a pass over the rows is laid out.
struct Plan {
  int lanes;  // threads that share a row: 8, 16, 64 or 256
  int parts, part;
  unsigned blocks;
};

// Rows that eight or sixteen threads or a wavefront take in one step share a block; where there are enough for all wavefronts, also those that a
// wavefront takes in four.  2^27 bytes of halves, us forward: rows of 64 by eight threads 58, by a wavefront 630; of 300 by sixteen 36, by a wavefront 111; of
// 2100 by a wavefront 36, by a block 73; of 8000 29 either way; distillation with 8 of 64 tokens, both passes, 207 by eight threads a row, 1342 by
// a wavefront.  Longer ones have a block each, or, where there are few, parts for four blocks a compute unit and a launch that joins
// them, if that saves a block five steps (three where likeliest tokens are looked for, whose list a block waits for in each step; then two parts are
// worth it, otherwise three).  us in parts and without: 4 rows of 32003 halves 7.0 and 7.0, of 50001 7.1 and 9.9, of 131101 7.2 and 19.6;
// 257 of 16001 8.2 and 5.9, of 50001 13.0 and 12.9, of 131101 22.8 and 30.7; 500 of 131101 floats 47.7 and 42.2.  With 8 alternatives 4
// rows of 16001 halves 9.3 and 9.1, of 32003 9.5 and 13.6, 257 of 50001 19.6 and 22.6, 500 of them 27.0 and 27.4.
template <typename T>
Plan plan_of(const Vocabulary &p, bool top) {
  constexpr int V = Piece<T>::V;
  const long long most = 1 << 22;
  if (!top && p.top <= 8 * kTurns && p.V <= 8 * V * kAtOnce) return Plan{8, 1, p.V, (unsigned)std::min<long long>(ceil_div(p.rows, 32), most)};
  if (!top && p.top <= 16 * kTurns && p.V <= 16 * V * kAtOnce) return Plan{16, 1, p.V, (unsigned)std::min<long long>(ceil_div(p.rows, 16), most)};
  const int steps = p.rows >= 16ll * runtime().props.multiProcessorCount ? 4 : 1;
  if (!top && p.V <= 64 * V * kAtOnce * steps) return Plan{64, 1, p.V, (unsigned)std::min<long long>(ceil_div(p.rows, 4), most)};
  const long long wanted = 4ll * runtime().props.multiProcessorCount / p.rows, piece = 256 * V, step = piece * kAtOnce;
  const long long parts = std::max<long long>(1, std::min<long long>(wanted, ceil_div(p.V, piece)));
  long long part = ceil_div(ceil_div(p.V, parts), piece) * piece;
  if (parts < (top ? 2 : 3) || ceil_div(p.V, step) - ceil_div(part, step) <= (top ? 2 : 4)) part = p.V;
  Plan plan{256, (int)ceil_div(p.V, part), (int)std::min<long long>(part, p.V), 0};
  plan.blocks = (unsigned)std::min<long long>(p.rows * plan.parts, most);
  return plan;
}

template <typename T, typename C, bool MEAN, bool TOP, typename End>
int over_rows(const Vocabulary &p, const void *logits, const End &end, void *top_scores, int32_t *top_ids) {
  const Plan plan = plan_of<T>(p, TOP);
  hipStream_t s = runtime().stream;
  Top w{plan.parts, plan.part, nullptr, nullptr, top_scores, top_ids};
  if (plan.parts > 1) {
    const size_t parts = (size_t)p.rows * plan.parts, sums = ceil_div(parts * sizeof(Sums<C>), 16) * 16, found = TOP ? parts * p.top : 0;
    char *space = nullptr;
    if (const int rc = workspace(sums + found * sizeof(Candidate<C>), (void **)&space)) return rc;
    w.partial = space, w.found = space + sums;
  }
  if (plan.lanes == 8) {
    if constexpr (!TOP) row_kernel<T, C, 8, MEAN, false, End><<<dim3(plan.blocks), dim3(256), 0, s>>>(p, w, (const T *)logits, end);
  } else if (plan.lanes == 16) {
    if constexpr (!TOP) row_kernel<T, C, 16, MEAN, false, End><<<dim3(plan.blocks), dim3(256), 0, s>>>(p, w, (const T *)logits, end);
  } else if (plan.lanes == 64) {
    if constexpr (!TOP) row_kernel<T, C, 64, MEAN, false, End><<<dim3(plan.blocks), dim3(256), 0, s>>>(p, w, (const T *)logits, end);
  } else {
    row_kernel<T, C, 256, MEAN, TOP, End><<<dim3(plan.blocks), dim3(256), 0, s>>>(p, w, (const T *)logits, end);
  }
  MG_HIP(hipGetLastError());
  if (plan.parts > 1) {
    row_join_kernel<T, C, MEAN, TOP, End><<<dim3((unsigned)std::min<long long>(p.rows, 1 << 22)), dim3(256), 0, s>>>(p, w, (const T *)logits, end);
    MG_HIP(hipGetLastError());
  }
  return MG_OK;
}

// ---- gradients --------------------------------------------------------------------------------------------------------------------
// As many pieces of a row as a block has on their way together, or eight or sixteen threads or a wavefront per row.  The rows come in the order opposite to the forward
// pass's: it has read the last of them last, and some of those are still near (4096 x 50000 halves, both passes 214 us and 231; distillation
// over 32000 144 and 153).
//
// PAST: a gradient that with its logits is more than the last-level cache (256 MB) holds is stored past it: what is stored there would have to go before
// the next kernel's reads come in.  us of both passes, and with a pass over the gradient behind them: 262 MB of halves 155 and 212, past it 127 and 190;
// 160 MB 84 and 123, 81 and 121; 128 MB 68 and 97, 66 and 99; 64 MB 37 and 52, 36 and 53.
template <typename T>
bool stores_past(const Vocabulary &p) {
  return (double)p.rows * p.V * sizeof(T) > 1.5e8;
}

template <typename T, typename C, int LANES, bool ENTROPY, bool PAST>
__global__ void __launch_bounds__(256) scores_bwd_kernel(Vocabulary p, int parts, const int32_t *__restrict__ ids, const T *__restrict__ logits,
                                                         const Row<C> *__restrict__ kept, const C *__restrict__ grad_scores,
                                                         const C *__restrict__ grad_entropy, T *__restrict__ dlogits) {
  typedef typename Piece<T>::Held Held;
  constexpr int V = Piece<T>::V, kStep = LANES * V * kAtOnce;
  const int lane = threadIdx.x & (LANES - 1);
  constexpr bool SHARED = LANES < 256;  // rows share a block
  const long long units = SHARED ? (p.rows + 256 / LANES - 1) / (256 / LANES) : p.rows * parts;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const long long nth = SHARED ? unit * (256 / LANES) + threadIdx.x / LANES : unit / parts;
    if (SHARED && nth >= p.rows) return;
    const long long r = p.rows - 1 - nth;
    const long long at = (SHARED ? 0 : (unit - nth * parts) * kStep) + lane * V;
    const T *z = logits + r * p.V;
    T *out = dlogits + r * p.V;
    Held held[kAtOnce];
    load_pieces<LANES>(held, z, at, p.V);
    const Row<C> row = kept[r];
    int id = grad_scores ? ids[r] : -1;
    if (id >= p.V) id = -1;
    const C g = id < 0 ? C(0) : grad_scores[r], h = ENTROPY ? grad_entropy[r] : C(0), inverse = 1 / row.s;
    const bool nothing = row.s == 0 || (id < 0 && !ENTROPY);
    // one value; the other way round, p (-g - h (t - a)), a row's own numbers would be formed for each
    auto gradient = [&](T value) {
      const C t = (C)value - row.m, share = exponential<T>(t) * inverse;
      C dz = -share * g;
      if (ENTROPY) dz -= share * ((share > 0 ? t : C(0)) - row.a) * h;
      return dz;
    };
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const long long d = at + (long long)u * LANES * V;
      if (d >= p.V) break;
      Held dz;
#pragma unroll
      for (int n = 0; n < V; ++n) dz[n] = nothing ? T(0) : (T)gradient(held[u][n]);
      const long long own = id - d;  // the token's place among them
      if (own >= 0 && own < V && !nothing) {
#pragma unroll
        for (int n = 0; n < V; ++n)
          if (n == own) dz[n] = (T)(gradient(held[u][n]) + g);
      }
      Piece<T>::template store<PAST>(out + d, p.V - d, dz);
    }
  }
}

// The threads that share a row, or those of each wavefront, write the teacher's tokens among their own values once more; nobody waits for another.
template <typename T, typename C, int LANES, bool PAST>
__global__ void __launch_bounds__(256) distillation_bwd_kernel(Vocabulary p, int parts, const int32_t *__restrict__ ids, const T *__restrict__ logits,
                                                               const Row<C> *__restrict__ kept, const C *__restrict__ shares,
                                                               const C *__restrict__ grad, T *__restrict__ dlogits) {
  typedef typename Piece<T>::Held Held;
  constexpr int V = Piece<T>::V, kStep = LANES * V * kAtOnce;
  const int lane = threadIdx.x & (LANES - 1);
  constexpr bool SHARED = LANES < 256;  // rows share a block
  const long long units = SHARED ? (p.rows + 256 / LANES - 1) / (256 / LANES) : p.rows * parts;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const long long nth = SHARED ? unit * (256 / LANES) + threadIdx.x / LANES : unit / parts;
    if (SHARED && nth >= p.rows) return;
    const long long r = p.rows - 1 - nth, from = SHARED ? 0 : (unit - nth * parts) * kStep, at = from + lane * V;
    const T *z = logits + r * p.V;
    T *out = dlogits + r * p.V;
    Held held[kAtOnce];
    load_pieces<LANES>(held, z, at, p.V);
    const Row<C> row = kept[r];
    const C per = (C)p.per, g = grad[r] * per, inverse = row.a / row.s;
    const bool nothing = row.s == 0 || row.a == 0;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const long long d = at + (long long)u * LANES * V;
      if (d >= p.V) break;
      Held dz;
#pragma unroll
      for (int n = 0; n < V; ++n) dz[n] = nothing ? T(0) : (T)(g * (exponential<T>(((C)held[u][n] - row.m) * per) * inverse));
      Piece<T>::template store<PAST>(out + d, p.V - d, dz);
    }
    if (nothing) continue;
    wave_sees();  // the same memory again, by other lanes
    for (int k = lane & 63; k < p.top; k += min(LANES, 64)) {
      const int id = ids[r * p.top + k];
      const C q = shares[r * p.top + k];
      const long long place = id - from;
      if (q < 0 || place < 0 || place >= kStep) continue;
      if (SHARED || (int)(place % (LANES * V)) / (64 * V) == (int)(threadIdx.x >> 6))
        out[id] = (T)(g * (exponential<T>(((C)z[id] - row.m) * per) * inverse - q));
    }
  }
}

int check(int dtype, int64_t rows, int64_t V, const char *who) {
  if (dtype != MG_F32 && dtype != MG_F64 && dtype != MG_F16) return fail(MG_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (rows < 0 || V < 1) return fail(MG_ERR_BAD_ARG, "%s: %lld rows of %lld logits", who, (long long)rows, (long long)V);
  if (rows > 0x7fffffff || V > (1 << 30)) return fail(MG_ERR_UNSUPPORTED, "%s: %lld rows of %lld logits", who, (long long)rows, (long long)V);
  return MG_OK;
}

int check_distillation(int dtype, int64_t rows, int64_t V, int64_t K, double temperature, const char *who) {
  if (const int rc = check(dtype, rows, V, who)) return rc;
  if (K < 1 || !(temperature >= 1e-30 && temperature <= 1e30))  // single precision holds it and its inverse
    return fail(MG_ERR_BAD_ARG, "%s: %lld tokens of the teacher's, temperature %g", who, (long long)K, temperature);
  if (K > kMostTaught) return fail(MG_ERR_UNSUPPORTED, "%s: %lld tokens of the teacher's (at most %d)", who, (long long)K, kMostTaught);
  return MG_OK;
}

// Calls f with a null pointer of the type that logits are stored in and one of the type sums are carried in.
template <typename F>
int with_types(int dtype, F f) {
  if (dtype == MG_F64) return f((double *)nullptr, (double *)nullptr);
  if (dtype == MG_F32) return f((float *)nullptr, (float *)nullptr);
  return f((_Float16 *)nullptr, (float *)nullptr);
}

// Calls f with the number of threads that share a row of a gradient, of whose tokens a teacher names K.
template <typename T, typename F>
void with_lanes(int64_t V, int64_t K, F f) {
  constexpr int one = Piece<T>::V * kAtOnce;
  if (K <= 8 * kTurns && V <= 8 * one) f(std::integral_constant<int, 8>{});
  else if (K <= 16 * kTurns && V <= 16 * one) f(std::integral_constant<int, 16>{});
  else if (V <= 64 * one) f(std::integral_constant<int, 64>{});
  else f(std::integral_constant<int, 256>{});
}
template <typename F>
void with_bool(bool value, F f) {
  if (value) f(std::true_type{});
  else f(std::false_type{});
}

}  // namespace

}  // namespace mg

using namespace mg;

extern "C" {

int mg_log_probabilities_fwd(int dtype, int64_t rows, int64_t V, int top, const int32_t *ids, const void *logits, void *scores, void *entropy, void *kept,
                             void *top_scores, int32_t *top_ids) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  if (const int rc = check(dtype, rows, V, "mg_log_probabilities_fwd")) return rc;
  if (top < 0 || top > V) return fail(MG_ERR_BAD_ARG, "mg_log_probabilities_fwd: the likeliest %d of %lld tokens", top, (long long)V);
  if (top > kMostTop) return fail(MG_ERR_UNSUPPORTED, "mg_log_probabilities_fwd: the likeliest %d tokens (at most %d)", top, kMostTop);
  if (rows == 0) return MG_OK;
  if (!logits || (scores && !ids) || (top && (!top_scores || !top_ids))) return fail(MG_ERR_BAD_ARG, "null pointer in mg_log_probabilities_fwd");
  const Vocabulary p{rows, (int)V, top, 1.0};
  return with_types(dtype, [&](auto *t, auto *c) {
    typedef std::remove_pointer_t<decltype(t)> T;
    typedef std::remove_pointer_t<decltype(c)> C;
    ScopedTiming timed(TAG_SCORES);
    const Scores<T, C> end{ids, (const T *)logits, (C *)scores, (C *)entropy, (Row<C> *)kept};
    if (entropy && top) return over_rows<T, C, true, true>(p, logits, end, top_scores, top_ids);
    if (entropy) return over_rows<T, C, true, false>(p, logits, end, nullptr, nullptr);
    if (top) return over_rows<T, C, false, true>(p, logits, end, top_scores, top_ids);
    return over_rows<T, C, false, false>(p, logits, end, nullptr, nullptr);
  });
}

int mg_log_probabilities_bwd(int dtype, int64_t rows, int64_t V, const int32_t *ids, const void *logits, const void *kept, const void *grad_scores,
                             const void *grad_entropy, void *dlogits) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  if (const int rc = check(dtype, rows, V, "mg_log_probabilities_bwd")) return rc;
  if (rows == 0) return MG_OK;
  if (!logits || !kept || !dlogits || (grad_scores && !ids) || (!grad_scores && !grad_entropy))
    return fail(MG_ERR_BAD_ARG, "null pointer in mg_log_probabilities_bwd");
  const Vocabulary p{rows, (int)V, 0, 1.0};
  return with_types(dtype, [&](auto *t, auto *c) {
    typedef std::remove_pointer_t<decltype(t)> T;
    typedef std::remove_pointer_t<decltype(c)> C;
    ScopedTiming timed(TAG_SCORES_BWD);
    auto run = [&](auto lanes, auto with_entropy, auto past) {
      const long long parts = ceil_div(V, lanes * Piece<T>::V * kAtOnce), blocks = lanes < 256 ? ceil_div(rows, 256 / lanes) : rows * parts;
      scores_bwd_kernel<T, C, lanes, with_entropy, past><<<dim3((unsigned)std::min<long long>(blocks, 1 << 22)), dim3(256), 0, runtime().stream>>>(
          p, (int)parts, ids, (const T *)logits, (const Row<C> *)kept, (const C *)grad_scores, (const C *)grad_entropy, (T *)dlogits);
    };
    with_lanes<T>(V, 0, [&](auto lanes) {
      with_bool(grad_entropy != nullptr, [&](auto with_entropy) { with_bool(stores_past<T>(p), [&](auto past) { run(lanes, with_entropy, past); }); });
    });
    MG_HIP(hipGetLastError());
    return (int)MG_OK;
  });
}

int mg_distillation_fwd(int dtype, int teacher_dtype, int64_t rows, int64_t V, int64_t K, double temperature, const void *logits, const int32_t *ids,
                        const void *teacher, void *loss, void *kept, void *shares) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  if (const int rc = check_distillation(dtype, rows, V, K, temperature, "mg_distillation_fwd")) return rc;
  if (teacher_dtype != dtype && !(dtype == MG_F16 && teacher_dtype == MG_F32))
    return fail(MG_ERR_UNSUPPORTED, "mg_distillation_fwd: a teacher of dtype %d for dtype %d", teacher_dtype, dtype);
  if (rows == 0) return MG_OK;
  if (!logits || !ids || !teacher || !loss) return fail(MG_ERR_BAD_ARG, "null pointer in mg_distillation_fwd");
  const Vocabulary p{rows, (int)V, (int)K, 1 / temperature};
  return with_types(dtype, [&](auto *t, auto *c) {
    typedef std::remove_pointer_t<decltype(t)> T;
    typedef std::remove_pointer_t<decltype(c)> C;
    ScopedTiming timed(TAG_DISTILLATION);
    if (teacher_dtype == dtype)
      return over_rows<T, C, false, false>(p, logits, Distillation<T, T, C>{ids, (const T *)logits, (const T *)teacher, (C *)loss, (Row<C> *)kept, (C *)shares}, nullptr, nullptr);
    return over_rows<T, C, false, false>(p, logits, Distillation<T, C, C>{ids, (const T *)logits, (const C *)teacher, (C *)loss, (Row<C> *)kept, (C *)shares}, nullptr, nullptr);
  });
}

int mg_distillation_bwd(int dtype, int64_t rows, int64_t V, int64_t K, double temperature, const void *logits, const int32_t *ids, const void *kept,
                        const void *shares, const void *grad, void *dlogits) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  if (const int rc = check_distillation(dtype, rows, V, K, temperature, "mg_distillation_bwd")) return rc;
  if (rows == 0) return MG_OK;
  if (!logits || !ids || !kept || !shares || !grad || !dlogits) return fail(MG_ERR_BAD_ARG, "null pointer in mg_distillation_bwd");
  const Vocabulary p{rows, (int)V, (int)K, 1 / temperature};
  return with_types(dtype, [&](auto *t, auto *c) {
    typedef std::remove_pointer_t<decltype(t)> T;
    typedef std::remove_pointer_t<decltype(c)> C;
    ScopedTiming timed(TAG_DISTILLATION_BWD);
    auto run = [&](auto lanes, auto past) {
      const long long parts = ceil_div(V, lanes * Piece<T>::V * kAtOnce), blocks = lanes < 256 ? ceil_div(rows, 256 / lanes) : rows * parts;
      distillation_bwd_kernel<T, C, lanes, past><<<dim3((unsigned)std::min<long long>(blocks, 1 << 22)), dim3(256), 0, runtime().stream>>>(
          p, (int)parts, ids, (const T *)logits, (const Row<C> *)kept, (const C *)shares, (const C *)grad, (T *)dlogits);
    };
    with_lanes<T>(V, K, [&](auto lanes) { with_bool(stores_past<T>(p), [&](auto past) { run(lanes, past); }); });
    MG_HIP(hipGetLastError());
    return (int)MG_OK;
  });
}

}  // extern "C"
