// Operands of attention on the matrix cores: tiles of rows in LDS, fragments, and the deal of blocks.
//
// All products run as D(32x32) += A(32xk) B(kx32), one wavefront each.  Lane l = 32 h + c (h = 0, 1) holds column c of D, at rows
// 8 (r / 4) + 4 h + r % 4 for r = 0..15.  A fragment holds eight values along k for row (of A) or column (of B) c, and the two halves
// of the wavefront hold sixteen between them.  The order of k is free as long as A and B agree:
//   over the head dimension: value j of half h is d = 16 step + 8 h + j, eight neighbours in memory;
//   over rows of a product's result: the registers 8 (step % 2) + j of a lane as they are, row 16 step + 8 (j / 4) + 4 h + j % 4 --
//   so weights and their gradients go from the accumulators of one product into the next one without a move between lanes.
// Float16 takes a fragment in one v_mfma_f32_32x32x16_f16, float32 in eight v_mfma_f32_32x32x2_f32.
#pragma once

#include <type_traits>

#include "attention_device.h"

namespace mg {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

#define MG_LDS __attribute__((address_space(3)))

constexpr unsigned kBeyond = 0x80000000u;  // a byte offset past the end of any buffer: reads as zero
constexpr float kLog2e = 1.44269504088896340736f;

template <typename T>
struct Fragment;

template <>
struct Fragment<_Float16> {
  typedef f16x8 V;
  static __device__ __forceinline__ f32x16 mma(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

template <>
struct Fragment<float> {
  typedef f32x8 V;
  static __device__ __forceinline__ f32x16 mma(V a, V b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// ROWS rows of DP values in LDS, in pieces of 16 bytes.  A row's pieces are permuted by the row's number, so that neither sixteen
// rows at one piece (fragments along the head dimension) nor four rows at four neighbouring pieces (fragments along rows) fall on
// the same banks twice.
template <typename T, int DP, int ROWS>
struct TileOf {
  static constexpr int kPieces = DP * (int)sizeof(T) / 16;  // of a row
  static constexpr int kRowBytes = DP * (int)sizeof(T);
  static constexpr int kBytes = ROWS * kRowBytes;
  typedef typename Fragment<T>::V V;

  static __device__ __forceinline__ int turn(int row) {
    if (sizeof(T) == 2) {
      if (kPieces == 16) return ((row & 3) << 2) | ((row >> 2) & 3);
      if (kPieces == 8) return ((row & 2) << 1) | ((row >> 2) & 3);
      return (row >> 2) & 3;  // 4 or 12
    }
    if (kPieces % 16 == 0) return ((row & 4) << 1) | ((row & 8) >> 1) | (row & 3);
    return (row >> 1) & 7;  // 8 or 24
  }

  // Brings rows that lie `stride` bytes apart straight into LDS, 16 bytes a lane; THREADS threads (a wavefront, or the block) take part.  A
  // thread's pieces of all rounds that begin a multiple of sixteen rows apart are permuted alike: one offset serves them.
  template <int THREADS>
  struct Loader {
    static constexpr int kRounds = (ROWS * kPieces + THREADS - 1) / THREADS;
    static constexpr int repeat() {
      for (int m = 1; m < kRounds; ++m)
        if (m * THREADS % (16 * kPieces) == 0) return m;
      return kRounds;
    }
    static constexpr int kOffsets = repeat();
    unsigned at[kOffsets], stride, dim;

    static __device__ __forceinline__ int slot(int round) { return round * THREADS + (int)(THREADS == 64 ? threadIdx.x & 63 : threadIdx.x); }

    // Pieces behind the `dim` bytes of a row are zeros; the one that the row's end cuts goes on into what follows it, which meets zeros of the
    // other operand (or lands in results that nobody stores).
    __device__ __forceinline__ Loader(unsigned stride, unsigned dim) : stride(stride), dim(dim) {
#pragma unroll
      for (int n = 0; n < kOffsets; ++n) {
        const int row = slot(n) / kPieces, piece = (slot(n) % kPieces) ^ turn(row);
        at[n] = (unsigned)piece * 16u < dim ? (unsigned)row * stride + (unsigned)piece * 16u : kBeyond;
      }
    }

    // Rows [0, ROWS) from `base` on to the tile at byte `lds`; rows from `last` on are zeros, and the last one's end is that of what is read.
    __device__ __forceinline__ void operator()(const char *base, int last, unsigned lds) const {
      if (last >= ROWS + (dim % 16 ? 1 : 0))
        rounds<false>(base, last, lds);
      else
        rounds<true>(base, last, lds);
    }

   private:
    template <bool CUT>
    __device__ __forceinline__ void rounds(const char *base, int last, unsigned lds) const {
      typedef MG_LDS void *LdsPointer;
      const int bytes = CUT ? last > 0 ? (last - 1) * (int)stride + (int)dim : 0 : 0x7fffffff;
      const __amdgpu_buffer_rsrc_t buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, bytes, 0x00020000);
      const int wave = THREADS == 64 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
      for (int n = 0; n < kRounds; ++n) {
        if (ROWS * kPieces % THREADS != 0 && n * THREADS + wave * 64 >= ROWS * kPieces) continue;
        unsigned from = at[n % kOffsets], more = (unsigned)(n / kOffsets * kOffsets * THREADS / kPieces) * stride;
        if (CUT) from = slot(n) / kPieces < last && from != kBeyond ? from + more : kBeyond, more = 0;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (LdsPointer)(unsigned long long)(lds + (unsigned)(n * THREADS + wave * 64) * 16u), 16, (int)from,
                                                 (int)more, 0, 0);
      }
    }
  };

  // Where a lane's fragments lie in a tile, but for what is the same in all lanes: pieces are permuted within groups of kGroup of a row, so
  // a step to another piece is an exclusive or within the group's bytes and an offset from group to group.
  static constexpr int kGroup = sizeof(T) == 2 ? (kPieces % 8 ? 4 : kPieces) : (kPieces % 16 ? 8 : 16);
  struct Place {
    unsigned along, across[sizeof(T) == 2 ? 2 : 8];
  };

  static __device__ __forceinline__ Place place(int lane) {
    const int h = lane >> 5, c = lane & 31;
    Place at;
    at.along = (unsigned)(c * kRowBytes + (((sizeof(T) == 2 ? h : 2 * h) ^ turn(c)) & (kGroup - 1)) * 16);
    if constexpr (sizeof(T) == 2) {
      // each sixteen lanes hand four rows of sixteen values to one another: lane 4 r + n reads row r at 4 n, lane m gets column m
      const int piece = 2 * ((lane & 31) >> 4) + ((lane & 3) >> 1);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int row = 8 * n + 4 * h + ((lane & 15) >> 2);
        at.across[n] = (unsigned)(row * kRowBytes + ((piece ^ turn(row)) & (kGroup - 1)) * 16 + (lane & 1) * 8);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = 8 * (j >> 2) + 4 * h + (j & 3);
        at.across[j] = (unsigned)(row * kRowBytes + (((c >> 2) ^ turn(row)) & (kGroup - 1)) * 16 + (c & 3) * 4);
      }
    }
    return at;
  }

  static __device__ __forceinline__ unsigned moved(unsigned at, int pieces) {
    return (at ^ (unsigned)(pieces % kGroup) * 16u) + (unsigned)(pieces / kGroup * kGroup) * 16u;
  }

  // Fragment `step` along the head dimension of the lane's row of rows 32 sub .. 32 sub + 31.  Tiles start on multiples of 1024 bytes; a
  // tile that lies a constant `beyond` another shares its addresses.
  static __device__ __forceinline__ V along(unsigned tile, const Place &place, int sub, int step, unsigned beyond = 0) {
    const unsigned at = tile + place.along, more = (unsigned)(32 * sub) * kRowBytes + beyond;
    if constexpr (sizeof(T) == 2) {
      return *(MG_LDS const f16x8 *)(unsigned long long)(moved(at, 2 * step) + more);
    } else {
      const f32x4 a = *(MG_LDS const f32x4 *)(unsigned long long)(moved(at, 4 * step) + more);
      const f32x4 b = *(MG_LDS const f32x4 *)(unsigned long long)(moved(at, 4 * step + 1) + more);
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }

  // Fragment `step` along the rows, for values 32 part .. 32 part + 31 of the head dimension (a value for each lane of a half).
  static __device__ __forceinline__ V across(unsigned tile, const Place &place, int part, int step, unsigned beyond = 0) {
    const unsigned more = (unsigned)(16 * step) * kRowBytes + beyond;
    V v;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const s16x4 q = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MG_LDS s16x4 *)(unsigned long long)(moved(tile + place.across[n], 4 * part) + more));
        const f16x4 f = __builtin_bit_cast(f16x4, q);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * n + j] = f[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = *(MG_LDS const float *)(unsigned long long)(moved(tile + place.across[j], 8 * part) + more);
    }
    return v;
  }
};

// Every load of this wave into LDS has landed, its LDS accesses and its stores are done; then all waves of the block are here.
__device__ __forceinline__ void all_landed() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// What the two halves of the wavefront hold for a column: lane c's value and lane 32 + c's, in both lanes.
struct Halves {
  float low, high;
};

__device__ __forceinline__ Halves halves_of(float v) {
  // The builtin's two results come out as one and the same in this compiler; the instruction wants two wait states behind what wrote its
  // operands, which nobody puts there for an asm statement.
  float low = v, high = v;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(low), "+v"(high));
  return Halves{low, high};
}

__device__ __forceinline__ float larger_half(float v) {
  const Halves both = halves_of(v);
  return __builtin_fmaxf(both.low, both.high);
}

__device__ __forceinline__ float sum_halves(float v) {
  const Halves both = halves_of(v);
  return both.low + both.high;
}

// Of 32 rows of queries, a row for each lane of a half: the keys that any of them sees [lo, hi), and those that all of them see
// [all_lo, all_hi) (rows beyond the last query count as seeing everything there, and nothing before).  The same in every lane.
struct Reach {
  int lo, hi, all_lo, all_hi;
};

__device__ __forceinline__ Reach reach_of(Span s, bool in) {
  const bool some = in && s.hi > s.lo;
  Reach r{some ? s.lo : 0x7fffffff, some ? s.hi : 0, in ? s.lo : 0, in ? s.hi : 0x7fffffff};
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    r.lo = min(r.lo, __shfl_xor(r.lo, m));
    r.hi = max(r.hi, __shfl_xor(r.hi, m));
    r.all_lo = max(r.all_lo, __shfl_xor(r.all_lo, m));
    r.all_hi = min(r.all_hi, __shfl_xor(r.all_hi, m));
  }
  return Reach{__builtin_amdgcn_readfirstlane(r.lo), __builtin_amdgcn_readfirstlane(r.hi), __builtin_amdgcn_readfirstlane(r.all_lo),
               __builtin_amdgcn_readfirstlane(r.all_hi)};
}

// Eight values of a row in memory as a fragment: zeros where the row or its values, whole fours, end.
template <typename T>
__device__ __forceinline__ typename Fragment<T>::V fragment_of(const T *row, int at, int dim, bool in) {
  typedef T Eight __attribute__((ext_vector_type(8), aligned(4 * sizeof(T)))), Four __attribute__((ext_vector_type(4)));
  typename Fragment<T>::V v = {};
  if (in && at + 8 <= dim) {
    const Eight held = *reinterpret_cast<const Eight *>(row + at);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = held[j];
  }
  if ((dim & 4) && in && at + 4 == dim) {
    const Four held = *reinterpret_cast<const Four *>(row + at);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = held[j];
  }
  return v;
}

// Four neighbouring values of a result to `to`; true if one of them is no number.
template <typename T>
__device__ __forceinline__ bool put_four(T *to, f32x4 value) {
  typedef T V __attribute__((ext_vector_type(4)));
  *reinterpret_cast<V *>(to) = __builtin_convertvector(value, V);
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) odd |= !(__builtin_fabsf(value[j]) < INFINITY);
  return odd;
}

__device__ __forceinline__ f32x4 four_of(const f32x16 &v, int r) { return f32x4{v[r], v[r + 1], v[r + 2], v[r + 3]}; }

// Rows of a tile of results as the registers of a lane hold them.
__device__ __forceinline__ int row_of(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

__device__ __forceinline__ f32x16 zeros() { return f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0}; }

// Registers 8 n .. 8 n + 7 as a fragment along the rows, and what rounding took off them as another.
template <typename T>
__device__ __forceinline__ typename Fragment<T>::V rows_of(const f32x16 &v, int n, typename Fragment<T>::V &more) {
  f32x8 part;
#pragma unroll
  for (int j = 0; j < 8; ++j) part[j] = v[8 * n + j];
  const auto near = __builtin_convertvector(part, typename Fragment<T>::V);
  if constexpr (sizeof(T) == 2) more = __builtin_convertvector(part - __builtin_convertvector(near, f32x8), typename Fragment<T>::V);
  return near;
}

// a times both: a float32 value in two of float16 keeps 22 bits (one is all of it in float32).  Weights and gradients of scores are multiplied so,
// and a result in float16 is off by its own rounding and no more.  Rounded to 11 bits weights would make out and dv off by 1.3 to 1.4 times that
// and, by what grad . out is off, dq and dk by 1.05 times; gradients of scores dq and dk by half as much again.  The third product of a tile forward and
// the sixth of dk and dv cost a tenth of a step: 8192 packed tokens, 16 heads of 128, 515 us against 568, 4 x 2048 of 16 over 4 with a cap 614 against 668.
template <typename T>
__device__ __forceinline__ f32x16 mma_of_two(typename Fragment<T>::V a, typename Fragment<T>::V b, typename Fragment<T>::V more, f32x16 c) {
  c = Fragment<T>::mma(a, b, c);
  if constexpr (sizeof(T) == 2) c = Fragment<T>::mma(a, more, c);
  return c;
}

// tanh of a lane's sixteen values.  Where all of the wavefront's are below 1/4, an odd polynomial (what float32's leaves out is below
// 2^-31 of x; float16's, two terms shorter, below 2^-19), which takes no quarter-rate instruction.  Else 1 - 2 / (e^2x + 1), which is off by
// 2^-24 where |x| is small: that is nothing next to weights in float16, float32 takes the polynomial there.
template <typename T>
__device__ __forceinline__ float tanh_small(float x) {
  const float y = x * x;
  float s = -0.0539682540f;                             // -17 / 315
  if (sizeof(T) == 4) {
    s = -0.00886323553f;                                // -1382 / 155925
    s = s * y + 0.0218694885f;                          // 62 / 2835
    s = s * y - 0.0539682540f;
  }
  s = s * y + 0.133333333f;
  s = s * y - 0.333333333f;
  return x + x * (s * y);
}

template <typename T>
__device__ __forceinline__ float tanh_any(float x) {
  const float e = __builtin_amdgcn_exp2f(x * (2 * kLog2e));  // infinity and 0 give +-1
  const float far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f);
  if (sizeof(T) == 2) return far;
  const float near = tanh_small<T>(x);
  return __builtin_fabsf(x) < 0.25f ? near : far;
}

template <typename T>
__device__ __forceinline__ void tanh_of_all(f32x16 &x) {
  float most = 0;
#pragma unroll
  for (int r = 0; r < 16; ++r) most = __builtin_fmaxf(most, __builtin_fabsf(x[r]));
  const bool small = !__any(!(most < 0.25f));
#pragma unroll
  for (int r = 0; r < 16; r += 4) {  // sixteen at once would take too many registers
    if (small) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[r + j] = tanh_small<T>(x[r + j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[r + j] = tanh_any<T>(x[r + j]);
    }
  }
}

// Weights are kept as 2^kLift times exp2(score - top): in float16 they are whole down to 2^-21 of the row's largest then, down to 2^-29 as `top` lags
// behind it, and their second parts down to 2^-31.  `top` follows the
// row's maximum only when that has grown by more than kSlack, so the sums are seldom scaled; 2^(kLift + kSlack) stays below 65504.
constexpr float kLift = 7.0f, kSlack = 8.0f;

// How scores are made of products, for one query head: factor * (tanh(bend * product), or the product) - slope * distance, in powers of two.
struct Scores {
  float bend, factor, slope;
};

__device__ __forceinline__ Scores scores_of(const Attention &p, int head) {
  return Scores{p.bend, (p.cap > 0 ? p.cap : p.scale) * kLog2e, p.slopes ? ((const float *)p.slopes)[head] * kLog2e : 0.0f};
}

// 32 queries, one in each lane's column (in both halves), on their way through tiles of SUBS times 32 keys: S^T = K Q^T has a query's scores in
// its lane (and the partner in the other half), so maximum and sum need no exchange but that one, and the weights are the right operand of
// out^T = V^T P^T as they lie.  BENT: scores have a cap (whose registers the others do without).
template <typename T, int DP, int SUBS, bool BENT>
struct Running {
  typedef TileOf<T, DP, 32 * SUBS> Tile;
  typedef typename Fragment<T>::V V;
  static constexpr int kSteps = DP / 16, kParts = DP / 32;

  f32x16 sums[kParts];
  float top = -INFINITY, total = 0;  // `total`: of this half's keys

  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int n = 0; n < kParts; ++n) sums[n] = zeros();
  }

  // Keys from `key0` on; `whole`: all columns see all of them.
  __device__ __forceinline__ void take(const Attention &p, const Scores &how, unsigned keys, unsigned values, const V (&rows)[kSteps], const Span &span,
                                       int key0, bool whole, const typename Tile::Place &place, int h) {
    f32x16 s[SUBS];
#pragma unroll
    for (int n = 0; n < SUBS; ++n) s[n] = zeros();
#pragma unroll
    for (int m = 0; m < kSteps; ++m)
#pragma unroll
      for (int n = 0; n < SUBS; ++n) s[n] = Fragment<T>::mma(Tile::along(keys, place, n, m), rows[m], s[n]);
    if constexpr (BENT) {
#pragma unroll
      for (int n = 0; n < SUBS; ++n) {
        s[n] *= how.bend;
        tanh_of_all<T>(s[n]);
      }
    }
    float factor = how.factor;
    if (p.slopes || !(factor > 0)) {
      const float away = (float)(span.place - key0 - 4 * h);
#pragma unroll
      for (int n = 0; n < SUBS; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] = s[n][r] * factor - how.slope * __builtin_fabsf(away - (float)(32 * n + row_of(r, 0)));
      factor = 1;
    }
    if (!whole) {
      const unsigned seen = (unsigned)(span.hi - span.lo);
      const int from = key0 + 4 * h - span.lo;
#pragma unroll
      for (int n = 0; n < SUBS; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] = (unsigned)(from + 32 * n + row_of(r, 0)) < seen ? s[n][r] : -INFINITY;
    }
    float most = s[0][0];
#pragma unroll
    for (int n = 0; n < SUBS; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) most = __builtin_fmaxf(most, s[n][r]);
    most = larger_half(most) * factor;
    if (__any(most > top + kSlack)) {  // also the first keys that a column sees
      const float now = __builtin_fmaxf(top, most), back = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - now);
      top = now;
      total *= back;
#pragma unroll
      for (int n = 0; n < kParts; ++n) sums[n] *= back;
    }
    const float base = top == -INFINITY ? 0.0f : top - kLift;
#pragma unroll
    for (int n = 0; n < SUBS; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r], factor, -base));
        total += s[n][r];
      }
    V weights[2 * SUBS], more[2 * SUBS];
#pragma unroll
    for (int m = 0; m < 2 * SUBS; ++m) weights[m] = rows_of<T>(s[m >> 1], m & 1, more[m]);
#pragma unroll
    for (int n = 0; n < kParts; ++n)
#pragma unroll
      for (int m = 0; m < 2 * SUBS; ++m) sums[n] = mma_of_two<T>(Tile::across(values, place, n, m), weights[m], more[m], sums[n]);
  }
};

// What the two kernels of the gradient need of each row, made in one pass over out, grad and v:
//   level_i = lse_i - shift             exp2(s_i - level_i) = 2^shift P_i
//   delta_i = grad_i . out_i            (with what the rounding of out took off)
//   spans of the rows, and for each chunk of `rows` rows their union and intersection
constexpr float kShift = 14.0f;  // 2^14 P in float16: whole down to 2^-28

struct Stats {
  float *level, *delta;  // (B, HQ, TQ)
  int *lo, *hi;          // (B, TQ)
  Reach *reach;          // (B, chunks of queries)
  int rows, chunks;
};

// Gradients of scores in float16: a lane's column is held at a power of two of its own, which follows its largest value so far (in both
// halves of the wavefront) and leaves that 2^8 of room, so that values down to 2^-21 of it keep all their digits and the sums are seldom
// scaled.  Float32 needs none of this.
struct Unit {
  float by = 0x1p100f;  // nothing seen yet
};

template <typename T, int PARTS>
__device__ __forceinline__ void in_units(Unit &unit, f32x16 &ds, f32x16 (&sums)[PARTS]) {
  if constexpr (sizeof(T) == 2) {
    float most = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) most = __builtin_fmaxf(most, __builtin_fabsf(ds[r]));
    most = larger_half(most);
    const bool over = most * unit.by > 0x1p15f;
    if (__any(over)) {
      const int e = min(max(261 - (int)(__builtin_bit_cast(unsigned, most) >> 23), 1), 254);  // 2^7 / 2^e of the largest
      const float now = over ? __builtin_bit_cast(float, e << 23) : unit.by, back = now / unit.by;
      unit.by = now;
#pragma unroll
      for (int n = 0; n < PARTS; ++n) sums[n] *= back;
    }
    ds *= unit.by;
  }
}

// From products s = q.k and dp = grad.v - delta of a tile to s = 2^shift P and dp = 2^shift dS / scale; `away`: place of the query less the key's,
// as they differ along r.  level(r): of registers r .. r + 3.
template <typename T, bool ROW_IS_KEY, bool BENT, typename Level>
__device__ __forceinline__ void gradients_of(const Attention &p, f32x16 &s, f32x16 &dp, const Scores &how, float away, Level level) {
  if constexpr (BENT) {
    s *= how.bend;
    tanh_of_all<T>(s);
    __builtin_amdgcn_sched_barrier(0);  // what follows, mixed with this, would not fit in the registers
    dp *= 1.0f - s * s;
    __builtin_amdgcn_sched_barrier(0);
  }
  if constexpr (ROW_IS_KEY) {
    float factor = how.factor;
    if (p.slopes) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = s[r] * factor - how.slope * __builtin_fabsf(away - (float)row_of(r, 0));
      factor = 1;
    }
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const f32x4 from = level(r);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[r + j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r + j], factor, -from[j]));
    }
  } else {  // the same with a product of its own: as above, the keys' kernel has two registers too few and takes 10% longer at 128 values a head
    s *= how.factor;
    if (p.slopes) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] -= how.slope * __builtin_fabsf(away + (float)row_of(r, 0));
    }
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const f32x4 from = level(r);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[r + j] = __builtin_amdgcn_exp2f(s[r + j] - from[j]);
    }
  }
  dp *= s;
}

// Products of 32 queries' gradients with 32 keys, summed into dq^T = K^T dS^T: a query in each lane's column.
template <typename T, int DP, int ROWS, bool BENT>
struct Pulled {
  typedef TileOf<T, DP, ROWS> Tile;
  typedef typename Fragment<T>::V V;
  static constexpr int kSteps = DP / 16, kParts = DP / 32;

  f32x16 sums[kParts];
  Unit unit;

  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int n = 0; n < kParts; ++n) sums[n] = zeros();
  }

  // Keys `from` .. from + 31, rows 32 sub on of the tile at `keys`; their values lie a tile behind.
  __device__ __forceinline__ void take(const Attention &p, const Scores &how, unsigned keys, int sub, const V (&rows)[kSteps], const V (&grads)[kSteps],
                                       float level, float delta, const Span &span, int from, bool whole, const typename Tile::Place &place, int h) {
    f32x16 s = zeros(), dp = zeros();
#pragma unroll
    for (int m = 0; m < kSteps; ++m) {
      s = Fragment<T>::mma(Tile::along(keys, place, sub, m), rows[m], s);
      dp = Fragment<T>::mma(Tile::along(keys, place, sub, m, Tile::kBytes), grads[m], dp);
    }
    dp -= delta;
    gradients_of<T, true, BENT>(p, s, dp, how, (float)(span.place - from - 4 * h), [&](int) { return f32x4{level, level, level, level}; });
    if (!whole) {
      const unsigned seen = (unsigned)(span.hi - span.lo);
      const int first = from + 4 * h - span.lo;
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = (unsigned)(first + row_of(r, 0)) < seen ? dp[r] : 0.0f;
    }
    in_units<T>(unit, dp, sums);
    V ds[2], more[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) ds[m] = rows_of<T>(dp, m, more[m]);
#pragma unroll
    for (int part = 0; part < kParts; ++part)
#pragma unroll
      for (int m = 0; m < 2; ++m) sums[part] = mma_of_two<T>(Tile::across(keys, place, part, 2 * sub + m), ds[m], more[m], sums[part]);
  }

  // What the sums are to be multiplied by.
  __device__ __forceinline__ float by(const Attention &p) const { return sizeof(T) == 2 ? p.scale / unit.by * 0x1p-14f : p.scale; }  // 2^-kShift
};

// f(head dimension in whole parts of 32, above 128 as 256 (float16 only), whether scores are bent), both known to the compiler.
template <typename T, typename F>
void with_shape(const Attention &p, F f) {
  auto with_dim = [&](auto bent) {
    switch ((p.D + 31) / 32) {
      case 1: return f(std::integral_constant<int, 32>{}, bent);
      case 2: return f(std::integral_constant<int, 64>{}, bent);
      case 3: return f(std::integral_constant<int, 96>{}, bent);
      case 4: return f(std::integral_constant<int, 128>{}, bent);
      default:
        if constexpr (sizeof(T) == 2) return f(std::integral_constant<int, 256>{}, bent);
    }
  };
  p.cap > 0 ? with_dim(std::true_type{}) : with_dim(std::false_type{});
}

// How the blocks of a launch are dealt out: `pairs` of a batch item and a key head, each with `heads` query heads and `tiles` row tiles.
// Blocks go to the eight XCDs in turn, so with a multiple of eight pairs each pair stays on one XCD and is read through one L2.  The last tiles,
// which see most where the mask is causal, come first: of one pair after the other where one fills an XCD, else of as many as do.  2 x 4096 causal
// tokens, 16 heads of 128 in float16, with the first tiles first and with the last: dk and dv 538 and 425 us, dq 326 and 274, forward 254 and 219.  Where
// all blocks run at once, two on a compute unit, the second half comes the other way round, so that the unit with most of the first gets least of
// it: 4 x 1024 behind a prefix, 8 heads of 64 in float32, dk and dv 112 to 100.
struct Deal {
  int pairs, heads, tiles;
  int beside;  // pairs of an XCD whose tiles are dealt in turn
  int folded;  // blocks, where all of them run at once; else 0
};

struct Dealt {
  int pair, head, tile;
};

constexpr int kSorted = 256;  // tiles of an item that are sorted by their work

inline Deal deal_of(const Attention &p, int heads, int tiles) {
  const int units = runtime().props.multiProcessorCount, pairs = p.B * p.HK, blocks = pairs * heads * tiles;
  // documents end where they like: sorted over two rounds of the units they leave less idle at the end, which for what is causal, on one pair's
  // keys at a time, costs 2% (4 x 2048 tokens, 16 heads over 4)
  const int fill = p.starts && tiles <= kSorted ? units / 2 : units / 4;
  return Deal{pairs, heads, tiles, std::max(1, std::min(pairs / 8, (int)ceil_div(fill, heads * tiles))), blocks > units && blocks <= 2 * units ? blocks : 0};
}

__device__ __forceinline__ Dealt dealt(const Deal &d, int block) {
  if (d.folded && block >= d.folded / 2) {  // in eights, as the XCDs take them
    const int first = (d.folded / 2 + 7) / 8 * 8, last = d.folded / 8 * 8;
    if (block >= first && block < last) block = first + (last - 8 - (block & ~7)) + (block & 7);
  }
  if (d.pairs % 8 == 0) {
    const int each = d.heads * d.tiles, turn = block >> 3, of_group = d.beside * each, group = turn / of_group, rest = turn - group * of_group;
    const int many = min(d.beside, d.pairs / 8 - group * d.beside) * d.heads, tile = rest / many, at = rest - tile * many;
    return Dealt{(group * d.beside + at / d.heads) * 8 + (block & 7), at % d.heads, d.tiles - 1 - tile};
  }
  const int many = d.pairs * d.heads, tile = block / many, rest = block - tile * many;
  return Dealt{rest / d.heads, rest % d.heads, d.tiles - 1 - tile};
}

// The tile of a batch item that is `rank`-th in work, where documents make that uneven; each wavefront finds it for itself, a tile a lane or
// four.  The work is an estimate by the tile's first and last row.  8192 tokens of five documents, 16 heads of 128, float16: dk and dv 313 to 275
// us, dq 168 to 166, forward 136 to 135.
template <bool KEYS, int EACH>
__device__ __forceinline__ int tile_of_rank(const Attention &p, int b, int rank, int tiles, int rows) {
  const int lane = threadIdx.x & 63, tokens = KEYS ? p.TK : p.TQ;
  int work[EACH], before[EACH] = {};
#pragma unroll
  for (int m = 0; m < EACH; ++m) {
    const int tile = tiles - 1 - lane - 64 * m, first = tile * rows, last = min(tokens, first + rows) - 1;
    work[m] = -1;
    if (tile < 0) continue;
    if (KEYS) {
      const long long items = (long long)b * p.TK;
      work[m] = max(p.ends[items + last] - (p.causal ? first : p.starts[items + first]), 0);
    } else {
      const Span from = span_of(p, b, first), to = span_of(p, b, last);
      work[m] = max(max(to.hi, from.hi) - (from.hi ? from.lo : to.lo), 0);
    }
    if (p.window) work[m] = (int)min((unsigned)work[m], window_of_rows(p.window, p.causal, rows));
  }
#pragma unroll
  for (int m = 0; m < EACH; ++m)
    for (int n = 0; n < min(64, tiles - 64 * m); ++n) {
      const int other = __builtin_amdgcn_readlane(work[m], n);
#pragma unroll
      for (int c = 0; c < EACH; ++c) before[c] += other > work[c] || (other == work[c] && 64 * m + n < 64 * c + lane);
    }
  int found = 0;
#pragma unroll
  for (int m = 0; m < EACH; ++m) {
    const unsigned long long here = __ballot(before[m] == rank && lane + 64 * m < tiles);
    if (here) found = 64 * m + __ffsll(here) - 1;
  }
  return __builtin_amdgcn_readfirstlane(tiles - 1 - found);
}

template <bool KEYS>
__device__ __forceinline__ int tile_of_rank(const Attention &p, int b, int rank, int tiles, int rows) {
  if (!p.starts || tiles > kSorted) return KEYS ? rank : tiles - 1 - rank;  // what is causal: the last see, the first are seen, most
  return tiles <= 64 ? tile_of_rank<KEYS, 1>(p, b, rank, tiles, rows) : tile_of_rank<KEYS, kSorted / 64>(p, b, rank, tiles, rows);
}

}  // namespace mg
