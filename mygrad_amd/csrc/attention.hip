// Attention with capped scores, a bias by distance and masks, and its gradient, for gfx950.
//
//   s_ij = scale * q_i . k_j                    s_ij = cap * tanh(s_ij / cap)   s_ij -= slope_h * |place_i - j|
//   P_ij = exp(s_ij) / sum_j exp(s_ij)  over the keys j that row i sees; lse_i = log2 of that sum is kept for the gradient
//   out_i = sum_j P_ij v_j                      (a row that sees no key: zeros, and no gradient from it)
//   dP_ij = g_i . v_j      D_i = g_i . out_i    dS_ij = P_ij (dP_ij - D_i) (1 - tanh^2) scale
//   dq_i = sum_j dS_ij k_j      dk_j = sum_i dS_ij q_i      dv_j = sum_i P_ij g_i   (over the heads that share key head j)
//
// The kernels in this file take any type, head dimension up to 256 and mask: a wavefront per row of the result, keys (or
// queries) over its lanes, sums in float32 (float64 for float64).  They serve double precision and what the kernels on the
// matrix cores do not take.  What a row does not see never enters its sums, so infinities and NaN there stay where they are.
#include "attention_row.h"
#include "attention_rows.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace mg {

namespace {

struct Mine {
  long long first;  // batch item * heads + head
  int row;
  bool in;
};

// A block takes four rows of one head: which of them is this wavefront's.
__device__ __forceinline__ Mine row_of_wave(int tokens) {
  const int tiles = (tokens + 3) / 4;
  Mine m;
  m.first = blockIdx.x / tiles;
  m.row = (int)(blockIdx.x - m.first * tiles) * 4 + (threadIdx.x >> 6);
  m.in = m.row < tokens;
  return m;
}

// A score for each lane, then a value of the result for each: bound by reading a row of keys a lane, which no two lanes share a line of.  8192 packed
// tokens, 16 heads of 128 in float16, forward and gradients: 83 ms (0.6 on tiles).
template <typename T, typename C>
__global__ void __launch_bounds__(256) attention_rows_kernel(Attention p, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                                                             T *__restrict__ out, _Float16 *__restrict__ rest, C *__restrict__ lse) {
  __shared__ C rows[4][kMaxDim];
  const Mine r = row_of_wave(p.TQ);
  if (r.in) attend_row<T, C>(p, (int)(r.first / p.HQ), (int)(r.first % p.HQ), r.row, rows[threadIdx.x >> 6], q, k, v, out, rest, lse);
}

// D_i, a wavefront per row.
template <typename T, typename C>
__global__ void __launch_bounds__(256) attention_delta_kernel(Attention p, const T *__restrict__ out, const _Float16 *__restrict__ rest,
                                                              const T *__restrict__ grad, C *__restrict__ delta) {
  const int lane = threadIdx.x & 63;
  const Mine r = row_of_wave(p.TQ);
  if (!r.in) return;
  const long long at = ((r.first / p.HQ * p.TQ + r.row) * p.HQ + r.first % p.HQ) * p.D;
  C sum = 0;
  for (int d = lane; d < p.D; d += 64) sum += ((C)out[at + d] + (rest ? (C)rest[at + d] / (C)kRest : C(0))) * (C)grad[at + d];
  sum = wave_sum(sum);
  if (lane == 0) delta[r.first * p.TQ + r.row] = sum;
}

template <typename T, typename C>
__global__ void __launch_bounds__(256) attention_dq_rows_kernel(Attention p, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                                                                const T *__restrict__ grad, const C *__restrict__ lse, const C *__restrict__ delta,
                                                                T *__restrict__ dq) {
  __shared__ C rows[4][2 * kMaxDim];
  const Mine r = row_of_wave(p.TQ);
  if (r.in) dq_row<T, C>(p, (int)(r.first / p.HQ), (int)(r.first % p.HQ), r.row, rows[threadIdx.x >> 6], q, k, v, grad, lse, delta, dq);
}

template <typename T, typename C>
__global__ void __launch_bounds__(256) attention_dkv_rows_kernel(Attention p, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                                                                 const T *__restrict__ grad, const C *__restrict__ lse, const C *__restrict__ delta,
                                                                 T *__restrict__ dk, T *__restrict__ dv) {
  __shared__ C rows[4][2 * kMaxDim];
  const Mine r = row_of_wave(p.TK);
  if (r.in) dkv_row<T, C>(p, (int)(r.first / p.HK), (int)(r.first % p.HK), r.row, rows[threadIdx.x >> 6], q, k, v, grad, lse, delta, dk, dv);
}

// Copies the t new tokens of each batch item to the places in the cache that end at its length, 16 bytes (or an element) a thread.  A launch's
// latency for the few tokens of a step: 6 us between events for 32 tokens of 8 heads of 128 as for one.
template <typename V>
__global__ void __launch_bounds__(256) cache_write_kernel(long long pieces, int row, int T, int capacity, const int32_t *__restrict__ lengths,
                                                          const V *__restrict__ k, const V *__restrict__ v, V *__restrict__ keys,
                                                          V *__restrict__ values) {
  for (long long n = (long long)blockIdx.x * 256 + threadIdx.x; n < pieces; n += (long long)gridDim.x * 256) {
    const long long token = n / row;
    const int b = (int)(token / T), place = lengths[b] - T + (int)(token - (long long)b * T);
    if (place < 0 || place >= capacity) continue;
    const long long to = ((long long)b * capacity + place) * row + (n - token * row);
    keys[to] = k[n];
    values[to] = v[n];
  }
}

template <typename T, typename C>
int forward_rows(const Attention &p, const void *q, const void *k, const void *v, void *out, void *rest, void *lse) {
  ScopedTiming timed(TAG_ATTENTION);
  attention_rows_kernel<T, C><<<dim3((unsigned)((long long)p.B * p.HQ * ceil_div(p.TQ, 4))), dim3(256), 0, runtime().stream>>>(
      p, (const T *)q, (const T *)k, (const T *)v, (T *)out, (_Float16 *)rest, (C *)lse);
  MG_HIP(hipGetLastError());
  return MG_OK;
}

template <typename T, typename C>
int backward_rows(const Attention &p, const void *q, const void *k, const void *v, const void *out, const void *rest, const void *lse,
                  const void *grad, void *dq, void *dk, void *dv) {
  hipStream_t s = runtime().stream;
  const dim3 rows((unsigned)((long long)p.B * p.HQ * ceil_div(p.TQ, 4))), keys((unsigned)((long long)p.B * p.HK * ceil_div(p.TK, 4)));
  void *delta = nullptr;
  const int rc = workspace((size_t)p.B * p.HQ * p.TQ * sizeof(C), &delta);
  if (rc) return rc;
  {
    ScopedTiming timed(TAG_ATTENTION_DELTA);
    attention_delta_kernel<T, C><<<rows, dim3(256), 0, s>>>(p, (const T *)out, (const _Float16 *)rest, (const T *)grad, (C *)delta);
    MG_HIP(hipGetLastError());
  }
  if (dq) {
    ScopedTiming timed(TAG_ATTENTION_DQ);
    attention_dq_rows_kernel<T, C><<<rows, dim3(256), 0, s>>>(p, (const T *)q, (const T *)k, (const T *)v, (const T *)grad, (const C *)lse,
                                                              (const C *)delta, (T *)dq);
    MG_HIP(hipGetLastError());
  }
  if (dk && p.TK) {
    ScopedTiming timed(TAG_ATTENTION_DKV);
    attention_dkv_rows_kernel<T, C><<<keys, dim3(256), 0, s>>>(p, (const T *)q, (const T *)k, (const T *)v, (const T *)grad, (const C *)lse,
                                                               (const C *)delta, (T *)dk, (T *)dv);
    MG_HIP(hipGetLastError());
  }
  return MG_OK;
}

int check_attention(const mg_attention_desc *d, Attention *p, const char *who, bool gradient) {
  if (!d) return fail(MG_ERR_BAD_ARG, "%s: null descriptor", who);
  if (d->dtype != MG_F32 && d->dtype != MG_F64 && d->dtype != MG_F16) return fail(MG_ERR_UNSUPPORTED, "%s: dtype %d", who, d->dtype);
  if (d->B < 0 || d->TQ < 0 || d->TK < 0 || d->HQ <= 0 || d->HK <= 0 || d->D <= 0 || d->HQ % d->HK != 0)
    return fail(MG_ERR_BAD_ARG, "%s: batch %lld, %lld queries, %lld keys, %lld heads, %lld key heads, dim %lld", who, (long long)d->B,
                (long long)d->TQ, (long long)d->TK, (long long)d->HQ, (long long)d->HK, (long long)d->D);
  if (d->D > kMaxDim) return fail(MG_ERR_UNSUPPORTED, "%s: a head dimension of %lld (at most %d)", who, (long long)d->D, kMaxDim);
  const int64_t most = 1 << 30;
  if (d->TQ >= most || d->TK >= most || d->HQ >= most || d->B >= most || d->B * d->HQ >= most || d->B * d->HQ * ceil_div(d->TQ, 4) >= (1 << 24) ||
      (gradient && d->B * d->HK * ceil_div(d->TK, 4) >= (1 << 24)))  // a wavefront per row
    return fail(MG_ERR_UNSUPPORTED, "%s: 2^26 rows of results or more", who);
  if (d->longest < 0 || d->mean < 0) return fail(MG_ERR_BAD_ARG, "%s: a longest length of %lld, a mean of %lld", who, (long long)d->longest, (long long)d->mean);
  if (d->window < 0 || d->window > most) return fail(MG_ERR_BAD_ARG, "%s: a window of %lld keys", who, (long long)d->window);
  if (!std::isfinite(d->scale) || !std::isfinite(d->cap) || d->cap < 0) return fail(MG_ERR_BAD_ARG, "%s: scale %g, cap %g", who, d->scale, d->cap);
  // in single precision quotients and products of the two stay numbers, and neither turns into zero or infinity
  if (d->dtype != MG_F64 && (std::fabs(d->scale) > 1e30 || d->cap > 1e30 || (d->cap > 0 && d->cap < 1e-30)))
    return fail(MG_ERR_UNSUPPORTED, "%s: scale %g, cap %g in single precision", who, d->scale, d->cap);
  if (!d->starts != !d->ends) return fail(MG_ERR_BAD_ARG, "%s: starts of documents without their ends, or the other way round", who);
  if (d->window && d->prefix) return fail(MG_ERR_BAD_ARG, "%s: a window and a prefix", who);
  p->B = (int)d->B, p->TQ = (int)d->TQ, p->TK = (int)d->TK, p->HQ = (int)d->HQ, p->HK = (int)d->HK, p->D = (int)d->D;
  p->group = p->HQ / p->HK;
  p->longest = d->longest ? (int)std::min(d->longest, d->TK) : p->TK;
  p->mean = d->mean ? (int)std::min<int64_t>(d->mean, p->longest) : p->longest;
  p->causal = d->causal != 0, p->window = (int)d->window;
  p->scale = (float)d->scale, p->cap = (float)d->cap;
  p->bend = d->cap > 0 ? (float)std::max(-(double)FLT_MAX, std::min((double)FLT_MAX, d->scale / d->cap)) : 0.0f;
  p->scale64 = d->scale, p->cap64 = d->cap;
  p->lengths = d->lengths, p->prefix = d->prefix, p->starts = d->starts, p->ends = d->ends, p->slopes = d->slopes;
  return MG_OK;
}

}  // namespace

}  // namespace mg

using namespace mg;

extern "C" {

int mg_attention_fwd(const mg_attention_desc *desc, const void *q, const void *k, const void *v, void *out, void *rest,
                     void *lse) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  Attention p{};
  const int rc = check_attention(desc, &p, "mg_attention_fwd", false);
  if (rc) return rc;
  if (p.B == 0 || p.TQ == 0) return MG_OK;
  if (!q || !out || (p.TK && (!k || !v))) return fail(MG_ERR_BAD_ARG, "null pointer in mg_attention_fwd");
  if (desc->dtype != MG_F16) rest = nullptr;
  if (desc->dtype == MG_F64) return forward_rows<double, double>(p, q, k, v, out, rest, lse);
  const uintptr_t ends = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)rest;
  if (p.TK && tiles_take(p, desc->dtype == MG_F16 ? 2 : 4, ends))
    return few_take(p, desc->dtype == MG_F16 ? 2 : 4) ? forward_few(p, desc->dtype, q, k, v, out, rest, lse) : forward_tiles(p, desc->dtype, q, k, v, out, rest, lse);
  if (desc->dtype == MG_F32) return forward_rows<float, float>(p, q, k, v, out, rest, lse);
  return forward_rows<_Float16, float>(p, q, k, v, out, rest, lse);
}

int mg_attention_bwd(const mg_attention_desc *desc, const void *q, const void *k, const void *v, const void *out, const void *rest,
                     const void *lse, const void *grad, void *dq, void *dk, void *dv) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  Attention p{};
  const int rc = check_attention(desc, &p, "mg_attention_bwd", true);
  if (rc) return rc;
  if (!dk != !dv) return fail(MG_ERR_BAD_ARG, "mg_attention_bwd: dk without dv, or the other way round");
  const size_t size = desc->dtype == MG_F64 ? 8 : desc->dtype == MG_F32 ? 4 : 2;
  if (p.B == 0 || p.TQ == 0) {
    const size_t bytes = (size_t)p.B * p.TK * p.HK * p.D * size;
    if (!dk || !bytes) return MG_OK;
    const int zeroed = mg_memset_zero(dk, bytes);
    return zeroed ? zeroed : mg_memset_zero(dv, bytes);
  }
  if (!q || !out || !lse || !grad || (p.TK && (!k || !v))) return fail(MG_ERR_BAD_ARG, "null pointer in mg_attention_bwd");
  if (desc->dtype != MG_F16) rest = nullptr;
  if (desc->dtype == MG_F64) return backward_rows<double, double>(p, q, k, v, out, rest, lse, grad, dq, dk, dv);
  const uintptr_t ends = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)rest | (uintptr_t)grad | (uintptr_t)dq | (uintptr_t)dk |
                         (uintptr_t)dv;
  if (p.TK && tiles_take(p, desc->dtype == MG_F16 ? 2 : 4, ends)) return backward_tiles(p, desc->dtype, q, k, v, out, rest, lse, grad, dq, dk, dv);
  if (desc->dtype == MG_F32) return backward_rows<float, float>(p, q, k, v, out, rest, lse, grad, dq, dk, dv);
  return backward_rows<_Float16, float>(p, q, k, v, out, rest, lse, grad, dq, dk, dv);
}

int mg_cache_write(int dtype, int64_t B, int64_t T, int64_t capacity, int64_t row, const int32_t *lengths, const void *k, const void *v,
                   void *keys, void *values) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  if (dtype != MG_F32 && dtype != MG_F64 && dtype != MG_F16) return fail(MG_ERR_UNSUPPORTED, "mg_cache_write: dtype %d", dtype);
  const int64_t most = 1 << 30;
  if (B < 0 || T < 0 || capacity < 0 || row < 0 || B >= most || T >= most || capacity >= most || row >= most)
    return fail(MG_ERR_BAD_ARG, "mg_cache_write: batch %lld, %lld tokens, capacity %lld, %lld values a token", (long long)B, (long long)T,
                (long long)capacity, (long long)row);
  if (B == 0 || T == 0 || row == 0) return MG_OK;
  if (!lengths || !k || !v || !keys || !values) return fail(MG_ERR_BAD_ARG, "null pointer in mg_cache_write");
  const int64_t size = dtype == MG_F64 ? 8 : dtype == MG_F32 ? 4 : 2;
  const uintptr_t ends = (uintptr_t)k | (uintptr_t)v | (uintptr_t)keys | (uintptr_t)values;
  const bool wide = row * size % 16 == 0 && ends % 16 == 0;
  if (B * T >= (1ll << 40) / row) return fail(MG_ERR_UNSUPPORTED, "mg_cache_write: 2^40 values or more");
  const int64_t piece = wide ? row * size / 16 : row, pieces = B * T * piece;
  const dim3 grid((unsigned)std::min<int64_t>(ceil_div(pieces, 256), 1 << 16)), block(256);
  hipStream_t s = runtime().stream;
  ScopedTiming timed(TAG_CACHE_WRITE);
  auto launch = [&](auto one) {
    using V = decltype(one);
    cache_write_kernel<V><<<grid, block, 0, s>>>(pieces, (int)piece, (int)T, (int)capacity, lengths, (const V *)k, (const V *)v, (V *)keys, (V *)values);
  };
  if (wide)
    launch(uint4{});
  else if (size == 8)
    launch(uint64_t{});
  else if (size == 4)
    launch(uint32_t{});
  else
    launch(uint16_t{});
  MG_HIP(hipGetLastError());
  return MG_OK;
}

}  // extern "C"
