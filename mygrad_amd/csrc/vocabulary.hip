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

namespace mg {

namespace {

constexpr int kMostTop = 128;      // likeliest tokens that are looked for
constexpr int kMostTaught = 256;   // a teacher's tokens for a row: a thread each

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

template <typename C>
__device__ __forceinline__ C block_max(C v, C *space) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
  for (int k = 32; k; k >>= 1) v = max(v, __shfl_xor(v, k));
  __syncthreads();
  if (lane == 0) space[wave] = v;
  __syncthreads();
  for (int w = 0; w < waves; ++w) v = max(v, space[w]);
  return v;
}

// m, s and a of a row that the whole block goes through.
template <typename T, typename C>
__device__ __forceinline__ Row<C> row_of(const Vocabulary &p, const T *z, bool with_mean, C *space) {
  const C per = (C)p.per;
  C most = -infinity<C>();
  for (int j = threadIdx.x; j < p.V; j += blockDim.x) most = max(most, (C)z[j]);
  most = block_max(most, space);
  if (most == -infinity<C>()) most = 0;
  C sums[2] = {0, 0};
  for (int j = threadIdx.x; j < p.V; j += blockDim.x) {
    const C t = ((C)z[j] - most) * per, e = exp(t);
    sums[0] += e;
    if (with_mean && e > 0) sums[1] += e * t;
  }
  block_add(sums, space);
  return Row<C>{most, sums[0], sums[0] > 0 ? sums[1] / sums[0] : C(0)};
}

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

// ---- log probabilities ----------------------------------------------------------------------------------------------------------
template <typename T, typename C>
__global__ void __launch_bounds__(256) scores_kernel(Vocabulary p, const int32_t *__restrict__ ids, const T *__restrict__ logits, C *__restrict__ scores,
                                                     C *__restrict__ entropy, Row<C> *__restrict__ kept, C *__restrict__ top_scores,
                                                     int32_t *__restrict__ top_ids) {
  __shared__ C space[32];
  const long long r = blockIdx.x;
  const T *z = logits + r * p.V;
  const Row<C> row = row_of(p, z, true, space);
  if (threadIdx.x == 0) {
    if (kept) kept[r] = row;
    if (scores) {
      const int id = ids[r];
      scores[r] = id < 0 || id >= p.V ? C(0) : log_probability<C>(row, (C)z[id], 1);
    }
    if (entropy) entropy[r] = row.s == 0 ? C(0) : log(row.s) - row.a;
  }
  typedef decltype(order_of(C(0))) Order;
  __shared__ Order best_value[4];
  __shared__ int best_place[4];
  Order last = 0;
  int after = -1;
  for (int k = 0; k < p.top; ++k) {
    Order value = 0;
    int place = 0x7fffffff;
    for (int j = threadIdx.x; j < p.V; j += 256) {
      const Order o = order_of((C)z[j]);
      const bool left = k == 0 || o < last || (o == last && j > after);
      if (left && (place == 0x7fffffff || o > value)) value = o, place = j;
    }
    for (int m = 32; m; m >>= 1) {
      const Order other = __shfl_xor(value, m);
      const int where = __shfl_xor(place, m);
      if (where != 0x7fffffff && (place == 0x7fffffff || other > value || (other == value && where < place))) value = other, place = where;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) best_value[threadIdx.x >> 6] = value, best_place[threadIdx.x >> 6] = place;
    __syncthreads();
    last = best_value[0], after = best_place[0];
    for (int w = 1; w < 4; ++w)
      if (best_place[w] != 0x7fffffff && (after == 0x7fffffff || best_value[w] > last || (best_value[w] == last && best_place[w] < after)))
        last = best_value[w], after = best_place[w];
    if (threadIdx.x == 0) {
      top_ids[r * p.top + k] = after;
      top_scores[r * p.top + k] = log_probability<C>(row, (C)z[after], 1);
    }
  }
}

template <typename T, typename C>
__global__ void __launch_bounds__(256) scores_bwd_kernel(Vocabulary p, const int32_t *__restrict__ ids, const T *__restrict__ logits,
                                                         const Row<C> *__restrict__ kept, const C *__restrict__ grad_scores,
                                                         const C *__restrict__ grad_entropy, T *__restrict__ dlogits) {
  const long long r = blockIdx.x;
  const T *z = logits + r * p.V;
  T *out = dlogits + r * p.V;
  const Row<C> row = kept[r];
  int id = grad_scores ? ids[r] : -1;
  if (id >= p.V) id = -1;
  const C g = id < 0 ? C(0) : grad_scores[r], h = grad_entropy ? grad_entropy[r] : C(0), inverse = 1 / row.s;
  const bool nothing = row.s == 0 || (id < 0 && !grad_entropy);
  for (int j = threadIdx.x; j < p.V; j += 256) {
    const C t = (C)z[j] - row.m, share = exp(t) * inverse;
    C dz = -share * g;
    if (grad_entropy) dz -= share * ((share > 0 ? t : C(0)) - row.a) * h;
    out[j] = nothing ? (T)0 : (T)(j == id ? dz + g : dz);
  }
}

// ---- distillation ---------------------------------------------------------------------------------------------------------------
// Thread k takes the teacher's k-th token; q goes to memory for the backward pass.
template <typename T, typename Y, typename C>
__global__ void __launch_bounds__(256) distillation_kernel(Vocabulary p, const int32_t *__restrict__ ids, const T *__restrict__ logits,
                                                           const Y *__restrict__ teacher, C *__restrict__ loss, Row<C> *__restrict__ kept,
                                                           C *__restrict__ shares) {
  __shared__ C space[32];
  const long long r = blockIdx.x;
  const T *z = logits + r * p.V;
  const C per = (C)p.per;
  Row<C> row = row_of(p, z, false, space);
  const int k = threadIdx.x;
  int id = k < p.top ? ids[r * p.top + k] : -1;
  if (id >= p.V) id = -1;
  const C y = id < 0 ? -infinity<C>() : (C)teacher[r * p.top + k];
  C most = block_max(y, space);
  if (most == -infinity<C>()) most = 0;
  const C u = (y - most) * per;
  C total[1] = {exp(u)};
  block_add(total, space);
  const C q = total[0] == 0 ? C(0) : exp(u) / total[0];
  const C zk = id < 0 ? C(0) : (C)z[id];
  C sum[1] = {q == 0 ? C(0) : q * ((u - log(total[0])) - log_probability<C>(row, zk, per))};
  block_add(sum, space);
  if (k < p.top && shares) shares[r * p.top + k] = q;
  if (k == 0) {
    loss[r] = sum[0];
    row.a = total[0] == 0 ? C(0) : total[0] / total[0];  // 1, or NaN
    if (kept) kept[r] = row;
  }
}

template <typename T, typename C>
__global__ void __launch_bounds__(256) distillation_bwd_kernel(Vocabulary p, const int32_t *__restrict__ ids, const T *__restrict__ logits,
                                                               const Row<C> *__restrict__ kept, const C *__restrict__ shares,
                                                               const C *__restrict__ grad, T *__restrict__ dlogits) {
  __shared__ int taught[kMostTaught];
  __shared__ C share_of[kMostTaught];
  const long long r = blockIdx.x;
  const T *z = logits + r * p.V;
  T *out = dlogits + r * p.V;
  const Row<C> row = kept[r];
  const int k = threadIdx.x;
  if (k < p.top) taught[k] = ids[r * p.top + k], share_of[k] = shares[r * p.top + k];
  __syncthreads();
  const C per = (C)p.per, g = grad[r] * per, inverse = row.a / row.s;
  const bool nothing = row.s == 0 || row.a == 0;
  for (int j = threadIdx.x; j < p.V; j += 256) out[j] = nothing ? (T)0 : (T)(g * exp(((C)z[j] - row.m) * per) * inverse);
  __syncthreads();  // the teacher's tokens are written once more, each by the first thread that has it
  if (k >= p.top || nothing) return;
  const int id = taught[k];
  if (id < 0 || id >= p.V) return;
  C q = 0;
  for (int n = 0; n < p.top; ++n)
    if (taught[n] == id) {
      if (n < k) return;
      q += share_of[n];
    }
  out[id] = (T)(g * (exp(((C)z[id] - row.m) * per) * inverse - q));
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
    scores_kernel<T, C><<<dim3((unsigned)rows), dim3(256), 0, runtime().stream>>>(p, ids, (const T *)logits, (C *)scores, (C *)entropy, (Row<C> *)kept,
                                                                                  (C *)top_scores, top_ids);
    MG_HIP(hipGetLastError());
    return (int)MG_OK;
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
    scores_bwd_kernel<T, C><<<dim3((unsigned)rows), dim3(256), 0, runtime().stream>>>(p, ids, (const T *)logits, (const Row<C> *)kept,
                                                                                      (const C *)grad_scores, (const C *)grad_entropy, (T *)dlogits);
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
    const dim3 grid((unsigned)rows);
    if (teacher_dtype == dtype)
      distillation_kernel<T, T, C><<<grid, dim3(256), 0, runtime().stream>>>(p, ids, (const T *)logits, (const T *)teacher, (C *)loss, (Row<C> *)kept, (C *)shares);
    else
      distillation_kernel<T, C, C><<<grid, dim3(256), 0, runtime().stream>>>(p, ids, (const T *)logits, (const C *)teacher, (C *)loss, (Row<C> *)kept, (C *)shares);
    MG_HIP(hipGetLastError());
    return (int)MG_OK;
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
    distillation_bwd_kernel<T, C><<<dim3((unsigned)rows), dim3(256), 0, runtime().stream>>>(p, ids, (const T *)logits, (const Row<C> *)kept,
                                                                                            (const C *)shares, (const C *)grad, (T *)dlogits);
    MG_HIP(hipGetLastError());
    return (int)MG_OK;
  });
}

}  // extern "C"
