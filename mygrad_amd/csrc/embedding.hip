// Rows of a table by token, and the gradient of the table, for gfx950.
//
//   y[n] = scale W[ids[n]]  (zeros where ids[n] < 0)          dW[v] = scale * sum of grad[n] over the n with ids[n] = v, in their order
#include "internal.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

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

// A block per token.
template <typename T>
__global__ void __launch_bounds__(256) embedding_kernel(Embedding p, const int32_t *__restrict__ ids, const T *__restrict__ weight, T *__restrict__ out) {
  const int id = ids[blockIdx.x];
  const bool there = id >= 0 && id < p.rows;
  const T *row = weight + (there ? id : 0) * p.D;
  T *y = out + blockIdx.x * p.D;
  for (long long d = threadIdx.x; d < p.D; d += 256) y[d] = there ? (T)((Scaled<T>)row[d] * (Scaled<T>)p.scale) : (T)0;
}

// A block per row of the table, which looks at all tokens.
template <typename T, typename C>
__global__ void __launch_bounds__(256) embedding_bwd_kernel(Embedding p, const int32_t *__restrict__ ids, const T *__restrict__ grad, T *__restrict__ dweight) {
  const int row = blockIdx.x;
  for (long long d = threadIdx.x; d < p.D; d += 256) {
    C sum = 0;
    for (long long n = 0; n < p.tokens; ++n)
      if (ids[n] == row) sum += (C)grad[n * p.D + d];
    dweight[row * p.D + d] = (T)((Scaled<T>)sum * (Scaled<T>)p.scale);
  }
}

int check(int dtype, int64_t tokens, int64_t rows, int64_t D, double scale, const char *who) {
  if (dtype != MG_F32 && dtype != MG_F64 && dtype != MG_F16) return fail(MG_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (tokens < 0 || rows < 0 || D < 0 || !(std::fabs(scale) <= 1e30))  // single precision holds it
    return fail(MG_ERR_BAD_ARG, "%s: %lld tokens, a table of %lld rows of %lld values, scale %g", who, (long long)tokens, (long long)rows, (long long)D,
                scale);
  if (tokens > 0x7fffffff || rows > 0x7ffffffe || D > (1ll << 30))
    return fail(MG_ERR_UNSUPPORTED, "%s: %lld tokens, a table of %lld rows of %lld values", who, (long long)tokens, (long long)rows, (long long)D);
  return MG_OK;
}

template <typename T>
int forward(const Embedding &p, const int32_t *ids, const void *weight, void *out) {
  ScopedTiming timed(TAG_EMBEDDING);
  embedding_kernel<T><<<dim3((unsigned)p.tokens), dim3(256), 0, runtime().stream>>>(p, ids, (const T *)weight, (T *)out);
  MG_HIP(hipGetLastError());
  return MG_OK;
}

template <typename T, typename C>
int backward(const Embedding &p, const int32_t *ids, const void *grad, void *dweight) {
  ScopedTiming timed(TAG_EMBEDDING_BWD);
  embedding_bwd_kernel<T, C><<<dim3((unsigned)p.rows), dim3(256), 0, runtime().stream>>>(p, ids, (const T *)grad, (T *)dweight);
  MG_HIP(hipGetLastError());
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
