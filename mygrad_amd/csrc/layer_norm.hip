// Layer norm and its gradient for gfx950.
//
//   mu = mean x     d = x - mu     r = 1 / sqrt(mean(d^2) + eps)     n = d r     y = w n + b     (over the D values of a row)
//   u = w grad      dx = r (u - mean(u) - n mean(u n))               dw = sum grad n             db = sum grad   (over the rows)
//
// The mean is taken twice: x - mean is exact to a unit of itself where a row lies far from zero, so the mean of what is left, and the
// variance around it, are those of the row to single precision whatever its offset.
#include "row_device.h"

#include <algorithm>
#include <cmath>

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

// Of a row that the whole block goes through.
template <typename T, typename C>
__device__ __forceinline__ Moments<C> moments_of(const LayerNorm &p, const T *row, C *space) {
  C sum[1] = {0};
  for (long long d = threadIdx.x; d < p.D; d += blockDim.x) sum[0] += (C)row[d];
  block_add(sum, space);
  const C shift = sum[0] / (C)p.D;
  C both[2] = {0, 0};
  for (long long d = threadIdx.x; d < p.D; d += blockDim.x) {
    const C v = (C)row[d] - shift;
    both[0] += v, both[1] += v * v;
  }
  block_add(both, space);
  const C mean = both[0] / (C)p.D;
  return Moments<C>{shift, mean, 1 / sqrt(max(both[1] / (C)p.D - mean * mean, C(0)) + (C)p.eps)};
}

// ---- a block per row, which it goes through three times ------------------------------------------------------------------------
template <typename T, typename C>
__global__ void __launch_bounds__(256) layer_norm_kernel(LayerNorm p, const T *__restrict__ x, const T *__restrict__ w, const T *__restrict__ b,
                                                         T *__restrict__ y) {
  __shared__ C space[32];
  const T *row = x + blockIdx.x * p.D;
  T *out = y + blockIdx.x * p.D;
  const Moments<C> m = moments_of(p, row, space);
  for (long long d = threadIdx.x; d < p.D; d += 256)
    out[d] = (T)(((C)row[d] - m.shift - m.mean) * m.r * (w ? (C)w[d] : C(1)) + (b ? (C)b[d] : C(0)));
}

// dx, and mean and r of each row for the sums over rows.
template <typename T, typename C>
__global__ void __launch_bounds__(256) layer_norm_dx_kernel(LayerNorm p, const T *__restrict__ x, const T *__restrict__ w, const T *__restrict__ grad,
                                                            T *__restrict__ dx, Moments<C> *__restrict__ moments) {
  __shared__ C space[32];
  const T *row = x + blockIdx.x * p.D, *g = grad + blockIdx.x * p.D;
  const Moments<C> m = moments_of(p, row, space);
  if (moments && threadIdx.x == 0) moments[blockIdx.x] = m;
  if (!dx) return;
  C sums[2] = {0, 0};
  for (long long d = threadIdx.x; d < p.D; d += 256) {
    const C u = (C)g[d] * (w ? (C)w[d] : C(1));
    sums[0] += u, sums[1] += u * (((C)row[d] - m.shift - m.mean) * m.r);
  }
  block_add(sums, space);
  const C first = sums[0] / (C)p.D, second = sums[1] / (C)p.D;
  for (long long d = threadIdx.x; d < p.D; d += 256) {
    const C n = ((C)row[d] - m.shift - m.mean) * m.r;
    dx[blockIdx.x * p.D + d] = (T)(m.r * ((C)g[d] * (w ? (C)w[d] : C(1)) - first - n * second));
  }
}

// Sums over the rows of one share (blockIdx.y): a thread per column.
template <typename T, typename C>
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(LayerNorm p, long long share, const T *__restrict__ x, const T *__restrict__ grad,
                                                                 const Moments<C> *__restrict__ moments, double *__restrict__ parts) {
  const long long d = (long long)blockIdx.x * 256 + threadIdx.x;
  if (d >= p.D) return;
  const long long from = blockIdx.y * share, to = min(p.rows, from + share);
  double dw = 0, db = 0;
  for (long long row = from; row < to; ++row) {
    const Moments<C> m = moments[row];
    const C g = (C)grad[row * p.D + d];
    dw += (double)(g * (((C)x[row * p.D + d] - m.shift - m.mean) * m.r));
    db += (double)g;
  }
  parts[(2ll * blockIdx.y) * p.D + d] = dw;
  parts[(2ll * blockIdx.y + 1) * p.D + d] = db;
}

template <typename T>
__global__ void __launch_bounds__(256) layer_norm_join_kernel(long long D, int shares, const double *__restrict__ parts, T *__restrict__ dw,
                                                              T *__restrict__ db) {
  const long long d = (long long)blockIdx.x * 256 + threadIdx.x;
  if (d >= D) return;
  double sums[2] = {0, 0};
  for (int n = 0; n < shares; ++n) sums[0] += parts[2ll * n * D + d], sums[1] += parts[(2ll * n + 1) * D + d];
  if (dw) dw[d] = (T)sums[0];
  if (db) db[d] = (T)sums[1];
}

template <typename T, typename C>
int forward(const LayerNorm &p, const void *x, const void *w, const void *b, void *y) {
  ScopedTiming timed(TAG_LAYER_NORM);
  layer_norm_kernel<T, C><<<dim3((unsigned)p.rows), dim3(256), 0, runtime().stream>>>(p, (const T *)x, (const T *)w, (const T *)b, (T *)y);
  MG_HIP(hipGetLastError());
  return MG_OK;
}

template <typename T, typename C>
int backward(const LayerNorm &p, const void *x, const void *w, const void *grad, void *dx, void *dw, void *db) {
  hipStream_t s = runtime().stream;
  const bool columns = dw || db;
  const long long share = std::max<long long>(ceil_div(p.rows, 256), 16), shares = ceil_div(p.rows, share);
  char *space = nullptr;
  const size_t sums = columns ? (size_t)(2 * shares * p.D) * sizeof(double) : 0;
  if (columns) {
    const int rc = workspace(sums + (size_t)p.rows * sizeof(Moments<C>), (void **)&space);
    if (rc) return rc;
  }
  ScopedTiming timed(TAG_LAYER_NORM_BWD);
  Moments<C> *moments = columns ? (Moments<C> *)(space + sums) : nullptr;
  layer_norm_dx_kernel<T, C><<<dim3((unsigned)p.rows), dim3(256), 0, s>>>(p, (const T *)x, (const T *)w, (const T *)grad, (T *)dx, moments);
  MG_HIP(hipGetLastError());
  if (!columns) return MG_OK;
  const unsigned across = (unsigned)ceil_div(p.D, 256);
  layer_norm_columns_kernel<T, C><<<dim3(across, (unsigned)shares), dim3(256), 0, s>>>(p, share, (const T *)x, (const T *)grad, moments, (double *)space);
  MG_HIP(hipGetLastError());
  layer_norm_join_kernel<T><<<dim3(across), dim3(256), 0, s>>>(p.D, (int)shares, (const double *)space, (T *)dw, (T *)db);
  MG_HIP(hipGetLastError());
  return MG_OK;
}

int check(int dtype, int64_t rows, int64_t D, double eps, const char *who) {
  if (dtype != MG_F32 && dtype != MG_F64 && dtype != MG_F16) return fail(MG_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (rows < 0 || D <= 0 || !(eps >= 0) || !std::isfinite(eps))
    return fail(MG_ERR_BAD_ARG, "%s: %lld rows of %lld values, eps %g", who, (long long)rows, (long long)D, eps);
  if (rows > 0x7fffffff || D > (1ll << 30)) return fail(MG_ERR_UNSUPPORTED, "%s: %lld rows of %lld values", who, (long long)rows, (long long)D);
  return MG_OK;
}

}  // namespace

}  // namespace mg

using namespace mg;

extern "C" {

int mg_layer_norm_fwd(int dtype, int64_t rows, int64_t D, double eps, const void *x, const void *weight, const void *bias, void *y) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  const int rc = check(dtype, rows, D, eps, "mg_layer_norm_fwd");
  if (rc || rows == 0) return rc;
  if (!x || !y) return fail(MG_ERR_BAD_ARG, "null pointer in mg_layer_norm_fwd");
  const LayerNorm p{rows, D, eps};
  if (dtype == MG_F64) return forward<double, double>(p, x, weight, bias, y);
  if (dtype == MG_F32) return forward<float, float>(p, x, weight, bias, y);
  return forward<_Float16, float>(p, x, weight, bias, y);
}

int mg_layer_norm_bwd(int dtype, int64_t rows, int64_t D, double eps, const void *x, const void *weight, const void *grad, void *dx, void *dweight,
                      void *dbias) {
  std::lock_guard<std::recursive_mutex> guard(api_mutex());
  MG_REQUIRE_INIT();
  const int rc = check(dtype, rows, D, eps, "mg_layer_norm_bwd");
  if (rc) return rc;
  if (!dx && !dweight && !dbias) return fail(MG_ERR_BAD_ARG, "mg_layer_norm_bwd: no gradient is wanted");
  if (rows == 0) {
    const size_t bytes = (size_t)D * (dtype == MG_F64 ? 8 : dtype == MG_F32 ? 4 : 2);
    for (void *out : {dweight, dbias})
      if (out)
        if (const int status = mg_memset_zero(out, bytes)) return status;
    return MG_OK;
  }
  if (!x || !grad) return fail(MG_ERR_BAD_ARG, "null pointer in mg_layer_norm_bwd");
  const LayerNorm p{rows, D, eps};
  if (dtype == MG_F64) return backward<double, double>(p, x, weight, grad, dx, dweight, dbias);
  if (dtype == MG_F32) return backward<float, float>(p, x, weight, grad, dx, dweight, dbias);
  return backward<_Float16, float>(p, x, weight, grad, dx, dweight, dbias);
}

}  // extern "C"
