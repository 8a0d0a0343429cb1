// Layer norm, forward and backward.
#include <math.h>

#include "types.cuh"

namespace b2 {

constexpr int kLnThreads = 256;

// Sum over the block, the same bits in every thread: shuffles within a warp, then the warps' sums in order.
__device__ __forceinline__ float ln_block_sum(float v, float *scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kLnThreads / 32; ++i) s += scratch[i];
  return s;
}

// One block per row, the row read three times.  The second reading sums the distances from the first mean as well as
// their squares: what the first mean was off by is taken out of both.
template <class T, class P>
__global__ void __launch_bounds__(kLnThreads) layernorm_kernel(int64_t rows, int64_t cols, float eps, const T *x, int64_t ldx,
                                                               const P *gamma, const P *beta, T *y, int64_t ldy, float *mean,
                                                               float *rstd) {
  __shared__ float scratch[kLnThreads / 32];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * ldx;
    T *yr = y + row * ldy;
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < cols; i += kLnThreads) s += to_f32(xr[i]);
    float m = ln_block_sum(s, scratch) / (float)cols;
    float d1 = 0.f, d2 = 0.f;
    for (int64_t i = threadIdx.x; i < cols; i += kLnThreads) {
      const float d = to_f32(xr[i]) - m;
      d1 += d;
      d2 = fmaf(d, d, d2);
    }
    d1 = ln_block_sum(d1, scratch) / (float)cols;
    d2 = ln_block_sum(d2, scratch) / (float)cols;
    m += d1;
    const float r = 1.f / sqrtf(fmaf(-d1, d1, d2) + eps);
    if (threadIdx.x == 0) {
      if (mean) mean[row] = m;
      if (rstd) rstd[row] = r;
    }
    for (int64_t i = threadIdx.x; i < cols; i += kLnThreads) {
      const float h = (to_f32(xr[i]) - m) * r;
      yr[i] = from_f32<T>(fmaf(h, gamma ? to_f32(gamma[i]) : 1.f, beta ? to_f32(beta[i]) : 0.f));
    }
  }
}

template <class T, class P>
__global__ void __launch_bounds__(kLnThreads) layernorm_dx_kernel(int64_t rows, int64_t cols, const T *dy, int64_t lddy, const T *x,
                                                                  int64_t ldx, const P *gamma, const float *mean,
                                                                  const float *rstd, T *dx, int64_t lddx) {
  __shared__ float scratch[kLnThreads / 32];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * ldx, *gr = dy + row * lddy;
    const float m = mean[row], r = rstd[row];
    float a = 0.f, b = 0.f;
    for (int64_t i = threadIdx.x; i < cols; i += kLnThreads) {
      const float u = to_f32(gr[i]) * (gamma ? to_f32(gamma[i]) : 1.f);
      a += u;
      b = fmaf(u, (to_f32(xr[i]) - m) * r, b);
    }
    a = ln_block_sum(a, scratch) / (float)cols;
    b = ln_block_sum(b, scratch) / (float)cols;
    for (int64_t i = threadIdx.x; i < cols; i += kLnThreads) {
      const float u = to_f32(gr[i]) * (gamma ? to_f32(gamma[i]) : 1.f);
      const float h = (to_f32(xr[i]) - m) * r;
      dx[row * lddx + i] = from_f32<T>(r * (u - fmaf(h, b, a)));
    }
  }
}

// Partial sums over rows: block (c, p) sums the rows p, p + parts, ... of 256 columns.
template <class T>
__global__ void __launch_bounds__(kLnThreads) layernorm_dparams_kernel(int64_t rows, int64_t cols, const T *dy, int64_t lddy,
                                                                       const T *x, int64_t ldx, const float *mean,
                                                                       const float *rstd, float *partial) {
  const int64_t c = (int64_t)blockIdx.x * kLnThreads + threadIdx.x;
  if (c >= cols) return;
  float g = 0.f, b = 0.f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float v = to_f32(dy[row * lddy + c]);
    g = fmaf(v, (to_f32(x[row * ldx + c]) - mean[row]) * rstd[row], g);
    b += v;
  }
  partial[((int64_t)blockIdx.y * 2) * cols + c] = g;
  partial[((int64_t)blockIdx.y * 2 + 1) * cols + c] = b;
}

template <class P>
__global__ void __launch_bounds__(kLnThreads) layernorm_reduce_kernel(int parts, int64_t cols, const float *partial, P *dgamma,
                                                                      P *dbeta) {
  const int64_t c = (int64_t)blockIdx.x * kLnThreads + threadIdx.x;
  if (c >= cols) return;
  float g = 0.f, b = 0.f;
  for (int p = 0; p < parts; ++p) {
    g += partial[((int64_t)p * 2) * cols + c];
    b += partial[((int64_t)p * 2 + 1) * cols + c];
  }
  if (dgamma) dgamma[c] = from_f32<P>(g);
  if (dbeta) dbeta[c] = from_f32<P>(b);
}

// Blocks that share the rows of the gradient sums.
static int64_t ln_parts(int64_t rows) { return rows < 148 ? rows : 148; }

}  // namespace b2

using namespace b2;

extern "C" {

int b2_layernorm(b2_handle h, int64_t rows, int64_t cols, float eps, int type, const void *x, int64_t ldx, int param_type,
                 const void *gamma, const void *beta, void *y, int64_t ldy, float *mean, float *rstd, void *stream) {
  const int tb = type_bytes(type), pb = type_bytes(param_type);
  B2_REQUIRE(tb != 0, B2_ERR_INVALID_ARG, "b2_layernorm: unknown type %d", type);
  B2_REQUIRE(param_type == B2_F32 || param_type == type, B2_ERR_INVALID_ARG,
             "b2_layernorm: param_type %d is neither B2_F32 nor the type %d of x", param_type, type);
  B2_REQUIRE(rows >= 0 && cols >= 1 && cols <= INT32_MAX, B2_ERR_INVALID_ARG, "b2_layernorm: bad shape %lld x %lld", (long long)rows,
             (long long)cols);
  B2_REQUIRE(ldx >= cols && ldy >= cols, B2_ERR_INVALID_ARG, "b2_layernorm: ldx = %lld or ldy = %lld is less than cols = %lld",
             (long long)ldx, (long long)ldy, (long long)cols);
  B2_REQUIRE(eps >= 0.f && isfinite(eps), B2_ERR_INVALID_ARG, "b2_layernorm: eps = %g is negative or not finite", (double)eps);
  if (rows == 0) return B2_OK;
  B2_REQUIRE(x != nullptr && y != nullptr, B2_ERR_INVALID_ARG, "b2_layernorm: x or y is NULL");
  B2_REQUIRE((((uintptr_t)x | (uintptr_t)y) & (tb - 1)) == 0 && (((uintptr_t)gamma | (uintptr_t)beta) & (pb - 1)) == 0 &&
                 (((uintptr_t)mean | (uintptr_t)rstd) & 3) == 0,
             B2_ERR_INVALID_ARG, "b2_layernorm: a pointer is not aligned to its element type");
  B2_REQUIRE((x == y && ldx == ldy) || !matrices_overlap(x, rows, cols * tb, ldx * tb, y, rows, cols * tb, ldy * tb),
             B2_ERR_INVALID_ARG, "b2_layernorm: y overlaps x (only y == x with ldy == ldx may share memory)");
  B2_CONTEXT(ctx, h, "b2_layernorm");
  const int64_t cap = (int64_t)ctx->sm_count * 8;
  const int grid = (int)(rows < cap ? rows : cap);
  auto launch = [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    layernorm_kernel<T, P><<<grid, kLnThreads, 0, (cudaStream_t)stream>>>(rows, cols, eps, (const T *)x, ldx, (const P *)gamma,
                                                                          (const P *)beta, (T *)y, ldy, mean, rstd);
    return 0;
  };
  with_type(type, [&](auto t) { return param_type == type ? launch(t, t) : launch(t, float()); });
  B2_CUDA(cudaGetLastError());
  return B2_OK;
}

size_t b2_layernorm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)ln_parts(rows) * 2 * (size_t)cols * sizeof(float);
}

int b2_layernorm_backward(b2_handle h, int64_t rows, int64_t cols, int type, const void *dy, int64_t lddy, const void *x,
                          int64_t ldx, int param_type, const void *gamma, const float *mean, const float *rstd, void *dx,
                          int64_t lddx, void *dgamma, void *dbeta, void *workspace, size_t workspace_bytes, void *stream) {
  const int tb = type_bytes(type), pb = type_bytes(param_type);
  B2_REQUIRE(tb != 0, B2_ERR_INVALID_ARG, "b2_layernorm_backward: unknown type %d", type);
  B2_REQUIRE(param_type == B2_F32 || param_type == type, B2_ERR_INVALID_ARG,
             "b2_layernorm_backward: param_type %d is neither B2_F32 nor the type %d of x", param_type, type);
  B2_REQUIRE(rows >= 0 && cols >= 1 && cols <= INT32_MAX, B2_ERR_INVALID_ARG, "b2_layernorm_backward: bad shape %lld x %lld",
             (long long)rows, (long long)cols);
  B2_REQUIRE(lddy >= cols && ldx >= cols && (!dx || lddx >= cols), B2_ERR_INVALID_ARG,
             "b2_layernorm_backward: a leading dimension (dy %lld, x %lld, dx %lld) is less than cols = %lld", (long long)lddy,
             (long long)ldx, (long long)lddx, (long long)cols);
  const bool sums = dgamma || dbeta;
  if (!dx && !sums) return B2_OK;
  if (rows > 0) {
    B2_REQUIRE(dy != nullptr && x != nullptr && mean != nullptr && rstd != nullptr, B2_ERR_INVALID_ARG,
               "b2_layernorm_backward: dy, x, mean or rstd is NULL");
    B2_REQUIRE((((uintptr_t)dy | (uintptr_t)x | (uintptr_t)dx) & (tb - 1)) == 0 && (((uintptr_t)mean | (uintptr_t)rstd) & 3) == 0,
               B2_ERR_INVALID_ARG, "b2_layernorm_backward: a pointer is not aligned to its element type");
    B2_REQUIRE((dx == dy && lddx == lddy) || !matrices_overlap(dx, rows, cols * tb, lddx * tb, dy, rows, cols * tb, lddy * tb),
               B2_ERR_INVALID_ARG, "b2_layernorm_backward: dx overlaps dy (only dx == dy with lddx == lddy may share memory)");
    B2_REQUIRE(!matrices_overlap(dx, rows, cols * tb, lddx * tb, x, rows, cols * tb, ldx * tb), B2_ERR_INVALID_ARG,
               "b2_layernorm_backward: dx overlaps x");
  }
  B2_REQUIRE((((uintptr_t)gamma | (uintptr_t)dgamma | (uintptr_t)dbeta) & (pb - 1)) == 0, B2_ERR_INVALID_ARG,
             "b2_layernorm_backward: gamma, dgamma or dbeta is not aligned to its element type");
  const size_t need = sums ? b2_layernorm_backward_workspace_bytes(rows, cols) : 0;
  B2_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), B2_ERR_WORKSPACE,
             "b2_layernorm_backward: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
  B2_REQUIRE(need == 0 || ((uintptr_t)workspace & 15) == 0, B2_ERR_INVALID_ARG, "b2_layernorm_backward: workspace is not 16-byte aligned");
  B2_CONTEXT(ctx, h, "b2_layernorm_backward");
  cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {
    if (dgamma) B2_CUDA(cudaMemsetAsync(dgamma, 0, (size_t)cols * pb, s));
    if (dbeta) B2_CUDA(cudaMemsetAsync(dbeta, 0, (size_t)cols * pb, s));
    return B2_OK;
  }
  const int64_t cap = (int64_t)ctx->sm_count * 8;
  const int grid = (int)(rows < cap ? rows : cap);
  const int parts = (int)ln_parts(rows);
  const unsigned col_blocks = (unsigned)((cols + kLnThreads - 1) / kLnThreads);
  auto launch = [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    if (sums) {
      layernorm_dparams_kernel<T><<<dim3(col_blocks, parts), kLnThreads, 0, s>>>(rows, cols, (const T *)dy, lddy, (const T *)x, ldx,
                                                                                mean, rstd, (float *)workspace);
      layernorm_reduce_kernel<P><<<col_blocks, kLnThreads, 0, s>>>(parts, cols, (const float *)workspace, (P *)dgamma, (P *)dbeta);
    }
    if (dx)
      layernorm_dx_kernel<T, P><<<grid, kLnThreads, 0, s>>>(rows, cols, (const T *)dy, lddy, (const T *)x, ldx, (const P *)gamma, mean,
                                                            rstd, (T *)dx, lddx);
    return 0;
  };
  with_type(type, [&](auto t) { return param_type == type ? launch(t, t) : launch(t, float()); });
  B2_CUDA(cudaGetLastError());
  return B2_OK;
}

}  // extern "C"
