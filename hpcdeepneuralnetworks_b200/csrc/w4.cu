// 4-bit weights with group scales: quantise, expand, and the matrix-vector product of decoding steps.
#include <math.h>

#include "types.cuh"

namespace b2 {

constexpr int kW4MaxRows = 64;   // rows of x that b2_w4_matvec takes

__device__ __forceinline__ float w4_warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The integer nearest to w / s for s > 0, ties to even, as a float.  The quotient in FP32 names a candidate that is at most
// one off; the candidate's remainder, which an FMA leaves exact near a border, says whether a neighbour is nearer.  `inv` is
// 1 / s (finite: see w4_prescale).
__device__ __forceinline__ float w4_nearest(float w, float s, float inv) {
  float q = rintf(fminf(fmaxf(w * inv, -40.f), 40.f));
  const float r = fmaf(-q, s, w), half = 0.5f * s;
  const bool odd = ((int)q) & 1;
  if (r > half || (r == half && odd)) q += 1.f;
  else if (r < -half || (r == -half && odd)) q -= 1.f;
  return q;
}
// A power of two that keeps the reciprocal of a tiny scale finite and its half exact; weights of such a group are at most
// 16 scales large, so nothing overflows.
__device__ __forceinline__ float w4_prescale(float s) { return s < 0x1p-100f ? 0x1p100f : 1.f; }

template <class S>
__device__ __forceinline__ float w4_largest();
template <>
__device__ __forceinline__ float w4_largest<float>() {
  return 3.402823466e38f;
}
template <>
__device__ __forceinline__ float w4_largest<__nv_bfloat16>() {
  return 0x1.FEp127f;
}
template <>
__device__ __forceinline__ float w4_largest<__half>() {
  return 65504.f;
}

// The scale of a group whose values reach from lo <= 0 to hi >= 0, and its zero point.
template <class S>
__device__ __forceinline__ S w4_scale(float lo, float hi, bool with_zeros) {
  float s;
  if (with_zeros) {
    s = hi - lo;
    s = isinf(s) ? hi / 15.f - lo / 15.f : s / 15.f;   // the span of finite weights may pass FP32's range
  } else {
    s = fmaxf(hi, -lo) / 7.f;
  }
  return from_f32<S>(fminf(s, w4_largest<S>()));
}

// One warp per group, a byte (two codes) per lane and turn.
template <class T, class S>
__global__ void __launch_bounds__(256) w4_quantize_kernel(int64_t N, int64_t K, int group, const T *W, int64_t ldw, uint8_t *codes,
                                                          int64_t ldq, S *scales, uint8_t *zeros) {
  const int64_t groups = (K + group - 1) / group;
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t at = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); at < N * groups; at += warps) {
    const int64_t n = at / groups, k0 = (at - n * groups) * group;
    const int len = (int)(K - k0 < group ? K - k0 : group);
    const T *w = W + n * ldw + k0;
    float lo = 0.f, hi = 0.f;
    bool bad = false;
    for (int i = lane; i < len; i += 32) {
      const float v = to_f32(w[i]);
      lo = fminf(lo, v);
      hi = fmaxf(hi, v);
      bad |= !isfinite(v);
    }
    hi = w4_warp_max(hi);
    lo = -w4_warp_max(-lo);
    bad = __any_sync(0xffffffffu, bad);
    const S stored = bad ? from_f32<S>(__int_as_float(0x7fffffff)) : w4_scale<S>(lo, hi, zeros != nullptr);
    const float scale = to_f32(stored);
    const bool flat = !(scale > 0.f);   // 0, or NaN: every code is the zero point
    const float f = w4_prescale(scale), s = scale * f, inv = 1.f / s;
    float zero = 8.f;
    if (zeros && !flat) zero = fminf(fmaxf(w4_nearest(-lo * f, s, inv), 0.f), 15.f);
    const float lowest = zeros ? 0.f : 1.f;
    if (lane == 0) {
      scales[at] = stored;
      if (zeros) zeros[at] = (uint8_t)zero;
    }
    for (int b = lane; 2 * b < len; b += 32) {
      int c[2] = {(int)zero, 2 * b + 1 < len ? (int)zero : 0};
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (!flat && 2 * b + e < len)
          c[e] = (int)fminf(fmaxf(w4_nearest(to_f32(w[2 * b + e]) * f, s, inv) + zero, lowest), 15.f);
      codes[n * ldq + (k0 >> 1) + b] = (uint8_t)(c[0] | (c[1] << 4));
    }
  }
}

__device__ __forceinline__ float w4_zero(const uint8_t *zeros, int64_t at) { return zeros ? (float)(zeros[at] & 15) : 8.f; }

// One thread per element, in the order of the output.
template <class T, class S>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(int64_t N, int64_t K, int group, const uint8_t *codes, int64_t ldq,
                                                            const S *scales, const uint8_t *zeros, T *W, int64_t ldw,
                                                            int transpose) {
  const int64_t groups = (K + group - 1) / group;
  const int64_t step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < N * K; i += step) {
    const int64_t a = transpose ? i / N : i / K, b = i - a * (transpose ? N : K);
    const int64_t n = transpose ? b : a, k = transpose ? a : b;
    const int c = (codes[n * ldq + (k >> 1)] >> (4 * (k & 1))) & 15;
    const int64_t g = n * groups + k / group;
    W[a * ldw + b] = from_f32<T>(((float)c - w4_zero(zeros, g)) * to_f32(scales[g]));
  }
}

// One warp per output column n, up to 8 rows of x at a time.
constexpr int kW4Rows = 8;
template <class T, class S>
__global__ void __launch_bounds__(256) w4_matvec_kernel(int64_t M, int64_t N, int64_t K, int group, float alpha, const T *x, int64_t ldx,
                                                        const uint8_t *codes, int64_t ldq, const S *scales, const uint8_t *zeros,
                                                        float beta, T *y, int64_t ldy) {
  const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= N) return;
  const int lane = threadIdx.x & 31;
  const int64_t m0 = (int64_t)blockIdx.y * kW4Rows, groups = (K + group - 1) / group;
  float acc[kW4Rows] = {};
  if (alpha != 0.f) {
    for (int64_t b = lane; 2 * b < K; b += 32) {
      const uint8_t c = codes[n * ldq + b];
      const int64_t g = n * groups + 2 * b / group;
      const float s = to_f32(scales[g]), z = w4_zero(zeros, g);
      const float w0 = ((float)(c & 15) - z) * s, w1 = ((float)(c >> 4) - z) * s;
#pragma unroll
      for (int m = 0; m < kW4Rows; ++m) {
        if (m0 + m < M) {
          const T *xr = x + (m0 + m) * ldx + 2 * b;
          acc[m] = fmaf(to_f32(xr[0]), w0, acc[m]);
          if (2 * b + 1 < K) acc[m] = fmaf(to_f32(xr[1]), w1, acc[m]);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < kW4Rows; ++m) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
    if (lane == 0 && m0 + m < M) {
      T *to = y + (m0 + m) * ldy + n;
      const float v = alpha * acc[m];
      *to = from_f32<T>(beta != 0.f ? fmaf(beta, to_f32(*to), v) : v);
    }
  }
}

// The checks that the three calls share: sizes, types, the codes' rows.
static int w4_check(const char *who, int64_t N, int64_t K, int group, int type, int scale_type, const void *codes, int64_t ldq,
                    const void *scales) {
  B2_REQUIRE(N >= 0 && K >= 0 && N <= INT32_MAX && K <= INT32_MAX, B2_ERR_INVALID_ARG, "%s: bad shape %lld x %lld", who, (long long)N,
             (long long)K);
  B2_REQUIRE(group == 32 || group == 64 || group == 128 || group == 256, B2_ERR_INVALID_ARG, "%s: group %d is not 32, 64, 128 or 256",
             who, group);
  B2_REQUIRE(type_bytes(type) != 0 && type_bytes(scale_type) != 0, B2_ERR_INVALID_ARG, "%s: unknown type %d or scale type %d", who,
             type, scale_type);
  B2_REQUIRE(ldq >= (K + 1) / 2, B2_ERR_INVALID_ARG, "%s: ldq = %lld bytes is less than a row's %lld", who, (long long)ldq,
             (long long)((K + 1) / 2));
  B2_REQUIRE(N == 0 || K == 0 || (codes != nullptr && scales != nullptr), B2_ERR_INVALID_ARG, "%s: codes or scales is NULL", who);
  B2_REQUIRE(((uintptr_t)scales & (type_bytes(scale_type) - 1)) == 0, B2_ERR_INVALID_ARG, "%s: scales are not aligned to their type", who);
  return B2_OK;
}

template <class F>
static void w4_with_types(int type, int scale_type, F &&f) {
  with_type(type, [&](auto t) { return with_type(scale_type, [&](auto s) { f(t, s); return 0; }); });
}

}  // namespace b2

using namespace b2;

extern "C" {

int b2_w4_quantize(b2_handle h, int64_t N, int64_t K, int group, int type, const void *W, int64_t ldw, uint8_t *codes,
                   int64_t ldq, int scale_type, void *scales, uint8_t *zeros, void *stream) {
  const int st = w4_check("b2_w4_quantize", N, K, group, type, scale_type, codes, ldq, scales);
  if (st != B2_OK) return st;
  const int tb = type_bytes(type);
  B2_REQUIRE(ldw >= K, B2_ERR_INVALID_ARG, "b2_w4_quantize: ldw = %lld is less than K = %lld", (long long)ldw, (long long)K);
  if (N == 0 || K == 0) return B2_OK;
  B2_REQUIRE(W != nullptr && ((uintptr_t)W & (tb - 1)) == 0, B2_ERR_INVALID_ARG, "b2_w4_quantize: W is NULL or not aligned to its type");
  B2_REQUIRE(!matrices_overlap(W, N, K * tb, ldw * tb, codes, N, (K + 1) / 2, ldq), B2_ERR_INVALID_ARG,
             "b2_w4_quantize: codes overlap W");
  B2_CONTEXT(ctx, h, "b2_w4_quantize");
  const int64_t need = (N * ((K + group - 1) / group) + 7) / 8, cap = (int64_t)ctx->sm_count * 16;
  const int grid = (int)(need < cap ? need : cap);
  w4_with_types(type, scale_type, [&](auto t, auto s) {
    using T = decltype(t);
    using S = decltype(s);
    w4_quantize_kernel<T, S><<<grid, 256, 0, (cudaStream_t)stream>>>(N, K, group, (const T *)W, ldw, codes, ldq, (S *)scales, zeros);
  });
  B2_CUDA(cudaGetLastError());
  return B2_OK;
}

int b2_w4_dequantize(b2_handle h, int64_t N, int64_t K, int group, const uint8_t *codes, int64_t ldq, int scale_type,
                     const void *scales, const uint8_t *zeros, int type, void *W, int64_t ldw, int transpose, void *stream) {
  const int st = w4_check("b2_w4_dequantize", N, K, group, type, scale_type, codes, ldq, scales);
  if (st != B2_OK) return st;
  const int tb = type_bytes(type);
  B2_REQUIRE(ldw >= (transpose ? N : K), B2_ERR_INVALID_ARG, "b2_w4_dequantize: ldw = %lld is less than %lld", (long long)ldw,
             (long long)(transpose ? N : K));
  if (N == 0 || K == 0) return B2_OK;
  B2_REQUIRE(W != nullptr && ((uintptr_t)W & (tb - 1)) == 0, B2_ERR_INVALID_ARG, "b2_w4_dequantize: W is NULL or not aligned to its type");
  B2_REQUIRE(!matrices_overlap(W, transpose ? K : N, (transpose ? N : K) * tb, ldw * tb, codes, N, (K + 1) / 2, ldq), B2_ERR_INVALID_ARG,
             "b2_w4_dequantize: W overlaps the codes");
  B2_CONTEXT(ctx, h, "b2_w4_dequantize");
  const int64_t need = (N * K + 255) / 256, cap = (int64_t)ctx->sm_count * 32;
  const int grid = (int)(need < cap ? need : cap);
  w4_with_types(type, scale_type, [&](auto t, auto s) {
    using T = decltype(t);
    using S = decltype(s);
    w4_dequantize_kernel<T, S><<<grid, 256, 0, (cudaStream_t)stream>>>(N, K, group, codes, ldq, (const S *)scales, zeros, (T *)W, ldw,
                                                                      transpose);
  });
  B2_CUDA(cudaGetLastError());
  return B2_OK;
}

int b2_w4_matvec(b2_handle h, int64_t M, int64_t N, int64_t K, int group, float alpha, int type, const void *x, int64_t ldx,
                 const uint8_t *codes, int64_t ldq, int scale_type, const void *scales, const uint8_t *zeros, float beta,
                 void *y, int64_t ldy, void *stream) {
  const int st = w4_check("b2_w4_matvec", N, K, group, type, scale_type, codes, ldq, scales);
  if (st != B2_OK) return st;
  const int tb = type_bytes(type);
  B2_REQUIRE(M >= 0, B2_ERR_INVALID_ARG, "b2_w4_matvec: M = %lld is negative", (long long)M);
  B2_REQUIRE(M <= kW4MaxRows, B2_ERR_UNSUPPORTED,
             "b2_w4_matvec: M = %lld exceeds %d rows: expand the weights with b2_w4_dequantize and use b2_sgemm", (long long)M, kW4MaxRows);
  B2_REQUIRE(ldx >= K && ldy >= N, B2_ERR_INVALID_ARG, "b2_w4_matvec: ldx = %lld is less than K = %lld or ldy = %lld less than N = %lld",
             (long long)ldx, (long long)K, (long long)ldy, (long long)N);
  if (M == 0 || N == 0) return B2_OK;
  B2_REQUIRE(y != nullptr && (K == 0 || x != nullptr), B2_ERR_INVALID_ARG, "b2_w4_matvec: x or y is NULL");
  B2_REQUIRE((((uintptr_t)x | (uintptr_t)y) & (tb - 1)) == 0, B2_ERR_INVALID_ARG, "b2_w4_matvec: x or y is not aligned to its type");
  B2_REQUIRE(!matrices_overlap(x, M, K * tb, ldx * tb, y, M, N * tb, ldy * tb), B2_ERR_INVALID_ARG, "b2_w4_matvec: y overlaps x");
  B2_CONTEXT(ctx, h, "b2_w4_matvec");
  (void)ctx;
  const dim3 grid((unsigned)((N + 7) / 8), (unsigned)((M + kW4Rows - 1) / kW4Rows));
  w4_with_types(type, scale_type, [&](auto t, auto s) {
    using T = decltype(t);
    using S = decltype(s);
    w4_matvec_kernel<T, S><<<grid, 256, 0, (cudaStream_t)stream>>>(M, N, K, group, alpha, (const T *)x, ldx, codes, ldq,
                                                                  (const S *)scales, zeros, beta, (T *)y, ldy);
  });
  B2_CUDA(cudaGetLastError());
  return B2_OK;
}

}  // extern "C"
