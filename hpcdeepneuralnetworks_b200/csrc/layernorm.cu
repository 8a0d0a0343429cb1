// Layer norm, forward and backward: both are bound by memory (the forward pass reads x and writes y, the backward pass reads x
// and dy and writes dx), so every row is read once and kept in registers while its sums are formed.
//
// A row belongs to a warp (up to 1024 columns; 512 backward) or to a block; a thread holds up to kHeld elements of it, V neighbouring ones to
// an access.  V is the widest access that every row pointer, the pitches and cols allow (16 bytes, 4 bytes, one element), so that
// no row needs a head or a tail.  Longer rows are read again instead of held.
#include <math.h>

#include <initializer_list>
#include <type_traits>

#include "types.cuh"

namespace b2 {

template <int BYTES>
struct LnRaw;
template <>
struct LnRaw<16> {
  using type = uint4;
};
template <>
struct LnRaw<8> {
  using type = uint2;
};
template <>
struct LnRaw<4> {
  using type = uint32_t;
};
template <>
struct LnRaw<2> {
  using type = uint16_t;
};
// V elements of type T as one access, and their values.
template <class T, int V>
struct LnPack {
  using raw_t = typename LnRaw<V * sizeof(T)>::type;
  union {
    raw_t raw;
    T e[V];
  };
  __device__ __forceinline__ LnPack() {}
  __device__ __forceinline__ void load_stream(const T *p) { raw = __ldcs(reinterpret_cast<const raw_t *>(p)); }   // read once
  __device__ __forceinline__ void load(const T *p) { raw = *reinterpret_cast<const raw_t *>(p); }
  __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<raw_t *>(p) = raw; }
  __device__ __forceinline__ float get(int i) const { return to_f32(e[i]); }
  __device__ __forceinline__ void set(int i, float v) { e[i] = from_f32<T>(v); }
};
// V values of a parameter vector (16-byte accesses where V elements are that long or longer), or a constant without one.
template <class P, int V>
__device__ __forceinline__ void ln_params(float (&v)[V], const P *p, int64_t at, float without) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = without;
    return;
  }
  constexpr int W = V * (int)sizeof(P) > 16 ? 16 / (int)sizeof(P) : V;
#pragma unroll
  for (int i = 0; i < V; i += W) {
    LnPack<P, W> q;
    q.load(p + at + i);
#pragma unroll
    for (int k = 0; k < W; ++k) v[i + k] = q.get(k);
  }
}

// Sums over the threads that share a row, the same bits in each of them: shuffles within a warp, then, where a block shares
// it, the warps' sums in order.  `scratch` alternates between two arrays, so that one barrier per sum is enough.
template <bool WARP>
__device__ __forceinline__ float2 ln_sum2(float2 v, float2 *scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (WARP) return v;
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = (int)blockDim.x >> 5, lane = threadIdx.x & 31;
  v = lane < warps ? scratch[lane] : make_float2(0.f, 0.f);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return v;
}

// y = (x - mean) * rstd * gamma + beta.  The variance is that of the distances from a first mean, and what the first mean was
// off by (the mean of those distances) is taken out of both: a large mean costs no digits.
template <class T, class P, int V, int N, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) layernorm_kernel(int64_t rows, int cols, float eps, const T *x, int64_t ldx,
                                                                      const P *gamma, const P *beta, T *y, int64_t ldy,
                                                                      float *mean, float *rstd) {
  __shared__ float2 scratch[2][32];
  const int share = WARP ? 32 : (int)blockDim.x, tid = WARP ? (int)threadIdx.x & 31 : (int)threadIdx.x;
  const int units = cols / V;
  const float n = (float)cols;
  const int64_t step = WARP ? (int64_t)gridDim.x * 8 : (int64_t)gridDim.x;
  for (int64_t row = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : (int64_t)blockIdx.x; row < rows; row += step) {
    LnPack<T, V> v[N];
    const T *xr = x + row * ldx;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (tid + i * share < units) v[i].load_stream(xr + (int64_t)(tid + i * share) * V);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (tid + i * share < units) {
#pragma unroll
        for (int k = 0; k < V; ++k) s += v[i].get(k);
      }
    float m = ln_sum2<WARP>(make_float2(s, 0.f), scratch[0]).x / n;
    float2 d = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (tid + i * share < units) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float e = v[i].get(k) - m;
          d.x += e;
          d.y = fmaf(e, e, d.y);
        }
      }
    d = ln_sum2<WARP>(d, scratch[1]);
    const float off = d.x / n;
    m += off;
    const float r = 1.f / sqrtf(fmaf(-off, off, d.y / n) + eps);
    if (tid == 0) {
      if (mean) mean[row] = m;
      if (rstd) rstd[row] = r;
    }
    T *yr = y + row * ldy;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (tid + i * share < units) {
        float g[V], b[V];
        ln_params<P, V>(g, gamma, (int64_t)(tid + i * share) * V, 1.f);
        ln_params<P, V>(b, beta, (int64_t)(tid + i * share) * V, 0.f);
#pragma unroll
        for (int k = 0; k < V; ++k) v[i].set(k, fmaf((v[i].get(k) - m) * r, g[k], b[k]));
        v[i].store(yr + (int64_t)(tid + i * share) * V);
      }
  }
}

// The same for rows that are too long to hold: one block per row, read three times (from L2 after the first).
template <class T, class P, int V>
__global__ void __launch_bounds__(1024) layernorm_long_kernel(int64_t rows, int cols, float eps, const T *x, int64_t ldx, const P *gamma,
                                                              const P *beta, T *y, int64_t ldy, float *mean, float *rstd) {
  __shared__ float2 scratch[2][32];
  const float n = (float)cols;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * ldx;
    LnPack<T, V> v;
    float s = 0.f;
    for (int64_t i = (int64_t)threadIdx.x * V; i < cols; i += 1024 * V) {
      v.load(xr + i);
#pragma unroll
      for (int k = 0; k < V; ++k) s += v.get(k);
    }
    float m = ln_sum2<false>(make_float2(s, 0.f), scratch[0]).x / n;
    float2 d = make_float2(0.f, 0.f);
    for (int64_t i = (int64_t)threadIdx.x * V; i < cols; i += 1024 * V) {
      v.load(xr + i);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float e = v.get(k) - m;
        d.x += e;
        d.y = fmaf(e, e, d.y);
      }
    }
    d = ln_sum2<false>(d, scratch[1]);
    const float off = d.x / n;
    m += off;
    const float r = 1.f / sqrtf(fmaf(-off, off, d.y / n) + eps);
    if (threadIdx.x == 0) {
      if (mean) mean[row] = m;
      if (rstd) rstd[row] = r;
    }
    for (int64_t i = (int64_t)threadIdx.x * V; i < cols; i += 1024 * V) {
      float g[V], b[V];
      v.load(xr + i);
      ln_params<P, V>(g, gamma, i, 1.f);
      ln_params<P, V>(b, beta, i, 0.f);
#pragma unroll
      for (int k = 0; k < V; ++k) v.set(k, fmaf((v.get(k) - m) * r, g[k], b[k]));
      v.store(y + row * ldy + i);
    }
  }
}

// Backward: a block (or each warp of one) walks over rows of its own with the next row's loads under way, and keeps the sums
// dy * xhat and dy of its columns in registers over all of them; they end as one line of `partial` per block.
//   xhat = (x - mean) * rstd,  u = dy * gamma,  dx = rstd * (u - sum(u) / n - xhat * sum(u * xhat) / n)
// dx may be dy: a thread writes only what it has read.
template <class T, class P, int V, int N, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) layernorm_backward_kernel(int64_t rows, int cols, const T *dy, int64_t lddy, const T *x,
                                                                               int64_t ldx, const P *gamma, const float *mean,
                                                                               const float *rstd, T *dx, int64_t lddx,
                                                                               float *partial) {
  __shared__ float2 scratch[2][32];
  extern __shared__ float joined[];                // WARP: [2][cols], the warps' sums
  pdl_launch_dependents();
  const int share = WARP ? 32 : (int)blockDim.x, tid = WARP ? (int)threadIdx.x & 31 : (int)threadIdx.x;
  const int units = cols / V;
  const float inv = 1.f / (float)cols;
  const int64_t step = WARP ? (int64_t)gridDim.x * 8 : (int64_t)gridDim.x;
  float dg[N * V] = {}, db[N * V] = {};
  LnPack<T, V> xn[N], gn[N];
  float mn = 0.f, rn = 0.f;
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (tid + i * share < units) {
        xn[i].load_stream(x + row * ldx + (int64_t)(tid + i * share) * V);
        gn[i].load_stream(dy + row * lddy + (int64_t)(tid + i * share) * V);
      }
    mn = mean[row];
    rn = rstd[row];
  };
  int64_t row = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  if (row < rows) fetch(row);
  for (int turn = 0; row < rows; row += step, turn ^= 1) {
    LnPack<T, V> xc[N], gc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) xc[i] = xn[i], gc[i] = gn[i];
    const float m = mn, r = rn;
    if (row + step < rows) fetch(row + step);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (tid + i * share < units) {
        float g[V];
        ln_params<P, V>(g, gamma, (int64_t)(tid + i * share) * V, 1.f);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float d = gc[i].get(k), h = (xc[i].get(k) - m) * r, u = d * g[k];
          s.x += u;
          s.y = fmaf(u, h, s.y);
          dg[i * V + k] = fmaf(d, h, dg[i * V + k]);
          db[i * V + k] += d;
        }
      }
    if (dx) {
      s = ln_sum2<WARP>(s, scratch[turn]);
      const float a = s.x * inv, b = s.y * inv;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (tid + i * share < units) {
          float g[V];
          ln_params<P, V>(g, gamma, (int64_t)(tid + i * share) * V, 1.f);
          LnPack<T, V> out;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const float h = (xc[i].get(k) - m) * r, u = gc[i].get(k) * g[k];
            out.set(k, r * (u - fmaf(h, b, a)));
          }
          out.store(dx + row * lddx + (int64_t)(tid + i * share) * V);
        }
    }
  }
  if (!partial) return;
  float *line = partial + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (!WARP) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (tid + i * share < units) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          line[(tid + i * share) * V + k] = dg[i * V + k];
          line[cols + (tid + i * share) * V + k] = db[i * V + k];
        }
      }
  } else {
    for (int w = 0; w < 8; ++w) {                    // warp by warp, in order
      if ((int)(threadIdx.x >> 5) == w) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (tid + i * share < units) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
              const int c = (tid + i * share) * V + k;
              joined[c] = w ? joined[c] + dg[i * V + k] : dg[i * V + k];
              joined[cols + c] = w ? joined[cols + c] + db[i * V + k] : db[i * V + k];
            }
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * cols; c += 256) line[c] = joined[c];
  }
}

// Rows too long for that: their sums of u and u * xhat first (one block per row), then everything else by tiles of columns,
// each thread walking down V columns.
template <class T, class P, int V>
__global__ void __launch_bounds__(1024) layernorm_row_sums_kernel(int64_t rows, int cols, const T *dy, int64_t lddy, const T *x, int64_t ldx,
                                                                  const P *gamma, const float *mean, const float *rstd, float2 *out) {
  __shared__ float2 scratch[2][32];
  int turn = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    const float m = mean[row], r = rstd[row];
    float2 s = make_float2(0.f, 0.f);
    for (int64_t i = (int64_t)threadIdx.x * V; i < cols; i += 1024 * V) {
      LnPack<T, V> xv, gv;
      float g[V];
      xv.load(x + row * ldx + i);
      gv.load(dy + row * lddy + i);
      ln_params<P, V>(g, gamma, i, 1.f);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float u = gv.get(k) * g[k];
        s.x += u;
        s.y = fmaf(u, (xv.get(k) - m) * r, s.y);
      }
    }
    s = ln_sum2<false>(s, scratch[turn]);
    if (threadIdx.x == 0) out[row] = make_float2(s.x / (float)cols, s.y / (float)cols);
  }
}
template <class T, class P, int V>
__global__ void __launch_bounds__(128) layernorm_columns_kernel(int64_t rows, int cols, const T *dy, int64_t lddy, const T *x, int64_t ldx,
                                                                const P *gamma, const float *mean, const float *rstd,
                                                                const float2 *row_sums, T *dx, int64_t lddx, float *partial) {
  const int64_t c = ((int64_t)blockIdx.x * 128 + threadIdx.x) * V;
  if (c >= cols) return;
  float g[V], dg[V] = {}, db[V] = {};
  ln_params<P, V>(g, gamma, c, 1.f);
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    LnPack<T, V> xv, gv;
    xv.load_stream(x + row * ldx + c);
    gv.load_stream(dy + row * lddy + c);
    const float m = mean[row], r = rstd[row];
    const float2 s = dx ? row_sums[row] : make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float d = gv.get(k), h = (xv.get(k) - m) * r;
      dg[k] = fmaf(d, h, dg[k]);
      db[k] += d;
      xv.set(k, r * (d * g[k] - fmaf(h, s.y, s.x)));
    }
    if (dx) xv.store(dx + row * lddx + c);
  }
  if (!partial) return;
  float *line = partial + (int64_t)blockIdx.y * 2 * cols + c;
#pragma unroll
  for (int k = 0; k < V; ++k) line[k] = dg[k], line[cols + k] = db[k];
}

// dgamma and dbeta from the lines of partial sums: 32 columns per block, the lines shared out over 32 warps and joined in order.
template <class P>
__global__ void __launch_bounds__(1024) layernorm_reduce_kernel(int parts, int cols, const float *partial, P *dgamma, P *dbeta) {
  __shared__ float part[2][32][33];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float g = 0.f, b = 0.f;
  if (c < cols) {
    for (int p = warp; p < parts; p += 32) {
      g += partial[(int64_t)p * 2 * cols + c];
      b += partial[((int64_t)p * 2 + 1) * cols + c];
    }
  }
  part[0][warp][lane] = g;
  part[1][warp][lane] = b;
  __syncthreads();
  if (warp < 2 && c < cols) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) s += part[warp][w][lane];
    if (warp == 0 && dgamma) dgamma[c] = from_f32<P>(s);
    if (warp == 1 && dbeta) dbeta[c] = from_f32<P>(s);
  }
}

// ---- which form -------------------------------------------------------------------------------------
constexpr int kLnWarpCols = 1024;       // up to here a warp takes a row; backward, where a thread holds sums too, up to
constexpr int kLnWarpColsBackward = 512;
constexpr int kLnParts = 296;           // most lines of partial sums: two blocks on each of 148 SMs
// Elements of a row that a thread holds, by the width of its accesses: enough that 1024 threads take 32768 columns forward
// and 8192 backward (there the sums over rows are held too).
constexpr int ln_held(int v) { return v == 1 ? 16 : 32; }
constexpr int kLnHeldBackward = 8;
static int ln_backward_longest() { return 1024 * kLnHeldBackward; }

static int64_t ln_parts(int64_t rows, int64_t cols) {
  const int64_t blocks = cols <= kLnWarpColsBackward ? (rows + 7) / 8 : rows;
  return blocks < kLnParts ? blocks : kLnParts;
}

// Whether every address and pitch (in bytes) is a multiple of `bytes`; NULL is.
static bool ln_multiple(int64_t bytes, std::initializer_list<const void *> pointers, std::initializer_list<int64_t> pitches) {
  for (const void *p : pointers)
    if ((uintptr_t)p % bytes) return false;
  for (int64_t p : pitches)
    if (p % bytes) return false;
  return true;
}
// The widest access, in elements, for rows of `cols` elements of `tb` bytes at these places; parameters of pb bytes are read
// as many at a time (16 bytes at most).
static int ln_width(int64_t cols, int tb, int pb, std::initializer_list<const void *> rows, std::initializer_list<int64_t> pitches,
                    std::initializer_list<const void *> params) {
  for (int bytes : {16, 4}) {
    const int v = bytes / tb;
    if (v > 1 && cols % v == 0 && ln_multiple(bytes, rows, pitches) && ln_multiple(v * pb > 16 ? 16 : v * pb, params, {})) return v;
  }
  return 1;
}
template <class T, class F>
static void ln_with_width(int v, F &&f) {
  if (v == 16 / (int)sizeof(T)) f(std::integral_constant<int, 16 / (int)sizeof(T)>());
  else if (sizeof(T) == 2 && v == 2) f(std::integral_constant<int, 4 / (int)sizeof(T)>());
  else f(std::integral_constant<int, 1>());
}

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
  const int width = ln_width(cols, tb, pb, {x, y}, {ldx * tb, ldy * tb}, {gamma, beta});
  cudaStream_t s = (cudaStream_t)stream;
  auto launch = [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    ln_with_width<T>(width, [&](auto w) {
      constexpr int V = decltype(w)::value, kMost = ln_held(V) / V, kFew = kMost >= 4 ? kMost / 4 : 1;
      const int64_t units = cols / V;
      auto run = [&](auto kernel, int64_t blocks, int threads) {
        const int64_t cap = (int64_t)1 << 30;
        kernel<<<(unsigned)(blocks < cap ? blocks : cap), threads, 0, s>>>(rows, (int)cols, eps, (const T *)x, ldx, (const P *)gamma,
                                                                          (const P *)beta, (T *)y, ldy, mean, rstd);
      };
      // Few rows: as many threads to each as its length allows; else each thread holds as much as it can, and more rows share an SM.
      const bool few = rows <= 2 * ctx->sm_count;
      if (units <= 32 * kMost && cols <= kLnWarpCols && !(few && units > 32 * kFew)) {
        if (units <= 32 * kFew) run(layernorm_kernel<T, P, V, kFew, true>, (rows + 7) / 8, 256);
        else run(layernorm_kernel<T, P, V, kMost, true>, (rows + 7) / 8, 256);
      } else if (units <= 1024 * kFew && (few || units <= 128 * kFew)) {
        run(layernorm_kernel<T, P, V, kFew, false>, rows, (int)((units + 32 * kFew - 1) / (32 * kFew)) * 32);
      } else if (units <= 1024 * kMost) {
        run(layernorm_kernel<T, P, V, kMost, false>, rows, (int)((units + 32 * kMost - 1) / (32 * kMost)) * 32);
      } else {
        run(layernorm_long_kernel<T, P, V>, rows, 1024);
      }
    });
    return 0;
  };
  with_type(type, [&](auto t) { return param_type == type ? launch(t, t) : launch(t, float()); });
  B2_CUDA(cudaGetLastError());
  return B2_OK;
}

size_t b2_layernorm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  const size_t sums = (size_t)ln_parts(rows, cols) * 2 * (size_t)cols * sizeof(float);
  return (sums + 15) / 16 * 16 + (cols > ln_backward_longest() ? (size_t)rows * sizeof(float2) : 0);
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
  const bool is_long = cols > ln_backward_longest();
  const size_t need = sums || is_long ? b2_layernorm_backward_workspace_bytes(rows, cols) : 0;
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
  (void)ctx;
  const int parts = (int)ln_parts(rows, cols);
  const int width = ln_width(cols, tb, pb, {dy, x, dx}, {lddy * tb, ldx * tb, dx ? lddx * tb : 0}, {gamma});
  float *partial = sums ? (float *)workspace : nullptr;
  float2 *row_sums = is_long ? (float2 *)((char *)workspace + (need - (size_t)rows * sizeof(float2))) : nullptr;
  auto launch = [&](auto t, auto p) {
    using T = decltype(t);
    using P = decltype(p);
    ln_with_width<T>(width, [&](auto w) {
      constexpr int V = decltype(w)::value, kCta = V >= kLnHeldBackward ? 1 : kLnHeldBackward / V, kWarp = kLnWarpColsBackward / 32 / V,
                    kFew = kWarp >= 4 ? kWarp / 4 : 1;
      const int64_t units = cols / V;
      auto run = [&](auto kernel, int threads, size_t smem) {
        kernel<<<parts, threads, smem, s>>>(rows, (int)cols, (const T *)dy, lddy, (const T *)x, ldx, (const P *)gamma, mean, rstd, (T *)dx,
                                            lddx, partial);
      };
      if (cols <= kLnWarpColsBackward) {
        const size_t smem = (size_t)2 * cols * sizeof(float);
        if (units <= 32 * kFew) run(layernorm_backward_kernel<T, P, V, kFew, true>, 256, smem);
        else run(layernorm_backward_kernel<T, P, V, kWarp, true>, 256, smem);
      } else if (!is_long) {
        run(layernorm_backward_kernel<T, P, V, kCta, false>, (int)((units + 32 * kCta - 1) / (32 * kCta)) * 32, 0);
      } else {
        if (dx) {
          const int64_t blocks = rows < 1 << 30 ? rows : 1 << 30;
          layernorm_row_sums_kernel<T, P, V><<<(unsigned)blocks, 1024, 0, s>>>(rows, (int)cols, (const T *)dy, lddy, (const T *)x, ldx,
                                                                            (const P *)gamma, mean, rstd, row_sums);
        }
        layernorm_columns_kernel<T, P, V><<<dim3((unsigned)((units + 127) / 128), (unsigned)parts), 128, 0, s>>>(
            rows, (int)cols, (const T *)dy, lddy, (const T *)x, ldx, (const P *)gamma, mean, rstd, row_sums, (T *)dx, lddx, partial);
      }
    });
    if (sums) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)((cols + 31) / 32));
      cfg.blockDim = dim3(1024);
      cfg.stream = s;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // its blocks may start, and wait, before the sums are done
      attr[0].val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      return (int)cudaLaunchKernelEx(&cfg, layernorm_reduce_kernel<P>, parts, (int)cols, (const float *)partial, (P *)dgamma, (P *)dbeta);
    }
    return 0;
  };
  with_type(type, [&](auto t) { return param_type == type ? launch(t, t) : launch(t, float()); });
  B2_CUDA(cudaGetLastError());
  return B2_OK;
}

}  // extern "C"
