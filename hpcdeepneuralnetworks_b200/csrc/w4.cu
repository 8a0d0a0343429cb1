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

// ---- matrix-vector product -----------------------------------------------------------------------
// y = alpha * x * W^T + beta * y.  The codes are read once and decide the time, so everything else is arranged around
// streaming them; the arithmetic runs on mma.sync m16n8k16 (16 weight rows x 8 columns of x), which has room for 8 columns at
// the price of one.  (A tcgen05 tile would want 128 rows and operands rewritten to shared memory in 16 bits first; at
// 0.5 byte per weight the kernel is bound by reading and unpacking, not by the tensor cores.)
//
//   W[n][k] = (c - z) * s, so per group  sum_k W x = s * sum_k (c - z) x:
// the integers (c - z) are exact in both 16-bit types, their products with x are exact in the FP32 accumulator, and the
// scale, in FP32, multiplies a group's sum.  Unpacking: a code or-ed into the low mantissa bits of 8.0 (bf16) or 64.0 (f16)
// reads 8 + c/16 or 64 + c/16; subtracting the same number with z leaves (c - z)/16 exactly.  (The 1/16 keeps sums of x near
// the end of its range finite; it is undone on the final sum.)  Two codes four apart in a word come out of one mask, so the
// elements of x are stored paired (0,4) (1,5) (2,6) (3,7).
// FP32 x is cut into three bf16 terms of 8 bits each (by truncation: exact, and no overflow) that take a column each.
//
// A block covers kRows x kChunkK codes at a time, double buffered: codes by cp.async, x and scales through registers.  A warp
// multiplies 32 rows by 128 of k, 8 warps as WN (rows) x WK (k).  The k range is also cut over the CTAs of a cluster, whose
// sums meet in distributed shared memory in the order of the ranks: no atomics, no workspace.
constexpr int kMvThreads = 256;

template <class T>
struct MvType;   // the 16-bit type of the tensor-core operands, and how many columns a row of x takes
template <>
struct MvType<float> {
  using half_t = __nv_bfloat16;
  static constexpr int kParts = 3;
};
template <>
struct MvType<__nv_bfloat16> {
  using half_t = __nv_bfloat16;
  static constexpr int kParts = 1;
};
template <>
struct MvType<__half> {
  using half_t = __half;
  static constexpr int kParts = 1;
};

template <class T, int NB, int WN_>
struct MvTile {
  static constexpr int WN = WN_, WK = 8 / WN_;
  static constexpr int kRows = 32 * WN, kChunkK = 128 * WK;                    // 64 x 512 or 128 x 256
  static constexpr int kParts = MvType<T>::kParts;
  static constexpr int kM = 8 * NB / kParts;                                   // rows of x per block
  static constexpr int kCodeBytes = kRows * kChunkK / 2;                       // 16 KB
  static constexpr int kXBytes = kChunkK * 8 * NB * 2;
  static constexpr int kScaleBytes = kRows * (kChunkK / 32) * 4;               // room for groups of 32
  static constexpr int kZeroBytes = kRows * (kChunkK / 32);
  static constexpr int kBuffer = kCodeBytes + kXBytes + kScaleBytes + kZeroBytes;
  static constexpr int kSmem = 2 * kBuffer;
  static constexpr int kUnits = (kM * kChunkK / 8 + kMvThreads - 1) / kMvThreads;   // 8 elements of x per thread and turn
  static_assert(WK * kRows * 8 * NB * 4 + kM * kRows * 4 <= kSmem, "the sums reuse the buffers");
};

struct MvArgs {
  int64_t N, K, ldx, ldq, ldy, groups;
  int M, group_shift, chunks_per_cta, m_chunks, scale_type;
  float alpha, beta;
  const void *x;
  const uint8_t *codes, *zeros;
  const void *scales;
  void *y;
};

__device__ __forceinline__ float mv_scale(const void *scales, int type, int64_t at) {
  if (type == B2_F32) return ((const float *)scales)[at];
  if (type == B2_BF16) return to_f32(((const __nv_bfloat16 *)scales)[at]);
  return to_f32(((const __half *)scales)[at]);
}

__device__ __forceinline__ void cp_async_16(void *smem, const void *global, int bytes) {   // the rest of the 16 bytes is zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(global), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Bytes [at, at + 16) of a row of `width` bytes that may start anywhere, zero behind its end, without touching a byte outside.
__device__ __forceinline__ uint4 mv_load_any(const uint8_t *row, int64_t at, int64_t width) {
  union {
    uint32_t w[4];
    uint4 v;
  } out;
  const uint8_t *p = row + at;
  const int skew = (int)((uintptr_t)p & 3);
  if (at >= 4 && at + 20 <= width) {
    const uint32_t *q = reinterpret_cast<const uint32_t *>(p - skew);
    uint32_t prev = q[0];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t next = q[i + 1];
      out.w[i] = __funnelshift_r(prev, next, 8 * skew);
      prev = next;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out.w[i] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (at + 4 * i + j < width) out.w[i] |= (uint32_t)p[4 * i + j] << (8 * j);
    }
  }
  return out.v;
}

// 16 bits of x in pairs (0,4) (1,5) (2,6) (3,7) from 8 in order.
__device__ __forceinline__ uint4 mv_pair(const uint32_t (&h)[4]) {
  return make_uint4(__byte_perm(h[0], h[2], 0x5410), __byte_perm(h[0], h[2], 0x7632), __byte_perm(h[1], h[3], 0x5410),
                    __byte_perm(h[1], h[3], 0x7632));
}

// 8 elements of one row of x (k, k + 8) as they lie, zero behind K.
template <class T>
struct MvUnit {
  uint32_t w[sizeof(T) * 2];
  __device__ __forceinline__ void load(const T *row, int64_t k, int64_t K, bool vec) {
    if (vec && k + 8 <= K) {
      const uint4 *q = reinterpret_cast<const uint4 *>(row + k);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        const uint4 v = __ldg(q + i);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = k + i < K ? __float_as_uint(row[k + i]) : 0u;
    } else {
      const uint16_t *q = reinterpret_cast<const uint16_t *>(row);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = k + 2 * i < K ? q[k + 2 * i] : 0u;
        if (k + 2 * i + 1 < K) w[i] |= (uint32_t)q[k + 2 * i + 1] << 16;
      }
    }
  }
  // part p (0..2) of FP32: 8 bits of the mantissa each, what is left handed to the next call
  __device__ __forceinline__ uint4 part(int p) {
    uint32_t h[4];
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t lo = w[2 * i] & 0xffff0000u, hi = w[2 * i + 1] & 0xffff0000u;
        const float f0 = __uint_as_float(w[2 * i]), f1 = __uint_as_float(w[2 * i + 1]);
        if (p == 0) {
          if (f0 != f0) lo = 0x7fff0000u;      // a NaN whose upper half alone would read as infinity
          if (f1 != f1) hi = 0x7fff0000u;
        }
        h[i] = (lo >> 16) | hi;
        // an infinity or NaN is whole in the first part
        w[2 * i] = isfinite(f0) ? __float_as_uint(f0 - __uint_as_float(lo)) : 0u;
        w[2 * i + 1] = isfinite(f1) ? __float_as_uint(f1 - __uint_as_float(hi)) : 0u;
      }
    }
    return mv_pair(h);
  }
};

__device__ __forceinline__ void mv_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mv_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The zero point in the form that unpacking subtracts: 8 + z/16 (bf16), 64 + z/16 (f16), in both halves.
__device__ __forceinline__ uint32_t mv_zero(uint32_t z, __nv_bfloat16) { return 0x41004100u | z * 0x00010001u; }
__device__ __forceinline__ uint32_t mv_zero(uint32_t z, __half) { return 0x54005400u | z * 0x00010001u; }

// (c - z) / 16 of codes j and j + 4 of a word, j = 0..3.
__device__ __forceinline__ uint32_t mv_unpack(uint32_t w, int j, uint32_t zero, __nv_bfloat16) {
  const uint32_t v = ((w >> (4 * j)) & 0x000f000fu) | 0x41004100u;
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), *reinterpret_cast<const __nv_bfloat162 *>(&zero));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t mv_unpack(uint32_t w, int j, uint32_t zero, __half) {
  const uint32_t v = ((w >> (4 * j)) & 0x000f000fu) | 0x54005400u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&v), *reinterpret_cast<const __half2 *>(&zero));
  return *reinterpret_cast<const uint32_t *>(&r);
}

__device__ __forceinline__ float ld_shared_cluster_f32(uint32_t cluster_addr) { return __uint_as_float(ld_shared_cluster_u32(cluster_addr)); }

// ALIGNED: rows of codes start on 16-byte boundaries.  XVEC: so do the 8-element units of x.
template <class T, int NB, int WN, bool ALIGNED>
__global__ void __launch_bounds__(kMvThreads) w4_matvec_kernel(const MvArgs a, int xvec) {
  using Tile = MvTile<T, NB, WN>;
  using H = typename MvType<T>::half_t;
  constexpr int kChunkK = Tile::kChunkK, kRows = Tile::kRows, kRowBytes = kChunkK / 2, kRowUnits = kRowBytes / 16;
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int wn = warp % WN, wk = warp / WN;
  const int rank = (int)cluster_ctarank(), ctas = (int)(gridDim.y);
  // blockIdx.y is the rank within the cluster; blockIdx.x runs over the row blocks, the m chunks of one row block together
  const int64_t block = blockIdx.x / a.m_chunks;
  const int m0 = (int)(blockIdx.x % a.m_chunks) * Tile::kM;
  const int mm = a.M - m0 < Tile::kM ? a.M - m0 : Tile::kM;
  const int64_t n0 = block * kRows, width = (a.K + 1) >> 1;
  const int64_t first = (int64_t)rank * a.chunks_per_cta;
  int64_t chunks = (a.K + kChunkK - 1) / kChunkK - first;
  if (chunks > a.chunks_per_cta) chunks = a.chunks_per_cta;
  const int chunk_groups = kChunkK >> a.group_shift;
  const T *x = (const T *)a.x;

  auto codes_of = [&](int buf) { return smem + buf * Tile::kBuffer; };
  auto x_of = [&](int buf) { return smem + buf * Tile::kBuffer + Tile::kCodeBytes; };
  auto scales_of = [&](int buf) { return reinterpret_cast<float *>(smem + buf * Tile::kBuffer + Tile::kCodeBytes + Tile::kXBytes); };
  auto zeros_of = [&](int buf) { return smem + buf * Tile::kBuffer + Tile::kCodeBytes + Tile::kXBytes + Tile::kScaleBytes; };

  // codes of a chunk: 16-byte units, unit u of row r at place u ^ (r & 7), so that 8 rows' words of one unit lie in 32 banks
  auto fetch_codes = [&](int buf, int64_t chunk) {
    unsigned char *to = codes_of(buf);
#pragma unroll
    for (int i = 0; i < Tile::kCodeBytes / 16 / kMvThreads; ++i) {
      const int u = tid + i * kMvThreads, r = u / kRowUnits, c = u % kRowUnits;
      unsigned char *dst = to + r * kRowBytes + ((c ^ (r & 7)) << 4);
      const int64_t at = chunk * kRowBytes + 16 * c;
      const int64_t n = n0 + r;
      const int64_t left = n < a.N ? width - at : 0;
      if (ALIGNED) {
        const int bytes = left >= 16 ? 16 : left > 0 ? (int)left : 0;
        cp_async_16(dst, a.codes + (bytes ? n * a.ldq + at : 0), bytes);
      } else {
        *reinterpret_cast<uint4 *>(dst) = left > 0 ? mv_load_any(a.codes + n * a.ldq, at, width) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  MvUnit<T> held[Tile::kUnits];
  auto fetch_x = [&](int64_t chunk) {
#pragma unroll
    for (int i = 0; i < Tile::kUnits; ++i) {
      const int u = tid + i * kMvThreads, m = u / (kChunkK / 8), c = u % (kChunkK / 8);
      if (m < mm) held[i].load(x + (int64_t)(m0 + m) * a.ldx, chunk * kChunkK + 8 * c, a.K, xvec != 0);
    }
  };
  // unit (block b of 32, word t) of column n at ((b * NB * 8) + n) * 4 + t: a warp's fragment load is 512 bytes in a row
  auto put_x = [&](int buf) {
    uint4 *to = reinterpret_cast<uint4 *>(x_of(buf));
#pragma unroll
    for (int i = 0; i < Tile::kUnits; ++i) {
      const int u = tid + i * kMvThreads, m = u / (kChunkK / 8), c = u % (kChunkK / 8);
      if (m < mm) {
#pragma unroll
        for (int p = 0; p < Tile::kParts; ++p) to[(((c >> 2) * NB * 8) + m * Tile::kParts + p) * 4 + (c & 3)] = held[i].part(p);
      }
    }
  };
  auto fetch_scales = [&](int buf, int64_t chunk) {
    float *sc = scales_of(buf);
    unsigned char *ze = zeros_of(buf);
    for (int i = tid; i < kRows * chunk_groups; i += kMvThreads) {
      const int r = i / chunk_groups, q = i % chunk_groups;
      const int64_t n = n0 + r, at = chunk * chunk_groups + q;
      const bool in = n < a.N && at < a.groups;
      sc[r * (kChunkK / 32) + q] = in ? mv_scale(a.scales, a.scale_type, n * a.groups + at) : 0.f;
      ze[r * (kChunkK / 32) + q] = in && a.zeros ? a.zeros[n * a.groups + at] & 15 : 8;
    }
  };

  float total[2][NB][4] = {};
  const int cols = mm * Tile::kParts;   // columns of x in use
  if (chunks > 0) {
    fetch_codes(0, first);
    fetch_x(first);
    fetch_scales(0, first);
    put_x(0);
    cp_async_wait_all();
    __syncthreads();
    for (int64_t c = 0; c < chunks; ++c) {
      const int buf = (int)(c & 1);
      const bool more = c + 1 < chunks;
      if (more) {
        fetch_codes(buf ^ 1, first + c + 1);
        fetch_x(first + c + 1);
      }
      const unsigned char *codes = codes_of(buf) + (wn * 32) * kRowBytes;
      const uint4 *xs = reinterpret_cast<const uint4 *>(x_of(buf));
      const float *sc = scales_of(buf) + wn * 32 * (kChunkK / 32);
      const unsigned char *ze = zeros_of(buf) + wn * 32 * (kChunkK / 32);
      float acc[2][NB][4] = {};
#pragma unroll
      for (int b4 = 0; b4 < 4; ++b4) {
        const int b = wk * 4 + b4;                                // block of 32 k within the chunk
        const int grp = (b << 5) >> a.group_shift;
        uint4 xf[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) xf[nb] = nb * 8 + g < cols ? xs[((b * NB + nb) * 8 + g) * 4 + t] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
          const int r0 = rt * 16 + g;                             // and r0 + 8: the same place in the swizzle
          const int place = ((b ^ (g & 7)) << 4) + 4 * t;
          const uint32_t w0 = *reinterpret_cast<const uint32_t *>(codes + r0 * kRowBytes + place);
          const uint32_t w1 = *reinterpret_cast<const uint32_t *>(codes + (r0 + 8) * kRowBytes + place);
          const uint32_t z0 = mv_zero(ze[r0 * (kChunkK / 32) + grp], H()), z1 = mv_zero(ze[(r0 + 8) * (kChunkK / 32) + grp], H());
          uint32_t f[4] = {mv_unpack(w0, 0, z0, H()), mv_unpack(w1, 0, z1, H()), mv_unpack(w0, 1, z0, H()), mv_unpack(w1, 1, z1, H())};
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mv_mma(acc[rt][nb], f, xf[nb].x, xf[nb].y, H());
          uint32_t h[4] = {mv_unpack(w0, 2, z0, H()), mv_unpack(w1, 2, z1, H()), mv_unpack(w0, 3, z0, H()), mv_unpack(w1, 3, z1, H())};
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mv_mma(acc[rt][nb], h, xf[nb].z, xf[nb].w, H());
        }
        // the end of a group, or of the warp's part of one
        if (b4 == 3 || (((b + 1) << 5) & ((1 << a.group_shift) - 1)) == 0) {
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) {
            const float s0 = sc[(rt * 16 + g) * (kChunkK / 32) + grp], s1 = sc[(rt * 16 + g + 8) * (kChunkK / 32) + grp];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                total[rt][nb][i] = fmaf(i < 2 ? s0 : s1, acc[rt][nb][i], total[rt][nb][i]);
                acc[rt][nb][i] = 0.f;
              }
            }
          }
        }
      }
      if (more) {
        fetch_scales(buf ^ 1, first + c + 1);
        put_x(buf ^ 1);
      }
      cp_async_wait_all();
      __syncthreads();
    }
  }

  // sums of the block: over the k parts of the warps, then over the terms of an FP32 x
  float *parts = reinterpret_cast<float *>(smem);                       // [WK][8 NB][kRows]
  float *sums = parts + Tile::WK * 8 * NB * kRows;                      // [kM][kRows]
#pragma unroll
  for (int rt = 0; rt < 2; ++rt)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        parts[(wk * 8 * NB + nb * 8 + 2 * t + (i & 1)) * kRows + wn * 32 + rt * 16 + g + (i >> 1) * 8] = total[rt][nb][i];
  __syncthreads();
  for (int i = tid; i < mm * kRows; i += kMvThreads) {
    const int m = i / kRows, r = i % kRows;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < Tile::WK; ++k)
#pragma unroll
      for (int p = 0; p < Tile::kParts; ++p) s += parts[(k * 8 * NB + m * Tile::kParts + p) * kRows + r];
    sums[i] = s;
  }
  if (ctas > 1) cluster_sync_all();
  else __syncthreads();
  // outputs, shared out over the cluster; every rank's sum in the order of the ranks
  for (int i = tid + rank * kMvThreads; i < mm * kRows; i += kMvThreads * ctas) {
    const int m = i / kRows;
    const int64_t n = n0 + i % kRows;
    float s = 0.f;
    if (ctas > 1) {
      for (int q = 0; q < ctas; ++q) s += ld_shared_cluster_f32(mapa_u32(smem_u32(sums + i), (uint32_t)q));
    } else {
      s = sums[i];
    }
    if (n < a.N) {
      T *to = (T *)a.y + (int64_t)(m0 + m) * a.ldy + n;
      const float v = a.alpha * (16.f * s);
      *to = from_f32<T>(a.beta != 0.f ? fmaf(a.beta, to_f32(*to), v) : v);
    }
  }
  if (ctas > 1) cluster_sync_all();   // nobody leaves while its sums may still be read
}

template <class T, int NB, int WN, bool ALIGNED>
static int w4_matvec_launch(Context *ctx, MvArgs a, bool xvec, cudaStream_t s) {
  using Tile = MvTile<T, NB, WN>;
  const auto kernel = w4_matvec_kernel<T, NB, WN, ALIGNED>;
  const int st = ensure_func_attributes((const void *)kernel, ctx->device, Tile::kSmem);
  if (st != B2_OK) return st;
  a.m_chunks = (a.M + Tile::kM - 1) / Tile::kM;
  const int64_t blocks = ((a.N + Tile::kRows - 1) / Tile::kRows) * a.m_chunks;
  const int64_t chunks = (a.K + Tile::kChunkK - 1) / Tile::kChunkK;
  B2_REQUIRE(blocks <= INT32_MAX, B2_ERR_UNSUPPORTED, "b2_w4_matvec: N = %lld is too large", (long long)a.N);
  // CTAs of a cluster: up to 8, as long as each has a chunk
  int ctas = 1;
  while (ctas < 8 && 2 * ctas <= chunks && blocks * ctas < (int64_t)ctx->sm_count * 8) ctas *= 2;
  a.chunks_per_cta = (int)((chunks + ctas - 1) / ctas);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, (unsigned)ctas);
  cfg.blockDim = dim3(kMvThreads);
  cfg.dynamicSmemBytes = Tile::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = (unsigned)ctas;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B2_CUDA(cudaLaunchKernelEx(&cfg, kernel, (const MvArgs)a, xvec ? 1 : 0));
  return B2_OK;
}

template <class T, bool ALIGNED>
static int w4_matvec_rows(Context *ctx, const MvArgs &a, bool xvec, cudaStream_t s) {
  if constexpr (sizeof(T) == 4) {
    if (a.M <= 2) return w4_matvec_launch<T, 1, 2, ALIGNED>(ctx, a, xvec, s);
    return w4_matvec_launch<T, 3, 4, ALIGNED>(ctx, a, xvec, s);
  } else {
    if (a.M <= 8) return w4_matvec_launch<T, 1, 2, ALIGNED>(ctx, a, xvec, s);
    if (a.M <= 16) return w4_matvec_launch<T, 2, 4, ALIGNED>(ctx, a, xvec, s);
    return w4_matvec_launch<T, 4, 4, ALIGNED>(ctx, a, xvec, s);
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
  MvArgs a = {};
  a.N = N, a.K = alpha != 0.f ? K : 0, a.ldx = ldx, a.ldq = ldq, a.ldy = ldy, a.groups = (K + group - 1) / group;
  a.M = (int)M, a.scale_type = scale_type, a.alpha = alpha, a.beta = beta;
  a.group_shift = group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : 8;
  a.x = x, a.codes = codes, a.zeros = zeros, a.scales = scales, a.y = y;
  const bool aligned = (((uintptr_t)codes | (uintptr_t)ldq) & 15) == 0;
  const bool xvec = (((uintptr_t)x | (uintptr_t)(ldx * tb)) & 15) == 0;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    return aligned ? w4_matvec_rows<T, true>(ctx, a, xvec, (cudaStream_t)stream) : w4_matvec_rows<T, false>(ctx, a, xvec, (cudaStream_t)stream);
  });
}

}  // extern "C"
