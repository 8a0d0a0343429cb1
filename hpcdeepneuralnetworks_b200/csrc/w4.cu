// 4-bit weights with group scales: quantise, expand, and the matrix-vector product of decoding steps.
#include <math.h>

#include <mutex>
#include <type_traits>

#include "types.cuh"

namespace b2 {

constexpr int kW4MaxRows = 64;   // rows of x that b2_w4_matvec takes
constexpr int64_t kW4MaxK = 1 << 27;   // and their length: units of a row are counted in 32 bits

__device__ __forceinline__ float w4_warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// The larger and the smaller of two, NaN if either is.
__device__ __forceinline__ float w4_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float w4_min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Two FP32 values to an instruction.
__device__ __forceinline__ uint64_t w4_two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 w4_both(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t w4_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t w4_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t w4_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The integer nearest to w / s for s > 0, ties to even, as a float.  The quotient in FP32 names a candidate that is at most
// one off; the candidate's remainder, which an FMA leaves exact near a border, says whether a neighbour is nearer.  `inv` is
// 1 / s (finite: see w4_prescale), `half` is s / 2.  Adding and taking away 1.5 * 2^23 rounds to an even integer as rintf does,
// and leaves the integer's parity in the lowest bit of the sum.
__device__ __forceinline__ float w4_nearest(float w, float s, float half, float inv) {
  const float big = fminf(fmaxf(w * inv, -40.f), 40.f) + 12582912.f;
  const float q = big - 12582912.f, r = fmaf(-q, s, w);
  if (fabsf(r) < half) return q;
  const bool odd = __float_as_uint(big) & 1u;
  if (r > half || (r == half && odd)) return q + 1.f;
  if (r < -half || (r == -half && odd)) return q - 1.f;
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

// V elements in order as FP32 (V a multiple of 2; one access of 16 bytes per 16 / sizeof(T) of them).
template <class T, int V>
__device__ __forceinline__ void w4_load(float (&v)[V], const T *p) {
  constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < V; i += PER) {
    union {
      uint4 q;
      T e[PER];
    } u;
    u.q = __ldcs(reinterpret_cast<const uint4 *>(p + i));
#pragma unroll
    for (int k = 0; k < PER; ++k) v[i + k] = to_f32(u.e[k]);
  }
}

// Quantising should be bound by reading W, and is by its 22 instructions per element, which take 82 % of the issue slots (8192 x 8192
// bf16: 45 us, 3.8 TB/s; a copy of those bytes takes 26).  group / 16 lanes share a group, 16
// elements (8 bytes of codes) each: a group's extremes take log2(group / 16) shuffles.  Nearly every element's code is what the
// magic addition in w4_nearest gives at once: w / s + 1.5 * 2^23 holds it in its low bits.  Elements that are not nearer than
// s / 2 to their codes' values (with 16-bit weights a third of the warps meet one that is exactly s / 2 away), and all of a group
// that needs more care (a scale that is 0, tiny or clamped), are given to w4_nearest, one by one.
// ALIGN: what W's rows and pitch are a multiple of, 16, 4 or 2 bytes.  Below 16 a warp's 512 elements pass through shared memory,
// so that its accesses lie side by side (8192 x 8190 bf16: 253 us with each lane reading its own elements); likewise its codes
// where rows of codes do not start on 8 bytes (QVEC = false).
template <class T, class S, bool ZEROS, int ALIGN, bool QVEC>
__global__ void __launch_bounds__(256) w4_quantize_kernel(int64_t N, int64_t K, int group_shift, const T *W, int64_t ldw, uint8_t *codes,
                                                          int64_t ldq, S *scales, uint8_t *zeros) {
  constexpr int PER = ALIGN / (int)sizeof(T) < 1 ? 1 : ALIGN / (int)sizeof(T);      // elements per access of a staged row
  constexpr int kPitch = 17;
  __shared__ float staged[ALIGN < 16 ? 8 : 1][ALIGN < 16 ? 32 * kPitch : 1];         // [warp][lane][16]
  __shared__ uint2 coded[QVEC ? 1 : 8][QVEC ? 1 : 32];
  const int lane = (threadIdx.y * blockDim.x + threadIdx.x) & 31, warp = (threadIdx.y * blockDim.x + threadIdx.x) >> 5;
  const bool wide = blockDim.x >= 32;                                     // a warp's lanes lie in one row
  const int64_t groups = (K + (1 << group_shift) - 1) >> group_shift;
  const int lanes = 1 << (group_shift - 4);                               // of a group: 2, 4, 8, 16
  const int64_t row_units = groups << (group_shift - 4);                  // units of 16 elements, whole groups
  // blockDim.x threads to a row (a power of two, not less than a group's lanes), blockDim.y rows to a block; all threads of a
  // block take every turn, so that shuffles see every lane
  for (int64_t nb = (int64_t)blockIdx.y * blockDim.y; nb < N; nb += (int64_t)gridDim.y * blockDim.y) {
    const int64_t n = nb + threadIdx.y;
    for (int64_t ub = (int64_t)blockIdx.x * blockDim.x; ub < row_units; ub += (int64_t)gridDim.x * blockDim.x) {
      if ((ALIGN < 16 || !QVEC) && wide && ub + (threadIdx.x & ~31u) >= row_units) continue;      // a whole warp behind the row
      const int64_t u = ub + threadIdx.x, k0 = u * 16;
      const int64_t left = n < N ? K - k0 : 0;
      const int len = left >= 16 ? 16 : left > 0 ? (int)left : 0;
      const T *w = W + n * ldw + k0;
      float v[16];
      if (ALIGN == 16 && len == 16) {
        w4_load<T, 16>(v, w);
      } else if (ALIGN < 16 && wide) {
        // the warp's elements from k0 of its first lane on
        const int64_t from = k0 - 16 * lane, behind = n < N ? K - from : 0;
        const T *row = W + (n < N ? n * ldw + from : 0);
        const int end = behind > 512 ? 512 : (int)behind;
        union Access {
          T e[PER];
          uint32_t word;
        } got[16 / PER];
        if (end == 512) {      // all loads before the first use
#pragma unroll
          for (int i = 0; i < 16 / PER; ++i) {
            const T *p = row + (i * 32 + lane) * PER;
            if (PER > 1) got[i].word = __ldcs(reinterpret_cast<const unsigned int *>(p));
            else got[i].e[0] = *p;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16 / PER; ++i)
#pragma unroll
            for (int q = 0; q < PER; ++q) {
              const int e = (i * 32 + lane) * PER + q;
              got[i].e[q] = e < end ? row[e] : from_f32<T>(0.f);
            }
        }
#pragma unroll
        for (int i = 0; i < 16 / PER; ++i)
#pragma unroll
          for (int q = 0; q < PER; ++q) {
            const int e = (i * 32 + lane) * PER + q;
            staged[warp][(e >> 4) * kPitch + (e & 15)] = to_f32(got[i].e[q]);
          }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = staged[warp][lane * kPitch + i];
        __syncwarp();
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = i < len ? to_f32(w[i]) : 0.f;
      }
      float lo = 0.f, hi = 0.f;                                           // without zeros: hi = largest magnitude
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        hi = w4_max_nan(hi, ZEROS ? v[i] : fabsf(v[i]));
        if (ZEROS) lo = w4_min_nan(lo, v[i]);
      }
      for (int o = 1; o < lanes; o <<= 1) {
        hi = w4_max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        if (ZEROS) lo = w4_min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      }
      if (len <= 0 && (QVEC || !wide)) continue;                          // nothing to write; a group's first lane has elements
      const bool bad = !isfinite(hi) || (ZEROS && !isfinite(lo));
      const S stored = bad ? from_f32<S>(__int_as_float(0x7fffffff)) : w4_scale<S>(lo, hi, ZEROS);
      const float scale = to_f32(stored);
      const bool flat = !(scale > 0.f);                                   // 0, or NaN: every code is the zero point
      const float f = w4_prescale(scale), s = scale * f, inv = 1.f / s, half = 0.5f * s;
      float zero = 8.f;
      if (ZEROS && !flat) zero = fminf(fmaxf(w4_nearest(-lo * f, s, half, inv), 0.f), 15.f);
      if ((u & (lanes - 1)) == 0 && (QVEC || len > 0)) {
        const int64_t at = n * groups + (u >> (group_shift - 4));
        scales[at] = stored;
        if (ZEROS) zeros[at] = (uint8_t)zero;
      }
      uint32_t out[2] = {0, 0};
      // the quick way: 1.5 * 2^23 + zero - 8 is even or odd as zero is, which only ties would tell apart
      uint32_t unsure = !flat && f == 1.f && (ZEROS || hi * inv < 7.4f) ? 0u : 0xffffu;
      if (!QVEC && len <= 0) unsure = 0;
      const float magic = 12582912.f;
      const uint64_t inv2 = w4_two(inv, inv), magic2 = w4_two(magic, magic), minus2 = w4_two(-magic, -magic), s2 = w4_two(-s, -s);
      const float least = magic - zero, most = magic + 15.f - zero;
      const uint32_t base = __float_as_uint(magic) - (uint32_t)(int)zero;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const uint64_t x = w4_two(v[i], v[i + 1]);
        const uint64_t big = w4_fma(x, inv2, magic2);                     // rounded once, to an integer
        const float2 r = w4_both(w4_fma(w4_add(big, minus2), s2, x));
        if (!(fabsf(r.x) < half) && (QVEC || len > 0)) unsure |= 1u << i;
        if (!(fabsf(r.y) < half) && (QVEC || len > 0)) unsure |= 2u << i;
        float2 b = w4_both(big);
        if (ZEROS) b = make_float2(fminf(fmaxf(b.x, least), most), fminf(fmaxf(b.y, least), most));
        // (where the quick way is not taken at all these bits are nonsense, and every code is set below)
        out[i >> 3] += ((__float_as_uint(b.x) - base) << (4 * (i & 7))) + ((__float_as_uint(b.y) - base) << (4 * (i & 7) + 4));
      }
      while (unsure) {
        const int i = __ffs((int)unsure) - 1;
        unsure &= unsure - 1;
        float e = v[0];
#pragma unroll
        for (int k = 1; k < 16; ++k) e = i == k ? v[k] : e;
        const float c = flat ? zero : fminf(fmaxf(w4_nearest(e * f, s, half, inv) + zero, ZEROS ? 0.f : 1.f), 15.f);
        const uint32_t shift = 4 * (i & 7), fresh = (uint32_t)c << shift, keep = ~(15u << shift);
        if (i < 8) out[0] = (out[0] & keep) | fresh;
        else out[1] = (out[1] & keep) | fresh;
      }
      uint8_t *to = codes + n * ldq + (k0 >> 1);
      if (QVEC && len == 16) {
        *reinterpret_cast<uint2 *>(to) = make_uint2(out[0], out[1]);
        continue;
      }
      if (len & 1) out[len >> 3] &= ~(0xf0u << (8 * ((len >> 1) & 3)));     // the half byte behind an odd row is 0
      if (!QVEC && wide) {
        coded[warp][lane] = make_uint2(out[0], out[1]);
        __syncwarp();
        const unsigned char *bytes = reinterpret_cast<const unsigned char *>(coded[warp]);
        const int64_t from = (k0 - 16 * lane) >> 1, behind = n < N ? ((K + 1) >> 1) - from : 0;
        uint8_t *const first = codes + n * ldq + from + lane;
        const int end = (behind > 256 ? 256 : (int)behind) - lane;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i * 32 < end) first[i * 32] = bytes[i * 32 + lane];
        __syncwarp();
      } else {
        for (int i = 0; 2 * i < len; ++i) to[i] = (uint8_t)(out[i >> 2] >> (8 * (i & 3)));
      }
    }
  }
}

__device__ __forceinline__ float w4_zero(const uint8_t *zeros, int64_t at) { return zeros ? (float)(zeros[at] & 15) : 8.f; }

// 8 codes of a word as FP32: (c - z) * scale, in order.  The even codes are masked out as bytes, the odd ones likewise after a
// shift; a byte under 2^23's upper three reads 2^23 + c, and the difference with 2^23 + z is exact.
__device__ __forceinline__ void w4_expand(float (&v)[8], uint32_t word, float scale, float zero) {
  const uint32_t even = word & 0x0f0f0f0fu, odd = (word >> 4) & 0x0f0f0f0fu;
  const uint64_t less = w4_two(-8388608.f - zero, -8388608.f - zero), by = w4_two(scale, scale);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = __uint_as_float(__byte_perm(even, 0x4b000000u, 0x7440 + i)), b = __uint_as_float(__byte_perm(odd, 0x4b000000u, 0x7440 + i));
    const float2 r = w4_both(w4_mul(w4_add(w4_two(a, b), less), by));
    v[2 * i] = r.x, v[2 * i + 1] = r.y;
  }
}

// Four bytes at an offset of a row of `width` bytes that may start anywhere, zero behind its end; no byte outside is touched.
__device__ __forceinline__ uint32_t w4_word(const uint8_t *row, int64_t at, int64_t width) {
  const uint8_t *p = row + at;
  const int skew = (int)((uintptr_t)p & 3);
  if (at >= 4 && at + 8 <= width) {
    const uint32_t *q = reinterpret_cast<const uint32_t *>(p - skew);
    return __funnelshift_r(q[0], q[1], 8 * skew);
  }
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i < width) word |= (uint32_t)p[i] << (8 * i);
  return word;
}

// Expanding is bound by writing W (8192 x 8192 to bf16: 37 us, 4.6 TB/s, of a copy's 6.5).  Rows as they lie: a thread takes 8 codes (one word) to 8 elements, four such units in flight.
// CVEC: words of codes start on 4 bytes.  WVEC: 16 bytes of W start on 16; otherwise a warp's 256 elements pass through shared
// memory, so that its stores lie side by side (8192 x 8190 bf16: 57 us; 171 with each lane writing its own elements).
template <class T, class S, bool CVEC, bool WVEC>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(int64_t N, int64_t K, int group_shift, const uint8_t *codes, int64_t ldq,
                                                            const S *scales, const uint8_t *zeros, T *W, int64_t ldw) {
  constexpr int kFlight = 4;
  struct alignas(16) Eight {
    T e[8];
  };
  __shared__ Eight staged[WVEC ? 1 : 8][WVEC ? 1 : 32];
  const int64_t groups = (K + (1 << group_shift) - 1) >> group_shift, width = (K + 1) >> 1;
  // within a row 32 bits do (K < 2^31); a row's units are fewer than 2^28, and kFlight steps fewer than 2^30
  const uint32_t units = (uint32_t)((K + 7) >> 3), step = gridDim.x * blockDim.x, k32 = (uint32_t)K;
  const int lane = (threadIdx.y * blockDim.x + threadIdx.x) & 31, warp = (threadIdx.y * blockDim.x + threadIdx.x) >> 5;
  const bool wide = blockDim.x >= 32;                                     // a warp's lanes lie in one row
  // every thread takes every turn: warps work together
  for (int64_t nb = (int64_t)blockIdx.y * blockDim.y; nb < N; nb += (int64_t)gridDim.y * blockDim.y) {
    const int64_t n = nb + threadIdx.y;
    const uint32_t mine = n < N ? units : 0;
    const uint8_t *row = codes + n * ldq;
    const S *scale_row = scales + n * groups;
    const uint8_t *zero_row = zeros ? zeros + n * groups : nullptr;
    T *out = W + n * ldw;
    for (uint32_t ub = blockIdx.x * blockDim.x; ub < units; ub += kFlight * step) {
      uint32_t word[kFlight];
      float scale[kFlight], zero[kFlight];
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        const uint32_t u = ub + threadIdx.x + i * step;
        word[i] = 0;
        scale[i] = zero[i] = 0.f;
        if (u < mine) {
          if (CVEC && 8 * u + 8 <= k32) word[i] = __ldcs(reinterpret_cast<const unsigned int *>(row + 4 * u));
          else word[i] = w4_word(row, 4 * u, width);
          scale[i] = to_f32(scale_row[(8 * u) >> group_shift]);
          zero[i] = zero_row ? (float)(zero_row[(8 * u) >> group_shift] & 15) : 8.f;
        }
      }
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        const uint32_t u = ub + threadIdx.x + i * step;
        if (ub + i * step >= units) break;                       // for the whole block
        float v[8];
        w4_expand(v, word[i], scale[i], zero[i]);
        union {
          Eight all;
          uint4 q[sizeof(T) / 2];
        } o;
#pragma unroll
        for (int k = 0; k < 8; ++k) o.all.e[k] = from_f32<T>(v[k]);
        T *to = out + 8 * u;
        if (WVEC && 8 * u + 8 <= k32) {
          if (u < mine) {
#pragma unroll
            for (int q = 0; q < (int)sizeof(T) / 2; ++q) __stcs(reinterpret_cast<uint4 *>(to) + q, o.q[q]);
          }
        } else if (!WVEC && wide) {
          staged[warp][lane] = o.all;
          __syncwarp();
          const T *flat = reinterpret_cast<const T *>(staged[warp]);
          const int64_t from = 8 * (int64_t)(u - lane), behind = n < N ? K - from : 0;
          T *const first = out + from + lane;
          const int end = (behind > 256 ? 256 : (int)behind) - lane;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k * 32 < end) first[k * 32] = flat[k * 32 + lane];
          __syncwarp();
        } else if (u < mine) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (8 * u + k < k32) to[k] = o.all.e[k];
        }
      }
    }
  }
}

// Transposed: tiles of 64 rows n x 64 of k through shared memory, so that codes are read along k and W is written along n.
// A thread expands 16 codes (8 bytes) of one row into a column of the tile; a row of the tile goes out as 64 elements along n,
// two of 16 bits to an access where W allows (PAIR).  6144 x 6144 to FP32: 37 us, 4.6 TB/s; 8192 x 8192 to bf16, whose rows of a tile
// are 128 bytes: 56 us.
template <class T, class S, bool VEC, bool PAIR>
__global__ void __launch_bounds__(256) w4_transpose_kernel(int64_t N, int64_t K, int group_shift, const uint8_t *codes, int64_t ldq,
                                                           const S *scales, const uint8_t *zeros, T *W, int64_t ldw) {
  __shared__ float tile[64][65];                // [k][n]
  const int64_t groups = (K + (1 << group_shift) - 1) >> group_shift;
  const int64_t k_tiles = (K + 63) >> 6, n_tiles = (N + 63) >> 6;
  // thread: row threadIdx.x / 4 of a tile, 16 codes from (threadIdx.x % 4) * 16 on; the next tile's are fetched while this one's go out
  const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
  uint32_t word[2];
  float scale, zero;
  auto fetch = [&](int64_t n_tile, int64_t k_tile) {
    const int64_t n = n_tile * 64 + r, k = k_tile * 64 + c;
    word[0] = word[1] = 0;
    scale = zero = 0.f;
    if (n < N && k < K) {
      const uint8_t *from = codes + n * ldq + (k >> 1);
      if (VEC && k + 16 <= K) {
        const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(from));
        word[0] = v.x, word[1] = v.y;
      } else {
        word[0] = w4_word(codes + n * ldq, k >> 1, (K + 1) >> 1);
        word[1] = w4_word(codes + n * ldq, (k >> 1) + 4, (K + 1) >> 1);
      }
      const int64_t g = n * groups + (k >> group_shift);
      scale = to_f32(scales[g]);
      zero = w4_zero(zeros, g);
    }
  };
  const int64_t n_step = gridDim.x % n_tiles, k_step = gridDim.x / n_tiles;
  int64_t n_tile = blockIdx.x % n_tiles, k_tile = blockIdx.x / n_tiles;
  fetch(n_tile, k_tile);
  while (k_tile < k_tiles) {
    const int64_t n0 = n_tile * 64, k0 = k_tile * 64;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[8];
      w4_expand(v, word[h], scale, zero);
#pragma unroll
      for (int i = 0; i < 8; ++i) tile[c + 8 * h + i][r] = v[i];
    }
    __syncthreads();
    n_tile += n_step, k_tile += k_step;
    if (n_tile >= n_tiles) n_tile -= n_tiles, ++k_tile;
    fetch(n_tile, k_tile);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t k = k0 + warp * 8 + i;
      if (k < K) {
        if constexpr (PAIR) {
          const int64_t n = n0 + 2 * lane;
          union {
            T e[2];
            uint32_t w;
          } o;
          o.e[0] = from_f32<T>(tile[warp * 8 + i][2 * lane]);
          o.e[1] = from_f32<T>(tile[warp * 8 + i][2 * lane + 1]);
          if (n + 1 < N) *reinterpret_cast<uint32_t *>(W + k * ldw + n) = o.w;
          else if (n < N) W[k * ldw + n] = o.e[0];
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int64_t n = n0 + h * 32 + lane;
            if (n < N) W[k * ldw + n] = from_f32<T>(tile[warp * 8 + i][h * 32 + lane]);
          }
        }
      }
    }
    __syncthreads();
  }
}

// ---- matrix-vector product -----------------------------------------------------------------------
// y = alpha * x * W^T + beta * y.  The codes are read once and should decide the time; what stands in the way is unpacking
// them, so the arithmetic is arranged to need nine instructions for eight codes.  It runs on mma.sync m16n8k16 (16 weight rows x
// 8 columns of x), which has room for 8 columns at the price of one; a tcgen05 tile would want its operands written back to
// shared memory in 16 bits first.
//
// Per group,  sum_k W x = s * sum_k (c - z) x.  The zero point is taken off while unpacking: taken off the sums it would leave, of an
// element of x that meets weight 0, the rounding of z x, and that may be more than all the rest of the group.  Operands are of the
// type that holds x exactly, and so are the differences c - z, whole numbers from -15 to 15.
//   bf16 and FP32 x: a code in the lowest bits of a 16-bit half IS the bf16 number c * 2^-133, four bits higher it is 16 c * 2^-133
//   (the first 256 bit patterns are the multiples of 2^-133); a mask and an FMA by 2^119 or 2^115 make (c - z) * 2^-14, exactly.  In
//   that unit the largest bf16 and 128 of the largest weights stay within FP32, and the smallest are not lost below it.  FP32 x is
//   cut into three bf16 terms of 8 bits, a column of the tile each: exact, but for what lies below 2^-135.
//   FP16 x: under 1024's upper bits a code reads 1024 + c, or 1024 + 16 c, and a subtraction or an FMA with 1/16 leaves c - z.
// Words w and w >> 8 give the pairs of codes (0,4) (1,5) (2,6) (3,7), and a small kernel in front (w4_x_kernel) pairs x alike.  All
// products are exact in FP32; group sums are FP32, scaled and added in FP32.
// An infinity or NaN in x is one in its column of the tile: it meets the exact weights, 0 among them, and stays in its row's outputs.
//
// A CTA streams tiles of 128 rows x 256 k (16 KB of codes and x of those k) through a ring of shared-memory stages.  Four
// producer warps fill it: one thread issues the TMA loads (codes with the 128-byte swizzle: the 16-byte unit u of row r lies at
// u ^ (r & 7), so that the words that a warp reads lie in 32 banks), the others fetch scales and zero points, eight groups of
// each row at a time.  Eight consumer warps, 4 (rows) x 2 (k), multiply 32 rows x 128 k each.  Where there are fewer row blocks
// than CTAs, the k range is cut over the CTAs of a cluster, whose sums meet over distributed shared memory in the order of the
// ranks: no atomics.
// Measured on the device: 1 x 4096^2 bf16 6.4 us and 1 x 8192^2 14.7, latency; 16 x 32768 x 8192 49 us = 2.9 TB/s (the loads alone
// take 30: unpacking and the waits around it decide; with the zero point taken off the sums instead, four instructions less per
// word, 45); 3 x 6144^2 FP32 15.2 us; 64 x 16384 x 4096 45 us, of which each of the two items of a row block unpacks the codes anew.
constexpr int kMvConsumers = 256, kMvProducers = 128, kMvThreads = kMvConsumers + kMvProducers;
constexpr int kMvRows = 128, kMvChunk = 256, kMvRowBytes = kMvChunk / 2;
constexpr int kMvPitch = kMvRows + 4;       // of the sums: 8 rows x 4 columns of a warp's store in 32 banks
constexpr int kMvWindow = 1024;             // scales and zero points held together: 8 groups of each row, the group / 32 chunks
constexpr int kMvWindows = 2;               // they span
constexpr int kMvMaxStages = 8, kMvBarrierBytes = 512 + 1024;   // barriers and flags, and room to align
constexpr int kMvXThreads = 128;

template <int NB, bool RESIDENT, bool ALIGNED>
struct MvTile {
  // rows of codes that start anywhere are held from the 16-byte boundary in front of them on, 9 units of 16 bytes
  static constexpr int kRowPitch = ALIGNED ? kMvRowBytes : kMvRowBytes + 16, kCodeBytes = kMvRows * kRowPitch;
  static constexpr int kXBytes = NB * kMvChunk * 8 * 2;            // x of one chunk
  static constexpr int kStage = RESIDENT ? kCodeBytes : (kCodeBytes + kXBytes + 1023) / 1024 * 1024;
  static constexpr int kSumBytes = 2 * 8 * NB * kMvPitch * 4;
  static constexpr int kCtasPerSm = NB <= 2 ? 2 : 1;
  static constexpr int kSmem = kCtasPerSm == 2 ? 115712 : 232448;   // what a CTA may have
};

// Columns that a row of x takes, blocks of 8 columns per item for M rows, rows per item.
static int mv_parts(int type) { return type == B2_F32 ? 3 : 1; }
static int mv_blocks(int64_t M, int type) { return M * mv_parts(type) <= 8 ? 1 : M * mv_parts(type) <= 16 ? 2 : 4; }
static int mv_rows(int nb, int type) { return 8 * nb / mv_parts(type); }
// Whether a product's CTAs lay x out themselves (RESIDENT): each keeps its part of k, cut over clusters of up to 8, in shared
// memory.  That saves a kernel and a workspace, and costs the same work in every row block's CTAs.
// (Device time against that through w4_x_kernel, groups of 128, bf16, K = 4096.  1 token, 64 to 1024 units: 5.0 / 5.8, 5.1 / 6.0, 5.9 /
// 6.5, 6.5 / 7.4, 768: 9.1 / 9.7, 1024: 10.4 / 10.0 us, 8192^2, 2048 units: 15.2 / 14.4.  8 tokens: 5.9 / 6.8, 5.9 / 6.8, 7.4 / 7.7, 7.7 /
// 8.3, 768: 10.0 / 10.2, 1024: 11.8 / 10.4, 2048: 18.1 / 15.2.  The host's share of a call: 4.5 / 8 us.)
constexpr int kMvResidentBytes = 32 * 1024;
constexpr int64_t kMvResidentWork = 600;       // row blocks x chunks (16 KB of codes each)
static bool mv_resident(int64_t M, int64_t N, int64_t K, int type) {
  const int nb = mv_blocks(M, type);
  const int64_t chunks = (K + kMvChunk - 1) / kMvChunk, per_cta = (chunks + 7) / 8;
  const int64_t blocks = (N + kMvRows - 1) / kMvRows;
  return nb == 1 && per_cta * kMvChunk * 8 * 2 <= kMvResidentBytes && blocks * chunks <= kMvResidentWork;
}

struct MvArgs {
  int64_t N, K, ldx, ldq, ldy, groups;
  int M, rows_per_item, parts, type, group_shift, scale_type;
  int stages, items, row_blocks, chunks, chunks_per_cta, vec;
  float alpha, beta;
  const void *x;
  const uint8_t *codes, *zeros;
  const void *scales;
  void *y;
  const unsigned char *image;      // [item's rows][chunk][kXBytes], unless the CTAs lay x out themselves
  int *status;
  unsigned int seq;
};

// x[k .. k + 8) of a row in FP32, zero behind K.
template <class T>
__device__ __forceinline__ void mv_load_x(float (&v)[8], const T *row, int64_t k, int64_t K, bool vec) {
  if (vec && k + 8 <= K) {
    union {
      uint4 q[sizeof(T) / 2];
      T e[8];
    } u;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u.q[i] = reinterpret_cast<const uint4 *>(row + k)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(u.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_f32(row[k + i]) : 0.f;
  }
}

// Lays one unit (8 elements, the `u`-th of its chunk) of columns col0.. out in a chunk's image: as FP16, or in `parts` bf16 terms,
// each the upper half of what the one before has left, and paired.  An infinity or NaN is the first term, and nothing is left of it.
template <bool BF16>
__device__ __forceinline__ void mv_put(unsigned char *chunk, const float (&e)[8], int u, int nb, int col0, int parts) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = e[i];
  for (int p = 0; p < parts; ++p) {
    const int col = col0 + p;
    union {
      uint16_t h[8];
      uint4 q;
    } out;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = 2 * (i & 3) + (i >> 2);      // pairs (0,4) (1,5) (2,6) (3,7)
      if constexpr (BF16) {
        const uint32_t top = isnan(r[i]) ? 0x7fff0000u : __float_as_uint(r[i]) & 0xffff0000u;
        out.h[at] = (uint16_t)(top >> 16);
        r[i] = isfinite(r[i]) ? r[i] - __uint_as_float(top) : 0.f;
      } else {
        out.h[at] = __half_as_ushort(__float2half_rn(r[i]));      // (x is FP16)
      }
    }
    reinterpret_cast<uint4 *>(chunk)[(((u >> 2) * nb + (col >> 3)) * 8 + (col & 7)) * 4 + (u & 3)] = out.q;
  }
}

// The images of all rows of x: a unit per thread, blockIdx.y the row.
template <class T>
__global__ void __launch_bounds__(kMvXThreads) w4_x_kernel(int64_t K, int64_t ldx, int vec, const T *x, int chunks, int nb, int rows_per_item,
                                                           unsigned char *image) {
  constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
  pdl_launch_dependents();
  const int m = blockIdx.y, item = m / rows_per_item, u = blockIdx.x * kMvXThreads + threadIdx.x;
  if (u >= chunks * (kMvChunk / 8)) return;
  float e[8];
  mv_load_x<T>(e, x + m * ldx, 8 * (int64_t)u, K, vec != 0);
  mv_put<!std::is_same<T, __half>::value>(image + ((int64_t)item * chunks + (u >> 5)) * (nb * kMvChunk * 8 * 2), e, u & 31, nb,
                                          (m - item * rows_per_item) * kParts, kParts);
}

// (w & mask) | bits in one instruction (left to itself the compiler makes two of it, having two constants)
__device__ __forceinline__ uint32_t mv_and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
  return r;
}
// d = a * b + (FIRST: 0, else d)
template <bool BF16, bool FIRST>
__device__ __forceinline__ void mv_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (FIRST) d[0] = d[1] = d[2] = d[3] = 0.f;
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What a group's zero point is held as, twice in 16 bits: what mv_even adds or takes off.
constexpr float kMvUnit = 0x1p-14f;      // of bf16 weights
template <bool BF16>
__device__ __forceinline__ uint32_t mv_zero(uint32_t z) {
  return BF16 ? (__float_as_uint(-(float)z * kMvUnit) >> 16) * 0x00010001u : 0x64006400u + z * 0x00010001u;
}
__device__ __forceinline__ uint32_t mv_fma_bf16(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// c - z of a word's codes 0 and 4 (even: in the lowest bits of its halves), or 1 and 5 (odd: four bits up).
template <bool BF16>
__device__ __forceinline__ uint32_t mv_even(uint32_t w, uint32_t zero) {
  if constexpr (BF16) return mv_fma_bf16(w & 0x000f000fu, 0x7b007b00u, zero);      // 2^119
  const uint32_t v = mv_and_or(w, 0x000f000fu, 0x64006400u);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&v), *reinterpret_cast<const __half2 *>(&zero));
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <bool BF16>
__device__ __forceinline__ uint32_t mv_odd(uint32_t w, uint32_t zero) {
  if constexpr (BF16) return mv_fma_bf16(w & 0x00f000f0u, 0x79007900u, zero);      // 2^115
  const uint32_t v = mv_and_or(w, 0x00f000f0u, 0x64006400u);
  const __half2 less = __hsub2(__float2half2_rn(960.f), *reinterpret_cast<const __half2 *>(&zero));      // -(64 + z)
  const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&v), __float2half2_rn(0.0625f), less);
  return *reinterpret_cast<const uint32_t *>(&r);
}

// A tensor map of `rows` rows of `cols` bytes, `pitch` bytes apart, in boxes of 128 bytes x box_rows.
static int mv_map(CUtensorMap *out, const void *base, int64_t cols, int64_t rows, int64_t pitch, int box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  B2_REQUIRE(fn != nullptr, B2_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, steps[2] = {1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void *)base, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  B2_REQUIRE(r == CUDA_SUCCESS, B2_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d (%lld x %lld, pitch %lld)", (int)r,
             (long long)rows, (long long)cols, (long long)pitch);
  return B2_OK;
}

// `bytes` (a multiple of 16, both addresses 16-byte aligned) from global to this CTA's shared memory, completion on an mbarrier.
__device__ __forceinline__ void bulk_load(void *smem_dst, const void *global, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)),
               "l"(global), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// 16 bytes by cp.async, the first `bytes` of them read and the others 0; the thread's arrival at a barrier once all its copies have
// landed; and the wait for them.
__device__ __forceinline__ void copy_async_16(void *smem_dst, const void *global, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem_dst)), "l"(global), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar_cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ uint32_t ld_shared_32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint4 ld_shared_128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ float ld_shared_cluster_f32(uint32_t cluster_addr) { return __uint_as_float(ld_shared_cluster_u32(cluster_addr)); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void mv_consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kMvConsumers) : "memory"); }

// A wait that runs out (about a second) is recorded for b2_check_status; from then on the thread waits no more but walks
// through the rest of its steps, so that every barrier still gets its arrivals and the launch ends, with wrong sums.
struct MvWait {
  int *status;
  unsigned int seq;
  bool alive = true;
  __device__ __forceinline__ void operator()(uint64_t *bar, uint32_t parity) {
    if (!mbar_try_wait(bar, parity)) slow(bar, parity);
  }
  __device__ __noinline__ void slow(uint64_t *bar, uint32_t parity) {
    if (alive && !mbar_wait(bar, parity)) fail();
  }
  __device__ __noinline__ void cluster(uint64_t *bar, uint32_t parity) {
    if (!alive || mbar_try_wait_cluster(bar, parity)) return;
    const uint64_t t0 = global_timer_ns();
    for (uint32_t i = 1; i < (1u << 22); ++i) {
      if (mbar_try_wait_cluster(bar, parity)) return;
      if ((i & 255u) == 0 && global_timer_ns() - t0 > 1000000000ull) break;
    }
    fail();
  }
  __device__ __noinline__ void fail() {
    alive = false;
    record_timeout(status, seq);
  }
};

// A place in a ring of buffers, and the parity of its turn.
struct MvRing {
  int at = 0, size;
  uint32_t phase = 0;
  __device__ __forceinline__ explicit MvRing(int n) : size(n) {}
  __device__ __forceinline__ void next() {
    if (++at == size) at = 0, phase ^= 1;
  }
};

__device__ __forceinline__ float mv_load_any_type(const void *p, int type, int64_t at) {
  if (type == B2_F32) return ((const float *)p)[at];
  if (type == B2_BF16) return to_f32(((const __nv_bfloat16 *)p)[at]);
  return to_f32(((const __half *)p)[at]);
}

// ALIGNED: rows of codes start on 16-byte boundaries (TMA); otherwise the producers copy them.
// RESIDENT: the consumers lay out x of this CTA's k themselves, before the first item; the ring brings codes alone.
// BLOCKS: blocks of 32 k in a group, or in the 128 of a longer one that a warp multiplies.
// BF16: operands in bf16 (for bf16 and FP32 x), else in FP16.
template <int NB, bool ALIGNED, bool RESIDENT, int BLOCKS, bool BF16>
__global__ void __launch_bounds__(kMvThreads, MvTile<NB, RESIDENT, ALIGNED>::kCtasPerSm)
    w4_matvec_kernel(const __grid_constant__ MvArgs a, const __grid_constant__ CUtensorMap code_map) {
  using Tile = MvTile<NB, RESIDENT, ALIGNED>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // the swizzle is one of addresses
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)cluster_ctarank(), ctas = (int)gridDim.y;        // blockIdx.y is the rank within the cluster
  const int first = rank * a.chunks_per_cta;
  int chunks = a.chunks - first;
  chunks = chunks < 0 ? 0 : chunks < a.chunks_per_cta ? chunks : a.chunks_per_cta;
  const int window_log = a.group_shift - 5;                                // chunks of a window: group / 32
  float2 *const windows = reinterpret_cast<float2 *>(smem + a.stages * Tile::kStage);    // [kMvWindows][row][8]: scale, mv_zero of the zero point
  unsigned char *const xs = reinterpret_cast<unsigned char *>(windows + kMvWindows * kMvWindow);   // RESIDENT: [chunk][kXBytes]
  float *const sums = reinterpret_cast<float *>(xs + (RESIDENT ? a.chunks_per_cta * Tile::kXBytes : 0));   // [2][8 NB][kMvPitch]
  uint64_t *const full = reinterpret_cast<uint64_t *>(reinterpret_cast<unsigned char *>(sums) + Tile::kSumBytes);
  uint64_t *const empty = full + kMvMaxStages, *const wfull = empty + kMvMaxStages, *const wempty = wfull + kMvWindows;
  uint64_t *const ready = wempty + kMvWindows, *const done = ready + 1;
  constexpr int kFillers = kMvProducers - 32;     // threads that write shared memory themselves

  if (tid == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], (ALIGNED || !RESIDENT ? 1 : 0) + (ALIGNED ? 0 : 2 * kFillers));
      mbar_init(&empty[s], kMvConsumers / 32);
    }
    for (int s = 0; s < kMvWindows; ++s) {
      mbar_init(&wfull[s], kFillers);
      mbar_init(&wempty[s], kMvConsumers / 32);
    }
    mbar_init(ready, ctas);
    mbar_init(done, ctas);
    mbar_fence_init();
  }
  __syncthreads();
  cluster_arrive();     // the wait comes before the first word to another CTA
  MvWait wait{a.status, a.seq};

  if (warp >= kMvConsumers / 32) {
    if (warp == kMvConsumers / 32) {
      if (lane == 0) {
        // (RESIDENT: an ordinary launch, and codes alone.)  Weights may be read at once: the kernel in front of this one, w4_x_kernel, began after all earlier work had ended.
        // Its own results, x, have to be waited for; the ring is filled with codes first.
        MvRing ring(a.stages);
        uint32_t sent = 0;
        const unsigned char *late[kMvMaxStages];
        bool waited = false;
        auto send_x = [&](int s, const unsigned char *from) {
          bulk_load(smem + s * Tile::kStage + Tile::kCodeBytes, from, Tile::kXBytes, &full[s]);
        };
        for (int item = blockIdx.x; item < a.items; item += gridDim.x) {
          const int mc = item / a.row_blocks, row = (item - mc * a.row_blocks) * kMvRows;
          const unsigned char *image = a.image + ((int64_t)mc * a.chunks + first) * Tile::kXBytes;
          for (int c = 0; c < chunks; ++c, ring.next(), image += Tile::kXBytes) {
            if (sent >= (uint32_t)a.stages) wait(&empty[ring.at], ring.phase ^ 1);
            if (!wait.alive) continue;
            if (ALIGNED || !RESIDENT) mbar_expect_tx(&full[ring.at], (ALIGNED ? Tile::kCodeBytes : 0) + (RESIDENT ? 0 : Tile::kXBytes));
            if (ALIGNED) tma_load_2d(smem + ring.at * Tile::kStage, &code_map, &full[ring.at], (first + c) * kMvRowBytes, row);
            if (RESIDENT) {
            } else if (waited) {
              send_x(ring.at, image);
            } else {
              late[sent] = image;
              const bool last = c + 1 == chunks && item + (int)gridDim.x >= a.items;
              if (sent + 1 == (uint32_t)a.stages || last) {
                pdl_wait();
                waited = true;
                for (uint32_t i = 0; i <= sent; ++i) send_x((int)i, late[i]);
              }
            }
            ++sent;
          }
        }
        ring_settle(full, a.stages, sent);      // nothing is in flight when the CTA leaves, whoever gave up waiting
      }
      __syncwarp();
    } else {
      const int me = tid - kMvConsumers - 32;
      MvRing ring(a.stages), window(kMvWindows);
      uint32_t filled = 0, opened = 0;
      for (int item = blockIdx.x; item < a.items; item += gridDim.x) {
        const int64_t n0 = (int64_t)(item % a.row_blocks) * kMvRows, n_rows = a.N - n0, width = (a.K + 1) >> 1;
        for (int c = 0; c < chunks; ++c) {
          const bool opens = (c & ((1 << window_log) - 1)) == 0;
          constexpr int kTurns = (kMvWindow + kFillers - 1) / kFillers, kRowStep = kFillers / 8;
          uint32_t scale[kTurns], zero[kTurns];
          if (opens) {
            // scales and zero points of a window: entry e is group e & 7 of row e >> 3, so a thread's group stays the same and
            // its rows lie kFillers / 8 apart; all loads before the first use
            const int64_t q = (((int64_t)(first + c) * kMvChunk) >> a.group_shift) + (me & 7);
            const int rows = n_rows < kMvRows ? (int)n_rows : kMvRows, mine = q < a.groups ? rows - (me >> 3) : 0;      // rows left
            const int64_t at = (n0 + (me >> 3)) * a.groups + q, row_step = kRowStep * a.groups;
#pragma unroll
            for (int i = 0; i < kTurns; ++i) scale[i] = 0, zero[i] = 8;
            if (a.scale_type == B2_F32) {
              const uint32_t *from = (const uint32_t *)a.scales + at;
#pragma unroll
              for (int i = 0; i < kTurns; ++i, from += row_step)
                if (i * kRowStep < mine) scale[i] = *from;
            } else {
              const uint16_t *from = (const uint16_t *)a.scales + at;
#pragma unroll
              for (int i = 0; i < kTurns; ++i, from += row_step)
                if (i * kRowStep < mine) scale[i] = *from;
            }
            if (a.zeros) {
              const uint8_t *from = a.zeros + at;
#pragma unroll
              for (int i = 0; i < kTurns; ++i, from += row_step)
                if (i * kRowStep < mine) zero[i] = *from & 15;
            }
          }
          if (!ALIGNED) {
            // 16 bytes at a time by cp.async, which arrives at the barrier when they have landed, cut off where the row ends.  In
            // front of a row a unit may bring bytes of the row before it along, but nothing from in front of the matrix.  Units
            // behind a row, and rows behind N, are left: x is 0 there, or nothing is written.
            if (filled >= (uint32_t)a.stages) wait(&empty[ring.at], ring.phase ^ 1);
            ++filled;
            unsigned char *const stage = smem + ring.at * Tile::kStage;
            const int64_t at = (int64_t)(first + c) * kMvRowBytes, before = n0 * a.ldq + at;      // bytes of the matrix in front of the tile
            const int rows = n_rows < kMvRows ? (int)n_rows : kMvRows, left = width - at < 256 ? (int)(width - at) : 256;
            const uint8_t *const tile = a.codes + before;
            auto unit = [&](const uint8_t *row, int r, int u) {
              const int from = 16 * u - (int)((uintptr_t)row & 15), bytes = left - from < 16 ? left - from : 16;      // from the tile's
              if (r < rows && bytes > 0 && (r >= 16 || row + from >= a.codes))
                copy_async_16(stage + r * Tile::kRowPitch + 16 * u, row + from, bytes);
            };
            // a thread's units are of one column and rows kFillers / 8 apart (known distances: the addresses are most of the work)
            const uint8_t *row = tile + (me >> 3) * a.ldq;
#pragma unroll
            for (int i = 0; i < (kMvRows * 8 + kFillers - 1) / kFillers; ++i, row += (kFillers / 8) * a.ldq) unit(row, (me >> 3) + i * (kFillers / 8), me & 7);
#pragma unroll
            for (int r = me; r < kMvRows; r += kFillers)      // the ninth, of rows that do not start on 16 bytes
              if ((uintptr_t)(tile + r * a.ldq) & 15) unit(tile + r * a.ldq, r, 8);
            if (before < 16) {      // the first rows (of 1 byte, 16 of them) byte by byte
#pragma unroll
              for (int i = 0; i < (256 + kFillers - 1) / kFillers; ++i) {
                const int r = (me + i * kFillers) >> 4, b = (me + i * kFillers) & 15, skew = (int)((uintptr_t)(tile + r * a.ldq) & 15);
                if (r < 16 && r < rows && before + r * a.ldq < skew && b >= skew && b - skew < left)
                  stage[r * Tile::kRowPitch + b] = tile[r * a.ldq + b - skew];
              }
            }
            copy_arrive(&full[ring.at]);
            mbar_arrive(&full[ring.at]);      // for what was stored
            ring.next();
          }
          if (opens) {
            if (opened >= kMvWindows) wait(&wempty[window.at], window.phase ^ 1);
            ++opened;
            float2 *to = windows + window.at * kMvWindow + me;
            if (a.scale_type != B2_F32) {
#pragma unroll
              for (int i = 0; i < kTurns; ++i)
                scale[i] = a.scale_type == B2_BF16 ? scale[i] << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)scale[i])));
            }
#pragma unroll
            for (int i = 0; i < kTurns; ++i)
              if ((i + 1) * kFillers <= kMvWindow || me + i * kFillers < kMvWindow) to[i * kFillers] = make_float2(__uint_as_float(scale[i]), __uint_as_float(mv_zero<BF16>(zero[i])));
            mbar_arrive(&wfull[window.at]);
            window.next();
          }
        }
      }
    }
    if (!ALIGNED) copy_wait_all();
    __syncwarp();
    cluster_wait();
  } else {
    const int g = lane >> 2, t = lane & 3, wn = warp & 3, wk = warp >> 2;
    uint32_t turn = 0;
    MvRing ring(a.stages), window(kMvWindows);
    const uint32_t smem_base = smem_u32(smem), xs_base = smem_u32(xs), windows_base = smem_u32(windows + ((wn * 32 + g) << 3));
    // ALIGNED: of this thread's words of row wn * 32 + g (and, at fixed distances, g + 8, ...) in a stage.  Otherwise of the first
    // of its words of rows g + 8 r, and by how many bits that word is off, set for each row block.
    uint32_t place[4], off[ALIGNED ? 1 : 4];
    if constexpr (ALIGNED) {
#pragma unroll
      for (int b4 = 0; b4 < 4; ++b4) place[b4] = (wn * 32 + g) * kMvRowBytes + (((wk * 4 + b4) ^ g) << 4) + 4 * t;
    }
    if constexpr (RESIDENT) {
      // x of this CTA's k, all rows of it (there is one item's worth): a warp takes a chunk of a row, a lane its unit of 8
      for (int at = warp; at < a.M * chunks; at += kMvConsumers / 32) {
        const int m = at / chunks, c = at - m * chunks;
        const int64_t k = (int64_t)(first + c) * kMvChunk + 8 * lane;
        float e[8];
        if (a.type == B2_F32) mv_load_x(e, (const float *)a.x + m * a.ldx, k, a.K, a.vec != 0);
        else if (a.type == B2_BF16) mv_load_x(e, (const __nv_bfloat16 *)a.x + m * a.ldx, k, a.K, a.vec != 0);
        else mv_load_x(e, (const __half *)a.x + m * a.ldx, k, a.K, a.vec != 0);
        mv_put<BF16>(xs + c * Tile::kXBytes, e, lane, NB, m * a.parts, a.parts);
      }
      mv_consumers_sync();
    }
    for (int item = blockIdx.x; item < a.items; item += gridDim.x, ++turn) {
      const int mc = item / a.row_blocks;
      float total[2][NB][4] = {};
      if constexpr (!ALIGNED) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = wn * 32 + g + 8 * r;
          const uint32_t skew = (uint32_t)(uintptr_t)(a.codes + ((int64_t)(item - mc * a.row_blocks) * kMvRows + row) * a.ldq) & 15u;
          place[r] = row * Tile::kRowPitch + wk * (kMvRowBytes / 2) + 4 * t + (skew & 12u);
          off[r] = 8 * (skew & 3u);
        }
      }
#pragma unroll 1
      for (int c = 0; c < chunks; ++c) {
        const int in_window = c & ((1 << window_log) - 1);
        if (in_window == 0) wait(&wfull[window.at], window.phase);
        wait(&full[ring.at], ring.phase);
        const uint32_t stage = smem_base + ring.at * Tile::kStage;
        const uint32_t image = RESIDENT ? xs_base + c * Tile::kXBytes : stage + Tile::kCodeBytes;
        const uint32_t xf = image + (wk * 4 * NB * 32 + lane) * 16;
        // this warp's first group of the window
        const uint32_t sz = windows_base + window.at * (kMvWindow * 8) + (((in_window * 8 + wk * 4) >> window_log) << 3);
        // the warp's 128 k in straight-line code
        {
#pragma unroll
          for (int b0 = 0; b0 < 4; b0 += BLOCKS) {
            float acc[2][NB][4];
            uint32_t zero[4];                                         // of rows g + 8 r
#pragma unroll
            for (int r = 0; r < 4; ++r) zero[r] = ld_shared_32(sz + (b0 / BLOCKS) * 8 + r * 8 * 64 + 4);
#pragma unroll
            for (int b4 = b0; b4 < b0 + BLOCKS; ++b4) {
              uint4 xv[NB];
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) xv[nb] = ld_shared_128(xf + (b4 * NB + nb) * 512);
#pragma unroll
              for (int rt = 0; rt < 2; ++rt) {
                uint32_t w0, w1;
                if constexpr (ALIGNED) {
                  const uint32_t at = stage + place[b4];
                  w0 = ld_shared_32(at + rt * 16 * kMvRowBytes), w1 = ld_shared_32(at + (rt * 16 + 8) * kMvRowBytes);
                } else {
                  const uint32_t at0 = stage + place[2 * rt] + 16 * b4, at1 = stage + place[2 * rt + 1] + 16 * b4;
                  w0 = __funnelshift_r(ld_shared_32(at0), ld_shared_32(at0 + 4), off[2 * rt]);
                  w1 = __funnelshift_r(ld_shared_32(at1), ld_shared_32(at1 + 4), off[2 * rt + 1]);
                }
                const uint32_t v0 = w0 >> 8, v1 = w1 >> 8;
                const uint32_t z0 = zero[2 * rt], z1 = zero[2 * rt + 1];
                const uint32_t f[4] = {mv_even<BF16>(w0, z0), mv_even<BF16>(w1, z1), mv_odd<BF16>(w0, z0), mv_odd<BF16>(w1, z1)};
                const uint32_t h[4] = {mv_even<BF16>(v0, z0), mv_even<BF16>(v1, z1), mv_odd<BF16>(v0, z0), mv_odd<BF16>(v1, z1)};
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                  if (b4 == b0) mv_mma<BF16, true>(acc[rt][nb], f, xv[nb].x, xv[nb].y);
                  else mv_mma<BF16, false>(acc[rt][nb], f, xv[nb].x, xv[nb].y);
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mv_mma<BF16, false>(acc[rt][nb], h, xv[nb].z, xv[nb].w);
              }
            }
            float scale[4];                                           // of rows g + 8 r
#pragma unroll
            for (int r = 0; r < 4; ++r) scale[r] = __uint_as_float(ld_shared_32(sz + (b0 / BLOCKS) * 8 + r * 8 * 64));
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  float &to = total[r >> 1][nb][2 * (r & 1) + i];
                  to = fmaf(scale[r], acc[r >> 1][nb][2 * (r & 1) + i], to);
                }
          }
        }
        const bool window_ends = in_window == (1 << window_log) - 1 || c + 1 == chunks;
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&empty[ring.at]);
          if (window_ends) mbar_arrive(&wempty[window.at]);
        }
        ring.next();
        if (window_ends) window.next();
      }

      __syncwarp();
      // the row block's sums: this CTA's two k halves side by side, then every rank's, in the order of the ranks
      if (turn == 0) cluster_wait();                                // every CTA's barriers are set up
      else if (ctas > 1) wait.cluster(done, (turn - 1) & 1);        // every CTA has read the sums of the block before
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int col = nb * 8 + 2 * t + i;
#pragma unroll
          for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int h = 0; h < 2; ++h) sums[(wk * 8 * NB + col) * kMvPitch + wn * 32 + rt * 16 + g + h * 8] = total[rt][nb][i + 2 * h];
        }
      mv_consumers_sync();
      if (ctas > 1) {
        if (tid < ctas) mbar_arrive_cluster(mapa_u32(smem_u32(ready), (uint32_t)tid));
        wait.cluster(ready, turn & 1);
      }
      const int m0 = mc * a.rows_per_item, mm = a.M - m0 < a.rows_per_item ? a.M - m0 : a.rows_per_item;
      const int64_t n0 = (int64_t)(item - mc * a.row_blocks) * kMvRows;
      if (!RESIDENT && turn == 0) pdl_wait();                       // the outputs come after everything in front of this kernel
      for (int i = tid + rank * kMvConsumers; i < mm * kMvRows; i += kMvConsumers * ctas) {
        const int m = i / kMvRows, r = i % kMvRows;
        if (n0 + r >= a.N) continue;
        float v = 0.f;
        if (a.chunks > 0) {
          for (int p = 0; p < a.parts; ++p) {
            const float *at = sums + (m * a.parts + p) * kMvPitch + r;
            float s = 0.f;
            if (ctas > 1) {
              for (int q = 0; q < ctas; ++q) {
                const uint32_t from = mapa_u32(smem_u32(at), (uint32_t)q);
                s += ld_shared_cluster_f32(from) + ld_shared_cluster_f32(from + 8 * NB * kMvPitch * 4);
              }
            } else {
              s = at[0] + at[8 * NB * kMvPitch];
            }
            v += s;
          }
          if constexpr (BF16) v *= 1.f / kMvUnit;
          v *= a.alpha;
        }
        const int64_t to = (int64_t)(m0 + m) * a.ldy + n0 + r;
        if (a.beta != 0.f) v = fmaf(a.beta, mv_load_any_type(a.y, a.type, to), v);
        if (a.type == B2_F32) ((float *)a.y)[to] = v;
        else if (a.type == B2_BF16) ((__nv_bfloat16 *)a.y)[to] = from_f32<__nv_bfloat16>(v);
        else ((__half *)a.y)[to] = from_f32<__half>(v);
      }
      mv_consumers_sync();
      if (ctas > 1 && tid < ctas) mbar_arrive_cluster(mapa_u32(smem_u32(done), (uint32_t)tid));
    }
  }
  __syncwarp();
  cluster_sync_all();     // nobody leaves while its sums may still be read or its barriers reached
}

// Clusters of `ctas` CTAs with `smem` bytes each that the device holds at once, asked once per kernel, size and device (and
// each time, should the table be full).
static int mv_clusters(const void *kernel, int device, int ctas, int smem, int *out) {
  struct Entry {
    const void *kernel;
    int device, ctas, smem, clusters;
  };
  static Entry known[512];
  static int count = 0;
  static std::mutex mu;
  std::lock_guard<std::mutex> lk(mu);
  for (int i = 0; i < count; ++i) {
    const Entry &e = known[i];
    if (e.kernel == kernel && e.device == device && e.ctas == ctas && e.smem == smem) {
      *out = e.clusters;
      return B2_OK;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1, (unsigned)ctas);
  cfg.blockDim = dim3(kMvThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = (unsigned)ctas;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  B2_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
  *out = n < 1 ? 1 : n;
  if (count < (int)(sizeof(known) / sizeof(known[0]))) known[count++] = {kernel, device, ctas, smem, *out};
  return B2_OK;
}

template <int NB, bool ALIGNED, bool RESIDENT, int BLOCKS, bool BF16>
static int w4_matvec_launch(Context *ctx, MvArgs a, cudaStream_t s) {
  using Tile = MvTile<NB, RESIDENT, ALIGNED>;
  const auto kernel = w4_matvec_kernel<NB, ALIGNED, RESIDENT, BLOCKS, BF16>;
  const int st = ensure_func_attributes((const void *)kernel, ctx->device, Tile::kSmem);
  if (st != B2_OK) return st;
  const int64_t row_blocks = (a.N + kMvRows - 1) / kMvRows;
  const int m_chunks = (a.M + a.rows_per_item - 1) / a.rows_per_item;
  B2_REQUIRE(row_blocks * m_chunks <= INT32_MAX / 2, B2_ERR_UNSUPPORTED, "b2_w4_matvec: N = %lld is too large", (long long)a.N);
  a.row_blocks = (int)row_blocks;
  a.items = (int)row_blocks * m_chunks;
  // CTAs of a cluster, each with a chunk at least: the number that makes the longest CTA shortest, counted in chunks, where a
  // row block's exchange counts as one more
  int ctas = 1, clusters = 1;
  int64_t shortest = INT64_MAX;
  for (int n = 1; n <= 8 && (n == 1 || n <= a.chunks); n *= 2) {
    const int64_t each = (a.chunks + n - 1) / n;
    if (RESIDENT && n < 8 && 2 * n <= a.chunks && each * Tile::kXBytes > kMvResidentBytes) continue;      // x would not fit
    int held = 1;
    const int e = mv_clusters((const void *)kernel, ctx->device, n, Tile::kSmem, &held);
    if (e != B2_OK) return e;
    if (held > a.items) held = a.items;
    const int64_t length = (int64_t)((a.items + held - 1) / held) * (each + 1) + (RESIDENT ? each : 0);
    if (length < shortest) shortest = length, ctas = n, clusters = held;
  }
  a.chunks_per_cta = (a.chunks + ctas - 1) / ctas;
  const int other = Tile::kSumBytes + kMvWindows * kMvWindow * 8 + kMvBarrierBytes + (RESIDENT ? a.chunks_per_cta * Tile::kXBytes : 0);
  a.stages = (Tile::kSmem - other) / Tile::kStage;
  if (a.stages > kMvMaxStages) a.stages = kMvMaxStages;
  const int64_t per_cta = (int64_t)a.chunks_per_cta * ((a.items + clusters - 1) / clusters);
  if (a.stages > per_cta) a.stages = per_cta > 0 ? (int)per_cta : 1;
  CUtensorMap code_map = {};
  if (ALIGNED && a.chunks > 0) {
    const int e = mv_map(&code_map, a.codes, (a.K + 1) / 2, a.N, a.ldq, kMvRows);
    if (e != B2_OK) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)clusters, (unsigned)ctas);
  cfg.blockDim = dim3(kMvThreads);
  cfg.dynamicSmemBytes = (size_t)(a.stages * Tile::kStage + other);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = (unsigned)ctas;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = RESIDENT || a.chunks == 0 ? 1 : 2;        // without w4_x_kernel in front there is nothing to overlap
  a.status = (int *)((char *)ctx->fixed + kFixedStatus);
  a.seq = next_launch_seq(ctx);
  B2_CUDA(cudaLaunchKernelEx(&cfg, kernel, (const MvArgs)a, (const CUtensorMap)code_map));
  return B2_OK;
}

template <int NB, bool RESIDENT, bool ALIGNED, bool BF16>
static int w4_matvec_groups(Context *ctx, const MvArgs &a, cudaStream_t s) {
  return a.group_shift == 5   ? w4_matvec_launch<NB, ALIGNED, RESIDENT, 1, BF16>(ctx, a, s)
         : a.group_shift == 6 ? w4_matvec_launch<NB, ALIGNED, RESIDENT, 2, BF16>(ctx, a, s)
                              : w4_matvec_launch<NB, ALIGNED, RESIDENT, 4, BF16>(ctx, a, s);
}
template <int NB, bool RESIDENT>
static int w4_matvec_forms(Context *ctx, const MvArgs &a, bool aligned, cudaStream_t s) {
  if (a.type != B2_F16) return aligned ? w4_matvec_groups<NB, RESIDENT, true, true>(ctx, a, s) : w4_matvec_groups<NB, RESIDENT, false, true>(ctx, a, s);
  return aligned ? w4_matvec_groups<NB, RESIDENT, true, false>(ctx, a, s) : w4_matvec_groups<NB, RESIDENT, false, false>(ctx, a, s);
}
static int w4_matvec_run(Context *ctx, const MvArgs &a, int nb, bool resident, bool aligned, cudaStream_t s) {
  if (resident) return w4_matvec_forms<1, true>(ctx, a, aligned, s);
  return nb == 1   ? w4_matvec_forms<1, false>(ctx, a, aligned, s)
         : nb == 2 ? w4_matvec_forms<2, false>(ctx, a, aligned, s)
                   : w4_matvec_forms<4, false>(ctx, a, aligned, s);
}

// The workspace of a product: the image of x.
static size_t mv_image_bytes(int64_t M, int64_t K, int type) {
  const int nb = mv_blocks(M, type);
  const int64_t items = (M + mv_rows(nb, type) - 1) / mv_rows(nb, type);
  return (size_t)(items * ((K + kMvChunk - 1) / kMvChunk)) * nb * (kMvChunk * 8 * 2);
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

static int w4_group_shift(int group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : 8; }

// Blocks of 256 threads over `units` of a row (x) and the rows (y): as many threads to a row, in powers of two, as it has units
// (at least `least`), the others to further rows.
struct W4Grid {
  dim3 grid, block;
  W4Grid(int64_t units, int64_t rows, int least) {
    int x = least;
    while (x < 256 && x < units) x *= 2;
    block = dim3(x, 256 / x);
    const int64_t gx = (units + x - 1) / x, gy = (rows + block.y - 1) / block.y;
    grid = dim3((unsigned)(gx < 1 << 20 ? gx : 1 << 20), (unsigned)(gy < 65535 ? gy : 65535));
  }
};

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
  (void)ctx;
  const int shift = w4_group_shift(group);
  const int64_t units = ((K + group - 1) / group) * (group / 16);
  const W4Grid g(units, N, group / 16);
  const uintptr_t place = (uintptr_t)W | (uintptr_t)(ldw * tb);
  const int align = (place & 15) == 0 ? 16 : (place & 3) == 0 ? 4 : 2;
  const bool qvec = (((uintptr_t)codes | (uintptr_t)ldq) & 7) == 0;
  cudaError_t launched = cudaSuccess;
  w4_with_types(type, scale_type, [&](auto t, auto s) {
    using T = decltype(t);
    using S = decltype(s);
    constexpr int kLeast = sizeof(T) == 4 ? 4 : 2;
    const auto pick = [&](auto z) {
      constexpr bool Z = decltype(z)::value;
      return align == 16  ? (qvec ? w4_quantize_kernel<T, S, Z, 16, true> : w4_quantize_kernel<T, S, Z, 16, false>)
             : align == 4 ? (qvec ? w4_quantize_kernel<T, S, Z, 4, true> : w4_quantize_kernel<T, S, Z, 4, false>)
                          : (qvec ? w4_quantize_kernel<T, S, Z, kLeast, true> : w4_quantize_kernel<T, S, Z, kLeast, false>);
    };
    const auto kernel = zeros ? pick(std::true_type()) : pick(std::false_type());
    launched = launch_kernel(kernel, g.grid, g.block, 0, (cudaStream_t)stream, N, K, shift, (const T *)W, ldw, codes, ldq, (S *)scales, zeros);
  });
  B2_CUDA(launched);
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
  const int shift = w4_group_shift(group);
  cudaError_t launched = cudaSuccess;
  w4_with_types(type, scale_type, [&](auto t, auto s) {
    using T = decltype(t);
    using S = decltype(s);
    if (transpose) {
      const int64_t tiles = ((N + 63) / 64) * ((K + 63) / 64), most = (int64_t)ctx->sm_count * 8;
      const unsigned grid = (unsigned)(tiles < most ? tiles : most);
      const bool vec = (((uintptr_t)codes | (uintptr_t)ldq) & 7) == 0;
      constexpr bool kPair = sizeof(T) == 2;
      const bool pair = kPair && (((uintptr_t)W | (uintptr_t)(ldw * tb)) & 3) == 0;
      const auto kernel = pair ? (vec ? w4_transpose_kernel<T, S, true, kPair> : w4_transpose_kernel<T, S, false, kPair>)
                               : (vec ? w4_transpose_kernel<T, S, true, false> : w4_transpose_kernel<T, S, false, false>);
      launched = launch_kernel(kernel, grid, 256, 0, (cudaStream_t)stream, N, K, shift, codes, ldq, (const S *)scales, zeros, (T *)W, ldw);
    } else {
      const W4Grid g((K + 31) / 32, N, 1);      // four units of 8 to a thread
      const bool cvec = (((uintptr_t)codes | (uintptr_t)ldq) & 3) == 0, wvec = (((uintptr_t)W | (uintptr_t)(ldw * tb)) & 15) == 0;
      const auto kernel = cvec ? (wvec ? w4_dequantize_kernel<T, S, true, true> : w4_dequantize_kernel<T, S, true, false>)
                               : (wvec ? w4_dequantize_kernel<T, S, false, true> : w4_dequantize_kernel<T, S, false, false>);
      launched = launch_kernel(kernel, g.grid, g.block, 0, (cudaStream_t)stream, N, K, shift, codes, ldq, (const S *)scales, zeros, (T *)W, ldw);
    }
  });
  B2_CUDA(launched);
  return B2_OK;
}

size_t b2_w4_matvec_workspace_bytes(int64_t M, int64_t N, int64_t K, int type) {
  if (M <= 0 || M > kW4MaxRows || N <= 0 || K <= 0 || N > INT32_MAX || K > kW4MaxK || type_bytes(type) == 0) return 0;
  if (mv_resident(M, N, K, type)) return 0;
  return mv_image_bytes(M, K, type);
}

int b2_w4_matvec(b2_handle h, int64_t M, int64_t N, int64_t K, int group, float alpha, int type, const void *x, int64_t ldx,
                 const uint8_t *codes, int64_t ldq, int scale_type, const void *scales, const uint8_t *zeros, float beta,
                 void *y, int64_t ldy, void *workspace, size_t workspace_bytes, void *stream) {
  const int st = w4_check("b2_w4_matvec", N, K, group, type, scale_type, codes, ldq, scales);
  if (st != B2_OK) return st;
  const int tb = type_bytes(type);
  B2_REQUIRE(M >= 0, B2_ERR_INVALID_ARG, "b2_w4_matvec: M = %lld is negative", (long long)M);
  B2_REQUIRE(M <= kW4MaxRows, B2_ERR_UNSUPPORTED,
             "b2_w4_matvec: M = %lld exceeds %d rows: expand the weights with b2_w4_dequantize and use b2_sgemm", (long long)M, kW4MaxRows);
  B2_REQUIRE(K <= kW4MaxK, B2_ERR_UNSUPPORTED, "b2_w4_matvec: K = %lld exceeds %lld", (long long)K, (long long)kW4MaxK);
  B2_REQUIRE(ldx >= K && ldy >= N, B2_ERR_INVALID_ARG, "b2_w4_matvec: ldx = %lld is less than K = %lld or ldy = %lld less than N = %lld",
             (long long)ldx, (long long)K, (long long)ldy, (long long)N);
  if (M == 0 || N == 0) return B2_OK;
  B2_REQUIRE(y != nullptr && (K == 0 || x != nullptr), B2_ERR_INVALID_ARG, "b2_w4_matvec: x or y is NULL");
  B2_REQUIRE((((uintptr_t)x | (uintptr_t)y) & (tb - 1)) == 0, B2_ERR_INVALID_ARG, "b2_w4_matvec: x or y is not aligned to its type");
  B2_REQUIRE(!matrices_overlap(x, M, K * tb, ldx * tb, y, M, N * tb, ldy * tb), B2_ERR_INVALID_ARG, "b2_w4_matvec: y overlaps x");
  const size_t need = b2_w4_matvec_workspace_bytes(M, N, K, type);
  B2_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), B2_ERR_WORKSPACE,
             "b2_w4_matvec: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
  B2_REQUIRE(need == 0 || ((uintptr_t)workspace & 15) == 0, B2_ERR_INVALID_ARG, "b2_w4_matvec: workspace is not 16-byte aligned");
  B2_CONTEXT(ctx, h, "b2_w4_matvec");
  cudaStream_t s = (cudaStream_t)stream;
  MvArgs a = {};
  a.N = N, a.K = alpha != 0.f ? K : 0, a.ldx = ldx, a.ldq = ldq, a.ldy = ldy, a.groups = (K + group - 1) / group;
  a.M = (int)M, a.type = type, a.scale_type = scale_type, a.alpha = alpha, a.beta = beta;
  a.group_shift = w4_group_shift(group);
  a.x = x, a.codes = codes, a.zeros = zeros, a.scales = scales, a.y = y;
  const int nb = mv_blocks(M, type);
  a.parts = mv_parts(type);
  a.rows_per_item = mv_rows(nb, type);
  a.chunks = (int)((a.K + kMvChunk - 1) / kMvChunk);
  a.vec = (((uintptr_t)x | (uintptr_t)(ldx * tb)) & 15) == 0;
  const bool resident = mv_resident(M, N, K, type);
  if (a.chunks > 0 && !resident) {
    a.image = (unsigned char *)workspace;
    cudaError_t launched = cudaSuccess;
    with_type(type, [&](auto t) {
      using T = decltype(t);
      const int64_t units = (int64_t)a.chunks * (kMvChunk / 8);
      launched = launch_kernel(w4_x_kernel<T>, dim3((unsigned)((units + kMvXThreads - 1) / kMvXThreads), (unsigned)M), kMvXThreads, 0, s, K, ldx,
                               a.vec, (const T *)x, a.chunks, nb, a.rows_per_item, (unsigned char *)workspace);
      return 0;
    });
    B2_CUDA(launched);
  }
  const bool aligned = (((uintptr_t)codes | (uintptr_t)ldq) & 15) == 0;
  return w4_matvec_run(ctx, a, nb, resident, aligned, s);
}

}  // extern "C"
