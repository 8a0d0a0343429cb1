// 4-bit weights with group scales: quantise, expand, and the matrix-vector product of decoding steps.
#include <math.h>

#include <mutex>
#include <type_traits>
#include <vector>

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
// A CTA streams tiles of 128 rows x 256 k (16 KB of codes) through a ring of shared-memory stages.  Four producer warps fill
// it: one thread issues the TMA loads of the codes (128-byte swizzle: the 16-byte unit u of row r lies at u ^ (r & 7), so that
// the words that a warp reads lie in 32 banks), the others fetch scales and zero points, eight groups of each row at a time.  Eight consumer warps, 4 (rows) x 2
// (k), multiply 32 rows x 128 k each.  The k range is cut over the CTAs of a cluster, each of which keeps its part of x, already
// cut and paired, in shared memory while it walks over row blocks; the sums of a row block meet over distributed shared memory
// in the order of the ranks: no atomics, no workspace.
constexpr int kMvConsumers = 256, kMvProducers = 128, kMvThreads = kMvConsumers + kMvProducers;
constexpr int kMvRows = 128, kMvChunk = 256, kMvRowBytes = kMvChunk / 2, kMvCodeBytes = kMvRows * kMvRowBytes;
constexpr int kMvPitch = kMvRows + 4;       // of the sums: 8 rows x 4 columns of a warp's store in 32 banks
constexpr int kMvWindow = 1024;             // scales and zero points held together: 8 groups of each row, the group / 32 chunks
constexpr int kMvWindows = 2;               // they span
constexpr int kMvMaxStages = 8, kMvBarrierBytes = 256 + 1024;   // barriers, and room to align

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

template <class T, int NB>
struct MvTile {
  static constexpr int kParts = MvType<T>::kParts;
  static constexpr bool kStream = kParts == 1;                      // 16-bit x comes through the ring as it lies in memory
  static constexpr int kM = 8 * NB / kParts;                        // rows of x per item
  static constexpr int kXBytes = kMvChunk * 8 * NB * 2;             // x of one chunk
  static constexpr int kStage = kMvCodeBytes + (kStream ? kXBytes : 0);
  static constexpr int kSumBytes = 2 * 8 * NB * kMvPitch * 4;
  static constexpr int kCtasPerSm = NB <= 2 ? 2 : 1;
  static constexpr int kSmem = kCtasPerSm == 2 ? 115712 : 232448;   // what a CTA may have
  static constexpr int kXLargest = kStream ? 0 : kCtasPerSm == 2 ? 32768 : 65536;
};

struct MvArgs {
  int64_t N, K, ldx, ldq, ldy, groups;
  int M, group_shift, scale_type, xvec;
  int stages, items, row_blocks, chunks_per_cta, panel_chunks;   // a panel: the chunks whose x is held at a time
  float alpha, beta;
  const void *x;
  const uint8_t *codes, *zeros;
  const void *scales;
  void *y;
  int *status;
  unsigned int seq;
};

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
__device__ __forceinline__ uint4 mv_pair(uint4 h) {
  return make_uint4(__byte_perm(h.x, h.z, 0x5410), __byte_perm(h.x, h.z, 0x7632), __byte_perm(h.y, h.w, 0x5410),
                    __byte_perm(h.y, h.w, 0x7632));
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
    return mv_pair(make_uint4(h[0], h[1], h[2], h[3]));
  }
};

__device__ __forceinline__ void mv_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mv_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The zero point in the form that unpacking subtracts: 8 + z/16 (bf16), 64 + z/16 (f16), in both halves.
__device__ __forceinline__ uint32_t mv_zero(uint32_t z, __nv_bfloat16) { return 0x41004100u | z * 0x00010001u; }
__device__ __forceinline__ uint32_t mv_zero(uint32_t z, __half) { return 0x54005400u | z * 0x00010001u; }

// (w & mask) | bits in one instruction (left to itself the compiler makes two of it, having two constants: 69.5 us for 63.3)
__device__ __forceinline__ uint32_t mv_and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
  return r;
}
// (c - z) / 16 of codes j and j + 4 of a word, j = 0..3.
__device__ __forceinline__ uint32_t mv_unpack(uint32_t w, int j, uint32_t zero, __nv_bfloat16) {
  const uint32_t v = mv_and_or(w >> (4 * j), 0x000f000fu, 0x41004100u);
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), *reinterpret_cast<const __nv_bfloat162 *>(&zero));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t mv_unpack(uint32_t w, int j, uint32_t zero, __half) {
  const uint32_t v = mv_and_or(w >> (4 * j), 0x000f000fu, 0x54005400u);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&v), *reinterpret_cast<const __half2 *>(&zero));
  return *reinterpret_cast<const uint32_t *>(&r);
}

__device__ __forceinline__ float ld_shared_cluster_f32(uint32_t cluster_addr) { return __uint_as_float(ld_shared_cluster_u32(cluster_addr)); }

// A tensor map of `rows` rows of `cols` elements, `pitch` bytes apart, in boxes of 128 bytes x box_rows.
static int mv_map(CUtensorMap *out, CUtensorMapDataType type, int elem, const void *base, int64_t cols, int64_t rows, int64_t pitch,
                  int box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  B2_REQUIRE(fn != nullptr, B2_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {(cuuint32_t)(128 / elem), (cuuint32_t)box_rows}, steps[2] = {1, 1};
  const CUresult r = fn(out, type, 2, (void *)base, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  B2_REQUIRE(r == CUDA_SUCCESS, B2_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d (%lld x %lld, pitch %lld)", (int)r,
             (long long)rows, (long long)cols, (long long)pitch);
  return B2_OK;
}

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
    if (alive && !mbar_wait(bar, parity)) fail();
  }
  __device__ __forceinline__ void cluster(uint64_t *bar, uint32_t parity) {
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

// ALIGNED: rows of codes start on 16-byte boundaries (TMA); otherwise the producers copy them.
// A place in a ring of buffers, and the parity of its turn.
struct MvRing {
  int at = 0, size;
  uint32_t phase = 0;
  __device__ __forceinline__ explicit MvRing(int n) : size(n) {}
  __device__ __forceinline__ void next() {
    if (++at == size) at = 0, phase ^= 1;
  }
};

template <class T, int NB, bool ALIGNED>
__global__ void __launch_bounds__(kMvThreads, MvTile<T, NB>::kCtasPerSm)
    w4_matvec_kernel(const MvArgs a, const __grid_constant__ CUtensorMap code_map, const __grid_constant__ CUtensorMap x_map) {
  using Tile = MvTile<T, NB>;
  using H = typename MvType<T>::half_t;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // the swizzle is one of addresses
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)cluster_ctarank(), ctas = (int)gridDim.y;        // blockIdx.y is the rank within the cluster
  const int first = rank * a.chunks_per_cta;
  int chunks = (int)((a.K + kMvChunk - 1) / kMvChunk) - first;
  chunks = chunks < 0 ? 0 : chunks < a.chunks_per_cta ? chunks : a.chunks_per_cta;
  const int window_log = a.group_shift - 5;                                // chunks of a window: group / 32
  const int64_t width = (a.K + 1) >> 1;
  float2 *const windows = reinterpret_cast<float2 *>(smem + a.stages * Tile::kStage);    // [kMvWindows][row][8]
  unsigned char *const xs = reinterpret_cast<unsigned char *>(windows + kMvWindows * kMvWindow);   // [chunk][block of 32][NB][column][word] x 16 bytes
  float *const sums = reinterpret_cast<float *>(xs + a.panel_chunks * Tile::kXBytes);   // [2][8 NB][kMvPitch]
  uint64_t *const full = reinterpret_cast<uint64_t *>(reinterpret_cast<unsigned char *>(sums) + Tile::kSumBytes);
  uint64_t *const empty = full + kMvMaxStages, *const wfull = empty + kMvMaxStages, *const wempty = wfull + kMvWindows;
  uint64_t *const xfull = wempty + kMvWindows, *const xempty = xfull + 1, *const ready = xfull + 2, *const done = xfull + 3;
  constexpr int kFillers = ALIGNED ? kMvProducers - 32 : kMvProducers;     // threads that write shared memory themselves

  if (tid == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], ALIGNED ? (Tile::kStream && !a.xvec ? 1 + kFillers : 1) : kFillers);
      mbar_init(&empty[s], kMvConsumers / 32);
    }
    for (int s = 0; s < kMvWindows; ++s) {
      mbar_init(&wfull[s], kFillers);
      mbar_init(&wempty[s], kMvConsumers / 32);
    }
    mbar_init(xfull, kFillers);
    mbar_init(xempty, kMvConsumers / 32);
    mbar_init(ready, ctas);
    mbar_init(done, ctas);
    mbar_fence_init();
  }
  __syncthreads();
  cluster_arrive();     // the wait comes before the first word to another CTA
  MvWait wait{a.status, a.seq};

  if (warp >= kMvConsumers / 32) {
    if (ALIGNED && warp == kMvConsumers / 32) {
      if (lane == 0) {
        MvRing ring(a.stages);
        uint32_t sent = 0;
        for (int item = blockIdx.x; item < a.items; item += gridDim.x) {
          const int mc = item / a.row_blocks, row = (item - mc * a.row_blocks) * kMvRows;
          for (int c = 0; c < chunks; ++c, ring.next()) {
            if (sent >= (uint32_t)a.stages) wait(&empty[ring.at], ring.phase ^ 1);
            if (!wait.alive) continue;
            unsigned char *stage = smem + ring.at * Tile::kStage;
            mbar_expect_tx(&full[ring.at], kMvCodeBytes + (Tile::kStream && a.xvec ? Tile::kXBytes : 0));
            tma_load_2d(stage, &code_map, &full[ring.at], (first + c) * kMvRowBytes, row);
            if (Tile::kStream && a.xvec) {      // columns that are not used lie behind M: zeros
#pragma unroll
              for (int q = 0; q < kMvChunk / 64; ++q)
                tma_load_2d(stage + kMvCodeBytes + q * (Tile::kXBytes / 4), &x_map, &full[ring.at], (first + c) * kMvChunk + 64 * q, mc * Tile::kM);
            }
            ++sent;
          }
        }
        ring_settle(full, a.stages, sent);      // nothing is in flight when the CTA leaves, whoever gave up waiting
      }
      __syncwarp();
    } else {
      const int me = tid - kMvConsumers - (ALIGNED ? 32 : 0);
      MvRing ring(a.stages), window(kMvWindows);
      uint32_t filled = 0, opened = 0, xcount = 0;
      int held_mc = -1, held_panel = -1;
      for (int item = blockIdx.x; item < a.items; item += gridDim.x) {
        const int mc = item / a.row_blocks, m0 = mc * Tile::kM;
        const int64_t n0 = (int64_t)(item - mc * a.row_blocks) * kMvRows;
        int panel = 0, in_panel = 0;
        for (int c = 0; c < chunks; ++c) {
          if (!Tile::kStream && (mc != held_mc || panel != held_panel)) {      // this panel's x: 8 elements of k per thread and turn, zeros in unused columns
            held_mc = mc, held_panel = panel;
            if (xcount > 0) wait(xempty, (xcount - 1) & 1);
            ++xcount;
            const int left = chunks - c, n_chunks = left < a.panel_chunks ? left : a.panel_chunks;
            const int64_t k0 = (int64_t)(first + c) * kMvChunk;
            uint4 *to = reinterpret_cast<uint4 *>(xs);
            const int units = n_chunks * (kMvChunk / 8);
            // unit v: 8 elements of k of row v / units; several in flight per thread
            constexpr int kFlight = sizeof(T) == 4 ? 2 : 4, kXRows = (8 * NB + Tile::kParts - 1) / Tile::kParts;
            for (int v0 = me; v0 < kXRows * units; v0 += kFlight * kFillers) {
              MvUnit<T> v[kFlight];
#pragma unroll
              for (int i = 0; i < kFlight; ++i) {
                const int at = v0 + i * kFillers, m = at / units, u = at - m * units;
                v[i] = MvUnit<T>{};
                if (m < Tile::kM && m0 + m < a.M) v[i].load((const T *)a.x + (int64_t)(m0 + m) * a.ldx, k0 + 8 * u, a.K, a.xvec != 0);
              }
#pragma unroll
              for (int i = 0; i < kFlight; ++i) {
                const int at = v0 + i * kFillers, m = at / units, u = at - m * units;
#pragma unroll
                for (int p = 0; p < Tile::kParts; ++p) {
                  const int col = m * Tile::kParts + p;
                  const uint4 h = v[i].part(p);
                  if (col < 8 * NB) to[(((u >> 2) * NB + (col >> 3)) * 8 + (col & 7)) * 4 + (u & 3)] = h;
                }
              }
            }
            mbar_arrive(xfull);
          }
          if ((c & ((1 << window_log) - 1)) == 0) {
            // scales and zero points of a window: entry e is group e & 7 of row e >> 3; all loads before the first use
            constexpr int kTurns = (kMvWindow + kFillers - 1) / kFillers;
            uint32_t scale[kTurns], zero[kTurns];
            const int64_t q0 = ((int64_t)(first + c) * kMvChunk) >> a.group_shift;
            const int count = a.groups - q0 < 8 ? (int)(a.groups - q0) : 8;
            const int64_t n_rows = a.N - n0;
            const int64_t base = n0 * a.groups + q0;
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
              const int e = me + i * kFillers, r = e >> 3, q = e & 7;
              const bool in = e < kMvWindow && r < n_rows && q < count;
              const int64_t at = in ? base + r * a.groups + q : 0;
              scale[i] = a.scale_type == B2_F32 ? ((const uint32_t *)a.scales)[at] : ((const uint16_t *)a.scales)[at];
              zero[i] = a.zeros ? a.zeros[at] : 8;
              if (!in) scale[i] = 0;
            }
            if (opened >= kMvWindows) wait(&wempty[window.at], window.phase ^ 1);
            ++opened;
            float2 *to = windows + window.at * kMvWindow;
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
              const int e = me + i * kFillers;
              const float s = a.scale_type == B2_F32    ? __uint_as_float(scale[i])
                              : a.scale_type == B2_BF16 ? __uint_as_float(scale[i] << 16)
                                                        : __half2float(__ushort_as_half((unsigned short)scale[i]));
              if (e < kMvWindow) to[e] = make_float2(s, __uint_as_float(mv_zero(zero[i] & 15, H())));
            }
            mbar_arrive(&wfull[window.at]);
            window.next();
          }
          if (!ALIGNED || (Tile::kStream && !a.xvec)) {
            if (filled >= (uint32_t)a.stages) wait(&empty[ring.at], ring.phase ^ 1);
            ++filled;
            unsigned char *stage = smem + ring.at * Tile::kStage;
            if constexpr (Tile::kStream) {        // as the TMA would lay it: 128-byte rows of 64 k, 16-byte unit u at u ^ (row & 7)
              const int64_t k0 = (int64_t)(first + c) * kMvChunk;
              constexpr int kFlight = 4;
              for (int v0 = me; v0 < 8 * NB * 32; v0 += kFlight * kFillers) {
                MvUnit<T> v[kFlight];
#pragma unroll
                for (int i = 0; i < kFlight; ++i) {
                  const int m = (v0 + i * kFillers) >> 5, u = (v0 + i * kFillers) & 31;
                  v[i] = MvUnit<T>{};
                  if (m < 8 * NB && m0 + m < a.M) v[i].load((const T *)a.x + (int64_t)(m0 + m) * a.ldx, k0 + 8 * u, a.K, a.xvec != 0);
                }
#pragma unroll
                for (int i = 0; i < kFlight; ++i) {
                  const int m = (v0 + i * kFillers) >> 5, u = (v0 + i * kFillers) & 31;
                  if (m < 8 * NB)
                    *reinterpret_cast<uint4 *>(stage + kMvCodeBytes + (u >> 3) * (Tile::kXBytes / 4) + m * 128 + (((u & 7) ^ (m & 7)) << 4)) =
                        make_uint4(v[i].w[0], v[i].w[1], v[i].w[2], v[i].w[3]);
                }
              }
            }
            if (!ALIGNED) {
              const int64_t at = (int64_t)(first + c) * kMvRowBytes;
              for (int u = me; u < kMvCodeBytes / 16; u += kFillers) {
                const int r = u >> 3, cc = u & 7;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (n0 + r < a.N && at + 16 * cc < width) v = mv_load_any(a.codes + (n0 + r) * a.ldq, at + 16 * cc, width);
                *reinterpret_cast<uint4 *>(stage + r * kMvRowBytes + ((cc ^ (r & 7)) << 4)) = v;
              }
            }
            mbar_arrive(&full[ring.at]);
            ring.next();
          }
          if (++in_panel == a.panel_chunks) in_panel = 0, ++panel;
        }
      }
    }
    __syncwarp();
    cluster_wait();
  } else {
    const int g = lane >> 2, t = lane & 3, wn = warp & 3, wk = warp >> 2;
    // A column of the tensor-core tile holds this row of a streamed x: two neighbouring lanes of a load 4 rows apart, so that
    // its quarter warps fall into different halves of the banks.
    const int xcol = (g >> 1) + 4 * (g & 1);
    uint32_t xcount = 0, turn = 0;
    MvRing ring(a.stages), window(kMvWindows);
    int held_mc = -1, held_panel = -1;
    for (int item = blockIdx.x; item < a.items; item += gridDim.x, ++turn) {
      const int mc = item / a.row_blocks;
      int panel = 0, in_panel = 0;
      float total[2][NB][4] = {};
      for (int c = 0; c < chunks; ++c) {
        if (!Tile::kStream && (mc != held_mc || panel != held_panel)) {
          if (held_mc >= 0) {
            __syncwarp();
            if (lane == 0) mbar_arrive(xempty);
          }
          held_mc = mc, held_panel = panel;
          wait(xfull, xcount & 1);
          ++xcount;
        }
        const int in_window = c & ((1 << window_log) - 1);
        if (in_window == 0) wait(&wfull[window.at], window.phase);
        wait(&full[ring.at], ring.phase);
        const unsigned char *const stage = smem + ring.at * Tile::kStage;
        const unsigned char *codes = stage + (wn * 32 + g) * kMvRowBytes + 4 * t;
        const uint4 *xf = reinterpret_cast<const uint4 *>(xs) + in_panel * (Tile::kXBytes / 16) + lane;
        const unsigned char *xr = stage + kMvCodeBytes + xcol * 128;
        const float2 *sz = windows + window.at * kMvWindow + ((wn * 32 + g) << 3);
        const int block0 = in_window * 8 + wk * 4;                    // this warp's first block of 32 k within the window
        // the warp's 128 k in straight-line code, BLOCKS blocks of 32 to a group (or to the warp's part of one)
        auto multiply = [&](auto blocks) {
          constexpr int BLOCKS = decltype(blocks)::value;
#pragma unroll
          for (int b0 = 0; b0 < 4; b0 += BLOCKS) {
            float sc[4], acc[2][NB][4] = {};
            uint32_t z[4];
            const float2 *from = sz + ((block0 + b0) >> window_log);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float2 v = from[(8 * r) << 3];
              sc[r] = v.x, z[r] = __float_as_uint(v.y);
            }
#pragma unroll
            for (int b4 = b0; b4 < b0 + BLOCKS; ++b4) {
              const int b = wk * 4 + b4;
              uint4 xv[NB];
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) {
                if constexpr (Tile::kStream) {
                  // (wk * 4 + b4) >> 1 and & 1, with b4 known
                  const int unit = ((b4 & 1) * 4 + t) ^ xcol;
                  xv[nb] = mv_pair(*reinterpret_cast<const uint4 *>(xr + (wk * 2 + (b4 >> 1)) * (Tile::kXBytes / 4) + nb * 1024 + (unit << 4)));
                } else {
                  xv[nb] = xf[(b * NB + nb) * 32];
                }
              }
#pragma unroll
              for (int rt = 0; rt < 2; ++rt) {
                const int place = (b ^ g) << 4;                     // rows g, g + 8, ... have one place
                const uint32_t w0 = *reinterpret_cast<const uint32_t *>(codes + (rt * 16) * kMvRowBytes + place);
                const uint32_t w1 = *reinterpret_cast<const uint32_t *>(codes + (rt * 16 + 8) * kMvRowBytes + place);
                const uint32_t z0 = z[2 * rt], z1 = z[2 * rt + 1];
                const uint32_t f[4] = {mv_unpack(w0, 0, z0, H()), mv_unpack(w1, 0, z1, H()), mv_unpack(w0, 1, z0, H()), mv_unpack(w1, 1, z1, H())};
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mv_mma(acc[rt][nb], f, xv[nb].x, xv[nb].y, H());
                const uint32_t h[4] = {mv_unpack(w0, 2, z0, H()), mv_unpack(w1, 2, z1, H()), mv_unpack(w0, 3, z0, H()), mv_unpack(w1, 3, z1, H())};
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mv_mma(acc[rt][nb], h, xv[nb].z, xv[nb].w, H());
              }
            }
#pragma unroll
            for (int rt = 0; rt < 2; ++rt)
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 4; ++i) total[rt][nb][i] = fmaf(sc[2 * rt + (i >> 1)], acc[rt][nb][i], total[rt][nb][i]);
          }
        };
        if (a.group_shift >= 7) multiply(std::integral_constant<int, 4>());
        else if (a.group_shift == 6) multiply(std::integral_constant<int, 2>());
        else multiply(std::integral_constant<int, 1>());
        const bool window_ends = in_window == (1 << window_log) - 1 || c + 1 == chunks;
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&empty[ring.at]);
          if (window_ends) mbar_arrive(&wempty[window.at]);
        }
        ring.next();
        if (window_ends) window.next();
        if (++in_panel == a.panel_chunks) in_panel = 0, ++panel;
      }

      __syncwarp();
      // the row block's sums: this CTA's two k halves side by side, then every rank's, in the order of the ranks
      if (turn == 0) cluster_wait();                                // every CTA's barriers are set up
      else if (ctas > 1) wait.cluster(done, (turn - 1) & 1);        // every CTA has read the sums of the block before
#pragma unroll
      for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int col = 2 * t + (i & 1), m = Tile::kStream ? (col >> 1) + 4 * (col & 1) : col;
            sums[(wk * 8 * NB + nb * 8 + m) * kMvPitch + wn * 32 + rt * 16 + g + (i >> 1) * 8] = total[rt][nb][i];
          }
      mv_consumers_sync();
      if (ctas > 1) {
        if (tid < ctas) mbar_arrive_cluster(mapa_u32(smem_u32(ready), (uint32_t)tid));
        wait.cluster(ready, turn & 1);
      }
      const int m0 = mc * Tile::kM, mm = a.M - m0 < Tile::kM ? a.M - m0 : Tile::kM;
      const int64_t n0 = (int64_t)(item - mc * a.row_blocks) * kMvRows;
      for (int i = tid + rank * kMvConsumers; i < mm * kMvRows; i += kMvConsumers * ctas) {
        const int m = i / kMvRows, r = i % kMvRows;
        const float *at = sums + m * Tile::kParts * kMvPitch + r;
        float v = 0.f;
        if (ctas > 1) {
          for (int q = 0; q < ctas; ++q) {
            const uint32_t from = mapa_u32(smem_u32(at), (uint32_t)q);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int p = 0; p < Tile::kParts; ++p) v += ld_shared_cluster_f32(from + (k * 8 * NB + p) * kMvPitch * 4);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int p = 0; p < Tile::kParts; ++p) v += at[(k * 8 * NB + p) * kMvPitch];
        }
        if (n0 + r < a.N) {
          T *to = (T *)a.y + (int64_t)(m0 + m) * a.ldy + n0 + r;
          v = a.alpha * (16.f * v);
          *to = from_f32<T>(a.beta != 0.f ? fmaf(a.beta, to_f32(*to), v) : v);
        }
      }
      mv_consumers_sync();
      if (ctas > 1 && tid < ctas) mbar_arrive_cluster(mapa_u32(smem_u32(done), (uint32_t)tid));
    }
  }
  __syncwarp();
  cluster_sync_all();     // nobody leaves while its sums may still be read or its barriers reached
}

// Clusters of `ctas` CTAs with `smem` bytes each that the device holds at once, asked once per kernel, size and device.
static int mv_clusters(const void *kernel, int device, int ctas, int smem, int *out) {
  struct Entry {
    const void *kernel;
    int device, ctas, smem, clusters;
  };
  static std::vector<Entry> known;
  static std::mutex mu;
  std::lock_guard<std::mutex> lk(mu);
  for (const Entry &e : known)
    if (e.kernel == kernel && e.device == device && e.ctas == ctas && e.smem == smem) {
      *out = e.clusters;
      return B2_OK;
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
  known.push_back({kernel, device, ctas, smem, n < 1 ? 1 : n});
  *out = n < 1 ? 1 : n;
  return B2_OK;
}

template <class T, int NB, bool ALIGNED>
static int w4_matvec_launch(Context *ctx, MvArgs a, cudaStream_t s) {
  using Tile = MvTile<T, NB>;
  const auto kernel = w4_matvec_kernel<T, NB, ALIGNED>;
  const int st = ensure_func_attributes((const void *)kernel, ctx->device, Tile::kSmem);
  if (st != B2_OK) return st;
  const int64_t row_blocks = (a.N + kMvRows - 1) / kMvRows, chunks = (a.K + kMvChunk - 1) / kMvChunk;
  const int m_chunks = (a.M + Tile::kM - 1) / Tile::kM;
  B2_REQUIRE(row_blocks * m_chunks <= INT32_MAX / 2, B2_ERR_UNSUPPORTED, "b2_w4_matvec: N = %lld is too large", (long long)a.N);
  a.row_blocks = (int)row_blocks;
  a.items = (int)row_blocks * m_chunks;
  // CTAs of a cluster, each with a chunk at least: the number that makes the longest CTA shortest, counted in chunks.  A row
  // block's exchange counts as one more, and so does bringing x of a chunk into shared memory: once if all of a CTA's part
  // fits, for every row block if not.
  const int largest = Tile::kXLargest / Tile::kXBytes;
  int ctas = 1, clusters = 1;
  int64_t shortest = INT64_MAX;
  for (int n = 1; n <= 8 && (n == 1 || n <= chunks); n *= 2) {
    int held = 1;
    const int e = mv_clusters((const void *)kernel, ctx->device, n, Tile::kSmem, &held);
    if (e != B2_OK) return e;
    if (held > a.items) held = a.items;
    const int64_t turns = (a.items + held - 1) / held, each = (chunks + n - 1) / n;
    const int64_t length = turns * (each + 1) + (Tile::kStream ? 0 : each <= largest ? each : turns * each);
    if (length < shortest) shortest = length, ctas = n, clusters = held;
  }
  a.chunks_per_cta = (int)((chunks + ctas - 1) / ctas);
  a.panel_chunks = a.chunks_per_cta < largest ? a.chunks_per_cta : largest;
  const int other = a.panel_chunks * Tile::kXBytes + Tile::kSumBytes + kMvWindows * kMvWindow * 8 + kMvBarrierBytes;
  a.stages = (Tile::kSmem - other) / Tile::kStage;
  if (a.stages > kMvMaxStages) a.stages = kMvMaxStages;
  const int64_t per_cta = (int64_t)a.chunks_per_cta * ((a.items + clusters - 1) / clusters);
  if (a.stages > per_cta) a.stages = per_cta > 0 ? (int)per_cta : 1;
  CUtensorMap code_map = {}, x_map = {};
  if (ALIGNED && a.K > 0) {
    int e = mv_map(&code_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.codes, (a.K + 1) / 2, a.N, a.ldq, kMvRows);
    if (e == B2_OK && Tile::kStream && a.xvec)
      e = mv_map(&x_map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, a.x, a.K, a.M, a.ldx * 2, 8 * NB);
    if (e != B2_OK) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)clusters, (unsigned)ctas);
  cfg.blockDim = dim3(kMvThreads);
  cfg.dynamicSmemBytes = (size_t)(a.stages * Tile::kStage + other);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = (unsigned)ctas;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  a.status = (int *)((char *)ctx->fixed + kFixedStatus);
  a.seq = next_launch_seq(ctx);
  B2_CUDA(cudaLaunchKernelEx(&cfg, kernel, (const MvArgs)a, (const CUtensorMap)code_map, (const CUtensorMap)x_map));
  return B2_OK;
}

template <class T, bool ALIGNED>
static int w4_matvec_rows(Context *ctx, const MvArgs &a, cudaStream_t s) {
  if constexpr (sizeof(T) == 4) {
    if (a.M <= 2) return w4_matvec_launch<T, 1, ALIGNED>(ctx, a, s);
    if (a.M <= 5) return w4_matvec_launch<T, 2, ALIGNED>(ctx, a, s);
    return w4_matvec_launch<T, 3, ALIGNED>(ctx, a, s);
  } else {
    if (a.M <= 8) return w4_matvec_launch<T, 1, ALIGNED>(ctx, a, s);
    if (a.M <= 16) return w4_matvec_launch<T, 2, ALIGNED>(ctx, a, s);
    return w4_matvec_launch<T, 4, ALIGNED>(ctx, a, s);
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
  a.xvec = (((uintptr_t)x | (uintptr_t)(ldx * tb)) & 15) == 0;
  return with_type(type, [&](auto t) {
    using T = decltype(t);
    return aligned ? w4_matvec_rows<T, true>(ctx, a, (cudaStream_t)stream) : w4_matvec_rows<T, false>(ctx, a, (cudaStream_t)stream);
  });
}

}  // extern "C"
