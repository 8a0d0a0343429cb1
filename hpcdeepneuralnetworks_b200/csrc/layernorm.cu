// Layer norm, forward and backward: both are bound by memory (the forward pass reads x and writes y, the backward pass reads x
// and dy and writes dx), so every row is read once and kept in registers while its sums are formed.
//
// A row belongs to a team of warps, a thread holds up to 32 elements of it (16 backward), V neighbouring ones to an access.  V is
// the widest access that every row pointer, the pitches and cols allow (16 bytes, 4 bytes, one element); rows that fit none but
// are off by the same amount in all matrices are taken in 16 bytes with their ends masked (PHASED).  Longer rows are read again
// instead of held.
// Measured, device time: forward 16384 x 4096 bf16 48.2 us (5.6 TB/s of the 268 MB it must move, 0.86 of a copy), 8192 x 4095
// 43 us; 8 x 4096 2.7 us, a launch's latency.  Backward 16384 x 4096 68.4 us (5.9 TB/s, 0.91), 8192 x 4095 64 us, 5003 x 1027 FP32
// 20.5 us, 64 x 4096 6.6 us.  Both run at memory speed where rows are whole accesses and there are waves of them; what holds the others back is the
// latency of a row's two sums, with 10 to 16 warps to an SM.
#include <math.h>

#include <initializer_list>
#include <mutex>
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
// W = 1 or 2 FP32 values that are worked on together: sm_100 adds, multiplies and fuses two at a time, and these kernels spend
// as many issue slots on arithmetic as the memory leaves them.
template <int W>
struct LnF;
template <>
struct LnF<1> {
  float v;
  __device__ __forceinline__ LnF() {}
  __device__ __forceinline__ explicit LnF(float a) : v(a) {}
  __device__ __forceinline__ LnF operator+(LnF o) const { return LnF(__fadd_rn(v, o.v)); }
  __device__ __forceinline__ LnF operator*(LnF o) const { return LnF(__fmul_rn(v, o.v)); }
  __device__ __forceinline__ float sum() const { return v; }
};
__device__ __forceinline__ LnF<1> ln_fma(LnF<1> a, LnF<1> b, LnF<1> c) { return LnF<1>(__fmaf_rn(a.v, b.v, c.v)); }
template <>
struct LnF<2> {
  uint64_t v;
  __device__ __forceinline__ LnF() {}
  __device__ __forceinline__ LnF(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit LnF(float a) : LnF(a, a) {}
  __device__ __forceinline__ float2 both() const {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
  }
  __device__ __forceinline__ LnF operator+(LnF o) const {
    LnF r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(v), "l"(o.v));
    return r;
  }
  __device__ __forceinline__ LnF operator*(LnF o) const {
    LnF r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(v), "l"(o.v));
    return r;
  }
  __device__ __forceinline__ float sum() const {
    const float2 r = both();
    return r.x + r.y;
  }
};
__device__ __forceinline__ LnF<2> ln_fma(LnF<2> a, LnF<2> b, LnF<2> c) {
  LnF<2> r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// V elements of type T as one access, and their values, W at a time.
template <class T, int V>
struct LnPack {
  using raw_t = typename LnRaw<V * sizeof(T)>::type;
  static constexpr int W = V >= 2 ? 2 : 1, kParts = V / W;
  using F = LnF<W>;
  union {
    raw_t raw;
    T e[V];
    uint32_t words[V * sizeof(T) >= 4 ? V * sizeof(T) / 4 : 1];
  };
  __device__ __forceinline__ LnPack() {}
  __device__ __forceinline__ void load_stream(const T *p) { raw = __ldcs(reinterpret_cast<const raw_t *>(p)); }   // read once
  __device__ __forceinline__ void load(const T *p) { raw = *reinterpret_cast<const raw_t *>(p); }
  __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<raw_t *>(p) = raw; }
  __device__ __forceinline__ F get(int i) const {
    if constexpr (W == 1) return F(to_f32(e[0]));
    else if constexpr (sizeof(T) == 4) return F(e[2 * i], e[2 * i + 1]);
    else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&words[i]));
      return F(f.x, f.y);
    } else return F(__uint_as_float(words[i] << 16), __uint_as_float(words[i] & 0xffff0000u));
  }
  __device__ __forceinline__ void set(int i, F f) {
    if constexpr (W == 1) e[0] = from_f32<T>(f.v);
    else {
      const float2 r = f.both();
      if constexpr (sizeof(T) == 4) e[2 * i] = r.x, e[2 * i + 1] = r.y;
      else if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(r.x, r.y);
        words[i] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(r.x, r.y);
        words[i] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
  }
};
// V values of a parameter vector (16-byte accesses where V elements are that long or longer), or a constant without one.
template <class P, int V>
__device__ __forceinline__ void ln_params(LnF<(V >= 2 ? 2 : 1)> (&v)[V >= 2 ? V / 2 : 1], const P *p, int at, float without) {
  constexpr int W = V * (int)sizeof(P) > 16 ? 16 / (int)sizeof(P) : V;
  if (!p) {
#pragma unroll
    for (int i = 0; i < (V >= 2 ? V / 2 : 1); ++i) v[i] = LnF<(V >= 2 ? 2 : 1)>(without);
    return;
  }
#pragma unroll
  for (int i = 0; i < V; i += W) {
    LnPack<P, W> q;
    q.load(p + at + i);
#pragma unroll
    for (int k = 0; k < LnPack<P, W>::kParts; ++k) v[i / LnPack<P, W>::W + k] = q.get(k);
  }
}

// ---- teams --------------------------------------------------------------------------------------------
// A row belongs to a team of `share` threads, whole warps; a block holds blockDim.x / share teams, each with rows of its own.
// Each warp takes a run of the row, `turns` accesses of 32 lanes one behind the other: access i of a thread lies i * 32 * V
// elements behind its first, a distance that is known when the kernel is compiled (with the threads' number in it instead, the
// addresses took more instructions than the arithmetic).  FULL: every access of every thread lies within the row.
struct LnTeam {
  int team, teams, tid, warps, lane;
  int64_t step, first;      // a team's rows: first, first + step, ...
  __device__ __forceinline__ explicit LnTeam(int share) {
    team = (int)threadIdx.x / share;
    teams = (int)blockDim.x / share;
    tid = (int)threadIdx.x - team * share;
    warps = share >> 5;
    lane = threadIdx.x & 31;
    step = (int64_t)gridDim.x * teams;
    first = (int64_t)blockIdx.x * teams + team;
  }
  __device__ __forceinline__ int unit(int turns) const { return (tid >> 5) * 32 * turns + lane; }      // first unit of V elements
  // accesses of this thread that lie within the row
  __device__ __forceinline__ int valid(int units, int turns) const {
    const int n = (units - unit(turns) + 31) >> 5;
    return n < 0 ? 0 : n < turns ? n : turns;
  }
  __device__ __forceinline__ void sync() const { asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(32 * warps) : "memory"); }
};
using LnScratch = float[2][32];      // [value][warp of the block]

// Sums of two values over a team, the same bits in each thread, in a fixed order.  The lower half of a warp adds the first
// value and the upper half the second, which takes half the shuffles.  A caller's next sum uses another scratch, so that one
// barrier per sum is enough.
__device__ __forceinline__ float2 ln_sum2(float2 v, LnScratch &scratch, const LnTeam &t) {
  const bool up = t.lane & 16;
  float keep = (up ? v.y : v.x) + __shfl_xor_sync(0xffffffffu, up ? v.x : v.y, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) keep += __shfl_xor_sync(0xffffffffu, keep, o);
  if (t.warps > 1) {
    if ((t.lane & 15) == 0) scratch[up][threadIdx.x >> 5] = keep;
    t.sync();
    const float *from = &scratch[up][t.team * t.warps];
    const int w = t.lane & 15;
    keep = (w < t.warps ? from[w] : 0.f) + (w + 16 < t.warps ? from[w + 16] : 0.f);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) keep += __shfl_xor_sync(0xffffffffu, keep, o);
  }
  const float other = __shfl_xor_sync(0xffffffffu, keep, 16);
  return up ? make_float2(other, keep) : make_float2(keep, other);
}
__device__ __forceinline__ float ln_sum(float v, LnScratch &scratch, const LnTeam &t) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (t.warps > 1) {
    if (t.lane == 0) scratch[0][threadIdx.x >> 5] = v;
    t.sync();
    v = t.lane < t.warps ? scratch[0][t.team * t.warps + t.lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

// A parameter vector in FP32 in shared memory, [warp of a team][access][16 bytes of it][lane]: read from memory, two 16-byte
// halves of every 32 bytes apart, gamma and beta together took as long as x and y.
template <int V, int N>
struct LnWeights {
  static constexpr int G = V >= 4 ? 4 : V;      // elements per access
  using Pack = LnPack<float, G>;
  Pack *at;
  __device__ __forceinline__ LnWeights(float *base, const LnTeam &t)
      : at(reinterpret_cast<Pack *>(base) + (t.tid >> 5) * N * (V / G) * 32 + t.lane) {}
  // p: of the thread's first column; CUT: which of the columns lie in the row is to be looked at (others read some parameter)
  template <class P, bool CUT>
  __device__ __forceinline__ void put(const P *p, int col, int cols, int valid, float without) {
    for (int i = 0; i < N; ++i) {
      if (i >= valid && !CUT) break;
#pragma unroll
      for (int q = 0; q < V / G; ++q) {
        Pack w;
#pragma unroll
        for (int k = 0; k < G; ++k) {
          int c = i * 32 * V + q * G + k;
          if (CUT) c = min(max(c, -col), cols - 1 - col);
          w.e[k] = p ? to_f32(p[c]) : without;
        }
        at[(i * (V / G) + q) * 32] = w;
      }
    }
  }
  __device__ __forceinline__ void get(LnF<(V >= 2 ? 2 : 1)> (&v)[V >= 2 ? V / 2 : 1], int i) const {
#pragma unroll
    for (int q = 0; q < V / G; ++q) {
      const Pack w = at[(i * (V / G) + q) * 32];
#pragma unroll
      for (int k = 0; k < Pack::kParts; ++k) v[q * Pack::kParts + k] = w.get(k);
    }
  }
};

// Rows to come are fetched by cp.async, each thread's elements into places of its own, so that no barrier guards them:
// `kLnAhead` rows besides the one in hand, or none where a block's memory does not hold them.  (FP16 and bf16 elements that
// must be read one by one have no cp.async of their size and go through registers.)
constexpr int kLnAhead = 2;
__device__ __forceinline__ void ln_copy_async(void *smem, const void *global, int bytes) {
  if (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(global) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem)), "l"(global) : "memory");
}
__device__ __forceinline__ void ln_copy_async_16(void *smem, const void *global, int bytes) {      // the first `bytes`, and 0 behind them
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(global), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ln_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void ln_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// Clears the places of a thread's accesses outside the row, once: nothing is ever fetched there, and the loops over a row need no
// conditions (with one around each access: 16384 x 2052 FP32 backward 152 us instead of 86).
template <class Pack>
__device__ __forceinline__ void ln_clear(Pack *at, int slot, int slots, int valid, int accesses) {
  for (int s = 0; s < slots; ++s)
    for (int i = valid; i < accesses; ++i) {
      Pack zero;
      memset(&zero, 0, sizeof(zero));
      at[s * slot + i * 32] = zero;
    }
}

// PHASED: rows that start anywhere, in accesses of 16 bytes all the same.  The rows of all matrices start equally far behind a
// 16-byte boundary, a team's rows do so too (its step is a multiple of V rows), and a thread's accesses lie on the boundaries: a
// thread's columns stay the same from row to row.  A row's first access may begin with elements of the row before it, which
// count as 0, and its last is cut off where the row ends (0 again); both are written element by element.
template <int V>
struct LnPhase {
  int col, cols, shift;     // column of a thread's first element (in front of the row if negative); columns; V - 1 or less
  bool front, edge;         // the thread has the row's first access, and it is such a one; has the first or the last
  __device__ __forceinline__ LnPhase(int shift, int col, int cols, int valid) : col(col), cols(cols), shift(shift) {
    front = valid > 0 && col < 0;
    edge = front || (valid > 0 && col + (valid - 1) * 32 * V + V > cols);
  }
  __device__ __forceinline__ bool inside(int i, int e) const { return (unsigned)(col + i * 32 * V + e) < (unsigned)cols; }
  template <class T>
  __device__ __forceinline__ void fetch(void *smem, const T *from, int i) const {
    const int left = cols - (col + i * 32 * V);
    ln_copy_async_16(smem, from, left < V ? left * (int)sizeof(T) : 16);
  }
  // Parameters of access i; outside the row, some others (all loads at once, without conditions).
  template <class P>
  __device__ __forceinline__ void params(LnF<2> (&v)[V / 2 + (V == 1)], const P *p, int i, float without) const {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      const int c = col + i * 32 * V + 2 * k, c0 = min(max(c, 0), cols - 1), c1 = min(max(c + 1, 0), cols - 1);
      v[k] = p ? LnF<2>(to_f32(p[c0]), to_f32(p[c1])) : LnF<2>(without);
    }
  }
  template <class T>
  __device__ __forceinline__ void clear_front(LnPack<T, V> &p) const {
    if (front) {
#pragma unroll
      for (int e = 0; e < V - 1; ++e)
        if (e < shift) p.e[e] = from_f32<T>(0.f);
    }
  }
  template <class T>
  __device__ __forceinline__ void store(const LnPack<T, V> &out, T *to, int i) const {
    if (!edge) out.store(to);
    else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (inside(i, e)) to[e] = out.e[e];
    }
  }
};

// The variance of a row is that of the distances from a first mean, and what the first mean was off by (`off`, the mean of those
// distances) is taken out of both: a large mean costs no digits.  In a constant row, or one that varies by less than the last digits
// of its mean, square - off^2 is what the roundings of its two parts leave, of either sign: each is good to D * 2^-24 of itself, D =
// 48 + cols / 256 additions deep, together 3 D 2^-24 off^2, and what is below that counts as 0 (NaN is not).  So a constant row's
// rstd is 1 / sqrt(eps) and its outputs beta, whatever its value.  Forming the distances a second time would resolve spreads below a
// hundredth of the mean's last digit too; its code cost all rows 1 to 9 % in the best of the arrangements tried (this: 0 to 3 %).
__device__ __forceinline__ float ln_noise(int cols) { return ((float)cols * (3.f / 256.f) + 144.f) * 0x1p-24f; }
__device__ __forceinline__ float ln_variance(float off, float square, float noise) {
  const float v = fmaf(-off, off, square);
  return v < off * off * noise ? 0.f : v;
}

// y = (x - mean) * rstd * gamma + beta, E elements of the row per thread.
template <class T, class P, int V, int E, int THREADS, bool FULL, bool PHASED>
__global__ void __launch_bounds__(THREADS) layernorm_kernel(int64_t rows, int cols, int share, int turns, int ahead, float eps, const T *x,
                                                            int64_t ldx, const P *gamma, const P *beta, T *y, int64_t ldy, float *mean,
                                                            float *rstd) {
  using Pack = LnPack<T, V>;
  using F = typename Pack::F;
  constexpr int N = E / V, K = Pack::kParts;
  constexpr bool RING = V * sizeof(T) >= 4, ALL = FULL || RING;      // ALL: accesses outside the row read zeros
  // gamma and beta: in registers over the rows, in shared memory, or (the longest rows) read again for each row
  constexpr bool HOLD = E <= 16, SHARED = !HOLD && THREADS <= 512;
  __shared__ LnScratch scratch[2];
  extern __shared__ __align__(16) unsigned char dynamic[];
  const LnTeam t(share);
  if (FULL) turns = N;
  const int shift = PHASED ? (int)((uintptr_t)(x + t.first * ldx) & 15) / (int)sizeof(T) : 0;
  const int valid = FULL ? N : t.valid((cols + shift + V - 1) / V, turns);
  const int64_t col = (int64_t)t.unit(turns) * V - shift;
  const LnPhase<V> phase(shift, (int)col, cols, PHASED ? valid : 0);
  const float inv = 1.f / (float)cols, noise = ln_noise(cols);
  const T *px = x + t.first * ldx + col;                    // the next row to fetch
  T *py = y + t.first * ldy + col;
  const P *const pg = gamma ? gamma + col : nullptr, *const pb = beta ? beta + col : nullptr;
  const int64_t x_step = t.step * ldx, y_step = t.step * ldy;
  int64_t next = t.first;
  // RING: [ahead + 1][warp][N][lane], so that a thread's accesses are a known distance apart
  Pack *const ring = reinterpret_cast<Pack *>(dynamic) + (threadIdx.x >> 5) * 32 * N + t.lane;
  const int slot = (int)blockDim.x * N;
  Pack *fetched = ring, *in_hand = ring, *const ring_end = ring + (ahead + 1) * slot;
  Pack v[N];
  if constexpr (RING && !FULL) ln_clear(ring, slot, ahead + 1, valid, N);
  auto fetch = [&]() {
    if (next < rows) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (FULL || i < valid) {
          if constexpr (PHASED) phase.fetch(fetched + i * 32, px + i * 32 * V, i);
          else if constexpr (RING) ln_copy_async(fetched + i * 32, px + i * 32 * V, V * sizeof(T));
          else v[i].load_stream(px + i * 32 * V);
        }
    }
    if constexpr (RING) {
      ln_commit();
      fetched += slot;
      if (fetched == ring_end) fetched = ring;
    }
    next += t.step;
    px += x_step;
  };
  if constexpr (RING)
    for (int i = 0; i < ahead; ++i) fetch();
  F g[HOLD ? N : 1][K], b[HOLD ? N : 1][K];
  using Weights = LnWeights<V, N>;
  float *const shared_params = reinterpret_cast<float *>(dynamic + (RING ? (ahead + 1) * slot * sizeof(Pack) : 0));
  Weights weights_g(shared_params + (PHASED ? 2 * t.team * share * E : 0), t), weights_b(shared_params + (PHASED ? 2 * t.team + 1 : 1) * share * E, t);
  if constexpr (SHARED) {
    if (PHASED || t.team == 0) {
      weights_g.template put<P, PHASED>(pg, (int)col, cols, valid, 1.f);
      weights_b.template put<P, PHASED>(pb, (int)col, cols, valid, 0.f);
    }
    __syncthreads();
  }
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (FULL || i < valid) {
        if constexpr (PHASED) {
          phase.params(g[i], gamma, i, 1.f);
          phase.params(b[i], beta, i, 0.f);
        } else {
          ln_params<P, V>(g[i], pg, i * 32 * V, 1.f);
          ln_params<P, V>(b[i], pb, i * 32 * V, 0.f);
        }
      }
  }
  for (int64_t row = t.first; row < rows; row += t.step, py += y_step) {
    fetch();
    if constexpr (RING) {
      if (ahead == 2) ln_wait<2>();
      else if (ahead == 1) ln_wait<1>();
      else ln_wait<0>();
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = in_hand[i * 32];
      in_hand += slot;
      if (in_hand == ring_end) in_hand = ring;
    }
    if constexpr (PHASED) phase.clear_front(v[0]);
    F f[N * K], s(0.f);
    const F part(inv);      // each term is divided: sums of values near the type's largest stay within FP32
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || i < valid) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          f[i * K + k] = v[i].get(k);
          s = ln_fma(f[i * K + k], part, s);
        }
      }
    float m = ln_sum(s.sum(), scratch[0], t);
    F d1(0.f), d2(0.f);
    if constexpr (ALL && !FULL) {
      if (valid < N || (PHASED && phase.edge)) {      // what is outside the row lies at the mean
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int k = 0; k < K; ++k) {
            if constexpr (PHASED) {
              const float2 r = f[i * K + k].both();
              f[i * K + k] = F(i < valid && phase.inside(i, 2 * k) ? r.x : m, i < valid && phase.inside(i, 2 * k + 1) ? r.y : m);
            } else if (i >= valid) {
              f[i * K + k] = F(m);
            }
          }
      }
    }
    const F less(-m);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || i < valid) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const F e = f[i * K + k] + less;
          d1 = ln_fma(e, part, d1);
          d2 = ln_fma(e, e, d2);
        }
      }
    const float2 d = ln_sum2(make_float2(d1.sum(), d2.sum()), scratch[1], t);
    const float off = d.x;
    m += off;
    const float r = rsqrtf(ln_variance(off, d.y * inv, noise) + eps);
    if (t.tid == 0) {
      if (mean) mean[row] = m;
      if (rstd) rstd[row] = r;
    }
    const F minus(-m), by(r);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || i < valid) {
        if constexpr (SHARED) {
          weights_g.get(g[0], i);
          weights_b.get(b[0], i);
        } else if constexpr (!HOLD) {
          if (FULL || i < valid) {
            ln_params<P, V>(g[0], pg, i * 32 * V, 1.f);
            ln_params<P, V>(b[0], pb, i * 32 * V, 0.f);
          }
        }
        Pack out;
#pragma unroll
        for (int k = 0; k < K; ++k) out.set(k, ln_fma((f[i * K + k] + minus) * by, g[HOLD ? i : 0][k], b[HOLD ? i : 0][k]));
        if (FULL || i < valid) {
          if constexpr (PHASED) phase.store(out, py + i * 32 * V, i);
          else out.store(py + i * 32 * V);
        }
      }
  }
}

// The same for rows that are too long to hold: one block per row, read three times (from L2 after the first).
template <class T, class P, int V>
__global__ void __launch_bounds__(1024) layernorm_long_kernel(int64_t rows, int cols, float eps, const T *x, int64_t ldx, const P *gamma,
                                                              const P *beta, T *y, int64_t ldy, float *mean, float *rstd) {
  using F = typename LnPack<T, V>::F;
  constexpr int K = LnPack<T, V>::kParts;
  __shared__ LnScratch scratch[2];
  const LnTeam t(1024);
  const float inv = 1.f / (float)cols, noise = ln_noise(cols);
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * ldx;
    LnPack<T, V> v;
    F s(0.f);
    for (int64_t i = (int64_t)threadIdx.x * V; i < cols; i += 1024 * V) {
      v.load(xr + i);
#pragma unroll
      for (int k = 0; k < K; ++k) s = ln_fma(v.get(k), F(inv), s);
    }
    float m = ln_sum(s.sum(), scratch[0], t);
    F d1(0.f), d2(0.f);
    for (int64_t i = (int64_t)threadIdx.x * V; i < cols; i += 1024 * V) {
      v.load(xr + i);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const F e = v.get(k) + F(-m);
        d1 = ln_fma(e, F(inv), d1);
        d2 = ln_fma(e, e, d2);
      }
    }
    const float2 d = ln_sum2(make_float2(d1.sum(), d2.sum()), scratch[1], t);
    const float off = d.x;
    m += off;
    const float r = rsqrtf(ln_variance(off, d.y * inv, noise) + eps);
    if (threadIdx.x == 0) {
      if (mean) mean[row] = m;
      if (rstd) rstd[row] = r;
    }
    for (int64_t i = (int64_t)threadIdx.x * V; i < cols; i += 1024 * V) {
      F g[K], b[K];
      v.load(xr + i);
      ln_params<P, V>(g, gamma, (int)i, 1.f);
      ln_params<P, V>(b, beta, (int)i, 0.f);
#pragma unroll
      for (int k = 0; k < K; ++k) v.set(k, ln_fma((v.get(k) + F(-m)) * F(r), g[k], b[k]));
      v.store(y + row * ldy + i);
    }
  }
}

constexpr __host__ __device__ int ln_padded(int cols) { return cols + (cols >> 5) + 1; }

// Backward: a team walks over its rows and keeps the sums dy * xhat and dy of its columns in registers over all of them; the
// teams' sums meet in shared memory and end as one line of `partial` per block (team after team into one line: 600 x 4096 bf16
// 19.5 us instead of 11.6, 60 x 300 FP32 11.3 instead of 5.5).
//   xhat = (x - mean) * rstd,  u = dy * gamma,  dx = rstd * (u - sum(u) / n - xhat * sum(u * xhat) / n)
// dx may be dy: a thread writes only what it has read.
template <class T, class P, int V, int E, bool FULL, bool PHASED>
__global__ void __launch_bounds__(512, 1) layernorm_backward_kernel(int64_t rows, int cols, int share, int turns, const T *dy, int64_t lddy,
                                                                 const T *x, int64_t ldx, const P *gamma, const float *mean,
                                                                 const float *rstd, T *dx, int64_t lddx, float *partial) {
  using Pack = LnPack<T, V>;
  using F = typename Pack::F;
  constexpr int N = E / V, K = Pack::kParts, W = Pack::W;
  constexpr bool RING = V * sizeof(T) >= 4, ALL = FULL || RING;      // ALL: accesses outside the row read zeros
  // When x - mean is multiplied by rstd: at once costs an instruction less (16384 x 4096 bf16 68 us, late 73), late shortens the way to
  // the sums (FP32 rows that do not fill their team, 16384 x 2052: 79 us, at once 87; no difference where they do).
  constexpr bool LATE = sizeof(T) == 4 && V == 4 && !FULL && !PHASED;
  __shared__ LnScratch scratch[2];
  extern __shared__ __align__(16) unsigned char dynamic[];
  float *const joined = reinterpret_cast<float *>(dynamic);                // at the end: [team][2][ln_padded(cols)]
  pdl_launch_dependents();
  const LnTeam t(share);
  if (FULL) turns = N;
  LnWeights<V, N> weights(reinterpret_cast<float *>(dynamic + (RING ? (kLnAhead + 1) * 2 * N * sizeof(Pack) * blockDim.x : 0)) + (PHASED ? t.team * share * E : 0), t);
  const int shift = PHASED ? (int)((uintptr_t)(x + t.first * ldx) & 15) / (int)sizeof(T) : 0;
  const int valid = FULL ? N : t.valid((cols + shift + V - 1) / V, turns);
  const int64_t col = (int64_t)t.unit(turns) * V - shift;
  const LnPhase<V> phase(shift, (int)col, cols, PHASED ? valid : 0);
  const float inv = 1.f / (float)cols;
  F dg[N * K], db[N * K];
#pragma unroll
  for (int i = 0; i < N * K; ++i) dg[i] = F(0.f), db[i] = F(0.f);
  const T *px = x + t.first * ldx + col, *pg = dy + t.first * lddy + col;  // the next row to fetch
  const P *const pw = gamma ? gamma + col : nullptr;
  T *to = dx + t.first * lddx + col;
  const int64_t x_step = t.step * ldx, g_step = t.step * lddy, to_step = t.step * lddx;
  int64_t next = t.first;
  // RING: [kLnAhead + 1][warp][x, dy][N][lane]
  Pack *const ring = reinterpret_cast<Pack *>(dynamic) + (threadIdx.x >> 5) * 64 * N + t.lane;
  const int slot = (int)blockDim.x * 2 * N;
  Pack *fetched = ring, *in_hand = ring, *const ring_end = ring + (kLnAhead + 1) * slot;
  if constexpr (RING && !FULL) {
    ln_clear(ring, slot, kLnAhead + 1, valid, N);
    ln_clear(ring + N * 32, slot, kLnAhead + 1, valid, N);
  }
  Pack xn[RING ? 1 : N], gn[RING ? 1 : N];
  auto fetch = [&]() {
    if (next < rows) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (FULL || i < valid) {
          if constexpr (PHASED) {
            phase.fetch(fetched + i * 32, px + i * 32 * V, i);
            phase.fetch(fetched + (N + i) * 32, pg + i * 32 * V, i);
          } else if constexpr (RING) {
            ln_copy_async(fetched + i * 32, px + i * 32 * V, V * sizeof(T));
            ln_copy_async(fetched + (N + i) * 32, pg + i * 32 * V, V * sizeof(T));
          } else {
            xn[i].load_stream(px + i * 32 * V);
            gn[i].load_stream(pg + i * 32 * V);
          }
        }
    }
    if constexpr (RING) {
      ln_commit();
      fetched += slot;
      if (fetched == ring_end) fetched = ring;
    }
    next += t.step;
    px += x_step;
    pg += g_step;
  };
  if (PHASED || t.team == 0) weights.template put<P, ALL && !FULL>(pw, (int)col, cols, valid, 1.f);
  __syncthreads();
  // mean and rstd of this team's next 32 rows, a row per lane
  int64_t at = t.first + t.lane * t.step;
  float mean32 = at < rows ? mean[at] : 0.f, rstd32 = at < rows ? rstd[at] : 0.f, mean_next = 0.f, rstd_next = 0.f;
#pragma unroll
  for (int i = 0; i < (RING ? kLnAhead : 1); ++i) fetch();
  int turn = 0;
  for (int64_t row = t.first; row < rows; row += t.step, to += to_step, ++turn) {
    const float m = __shfl_sync(0xffffffffu, mean32, turn & 31), r = __shfl_sync(0xffffffffu, rstd32, turn & 31);
    if ((turn & 31) == 16) {                       // the 32 after these, well before they are needed
      at += 32 * t.step;
      mean_next = at < rows ? mean[at] : 0.f;
      rstd_next = at < rows ? rstd[at] : 0.f;
    }
    if ((turn & 31) == 31) mean32 = mean_next, rstd32 = rstd_next;
    Pack xc[N], gc[N];
    if constexpr (RING) {
      fetch();      // into the place that the row before this one left
      ln_wait<kLnAhead>();
#pragma unroll
      for (int i = 0; i < N; ++i)
        xc[i] = in_hand[i * 32], gc[i] = in_hand[(N + i) * 32];
      in_hand += slot;
      if (in_hand == ring_end) in_hand = ring;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) xc[i] = xn[i], gc[i] = gn[i];
      fetch();
    }
    // with h = xhat:  dx = u * rstd + (h * (-rstd * sum(u * h) / n) - rstd * sum(u) / n).  LATE: h is x - mean until dx is formed.
    // (rstd^2 must not be: it passes FP32 where rstd alone does not; nor 0 * sum(u * (x - mean)), which may have passed it.)
    if constexpr (PHASED) phase.clear_front(xc[0]), phase.clear_front(gc[0]);
    F h[N * K], u[N * K], s1(0.f), s2(0.f);
    const F minus(-m), by(r);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (ALL || i < valid) {
        F g[K];
        weights.get(g, i);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int q = i * K + k;
          const F d = gc[i].get(k);
          u[q] = d * g[k];
          s1 = s1 + u[q];
          db[q] = db[q] + d;
          h[q] = xc[i].get(k) + minus;
          if constexpr (!LATE) h[q] = h[q] * by;
          s2 = ln_fma(u[q], h[q], s2);
          dg[q] = ln_fma(LATE ? d * by : d, h[q], dg[q]);
        }
      }
    if (dx) {
      const float2 s = ln_sum2(make_float2(s1.sum(), s2.sum()), scratch[turn & 1], t);
      const F a(-r * (s.x * inv)), b(LATE ? (r == 0.f ? 0.f : -r * (r * s.y * inv)) : -r * (s.y * inv));
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (ALL || i < valid) {
          Pack out;
#pragma unroll
          for (int k = 0; k < K; ++k) out.set(k, ln_fma(u[i * K + k], by, ln_fma(LATE ? h[i * K + k] * by : h[i * K + k], b, a)));
          if (FULL || i < valid) {
            if constexpr (PHASED) phase.store(out, to + i * 32 * V, i);
            else out.store(to + i * 32 * V);
          }
        }
    }
  }
  if constexpr (RING) ln_wait<0>();
  if (!partial) return;
  // each team's sums side by side in shared memory, then a column's over the teams in their order; a word in 33 is skipped, which
  // spreads accesses V words apart over the banks
  float *const line = partial + (int64_t)blockIdx.x * 2 * cols, *const sums = joined + t.team * 2 * ln_padded(cols);
  __syncthreads();                                   // the ring's memory is used again
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (FULL || i < valid) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float two[2][2];
        if constexpr (W == 2) {
          const float2 p = dg[i * K + k].both(), q = db[i * K + k].both();
          two[0][0] = p.x, two[0][1] = p.y, two[1][0] = q.x, two[1][1] = q.y;
        } else {
          two[0][0] = dg[i * K + k].v, two[1][0] = db[i * K + k].v;
        }
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const int c = (int)col + i * 32 * V + k * W + e;
          if (PHASED && !phase.inside(i, k * W + e)) continue;
          sums[c + (c >> 5)] = two[0][e];
          sums[ln_padded(cols) + c + (c >> 5)] = two[1][e];
        }
      }
    }
  __syncthreads();
  for (int which = 0; which < 2; ++which)
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const float *from = joined + which * ln_padded(cols) + c + (c >> 5);
      float sum = from[0];
      for (int w = 1; w < t.teams; ++w) sum += from[w * 2 * ln_padded(cols)];
      line[which * cols + c] = sum;
    }
}

// Rows too long for that: their sums of u and u * xhat first (one block per row), then everything else by tiles of columns,
// each thread walking down V columns.  x and dy are read twice: 4096 x 16384 bf16 takes 125 us, 5.4 TB/s of that traffic and 2.0
// times what one reading would take (158 us with 1024 threads to a row and a line of sums for every 28 rows).  Going over the rows
// by panels that fit L2, both kernels for each, was slower: 191 us for panels of 48 MB, 164 for 80 MB; the kernels' ends cost more
// than the second reading.
// dx alone needs no second kernel and no place for the sums: the block that has a row's sums reads the row again, from L2 (DX).
constexpr int kLnSumThreads = 512;
template <class T, class P, int V, bool DX>
__global__ void __launch_bounds__(kLnSumThreads) layernorm_row_sums_kernel(int64_t rows, int cols, const T *dy, int64_t lddy, const T *x, int64_t ldx,
                                                                  const P *gamma, const float *mean, const float *rstd, float2 *out, T *dx,
                                                                  int64_t lddx) {
  using F = typename LnPack<T, V>::F;
  constexpr int K = LnPack<T, V>::kParts;
  __shared__ LnScratch scratch[2];
  const LnTeam t(kLnSumThreads);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    const float m = mean[row], r = rstd[row];
    F s1(0.f), s2(0.f);
#pragma unroll 4
    for (int64_t i = (int64_t)threadIdx.x * V; i < cols; i += kLnSumThreads * V) {
      LnPack<T, V> xv, gv;
      F g[K];
      xv.load(x + row * ldx + i);
      gv.load(dy + row * lddy + i);
      ln_params<P, V>(g, gamma, (int)i, 1.f);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const F u = gv.get(k) * g[k];
        s1 = s1 + u;
        s2 = ln_fma(u, (xv.get(k) + F(-m)) * F(r), s2);
      }
    }
    const float2 s = ln_sum2(make_float2(s1.sum(), s2.sum()), scratch[turn], t);
    if constexpr (DX) {
      const float2 by_n = make_float2(s.x / (float)cols, s.y / (float)cols);
      for (int64_t i = (int64_t)threadIdx.x * V; i < cols; i += kLnSumThreads * V) {      // (dx may be dy: each thread reads its own again)
        LnPack<T, V> xv, gv;
        F g[K];
        xv.load(x + row * ldx + i);
        gv.load(dy + row * lddy + i);
        ln_params<P, V>(g, gamma, (int)i, 1.f);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const F h = (xv.get(k) + F(-m)) * F(r);
          xv.set(k, F(r) * (gv.get(k) * g[k] + ln_fma(h, F(-by_n.y), F(-by_n.x))));
        }
        xv.store(dx + row * lddx + i);
      }
    } else if (threadIdx.x == 0) {
      out[row] = make_float2(s.x / (float)cols, s.y / (float)cols);
    }
  }
}
template <class T, class P, int V>
__global__ void __launch_bounds__(128) layernorm_columns_kernel(int64_t rows, int cols, const T *dy, int64_t lddy, const T *x, int64_t ldx,
                                                                const P *gamma, const float *mean, const float *rstd,
                                                                const float2 *row_sums, T *dx, int64_t lddx, float *partial) {
  const int64_t c = ((int64_t)blockIdx.x * 128 + threadIdx.x) * V;
  if (c >= cols) return;
  using F = typename LnPack<T, V>::F;
  constexpr int K = LnPack<T, V>::kParts, W = LnPack<T, V>::W;
  F g[K], dg[K], db[K];
#pragma unroll
  for (int k = 0; k < K; ++k) dg[k] = F(0.f), db[k] = F(0.f);
  ln_params<P, V>(g, gamma, (int)c, 1.f);
#pragma unroll 2
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    LnPack<T, V> xv, gv;
    xv.load_stream(x + row * ldx + c);
    gv.load_stream(dy + row * lddy + c);
    const float m = mean[row], r = rstd[row];
    const float2 s = dx ? row_sums[row] : make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const F d = gv.get(k), h = (xv.get(k) + F(-m)) * F(r);
      dg[k] = ln_fma(d, h, dg[k]);
      db[k] = db[k] + d;
      xv.set(k, F(r) * (d * g[k] + ln_fma(h, F(-s.y), F(-s.x))));
    }
    if (dx) xv.store(dx + row * lddx + c);
  }
  if (!partial) return;
  float *const line = partial + (int64_t)blockIdx.y * 2 * cols + c, *const second = line + cols;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if constexpr (W == 2) {
      const float2 p = dg[k].both(), q = db[k].both();
      line[2 * k] = p.x, line[2 * k + 1] = p.y, second[2 * k] = q.x, second[2 * k + 1] = q.y;
    } else {
      line[k] = dg[k].v, second[k] = db[k].v;
    }
  }
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
constexpr int kLnBlock = 384;           // threads of a block of several teams, forward
constexpr int kLnHeldBackward = 16;       // elements per thread, backward
constexpr int kLnLongestBackward = 8192;  // 512 threads of 16 elements, or 1024 of 8
// Most blocks, and lines of partial sums: three blocks on each of 148 SMs (as many as an SM may hold); the longest rows, whose lines are long and whose blocks
// share the columns, take about 1184 blocks of 1024 columns and give each 8 rows at least (300 x 16384 bf16: 34 -> 18 us).
static int64_t ln_parts(int64_t rows, int64_t cols) {
  int64_t most = 444;
  if (cols > kLnLongestBackward) {
    most = 1184 * 1024 / cols;
    if (most > rows / 8) most = rows / 8;
    if (most < 8) most = 8;
  }
  return rows < most ? rows : most;
}

// Whether every address and pitch (in bytes) is a multiple of `bytes`; NULL is.
static bool ln_multiple(int64_t bytes, std::initializer_list<const void *> pointers, std::initializer_list<int64_t> pitches) {
  for (const void *p : pointers)
    if ((uintptr_t)p % bytes) return false;
  for (int64_t p : pitches)
    if (p % bytes) return false;
  return true;
}
// Accesses per thread that take `units` of them over `share` threads.
static int ln_turns(int64_t units, int share) { return (int)((units + share - 1) / share); }

// Blocks of this size that an SM holds, asked once per kernel, size and device (and each time, should the table be full).
static int ln_blocks_per_sm(const void *kernel, int device, int threads, size_t smem, int *out) {
  struct Entry {
    const void *kernel;
    int device, threads;
    size_t smem;
    int blocks;
  };
  static Entry known[512];
  static int count = 0;
  static std::mutex mu;
  std::lock_guard<std::mutex> lk(mu);
  for (int i = 0; i < count; ++i) {
    const Entry &e = known[i];
    if (e.kernel == kernel && e.device == device && e.threads == threads && e.smem == smem) {
      *out = e.blocks;
      return B2_OK;
    }
  }
  int n = 0;
  B2_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem));
  *out = n < 1 ? 1 : n;
  if (count < (int)(sizeof(known) / sizeof(known[0]))) known[count++] = {kernel, device, threads, smem, *out};
  return B2_OK;
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
// Whether rows that are not multiples of 16 bytes can be taken as PHASED does: the matrices start on 16 bytes (so that what is
// in front of a row is the matrix's own) and their pitches are off by as much.
static bool ln_phased(std::initializer_list<const void *> matrices, std::initializer_list<int64_t> pitches) {
  for (int64_t p : pitches)
    if ((p - *pitches.begin()) % 16) return false;
  return ln_multiple(16, matrices, {});
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
  int width = ln_width(cols, tb, pb, {x, y}, {ldx * tb, ldy * tb}, {gamma, beta});
  const bool phased = width * tb < 16 && rows > 2 * ctx->sm_count && cols >= 128 && cols + 16 <= 512 * 32 && ln_phased({x, y}, {ldx * tb, ldy * tb});
  if (phased) width = 16 / tb;
  cudaStream_t s = (cudaStream_t)stream;
  auto launch = [&](auto t, auto p) -> int {
    using T = decltype(t);
    using P = decltype(p);
    int result = B2_OK;
    cudaError_t launched = cudaSuccess;
    ln_with_width<T>(width, [&](auto w) {
      constexpr int V = decltype(w)::value;
      // E elements per thread, teams of threads to a row in blocks of about 256
      auto run = [&](auto elements, auto bound, auto off) {
        constexpr int E = decltype(elements)::value, THREADS = decltype(bound)::value;
        constexpr bool PHASED = decltype(off)::value;
        const int64_t span = cols + (PHASED ? V - 1 : 0);
        const int share = (int)((span + 32 * E - 1) / (32 * E)) * 32, turns = ln_turns((span + V - 1) / V, share);
        const bool full = !PHASED && turns == E / V && cols == (int64_t)share * E;
        const auto kernel = full ? layernorm_kernel<T, P, V, E, THREADS, !PHASED, PHASED> : layernorm_kernel<T, P, V, E, THREADS, false, PHASED>;
        const int64_t fit = share <= (PHASED ? 192 : kLnBlock) ? (PHASED ? 192 : kLnBlock) / share : 1;
        const int teams = (int)(fit < rows ? fit : rows), threads = share * teams;
        const size_t row_bytes = V * sizeof(T) >= 4 ? (size_t)threads * E * sizeof(T) : 0;
        const size_t params = E > 16 && THREADS <= 512 ? (size_t)2 * (PHASED ? threads : share) * E * sizeof(float) : 0;
        // rows ahead: two, or as many as leave room for two blocks on an SM, or for one
        int ahead = kLnAhead;
        while (ahead > 0 && (ahead + 1) * row_bytes + params > 112 * 1024) --ahead;
        if (ahead == 0)
          for (ahead = kLnAhead; ahead > 0 && (ahead + 1) * row_bytes + params > 224 * 1024;) --ahead;
        const size_t smem = (ahead + 1) * row_bytes + params;
        const int64_t blocks = (rows + teams - 1) / teams;
        result = ensure_func_attributes((const void *)kernel, ctx->device, 224 * 1024);
        if (result != B2_OK) return;
        int held = 1;      // the blocks that the device holds at once walk over all rows
        result = ln_blocks_per_sm((const void *)kernel, ctx->device, threads, smem, &held);
        if (result != B2_OK) return;
        int64_t most = (int64_t)ctx->sm_count * held;
        if (PHASED && blocks > most) most = most / V * V;
        launched = launch_kernel(kernel, (unsigned)(blocks < most ? blocks : most), threads, smem, s, rows, (int)cols, share, turns, ahead, eps,
                                 (const T *)x, ldx, (const P *)gamma, (const P *)beta, (T *)y, ldy, mean, rstd);
      };
      constexpr int kFew = V == 8 ? 8 : 4, kMost = V >= 4 ? 32 : 16, kLong = V == 1 ? 16 : 32;
      using Half = std::integral_constant<int, 512>;
      using Full = std::integral_constant<int, 1024>;
      using Even = std::false_type;
      if constexpr (V == 16 / (int)sizeof(T)) {
        if (phased) {
          // 16 bytes against the widest access that fits: 8192 x 4095 bf16 62 -> 43 us (16 elements per thread: 80), 16384 x 2050
          // 70 -> 51, 8192 x 8001 FP32 127 -> 103, 40000 x 131 FP16 25.6 -> 16.2 (32 elements per thread: 29.8).  Shorter rows lose
          // (4000 x 67: 3.2 -> 4.7), and so do few rows, which the parameters' odd places delay (11 x 4097: 3.1 -> 4.9).
          if (cols + V <= 32 * V) run(std::integral_constant<int, V>(), Half(), std::true_type());      // a warp, one access each
          else run(std::integral_constant<int, 32>(), Half(), std::true_type());
          return;
        }
      }
      // Few rows: as many threads to each as its length allows; rows so short that a warp has enough with a few elements per
      // thread likewise.  Else each thread takes as much as it can hold: the fewer share a sum, the less it costs.
      if ((rows <= 2 * ctx->sm_count && cols <= 1024 * kFew) || cols <= 32 * kFew) run(std::integral_constant<int, kFew>(), Full(), Even());
      else if (cols <= 512 * kMost) run(std::integral_constant<int, kMost>(), Half(), Even());
      else if (cols <= 1024 * kLong) run(std::integral_constant<int, kLong>(), Full(), Even());
      else
        launched = launch_kernel(layernorm_long_kernel<T, P, V>, (unsigned)(rows < 1 << 30 ? rows : 1 << 30), 1024, 0, s, rows, (int)cols, eps,
                                 (const T *)x, ldx, (const P *)gamma, (const P *)beta, (T *)y, ldy, mean, rstd);
    });
    if (result == B2_OK) B2_CUDA(launched);
    return result;
  };
  return with_type(type, [&](auto t) { return param_type == type ? launch(t, t) : launch(t, float()); });
}

size_t b2_layernorm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  const size_t sums = (size_t)ln_parts(rows, cols) * 2 * (size_t)cols * sizeof(float);
  return (sums + 15) / 16 * 16 + (cols > kLnLongestBackward ? (size_t)rows * sizeof(float2) : 0);
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
  const bool is_long = cols > kLnLongestBackward;
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
  int parts = (int)ln_parts(rows, cols);
  int width = ln_width(cols, tb, pb, {dy, x, dx}, {lddy * tb, ldx * tb, dx ? lddx * tb : 0}, {gamma});
  const bool phased = width * tb < 16 && cols + 16 <= kLnLongestBackward && ln_phased({dy, x, dx}, {lddy * tb, ldx * tb, dx ? lddx * tb : ldx * tb});
  if (phased) width = 16 / tb;
  float *partial = sums ? (float *)workspace : nullptr;
  float2 *row_sums = is_long && sums ? (float2 *)((char *)workspace + (need - (size_t)rows * sizeof(float2))) : nullptr;
  auto launch = [&](auto t, auto p) -> int {
    using T = decltype(t);
    using P = decltype(p);
    int result = B2_OK;
    cudaError_t launched = cudaSuccess;
    ln_with_width<T>(width, [&](auto w) {
      constexpr int V = decltype(w)::value;
      if (!is_long) {
        // E elements per thread, and teams of threads to a row in blocks of about 256
        auto run = [&](auto elements, auto off) {
          constexpr int E = decltype(elements)::value;
          constexpr bool PHASED = decltype(off)::value;
          const int64_t span = cols + (PHASED ? V - 1 : 0);
          const int share = (int)((span + 32 * E - 1) / (32 * E)) * 32, turns = ln_turns((span + V - 1) / V, share);
          const bool full = !PHASED && turns == E / V && cols == (int64_t)share * E;
          const auto kernel = full ? layernorm_backward_kernel<T, P, V, E, !PHASED, PHASED> : layernorm_backward_kernel<T, P, V, E, false, PHASED>;
          const int64_t fit = share <= 256 ? 256 / share : 1;
          const int teams = (int)(fit < rows ? fit : rows), threads = share * teams;
          size_t smem = V * sizeof(T) >= 4 ? (size_t)(kLnAhead + 1) * 2 * E * sizeof(T) * threads : 0;
          smem += (size_t)(PHASED ? threads : share) * E * sizeof(float);       // gamma
          const size_t joined = (size_t)teams * 2 * ln_padded((int)cols) * sizeof(float);
          if (smem < joined) smem = joined;
          result = ensure_func_attributes((const void *)kernel, ctx->device, 224 * 1024);
          if (result != B2_OK) return;
          // A block per SM before any block takes a second turn, then two turns before there are more blocks: a line of sums per
          // block costs as much as a row or two (248 x 7424 FP32 17.5 -> 11.1 us with two turns, 2213 x 76 bf16 8.1 -> 6.3; with fewer
          // blocks than SMs it loses: 60 x 300 5.5 -> 6.1)
          const int64_t turn = (rows + teams - 1) / teams, wanted = turn <= ctx->sm_count ? turn : (turn + 1) / 2 < ctx->sm_count ? ctx->sm_count : (turn + 1) / 2;
          int held = 1;      // blocks that an SM holds at once (three where registers allow: 16384 x 2049 FP32 104 -> 94 us)
          result = ln_blocks_per_sm((const void *)kernel, ctx->device, threads, smem, &held);
          if (result != B2_OK) return;
          if ((int64_t)held * ctx->sm_count < parts) parts = held * ctx->sm_count;
          const int limit = parts;
          if (wanted < parts) parts = (int)wanted;
          if (PHASED && (int64_t)parts * teams < rows) parts = (parts + V - 1) / V * V;
          if (parts > limit) parts = (int64_t)limit * teams < rows ? limit / V * V : limit;
          launched = launch_kernel(kernel, parts, threads, smem, s, rows, (int)cols, share, turns, (const T *)dy, lddy, (const T *)x, ldx,
                                   (const P *)gamma, mean, rstd, (T *)dx, lddx, partial);
        };
        // Elements one by one take more registers and instructions each: fewer of them, in more threads (5003 x 1027 FP32: 35 -> 23 us)
        if constexpr (V == 16 / (int)sizeof(T)) {
          if (phased) {
            // 16 bytes against the widest access that fits, when this was chosen: 8192 x 4095 bf16 257 -> 73 us, 16384 x 2050 84 -> 63 (8
            // elements per thread: 93), 5003 x 1027 FP32 23.4 -> 21.9 (16 elements: 30.5), 40000 x 517 FP32 64 -> 59 (16: 108), 40000 x 131
            // FP16 47 -> 26.5 (16: 31); by now 64, 52, 20.5, 58 and 21
            if (cols + V <= (V == 4 ? 512 : 32) * 8) run(std::integral_constant<int, 8>(), std::true_type());
            else run(std::integral_constant<int, kLnHeldBackward>(), std::true_type());
            return;
          }
        }
        if (V == 1 && cols <= 512 * 8) run(std::integral_constant<int, (V == 1 ? 8 : kLnHeldBackward)>(), std::false_type());
        else run(std::integral_constant<int, kLnHeldBackward>(), std::false_type());
      } else {
        if (dx)
          launched = launch_kernel(sums ? layernorm_row_sums_kernel<T, P, V, false> : layernorm_row_sums_kernel<T, P, V, true>,
                                   (unsigned)(rows < 1 << 30 ? rows : 1 << 30), kLnSumThreads, 0, s, rows, (int)cols, (const T *)dy, lddy,
                                   (const T *)x, ldx, (const P *)gamma, mean, rstd, row_sums, (T *)dx, lddx);
        if (sums && launched == cudaSuccess)
          launched = launch_kernel(layernorm_columns_kernel<T, P, V>, dim3((unsigned)((cols / V + 127) / 128), (unsigned)parts), 128, 0, s, rows,
                                   (int)cols, (const T *)dy, lddy, (const T *)x, ldx, (const P *)gamma, mean, rstd, row_sums, (T *)dx, lddx, partial);
      }
    });
    if (result == B2_OK) B2_CUDA(launched);
    if (result == B2_OK && sums) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)((cols + 31) / 32));
      cfg.blockDim = dim3(1024);
      cfg.stream = s;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // its blocks may start, and wait, before the sums are done
      attr[0].val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      B2_CUDA(cudaLaunchKernelEx(&cfg, layernorm_reduce_kernel<P>, parts, (int)cols, (const float *)partial, (P *)dgamma, (P *)dbeta));
    }
    return result;
  };
  return with_type(type, [&](auto t) { return param_type == type ? launch(t, t) : launch(t, float()); });
}

}  // extern "C"
