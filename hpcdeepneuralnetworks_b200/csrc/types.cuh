// Element types of the layer-norm and 4-bit-weight operators: names, sizes, conversions to and from FP32 (rounding to
// nearest even, once, at the store), and the host-side argument checks they share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace b2 {

inline int type_bytes(int type) { return type == B2_F32 ? 4 : type == B2_BF16 || type == B2_F16 ? 2 : 0; }

// Whether two pitched matrices share an element: `rows` rows of `bytes` bytes, `pitch` bytes apart.  Views of one buffer
// with the same pitch may interleave (the halves of a row of 2 * cols); with other pitches any common span counts.
inline bool matrices_overlap(const void *a, int64_t rows_a, int64_t bytes_a, int64_t pitch_a, const void *b, int64_t rows_b,
                             int64_t bytes_b, int64_t pitch_b) {
  if (!a || !b || rows_a <= 0 || rows_b <= 0 || bytes_a <= 0 || bytes_b <= 0) return false;
  const intptr_t a0 = (intptr_t)a, b0 = (intptr_t)b;
  if (a0 + (rows_a - 1) * pitch_a + bytes_a <= b0 || b0 + (rows_b - 1) * pitch_b + bytes_b <= a0) return false;
  if (pitch_a != pitch_b) return true;
  int64_t d = (b0 - a0) % pitch_a;   // b's first column seen from a's rows
  if (d < 0) d += pitch_a;
  return !(d >= bytes_a && d + bytes_b <= pitch_a);
}

#ifdef __CUDACC__
// kernel<<<grid, block, smem, stream>>>(args...), with the launch's own status.  cudaGetLastError after such a launch would also
// report, for work that is on its way, what some earlier call of the thread has left behind.
template <class... P, class... A>
inline cudaError_t launch_kernel(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<A &&>(args)...);
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}

// Programmatic dependent launch: a kernel launched with the stream-serialization attribute may start while the one in front of
// it still runs; it waits for that one's end, and so for its results, in pdl_wait.
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Calls f with a value of the element type that `type` names; the type has been checked before.
template <class F>
inline int with_type(int type, F &&f) {
  if (type == B2_F32) return f(float());
  if (type == B2_BF16) return f(__nv_bfloat16());
  return f(__half());
}
#endif  // __CUDACC__

}  // namespace b2
