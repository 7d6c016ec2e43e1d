// Typed vector access shared by the memory-bound operators: N elements of bf16, fp16 or fp32 move in one load or
// store of N * sizeof(T) <= 16 bytes and are handled as fp32 in registers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

namespace mb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
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

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& p, float* f) {
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = to_f32(p.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
  const Pack<T, N> v = *reinterpret_cast<const Pack<T, N>*>(p);
  unpack<T, N>(v, f);
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
  Pack<T, N> v;
#pragma unroll
  for (int i = 0; i < N; ++i) v.v[i] = from_f32<T>(f[i]);
  *reinterpret_cast<Pack<T, N>*>(p) = v;
}

__device__ __forceinline__ float warp_reduce_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_reduce_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Sum over the CTA's kThreads threads, the same value in every thread; `red` holds kThreads / 32 floats and may be
// handed in again at once.
template <int kThreads>
__device__ __forceinline__ float block_reduce_sum(float v, float* red) {
  v = warp_reduce_sum(v);
  if (kThreads == 32) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_reduce_sum(lane < kThreads / 32 ? red[lane] : 0.f);
}
template <int kThreads>
__device__ __forceinline__ float block_reduce_max(float v, float* red) {
  v = warp_reduce_max(v);
  if (kThreads == 32) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_reduce_max(lane < kThreads / 32 ? red[lane] : -INFINITY);
}

inline bool is_aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

}  // namespace mb
