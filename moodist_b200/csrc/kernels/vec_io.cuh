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

// N elements as they lie in memory, in 32-bit words (a struct of 16-bit members is taken apart and put together again member by
// member in registers) or, alone, a 16-bit element. On a 16-byte boundary at most: eight fp32 weights beside eight 16-bit
// elements are two loads.
template <typename T, int N, bool kWords = sizeof(T) * N % 4 == 0>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
  uint32_t w[sizeof(T) * N / 4];
};
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack<T, N, false> {
  T v[N];
};

// Pairs are converted together: at most one instruction each way per 16-bit value (single conversions to 16 bits run at a
// quarter of the rate, and made bf16 rows take as long as fp32 rows of twice the bytes).
template <typename T>
__device__ __forceinline__ float2 pair_to_f32(uint32_t w);
template <>
__device__ __forceinline__ float2 pair_to_f32<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 pair_to_f32<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pair_from_f32(float a, float b);
template <>
__device__ __forceinline__ uint32_t pair_from_f32<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pair_from_f32<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T>
struct PairOf;
template <>
struct PairOf<__nv_bfloat16> {
  using type = __nv_bfloat162;
};
template <>
struct PairOf<__half> {
  using type = __half2;
};

template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& p, float* f) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = __uint_as_float(p.w[i]);
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 v = pair_to_f32<T>(p.w[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  } else {
    static_assert(N == 1, "one 16-bit element or pairs of them");
    f[0] = to_f32(p.v[0]);
  }
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> pack(const float* f) {
  Pack<T, N> p;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) p.w[i] = __float_as_uint(f[i]);
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) p.w[i] = pair_from_f32<T>(f[2 * i], f[2 * i + 1]);
  } else {
    p.v[0] = from_f32<T>(f[0]);
  }
  return p;
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> splat(float x) {
  float f[N];
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = x;
  return pack<T, N>(f);
}
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
  const Pack<T, N> v = *reinterpret_cast<const Pack<T, N>*>(p);
  unpack<T, N>(v, f);
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
  *reinterpret_cast<Pack<T, N>*>(p) = pack<T, N>(f);
}

// Two fp32 values in a register pair: one instruction adds, multiplies or fuses both.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ float2 split(F2 x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
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
inline bool is_aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

}  // namespace mb
