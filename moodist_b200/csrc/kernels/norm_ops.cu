// Layer normalisation over the last dimension, forward and backward, for bf16, fp16 and fp32 rows with an optional
// weight and bias (of the rows' type or fp32).
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) * r, y = xh * w + b
//   g  = dy * w,  dx = r * (g - mean(g) - xh * mean(g * xh)),  dw = sum over rows of dy * xh,  db = sum over rows of dy
//
// The variance is taken around the mean (a second walk over the row), so a row far from zero loses nothing; every sum is
// fp32. Bound by the bytes: x in and y out, x and dy in and dx out.
#include "kernels_api.h"
#include "vec_io.cuh"

#define MB_STREAM(s) reinterpret_cast<cudaStream_t>(s)

namespace {

using namespace mb;

inline int check_launch() { return cudaPeekAtLastError() == cudaSuccess ? MB_OK : MB_ERR_LAUNCH; }

// element i of a weight vector of type T or fp32 (a null pointer: `otherwise`)
template <typename T>
__device__ __forceinline__ float weight_at(const void* w, bool f32, int64_t i, float otherwise) {
  if (!w) return otherwise;
  return f32 ? reinterpret_cast<const float*>(w)[i] : to_f32(reinterpret_cast<const T*>(w)[i]);
}

constexpr int kThreads = 256;

template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads)
    layernorm_fwd_kernel(const T* __restrict__ x, const void* __restrict__ w, const void* __restrict__ b, T* __restrict__ y,
                         float* __restrict__ mean, float* __restrict__ rstd, int64_t rows, int64_t D, int64_t x_stride,
                         int64_t y_stride, float eps, bool w_f32) {
  __shared__ float red[kThreads / 32];
  const int64_t step = (int64_t)kThreads * kVec;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * x_stride;
    float f[kVec], s = 0.f;
    for (int64_t c = threadIdx.x * kVec; c < D; c += step) {
      load_vec<T, kVec>(xr + c, f);
#pragma unroll
      for (int k = 0; k < kVec; ++k) s += f[k];
    }
    const float mu = block_reduce_sum<kThreads>(s, red) / (float)D;
    s = 0.f;
    for (int64_t c = threadIdx.x * kVec; c < D; c += step) {
      load_vec<T, kVec>(xr + c, f);
#pragma unroll
      for (int k = 0; k < kVec; ++k) s += (f[k] - mu) * (f[k] - mu);
    }
    const float rs = rsqrtf(block_reduce_sum<kThreads>(s, red) / (float)D + eps);
    if (threadIdx.x == 0 && mean) {
      mean[r] = mu;
      rstd[r] = rs;
    }
    for (int64_t c = threadIdx.x * kVec; c < D; c += step) {
      load_vec<T, kVec>(xr + c, f);
#pragma unroll
      for (int k = 0; k < kVec; ++k)
        f[k] = (f[k] - mu) * rs * weight_at<T>(w, w_f32, c + k, 1.f) + weight_at<T>(b, w_f32, c + k, 0.f);
      store_vec<T, kVec>(y + r * y_stride + c, f);
    }
  }
}

template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads)
    layernorm_dx_kernel(const T* __restrict__ x, const void* __restrict__ w, const T* __restrict__ dy,
                        const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, int64_t rows,
                        int64_t D, int64_t x_stride, int64_t dy_stride, int64_t dx_stride, bool w_f32) {
  __shared__ float red[kThreads / 32];
  const int64_t step = (int64_t)kThreads * kVec;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mu = mean[r], rs = rstd[r];
    float fx[kVec], fd[kVec], s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x * kVec; c < D; c += step) {
      load_vec<T, kVec>(x + r * x_stride + c, fx);
      load_vec<T, kVec>(dy + r * dy_stride + c, fd);
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        const float g = fd[k] * weight_at<T>(w, w_f32, c + k, 1.f);
        s1 += g;
        s2 += g * (fx[k] - mu) * rs;
      }
    }
    s1 = block_reduce_sum<kThreads>(s1, red) / (float)D;
    s2 = block_reduce_sum<kThreads>(s2, red) / (float)D;
    for (int64_t c = threadIdx.x * kVec; c < D; c += step) {
      load_vec<T, kVec>(x + r * x_stride + c, fx);
      load_vec<T, kVec>(dy + r * dy_stride + c, fd);
#pragma unroll
      for (int k = 0; k < kVec; ++k)
        fx[k] = rs * (fd[k] * weight_at<T>(w, w_f32, c + k, 1.f) - s1 - (fx[k] - mu) * rs * s2);
      store_vec<T, kVec>(dx + r * dx_stride + c, fx);
    }
  }
}

// partial[part][0][c] = sum of dy * xh, partial[part][1][c] = sum of dy, over the rows part, part + parts, ...
template <typename T>
__global__ void __launch_bounds__(kThreads)
    layernorm_dw_kernel(const T* __restrict__ x, const T* __restrict__ dy, const float* __restrict__ mean,
                        const float* __restrict__ rstd, float* __restrict__ partial, int64_t rows, int64_t D,
                        int64_t x_stride, int64_t dy_stride) {
  const int64_t c = blockIdx.x * (int64_t)kThreads + threadIdx.x;
  if (c >= D) return;
  float sw = 0.f, sb = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float d = to_f32(dy[r * dy_stride + c]);
    sw += d * (to_f32(x[r * x_stride + c]) - mean[r]) * rstd[r];
    sb += d;
  }
  partial[(int64_t)blockIdx.y * 2 * D + c] = sw;
  partial[((int64_t)blockIdx.y * 2 + 1) * D + c] = sb;
}

// dw[c], db[c] = sums of the partial rows, 32 columns of one of the two per CTA, eight warps side by side
template <typename T>
__global__ void __launch_bounds__(256)
    layernorm_dw_join_kernel(const float* __restrict__ partial, void* __restrict__ dw, void* __restrict__ db, int parts,
                             int64_t D, bool w_f32) {
  __shared__ float sm[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, which = blockIdx.y;
  void* out = which ? db : dw;
  if (!out) return;
  const int64_t c = blockIdx.x * 32ll + tx;
  float s = 0.f;
  if (c < D)
    for (int p = ty; p < parts; p += 8) s += partial[((int64_t)p * 2 + which) * D + c];
  sm[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < D) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += sm[k][tx];
    if (w_f32)
      reinterpret_cast<float*>(out)[c] = t;
    else
      reinterpret_cast<T*>(out)[c] = from_f32<T>(t);
  }
}

inline unsigned row_grid(int64_t rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

template <typename T>
int fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows, int64_t D,
        int64_t x_stride, int64_t y_stride, bool w_f32, float eps, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  const bool vec = D % kV == 0 && x_stride % kV == 0 && y_stride % kV == 0 && is_aligned(x, 16) && is_aligned(y, 16);
  auto k = vec ? layernorm_fwd_kernel<T, kV> : layernorm_fwd_kernel<T, 1>;
  k<<<row_grid(rows), kThreads, 0, s>>>((const T*)x, w, b, (T*)y, mean, rstd, rows, D, x_stride, y_stride, eps, w_f32);
  return check_launch();
}

template <typename T>
int bwd(const void* x, const void* w, const void* dy, const float* mean, const float* rstd, void* dx, void* dw, void* db,
        float* partial, int64_t rows, int64_t D, int64_t x_stride, int64_t dy_stride, int64_t dx_stride, bool w_f32,
        cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  if (dx) {
    const bool vec = D % kV == 0 && x_stride % kV == 0 && dy_stride % kV == 0 && dx_stride % kV == 0 && is_aligned(x, 16) &&
                     is_aligned(dy, 16) && is_aligned(dx, 16);
    auto k = vec ? layernorm_dx_kernel<T, kV> : layernorm_dx_kernel<T, 1>;
    k<<<row_grid(rows), kThreads, 0, s>>>((const T*)x, w, (const T*)dy, mean, rstd, (T*)dx, rows, D, x_stride, dy_stride,
                                          dx_stride, w_f32);
    if (check_launch()) return MB_ERR_LAUNCH;
  }
  if (dw || db) {
    const int parts = mb_layernorm_bwd_parts(rows, D);
    layernorm_dw_kernel<T><<<dim3((unsigned)((D + kThreads - 1) / kThreads), parts), kThreads, 0, s>>>(
        (const T*)x, (const T*)dy, mean, rstd, partial, rows, D, x_stride, dy_stride);
    if (check_launch()) return MB_ERR_LAUNCH;
    layernorm_dw_join_kernel<T><<<dim3((unsigned)((D + 31) / 32), 2), 256, 0, s>>>(partial, dw, db, parts, D, w_f32);
  }
  return check_launch();
}

}  // namespace

extern "C" int mb_layernorm_bwd_parts(int64_t rows, int64_t D) {
  const int64_t col_ctas = (D + kThreads - 1) / kThreads;
  int64_t parts = 148 * 8 / (col_ctas < 1 ? 1 : col_ctas);
  if (parts > rows) parts = rows;
  return (int)(parts < 1 ? 1 : parts);
}

extern "C" int mb_layernorm_fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows,
                                int64_t D, int64_t x_stride, int64_t y_stride, int dtype, int w_dtype, float eps,
                                void* stream) {
  if (rows <= 0) return MB_OK;
  if (D <= 0 || D > (1 << 30) || (w_dtype != dtype && w_dtype != MB_F32) || !mean != !rstd) return MB_ERR_ARG;
  const bool w32 = w_dtype == MB_F32;
  switch (dtype) {
    case MB_BF16: return fwd<__nv_bfloat16>(x, w, b, y, mean, rstd, rows, D, x_stride, y_stride, w32, eps, MB_STREAM(stream));
    case MB_F16: return fwd<__half>(x, w, b, y, mean, rstd, rows, D, x_stride, y_stride, w32, eps, MB_STREAM(stream));
    case MB_F32: return fwd<float>(x, w, b, y, mean, rstd, rows, D, x_stride, y_stride, w32, eps, MB_STREAM(stream));
    default: return MB_ERR_ARG;
  }
}

extern "C" int mb_layernorm_bwd(const void* x, const void* w, const void* dy, const float* mean, const float* rstd, void* dx,
                                void* dw, void* db, float* partial, int64_t rows, int64_t D, int64_t x_stride,
                                int64_t dy_stride, int64_t dx_stride, int dtype, int w_dtype, void* stream) {
  if (rows <= 0) return MB_OK;
  if (D <= 0 || D > (1 << 30) || (w_dtype != dtype && w_dtype != MB_F32)) return MB_ERR_ARG;
  const bool w32 = w_dtype == MB_F32;
  switch (dtype) {
    case MB_BF16:
      return bwd<__nv_bfloat16>(x, w, dy, mean, rstd, dx, dw, db, partial, rows, D, x_stride, dy_stride, dx_stride, w32, MB_STREAM(stream));
    case MB_F16:
      return bwd<__half>(x, w, dy, mean, rstd, dx, dw, db, partial, rows, D, x_stride, dy_stride, dx_stride, w32, MB_STREAM(stream));
    case MB_F32:
      return bwd<float>(x, w, dy, mean, rstd, dx, dw, db, partial, rows, D, x_stride, dy_stride, dx_stride, w32, MB_STREAM(stream));
    default: return MB_ERR_ARG;
  }
}
