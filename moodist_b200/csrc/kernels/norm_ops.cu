// Layer normalisation over the last dimension, forward and backward, for bf16, fp16 and fp32 rows with an optional
// weight and bias (of the rows' type or fp32).
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) * r, y = xh * w + b
//   g  = dy * w,  dx = r * (g - mean(g) - xh * mean(g * xh)),  dw = sum over rows of dy * xh,  db = sum over rows of dy
//
// The variance is taken around the mean (a second walk over the row), so a row far from zero loses nothing; every sum is
// fp32. Bound by the bytes: x in and y out, x and dy in and dx out.
//
// Rows of up to 16384 elements stay in registers between their statistics and their result, so every byte moves once. A
// thread holds 16 columns, the same ones in all rows of its CTA: weights and, in the backward pass, two sums per column stay in
// registers too. Up to four rows ahead are on their way into shared memory, each thread copying the vectors that it will
// read itself, so that no barrier guards them (one row ahead in registers left DRAM at 65 %: 24 KB in flight per SM).
// At 16 bits an element the instructions count as much as the bytes (18 of them per element and pass would take all of the
// time the bytes need), so the arithmetic is on pairs, two fp32 values per instruction. (A warp per row with up to 128 columns
// per lane was slower than three walks over memory: too few warps to hide its own latency.)
// 8192 x 4096 bf16: forward 23 us (5.8 TB/s), backward 47 us and 4 for joining the weight sums (4.3 TB/s); fp32: 45 us (5.9),
// 74 + 5 us (5.4). Widths that no 16-byte vector divides use the same kernels with single elements (8192 x 4095 bf16: 49 and
// 83 us). Longer rows take the loops (1024 x 20480 bf16: 35 and 85 us), which read them up to three times.
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

// dw[c], db[c] = sums of the partial rows, 32 columns of one of the two per CTA, 32 warps side by side
template <typename T>
__global__ void __launch_bounds__(1024)
    layernorm_dw_join_kernel(const float* __restrict__ partial, void* __restrict__ dw, void* __restrict__ db, int parts,
                             int64_t D, bool w_f32) {
  __shared__ float sm[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, which = blockIdx.y;
  void* out = which ? db : dw;
  if (!out) return;
  const int64_t c = blockIdx.x * 32ll + tx;
  float s = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int p = ty; p < parts; p += 32) s += partial[((int64_t)p * 2 + which) * D + c];
  }
  sm[ty][tx] = s;
  __syncthreads();
  // warp ty sums column ty
  const float sum = warp_reduce_sum(sm[tx][ty]);
  const int64_t col = blockIdx.x * 32ll + ty;
  if (tx == 0 && col < D) {
    if (w_f32)
      reinterpret_cast<float*>(out)[col] = sum;
    else
      reinterpret_cast<T*>(out)[col] = from_f32<T>(sum);
  }
}

// ---- rows in registers -------------------------------------------------------------------------------------------------

constexpr int kCols = 16, kPairs = kCols / 2;  // columns per thread

// A thread's columns of one row as they lie in memory: kCols / kVec vectors, vector i of thread t at column (i * kTpr + t) * kVec.
template <typename T, int kVec, int kTpr>
struct Held {
  static constexpr int kG = kCols / kVec;
  Pack<T, kVec> v[kG];
  __device__ __forceinline__ static int column(int t, int i) { return (i * kTpr + t) * kVec; }
  __device__ __forceinline__ void fill(float x) {
#pragma unroll
    for (int i = 0; i < kG; ++i) v[i] = splat<T, kVec>(x);
  }
  // columns from D up keep what they hold
  __device__ __forceinline__ void load(const T* row, int t, int D) {
#pragma unroll
    for (int i = 0; i < kG; ++i)
      if (column(t, i) < D) v[i] = *reinterpret_cast<const Pack<T, kVec>*>(row + column(t, i));
  }
  __device__ __forceinline__ void pairs(F2* f) const {
    float u[kCols];
#pragma unroll
    for (int i = 0; i < kG; ++i) unpack<T, kVec>(v[i], u + i * kVec);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) f[j] = f2(u[2 * j], u[2 * j + 1]);
  }
  __device__ __forceinline__ static void store(T* row, int t, int D, const F2* f) {
    float u[kCols];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const float2 p = split(f[j]);
      u[2 * j] = p.x;
      u[2 * j + 1] = p.y;
    }
#pragma unroll
    for (int i = 0; i < kG; ++i)
      if (column(t, i) < D) store_vec<T, kVec>(row + column(t, i), u + i * kVec);
  }
};
__device__ __forceinline__ void cp_async16(void* smem, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(global) : "memory");
}
// The rows that a thread is about to need, in order. Whole vectors travel kDepth rows ahead through the thread's own slots of
// shared memory; single elements one row ahead in registers.
template <typename T, int kVec, int kTpr, int kBlock, int kDepth>
struct Feed {
  using X = Held<T, kVec, kTpr>;
  static constexpr bool kAsync = sizeof(T) * kVec == 16;
  static constexpr int kBytes = kAsync ? kDepth * X::kG * kBlock * 16 : 0;
  X next;
  uint8_t* slots;
  int64_t r, last;  // the next row to request, the number of rows

  __device__ __forceinline__ void begin(uint8_t* smem, int64_t row, int64_t rows, int t, int D) {
    last = rows;
    r = row;
    if constexpr (kAsync) {
      slots = smem + threadIdx.x * 16;
      // columns past the row's end read as zero
#pragma unroll
      for (int d = 0; d < kDepth; ++d)
#pragma unroll
        for (int i = 0; i < X::kG; ++i)
          if (X::column(t, i) >= D) *reinterpret_cast<uint4*>(slots + (d * X::kG + i) * kBlock * 16) = make_uint4(0, 0, 0, 0);
    } else {
      next.fill(0.f);
    }
  }
  __device__ __forceinline__ void request(int slot, const T* x, int64_t stride, int64_t step, int t, int D) {
    if (r < last) {
      const T* row = x + r * stride;
      if constexpr (kAsync) {
#pragma unroll
        for (int i = 0; i < X::kG; ++i)
          if (X::column(t, i) < D) cp_async16(slots + (slot * X::kG + i) * kBlock * 16, row + X::column(t, i));
      } else {
        next.load(row, t, D);
      }
      r += step;
    }
  }
  // the row in `slot`. A slot may be asked for anew once the sums over its row are known: by then its values have been used.
  __device__ __forceinline__ void pairs(int slot, F2* f) {
    if constexpr (kAsync) {
#pragma unroll
      for (int i = 0; i < X::kG; ++i) next.v[i] = *reinterpret_cast<const Pack<T, kVec>*>(slots + (slot * X::kG + i) * kBlock * 16);
    }
    next.pairs(f);
  }
};
template <int kPending>
__device__ __forceinline__ void feed_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ void feed_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// rows ahead for `arrays` rows of kCols elements per thread: what fits the CTA's share of shared memory, four at most
constexpr int feed_depth(int elem, int block, int arrays) {
  const int stage = block * arrays * kCols * elem, fit = (block <= 256 ? 96 : 192) * 1024 / stage;
  return fit < 1 ? 1 : fit > 4 ? 4 : fit;
}

__device__ __forceinline__ float both(F2 x) {
  const float2 p = split(x);
  return p.x + p.y;
}

// The threads of one row: kTpr of the CTA's kBlock threads. Sums over them give every thread the same value; consecutive calls
// use the two halves of `red` in turn, so one barrier per call is enough.
template <int kTpr, int kBlock>
struct RowThreads {
  static constexpr int kWarps = kTpr / 32;
  __device__ static int index() { return threadIdx.x % kTpr; }
  __device__ static int group() { return threadIdx.x / kTpr; }
  __device__ static void sync() {
    if (kTpr == kBlock)
      __syncthreads();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(group() + 1), "n"(kTpr) : "memory");
  }
  __device__ static float sum(float v, float (*red)[2][kBlock / 32], int& turn) {
    v = warp_reduce_sum(v);
    if (kTpr == 32) return v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) red[turn][0][warp] = v;
    sync();
    v = red[turn][0][group() * kWarps + lane % kWarps];
#pragma unroll
    for (int o = kWarps / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    turn ^= 1;
    return v;
  }
  // two sums at once: the lower half warp takes the first, the upper one the second
  __device__ static float2 sum(float a, float b, float (*red)[2][kBlock / 32], int& turn) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4;
    float v = half ? b : a;
    v += __shfl_xor_sync(0xffffffffu, half ? a : b, 16);
#pragma unroll
    for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (kTpr > 32) {
      if ((lane & 15) == 0) red[turn][half][warp] = v;
      sync();
      const float* from = red[turn][half] + group() * kWarps;
      if (kWarps <= 16) {
        v = from[lane % kWarps];
#pragma unroll
        for (int o = kWarps / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      } else {
        v = from[lane & 15] + from[16 + (lane & 15)];
#pragma unroll
        for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      }
      turn ^= 1;
    }
    return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 16));
  }
};

template <typename T, typename W, int kVec, int kTpr, int kBlock>
__global__ void __launch_bounds__(kBlock, kBlock <= 256 && kVec == 8 && sizeof(W) == 2 ? 3 : 1)
    layernorm_fwd_reg_kernel(const T* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b, T* __restrict__ y,
                             float* __restrict__ mean, float* __restrict__ rstd, int64_t rows, int D, int64_t x_stride,
                             int64_t y_stride, float eps) {
  using Row = RowThreads<kTpr, kBlock>;
  using X = Held<T, kVec, kTpr>;
  constexpr int kDepth = kVec == 1 ? 1 : feed_depth(sizeof(T), kBlock, 1);
  using In = Feed<T, kVec, kTpr, kBlock, kDepth>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[2][2][kBlock / 32];
  const int t = Row::index();
  int turn = 0, slot = 0;
  const float inv_d = 1.f / (float)D;
  const int64_t step = (int64_t)gridDim.x * (kBlock / kTpr);
  int64_t r = blockIdx.x * (int64_t)(kBlock / kTpr) + Row::group();
  In in;
  in.begin(ring, r, rows, t, D);
#pragma unroll
  for (int d = 0; d < kDepth; ++d) {
    in.request(d, x, x_stride, step, t, D);
    feed_commit();
  }
  Held<W, kVec, kTpr> pw, pb;
  pw.fill(1.f);
  pb.fill(0.f);
  if (w) pw.load(w, t, D);
  if (b) pb.load(b, t, D);
  for (; r < rows; r += step) {
    F2 f[kPairs], s = f2(0.f);
    feed_wait<kDepth - 1>();
    in.pairs(slot, f);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) s = add2(s, f[j]);
    const float mu = Row::sum(both(s), red, turn) * inv_d;
    in.request(slot, x, x_stride, step, t, D);
    feed_commit();
    if (++slot == kDepth) slot = 0;
    const F2 minus = f2(-mu);
    s = f2(0.f);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) f[j] = add2(f[j], minus);
    if (D < kTpr * kCols) {
      // the columns past the end are no part of the variance
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const float2 p = split(f[j]);
        const int e0 = 2 * j, e1 = 2 * j + 1;
        f[j] = f2(X::column(t, e0 / kVec) < D ? p.x : 0.f, X::column(t, e1 / kVec) < D ? p.y : 0.f);
      }
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) s = fma2(f[j], f[j], s);
    const float rs = rsqrtf(Row::sum(both(s), red, turn) * inv_d + eps);
    if (t == 0 && mean) {
      mean[r] = mu;
      rstd[r] = rs;
    }
    F2 fw[kPairs], fb[kPairs];
    pw.pairs(fw);
    pb.pairs(fb);
    const F2 scale = f2(rs);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) f[j] = fma2(mul2(f[j], scale), fw[j], fb[j]);
    X::store(y + r * y_stride, t, D, f);
  }
}

// dx, and partial[cta][0][c] = sum of dy * xh, partial[cta][1][c] = sum of dy over the CTA's rows
template <typename T, typename W, int kVec, int kTpr, int kBlock>
__global__ void __launch_bounds__(kBlock, kBlock <= 256 && kVec > 1 ? 2 : 1)
    layernorm_bwd_reg_kernel(const T* __restrict__ x, const W* __restrict__ w, const T* __restrict__ dy,
                             const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
                             float* __restrict__ partial, int64_t rows, int D, int64_t x_stride, int64_t dy_stride,
                             int64_t dx_stride) {
  using Row = RowThreads<kTpr, kBlock>;
  using X = Held<T, kVec, kTpr>;
  constexpr int kGroups = kBlock / kTpr;
  constexpr int kDepth = kVec == 1 ? 1 : feed_depth(sizeof(T), kBlock, 2);
  using In = Feed<T, kVec, kTpr, kBlock, kDepth>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[2][2][kBlock / 32];
  const int t = Row::index(), group = Row::group();
  int turn = 0, slot = 0;
  const float inv_d = 1.f / (float)D;
  const int64_t step = (int64_t)gridDim.x * kGroups;
  int64_t r = blockIdx.x * (int64_t)kGroups + group;
  // columns past the row's end are zero in dy, which makes their every term zero
  In in_x, in_dy;
  in_x.begin(ring, r, rows, t, D);
  in_dy.begin(ring + In::kBytes, r, rows, t, D);
#pragma unroll
  for (int d = 0; d < kDepth; ++d) {
    in_x.request(d, x, x_stride, step, t, D);
    in_dy.request(d, dy, dy_stride, step, t, D);
    feed_commit();
  }
  float nmu = 0.f, nrs = 0.f;
  if (r < rows) {
    nmu = mean[r];
    nrs = rstd[r];
  }
  Held<W, kVec, kTpr> pw;
  pw.fill(1.f);
  if (w) pw.load(w, t, D);
  F2 sw[kPairs], sb[kPairs];
#pragma unroll
  for (int j = 0; j < kPairs; ++j) sw[j] = sb[j] = f2(0.f);
  for (; r < rows; r += step) {
    const float rs = nrs;
    const F2 minus = f2(-nmu), scale = f2(rs);
    F2 h[kPairs], g[kPairs], s0 = f2(0.f), s1 = f2(0.f);
    feed_wait<kDepth - 1>();
    in_x.pairs(slot, h);
    in_dy.pairs(slot, g);
    if (r + step < rows) {
      nmu = mean[r + step];
      nrs = rstd[r + step];
    }
    {
      F2 fw[kPairs];
      pw.pairs(fw);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        h[j] = mul2(add2(h[j], minus), scale);
        sw[j] = fma2(g[j], h[j], sw[j]);
        sb[j] = add2(sb[j], g[j]);
        g[j] = mul2(g[j], fw[j]);
        s0 = add2(s0, g[j]);
        s1 = fma2(g[j], h[j], s1);
      }
    }
    const float2 sums = Row::sum(both(s0), both(s1), red, turn);
    in_x.request(slot, x, x_stride, step, t, D);
    in_dy.request(slot, dy, dy_stride, step, t, D);
    feed_commit();
    if (++slot == kDepth) slot = 0;
    if (dx) {
      const F2 c1 = f2(-rs * sums.x * inv_d), c2 = f2(-rs * sums.y * inv_d);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) g[j] = fma2(g[j], scale, fma2(h[j], c2, c1));
      X::store(dx + r * dx_stride, t, D, g);
    }
  }
  if (!partial) return;
  float* out = partial + (int64_t)blockIdx.x * 2 * D;
  if (kGroups == 1) {
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const float2 a = split(sw[j]), c = split(sb[j]);
      const int c0 = X::column(t, 2 * j / kVec) + 2 * j % kVec, c1 = X::column(t, (2 * j + 1) / kVec) + (2 * j + 1) % kVec;
      if (c0 < D) out[c0] = a.x, out[D + c0] = c.x;
      if (c1 < D) out[c1] = a.y, out[D + c1] = c.y;
    }
  } else {
    // the CTA's groups add their sums up in turn
    __shared__ float joined[2][kGroups > 1 ? kTpr * kCols : 1];
    for (int q = 0; q < kGroups; ++q) {
      if (q == group) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const float2 a = split(sw[j]), c = split(sb[j]);
          const int c0 = X::column(t, 2 * j / kVec) + 2 * j % kVec, c1 = X::column(t, (2 * j + 1) / kVec) + (2 * j + 1) % kVec;
          joined[0][c0] = (q ? joined[0][c0] : 0.f) + a.x;
          joined[0][c1] = (q ? joined[0][c1] : 0.f) + a.y;
          joined[1][c0] = (q ? joined[1][c0] : 0.f) + c.x;
          joined[1][c1] = (q ? joined[1][c1] : 0.f) + c.y;
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < D; c += kBlock) {
      out[c] = joined[0][c];
      out[D + c] = joined[1][c];
    }
  }
}

constexpr int kSms = 148;

constexpr int feed_bytes(int elem, int block, int arrays) { return feed_depth(elem, block, arrays) * block * arrays * kCols * elem; }

// the shared memory of one kernel above 48 KB, allowed once per device
struct SmemSet {
  bool done[64] = {};
  template <typename K>
  bool allow(K kernel, int bytes) {
    int device = 0;
    if (bytes <= 48 * 1024) return true;
    if (cudaGetDevice(&device) != cudaSuccess || device >= 64) return false;
    if (!done[device]) done[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
    return done[device];
  }
};

inline unsigned row_grid(int64_t rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

// rows of fewer than 256 threads share a CTA
template <typename T, typename W>
int fwd_reg(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows, int64_t D,
            int64_t x_stride, int64_t y_stride, float eps, bool vec, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  int tpr = 32;
  while (tpr * kCols < D) tpr *= 2;
  const int block = tpr < 256 ? 256 : tpr, per = block / tpr;
  const int64_t ctas = (rows + per - 1) / per, most = (int64_t)kSms * (block <= 256 ? 3 : 1024 / block);
  const unsigned grid = (unsigned)(ctas < most ? ctas : most);
#define ROWS(TPR)                                                                                                             \
  case TPR: {                                                                                                                 \
    constexpr int kB = (TPR) < 256 ? 256 : (TPR);                                                                             \
    auto k = vec ? layernorm_fwd_reg_kernel<T, W, kV, TPR, kB> : layernorm_fwd_reg_kernel<T, W, 1, TPR, kB>;                  \
    const int smem = vec ? feed_bytes(sizeof(T), kB, 1) : 0;                                                                  \
    static SmemSet vec_set;                                                                                                   \
    if (vec && !vec_set.allow(k, smem)) return MB_ERR_LAUNCH;                                                                 \
    k<<<grid, kB, smem, s>>>((const T*)x, (const W*)w, (const W*)b, (T*)y, mean, rstd, rows, (int)D, x_stride, y_stride, eps); \
    break;                                                                                                                    \
  }
  switch (tpr) {
    ROWS(32) ROWS(64) ROWS(128) ROWS(256) ROWS(512) ROWS(1024)
  }
#undef ROWS
  return check_launch();
}

template <typename T>
int fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows, int64_t D,
        int64_t x_stride, int64_t y_stride, bool w_f32, float eps, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  const bool vec = D % kV == 0 && x_stride % kV == 0 && y_stride % kV == 0 && is_aligned(x, 16) && is_aligned(y, 16) &&
                   is_aligned(w, 16) && is_aligned(b, 16);
  if (D <= 16384) {
    if (w_f32) return fwd_reg<T, float>(x, w, b, y, mean, rstd, rows, D, x_stride, y_stride, eps, vec, s);
    return fwd_reg<T, T>(x, w, b, y, mean, rstd, rows, D, x_stride, y_stride, eps, vec, s);
  }
  auto k = vec ? layernorm_fwd_kernel<T, kV> : layernorm_fwd_kernel<T, 1>;
  k<<<row_grid(rows), kThreads, 0, s>>>((const T*)x, w, b, (T*)y, mean, rstd, rows, D, x_stride, y_stride, eps, w_f32);
  return check_launch();
}

// Threads per row in the backward pass (0: too long for registers).
inline int bwd_tpr(int64_t D) {
  if (D > 1024 * kCols) return 0;
  int tpr = 32;
  while (tpr * kCols < D) tpr *= 2;
  return tpr;
}
inline int bwd_ctas(int64_t rows, int tpr) {
  const int block = tpr < 256 ? 256 : tpr, per = block / tpr;
  const int64_t ctas = (rows + per - 1) / per, most = kSms * (block < 512 ? 512 / block : 1);
  return (int)(ctas < most ? ctas : most);
}

template <typename T, typename W>
int bwd_reg(const void* x, const void* w, const void* dy, const float* mean, const float* rstd, void* dx, float* sums,
            int64_t rows, int64_t D, int64_t x_stride, int64_t dy_stride, int64_t dx_stride, bool vec, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  const int tpr = bwd_tpr(D), grid = bwd_ctas(rows, tpr);
#define ROWS(TPR)                                                                                                             \
  case TPR: {                                                                                                                 \
    constexpr int kB = (TPR) < 256 ? 256 : (TPR);                                                                             \
    auto k = vec ? layernorm_bwd_reg_kernel<T, W, kV, TPR, kB> : layernorm_bwd_reg_kernel<T, W, 1, TPR, kB>;                  \
    const int smem = vec ? feed_bytes(sizeof(T), kB, 2) : 0;                                                                  \
    static SmemSet vec_set;                                                                                                   \
    if (vec && !vec_set.allow(k, smem)) return MB_ERR_LAUNCH;                                                                 \
    k<<<grid, kB, smem, s>>>((const T*)x, (const W*)w, (const T*)dy, mean, rstd, (T*)dx, sums, rows, (int)D, x_stride, dy_stride, \
                          dx_stride);                                                                                         \
    break;                                                                                                                    \
  }
  switch (tpr) {
    ROWS(32) ROWS(64) ROWS(128) ROWS(256) ROWS(512) ROWS(1024)
  }
#undef ROWS
  return check_launch();
}

template <typename T>
int bwd(const void* x, const void* w, const void* dy, const float* mean, const float* rstd, void* dx, void* dw, void* db,
        float* partial, int64_t rows, int64_t D, int64_t x_stride, int64_t dy_stride, int64_t dx_stride, bool w_f32,
        cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  const bool vec = D % kV == 0 && x_stride % kV == 0 && dy_stride % kV == 0 && dx_stride % kV == 0 && is_aligned(x, 16) &&
                   is_aligned(dy, 16) && is_aligned(dx, 16) && is_aligned(w, 16);
  const int parts = mb_layernorm_bwd_parts(rows, D);
  float* sums = dw || db ? partial : nullptr;
  if (bwd_tpr(D)) {
    const int rc = w_f32 ? bwd_reg<T, float>(x, w, dy, mean, rstd, dx, sums, rows, D, x_stride, dy_stride, dx_stride, vec, s)
                         : bwd_reg<T, T>(x, w, dy, mean, rstd, dx, sums, rows, D, x_stride, dy_stride, dx_stride, vec, s);
    if (rc) return rc;
  } else {
    if (dx) {
      auto k = vec ? layernorm_dx_kernel<T, kV> : layernorm_dx_kernel<T, 1>;
      k<<<row_grid(rows), kThreads, 0, s>>>((const T*)x, w, (const T*)dy, mean, rstd, (T*)dx, rows, D, x_stride, dy_stride,
                                            dx_stride, w_f32);
      if (check_launch()) return MB_ERR_LAUNCH;
    }
    if (sums) {
      layernorm_dw_kernel<T><<<dim3((unsigned)((D + kThreads - 1) / kThreads), parts), kThreads, 0, s>>>(
          (const T*)x, (const T*)dy, mean, rstd, partial, rows, D, x_stride, dy_stride);
      if (check_launch()) return MB_ERR_LAUNCH;
    }
  }
  if (sums) layernorm_dw_join_kernel<T><<<dim3((unsigned)((D + 31) / 32), 2), 1024, 0, s>>>(partial, dw, db, parts, D, w_f32);
  return check_launch();
}

}  // namespace

extern "C" int mb_layernorm_bwd_parts(int64_t rows, int64_t D) {
  if (const int tpr = bwd_tpr(D)) return bwd_ctas(rows < 1 ? 1 : rows, tpr);
  const int64_t col_ctas = (D + kThreads - 1) / kThreads;
  int64_t parts = kSms * 8 / (col_ctas < 1 ? 1 : col_ctas);
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
