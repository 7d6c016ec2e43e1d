// Distillation loss from a teacher's top entries, forward and backward.
//
//   p = softmax(top / tau) over the row's valid entries, q = softmax(z / tau) over the vocabulary
//   row   = (1 - hard) tau^2 sum_k p_k (log p_k - log q_{id_k}) + hard (logsumexp(z) - z_target)
//   dz_j  = (1 - hard) tau (q_j - sum_{k: id_k = j} p_k) + hard (softmax(z)_j - [j = target])
//
// Bound by the bytes of the logits: read by the forward pass, read again and written as the gradient by the backward pass.
// Sums and row statistics are fp32; sums have a fixed order, so the same inputs give the same bits.
#include "kernels_api.h"
#include "vec_io.cuh"

#define MB_STREAM(s) reinterpret_cast<cudaStream_t>(s)

namespace {

using namespace mb;

inline int check_launch() { return cudaPeekAtLastError() == cudaSuccess ? MB_OK : MB_ERR_LAUNCH; }

constexpr int kTopThreads = 128;
constexpr int kRowThreads = 512;

__device__ __forceinline__ int64_t id_at(const mb_distill_t& d, int64_t i) {
  return d.ids_i64 ? reinterpret_cast<const int64_t*>(d.ids)[i] : (int64_t)reinterpret_cast<const int32_t*>(d.ids)[i];
}
__device__ __forceinline__ float top_at(const mb_distill_t& d, int64_t i) {
  if (d.top_dtype == MB_F32) return reinterpret_cast<const float*>(d.top)[i];
  if (d.top_dtype == MB_BF16) return to_f32(reinterpret_cast<const __nv_bfloat16*>(d.top)[i]);
  return to_f32(reinterpret_cast<const __half*>(d.top)[i]);
}

// Entry i of row r takes part when its id names a word and its logit is not -inf (a teacher's mask); its logit goes to *t.
__device__ __forceinline__ bool entry(const mb_distill_t& d, int64_t i, float* t) {
  const int64_t id = id_at(d, i);
  if (id < 0 || id >= d.V) return false;
  *t = top_at(d, i);
  return *t != -INFINITY;
}

// One CTA per row: the teacher's probabilities over the valid entries (0 in the others), sum p log p, whether the row counts.
__global__ void __launch_bounds__(kTopThreads) distill_teacher_kernel(const mb_distill_t d) {
  __shared__ float red[kTopThreads / 32];
  const float inv_tau = 1.f / d.tau;
  for (int64_t r = blockIdx.x; r < d.rows; r += gridDim.x) {
    const int64_t base = r * d.K;
    bool counts = true;
    if (d.targets) {
      const int64_t t = d.targets[r];
      counts = t != d.ignore_index && t >= 0 && t < d.V;
    }
    float m = -INFINITY, any = 0.f;
    float t;
    for (int k = threadIdx.x; k < d.K; k += kTopThreads) {
      if (entry(d, base + k, &t)) {
        any = 1.f;
        m = fmaxf(m, t);
      }
    }
    m = block_reduce_max<kTopThreads>(m, red);
    any = block_reduce_max<kTopThreads>(any, red);
    const bool live = counts && any > 0.f;
    float s = 0.f, e = 0.f;
    for (int k = threadIdx.x; k < d.K; k += kTopThreads) {
      if (live && entry(d, base + k, &t)) {
        t = (t - m) * inv_tau;
        const float w = expf(t);
        s += w;
        if (!(w <= 0.f)) e += w * t;  // weight 0: t may have overflowed to -inf; NaN goes on
      }
    }
    s = block_reduce_sum<kTopThreads>(s, red);
    e = block_reduce_sum<kTopThreads>(e, red);
    const float inv = live ? 1.f / s : 0.f;
    for (int k = threadIdx.x; k < d.K; k += kTopThreads)
      d.p[base + k] = live && entry(d, base + k, &t) ? expf((t - m) * inv_tau) * inv : 0.f;
    if (threadIdx.x == 0) {
      d.live[r] = live;
      d.entropy[r] = live ? e * inv - logf(s) : 0.f;
    }
  }
}

// factor = scale, or scale over the number of rows that count (one CTA)
__global__ void __launch_bounds__(1024) distill_factor_kernel(const mb_distill_t d) {
  __shared__ int part[32];
  int n = 0;
  for (int64_t r = threadIdx.x; r < d.rows; r += 1024) n += d.live[r];
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x < 32) {
    n = __reduce_add_sync(0xffffffffu, part[threadIdx.x]);
    if (threadIdx.x == 0) d.factor[0] = d.mean ? d.scale / (float)(n > 0 ? n : 1) : d.scale;
  }
}

// one value joins a running maximum m and the sums of exp((z - m) / tau) and, with kHard, exp(z - m)
template <bool kHard>
__device__ __forceinline__ void join(float& m, float& st, float& s1, float om, float ost, float os1, float inv_tau) {
  const float nm = fmaxf(m, om);
  if (nm == -INFINITY) return;
  const float a = m == -INFINITY ? 0.f : __expf((m - nm) * inv_tau), b = om == -INFINITY ? 0.f : __expf((om - nm) * inv_tau);
  st = st * a + ost * b;
  if (kHard) {
    const float a1 = m == -INFINITY ? 0.f : __expf(m - nm), b1 = om == -INFINITY ? 0.f : __expf(om - nm);
    s1 = s1 * a1 + os1 * b1;
  }
  m = nm;
}

template <typename T, int kV, bool kHard>
__global__ void __launch_bounds__(kRowThreads) distill_row_kernel(const mb_distill_t d) {
  __shared__ float sm[3][kRowThreads / 32];
  __shared__ float red[kRowThreads / 32];
  const float inv_tau = 1.f / d.tau;
  for (int64_t r = blockIdx.x; r < d.rows; r += gridDim.x) {
    if (!d.live[r]) {
      if (threadIdx.x == 0) d.row_loss[r] = 0.f;
      continue;
    }
    const T* z = reinterpret_cast<const T*>(d.logits) + r * d.stride;
    float m = -INFINITY, st = 0.f, s1 = 0.f;
    for (int64_t c = threadIdx.x * kV; c < d.V; c += kRowThreads * kV) {
      float f[kV];
      load_vec<T, kV>(z + c, f);
      float lm = f[0];
#pragma unroll
      for (int k = 1; k < kV; ++k) lm = fmaxf(lm, f[k]);
      const float nm = fmaxf(m, lm);
      if (nm == -INFINITY) {
#pragma unroll
        for (int k = 0; k < kV; ++k)
          if (f[k] != f[k]) st = s1 = NAN;  // fmaxf drops NaN: the row has to show it
        continue;
      }
      float at = 0.f, a1 = 0.f;
#pragma unroll
      for (int k = 0; k < kV; ++k) {
        at += __expf((f[k] - nm) * inv_tau);
        if (kHard) a1 += __expf(f[k] - nm);
      }
      st = st * __expf((m - nm) * inv_tau) + at;
      if (kHard) s1 = s1 * __expf(m - nm) + a1;
      m = nm;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m, o), ot = __shfl_xor_sync(0xffffffffu, st, o);
      const float o1 = kHard ? __shfl_xor_sync(0xffffffffu, s1, o) : 0.f;
      join<kHard>(m, st, s1, om, ot, o1, inv_tau);
    }
    __syncthreads();
    if (lane == 0) {
      sm[0][warp] = m;
      sm[1][warp] = st;
      sm[2][warp] = s1;
    }
    __syncthreads();
    m = -INFINITY, st = 0.f, s1 = 0.f;
    for (int w = 0; w < kRowThreads / 32; ++w) join<kHard>(m, st, s1, sm[0][w], sm[1][w], sm[2][w], inv_tau);
    // cross entropy of the teacher's entries against q
    const float log_st = logf(st);
    float ce = 0.f;
    for (int k = threadIdx.x; k < d.K; k += kRowThreads) {
      const float p = d.p[r * d.K + k];
      if (p != 0.f) ce += p * ((to_f32(z[id_at(d, r * d.K + k)]) - m) * inv_tau - log_st);
    }
    ce = block_reduce_sum<kRowThreads>(ce, red);
    if (threadIdx.x == 0) {
      d.stats[r * 3] = m;
      d.stats[r * 3 + 1] = 1.f / st;
      d.stats[r * 3 + 2] = kHard ? 1.f / s1 : 0.f;
      float l = d.hard < 1.f ? (1.f - d.hard) * d.tau * d.tau * (d.entropy[r] - ce) : 0.f;
      if (kHard) l += d.hard * (logf(s1) + m - to_f32(z[d.targets[r]]));
      d.row_loss[r] = l;
    }
  }
}

// loss = factor * sum of the row losses, in a fixed order (one CTA)
__global__ void __launch_bounds__(1024) distill_sum_kernel(const mb_distill_t d) {
  __shared__ float red[32];
  float s = 0.f;
  for (int64_t r = threadIdx.x; r < d.rows; r += 1024) s += d.row_loss[r];
  s = block_reduce_sum<1024>(s, red);
  if (threadIdx.x == 0) d.loss[0] = s * d.factor[0];
}

template <typename T, int kV, bool kHard>
__global__ void __launch_bounds__(kRowThreads)
    distill_grad_kernel(const mb_distill_t d, const float* __restrict__ gout, T* __restrict__ grad, int64_t grad_stride) {
  const float inv_tau = 1.f / d.tau;
  const float sc = d.factor[0] * gout[0], a_soft = (1.f - d.hard) * d.tau * sc, a_hard = d.hard * sc;
  for (int64_t r = blockIdx.x; r < d.rows; r += gridDim.x) {
    const T* z = reinterpret_cast<const T*>(d.logits) + r * d.stride;
    T* g = grad + r * grad_stride;
    const bool live = d.live[r];
    const float m = live ? d.stats[r * 3] : 0.f;
    const float iq = live ? d.stats[r * 3 + 1] * a_soft : 0.f, i1 = live && kHard ? d.stats[r * 3 + 2] * a_hard : 0.f;
    auto slope = [&](float v) {
      float o = __expf((v - m) * inv_tau) * iq;
      if (kHard) o += __expf(v - m) * i1;
      return o;
    };
    for (int64_t c = threadIdx.x * kV; c < d.V; c += kRowThreads * kV) {
      float f[kV];
      if (live) load_vec<T, kV>(z + c, f);
#pragma unroll
      for (int k = 0; k < kV; ++k) f[k] = live ? slope(f[k]) : 0.f;
      store_vec<T, kV>(g + c, f);
    }
    if (!live) continue;
    __syncthreads();
    // the places that the teacher or the target names, each written once by the first entry that names it
    const int64_t t = kHard ? d.targets[r] : -1;
    for (int k = threadIdx.x; k < d.K + (kHard ? 1 : 0); k += kRowThreads) {
      const int64_t j = k < d.K ? id_at(d, r * d.K + k) : t;
      if (j < 0 || j >= d.V) continue;
      bool first = true;
      float p = 0.f;
      for (int i = 0; i < d.K && first; ++i) {
        if (id_at(d, r * d.K + i) != j) continue;
        if (i < k) first = false;
        p += d.p[r * d.K + i];
      }
      if (first) g[j] = from_f32<T>(slope(to_f32(z[j])) - p * a_soft - (j == t ? a_hard : 0.f));
    }
  }
}

inline unsigned row_grid(int64_t rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

template <typename T>
int fwd(const mb_distill_t& d, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  const bool vec = d.V % kV == 0 && d.stride % kV == 0 && is_aligned(d.logits, 16);
  auto k = d.hard > 0.f ? (vec ? distill_row_kernel<T, kV, true> : distill_row_kernel<T, 1, true>)
                        : (vec ? distill_row_kernel<T, kV, false> : distill_row_kernel<T, 1, false>);
  k<<<row_grid(d.rows), kRowThreads, 0, s>>>(d);
  return check_launch();
}

template <typename T>
int bwd(const mb_distill_t& d, const float* gout, void* grad, int64_t grad_stride, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(T);
  const bool vec = d.V % kV == 0 && d.stride % kV == 0 && grad_stride % kV == 0 && is_aligned(d.logits, 16) && is_aligned(grad, 16);
  auto k = d.hard > 0.f ? (vec ? distill_grad_kernel<T, kV, true> : distill_grad_kernel<T, 1, true>)
                        : (vec ? distill_grad_kernel<T, kV, false> : distill_grad_kernel<T, 1, false>);
  k<<<row_grid(d.rows), kRowThreads, 0, s>>>(d, gout, (T*)grad, grad_stride);
  return check_launch();
}

bool sane(const mb_distill_t& d) {
  return d.V > 0 && d.K > 0 && d.tau > 0.f && d.hard >= 0.f && d.hard <= 1.f && (d.hard == 0.f || d.targets || d.rows <= 0) &&
         (d.top_dtype == MB_F32 || d.top_dtype == MB_BF16 || d.top_dtype == MB_F16);
}

}  // namespace

extern "C" int mb_distill_fwd(const mb_distill_t* d, void* stream) {
  if (!sane(*d)) return MB_ERR_ARG;
  cudaStream_t s = MB_STREAM(stream);
  if (d->rows > 0) {
    distill_teacher_kernel<<<row_grid(d->rows), kTopThreads, 0, s>>>(*d);
    if (check_launch()) return MB_ERR_LAUNCH;
  }
  distill_factor_kernel<<<1, 1024, 0, s>>>(*d);
  if (check_launch()) return MB_ERR_LAUNCH;
  if (d->rows > 0) {
    int rc = MB_ERR_ARG;
    if (d->dtype == MB_BF16) rc = fwd<__nv_bfloat16>(*d, s);
    if (d->dtype == MB_F16) rc = fwd<__half>(*d, s);
    if (d->dtype == MB_F32) rc = fwd<float>(*d, s);
    if (rc) return rc;
  }
  distill_sum_kernel<<<1, 1024, 0, s>>>(*d);
  return check_launch();
}

extern "C" int mb_distill_bwd(const mb_distill_t* d, const float* gout, void* grad, int64_t grad_stride, void* stream) {
  if (!sane(*d)) return MB_ERR_ARG;
  if (d->rows <= 0) return MB_OK;
  switch (d->dtype) {
    case MB_BF16: return bwd<__nv_bfloat16>(*d, gout, grad, grad_stride, MB_STREAM(stream));
    case MB_F16: return bwd<__half>(*d, gout, grad, grad_stride, MB_STREAM(stream));
    case MB_F32: return bwd<float>(*d, gout, grad, grad_stride, MB_STREAM(stream));
    default: return MB_ERR_ARG;
  }
}
