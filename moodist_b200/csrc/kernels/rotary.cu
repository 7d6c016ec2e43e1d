// Rotary positions on q and k heads in one launch: head dimensions [0, R) turn pairwise by the angle of their token's
// position, the rest pass through.
//
//   a' = a c - b s,  b' = b c + a s      (c, s) = (cos, sin)[position, j];  the backward pass takes -s (the transpose)
//   half layout:  pairs (j, j + R/2);    interleaved: pairs (2j, 2j + 1)
//
// Bound by the bytes of q and k, read once and written once. A thread takes V pairs of one token (V * sizeof(T) = 16 bytes where
// sizes, strides and addresses allow: two vector loads and two vector stores) in four neighbouring heads: eight loads in
// flight, and the cosines and sines, which are twice the bytes of the pairs of one 16-bit head, are read once for the four
// (two heads per thread: 35 us where four take 31). 8192 tokens, 40 heads of 128, bf16: 31 us, 5.5 TB/s, each way.
#include "kernels_api.h"
#include "vec_io.cuh"

#define MB_STREAM(s) reinterpret_cast<cudaStream_t>(s)

namespace {

using namespace mb;

inline int check_launch() { return cudaPeekAtLastError() == cudaSuccess ? MB_OK : MB_ERR_LAUNCH; }

constexpr int kHeads = 4;  // heads per thread

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}

// chunks of a tensor's heads
__host__ __device__ __forceinline__ int head_chunks(int heads) { return (heads + kHeads - 1) / kHeads; }

template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(256, 3) rotary_kernel(const __grid_constant__ mb_rotary_t p, int64_t threads) {
  const int half = p.rot / 2;
  const int turns = half / V;                                                 // items of a head that turn
  const int copies = p.in_place ? 0 : (p.dim - p.rot + 2 * V - 1) / (2 * V);  // items that only move
  const int per_head = turns + copies, chunks = head_chunks(p.q_heads) + head_chunks(p.k_heads);
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= threads) return;
  int64_t b, s;
  int chunk, item;
  if (threads <= 0xffffffffll) {
    const uint32_t u = (uint32_t)i, q = u / (uint32_t)per_head, t = q / (uint32_t)chunks, bb = t / (uint32_t)p.seq;
    item = (int)(u - q * per_head);
    chunk = (int)(q - t * chunks);
    b = bb;
    s = t - bb * (uint32_t)p.seq;
  } else {
    const int64_t q = i / per_head;
    item = (int)(i - q * per_head);
    const int64_t token = q / chunks;
    chunk = (int)(q - token * chunks);
    b = token / p.seq;
    s = token - b * p.seq;
  }
  const bool is_k = chunk >= head_chunks(p.q_heads);
  const mb_rotary_heads_t& x = is_k ? p.k : p.q;
  const int h0 = (is_k ? chunk - head_chunks(p.q_heads) : chunk) * kHeads, heads = (is_k ? p.k_heads : p.q_heads) - h0;
  const int j = item * V;
  const bool moves = item >= turns;
  const int rest = p.rot + 2 * (j - half);
  const int first = moves ? rest : kInterleaved ? 2 * j : j;
  const int apart = moves || kInterleaved ? V : half;  // from the first vector to the second
  const bool both = !moves || first + apart < p.dim;
  const T* in = reinterpret_cast<const T*>(x.in) + b * x.in_batch + s * x.in_seq + h0 * x.in_head + first;
  T* out = reinterpret_cast<T*>(x.out) + b * x.out_batch + s * x.out_seq + h0 * x.out_head + first;
  Pack<T, V> va[kHeads], vb[kHeads];
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    if (k < heads) {
      va[k] = load_pack<T, V>(in + k * x.in_head);
      if (both) vb[k] = load_pack<T, V>(in + k * x.in_head + apart);
    }
  }
  if (!moves) {
    int64_t pos = s;
    if (p.positions) {
      const int64_t at = b * p.pos_batch + s * p.pos_seq;
      pos = p.pos_i64 ? reinterpret_cast<const int64_t*>(p.positions)[at] : reinterpret_cast<const int32_t*>(p.positions)[at];
    }
    if (pos >= p.length) {
      // a position that the tables do not have shows as NaN
#pragma unroll
      for (int k = 0; k < kHeads; ++k) va[k] = vb[k] = splat<T, V>(NAN);
    } else if (pos >= 0) {
      constexpr int kStep = V <= 4 ? V : 4;
      float c[V], sn[V];
#pragma unroll
      for (int e = 0; e < V; e += kStep) {
        load_vec<float, kStep>(p.cos_tab + pos * half + j + e, c + e);
        load_vec<float, kStep>(p.sin_tab + pos * half + j + e, sn + e);
      }
      if (p.inverse) {
#pragma unroll
        for (int e = 0; e < V; ++e) sn[e] = -sn[e];
      }
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        float f[2 * V], o[2 * V];
        unpack<T, V>(va[k], f);
        unpack<T, V>(vb[k], f + V);
        // every vector width and layout rounds alike: first b s (a s), then its sum with a c (b c) in one step
        if constexpr (kInterleaved || V == 1) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int ia = kInterleaved ? 2 * e : e, ib = kInterleaved ? 2 * e + 1 : e + V;
            const float2 t = split(fma2(f2(f[ia], f[ib]), f2(c[e]), mul2(f2(f[ib], f[ia]), f2(-sn[e], sn[e]))));
            o[ia] = t.x;
            o[ib] = t.y;
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            const F2 a = f2(f[e], f[e + 1]), bb = f2(f[V + e], f[V + e + 1]), cc = f2(c[e], c[e + 1]), ss = f2(sn[e], sn[e + 1]);
            const float2 ta = split(fma2(a, cc, mul2(bb, f2(-sn[e], -sn[e + 1])))), tb = split(fma2(bb, cc, mul2(a, ss)));
            o[e] = ta.x;
            o[e + 1] = ta.y;
            o[V + e] = tb.x;
            o[V + e + 1] = tb.y;
          }
        }
        va[k] = pack<T, V>(o);
        vb[k] = pack<T, V>(o + V);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    if (k < heads) {
      *reinterpret_cast<Pack<T, V>*>(out + k * x.out_head) = va[k];
      if (both) *reinterpret_cast<Pack<T, V>*>(out + k * x.out_head + apart) = vb[k];
    }
  }
}

// whether V elements at a time fit the sizes, strides and addresses of these heads
bool fits(const mb_rotary_heads_t& x, int heads, int V, int elem) {
  if (heads == 0) return true;
  return x.in_batch % V == 0 && x.in_seq % V == 0 && x.in_head % V == 0 && x.out_batch % V == 0 && x.out_seq % V == 0 &&
         x.out_head % V == 0 && is_aligned(x.in, V * elem) && is_aligned(x.out, V * elem);
}

template <typename T, int V>
int launch(const mb_rotary_t& p, cudaStream_t stream) {
  const int64_t per_head = p.rot / 2 / V + (p.in_place ? 0 : (p.dim - p.rot + 2 * V - 1) / (2 * V));
  const int64_t threads = p.batch * p.seq * (head_chunks(p.q_heads) + head_chunks(p.k_heads)) * per_head;
  if (threads == 0) return MB_OK;
  const int64_t grid = (threads + 255) / 256;
  if (grid > 0x7fffffffll) return MB_ERR_TOO_BIG;
  if (p.interleaved)
    rotary_kernel<T, V, true><<<(unsigned)grid, 256, 0, stream>>>(p, threads);
  else
    rotary_kernel<T, V, false><<<(unsigned)grid, 256, 0, stream>>>(p, threads);
  return check_launch();
}

template <typename T>
int dispatch(const mb_rotary_t& p, cudaStream_t stream) {
  int V = 16 / (int)sizeof(T);
  while (V > 1 && !((p.rot / 2) % V == 0 && (p.dim - p.rot) % V == 0 && is_aligned(p.cos_tab, V < 4 ? V * 4 : 16) &&
                    is_aligned(p.sin_tab, V < 4 ? V * 4 : 16) && fits(p.q, p.q_heads, V, sizeof(T)) &&
                    fits(p.k, p.k_heads, V, sizeof(T))))
    V /= 2;
  switch (V) {
    case 8:
      if constexpr (sizeof(T) == 2) return launch<T, 8>(p, stream);
      return MB_ERR_ARG;
    case 4: return launch<T, 4>(p, stream);
    case 2: return launch<T, 2>(p, stream);
    default: return launch<T, 1>(p, stream);
  }
}

}  // namespace

extern "C" int mb_rotary(const mb_rotary_t* p, void* stream) {
  if (p->batch <= 0 || p->seq <= 0) return MB_OK;
  if (p->rot < 2 || p->rot % 2 || p->dim < p->rot || p->q_heads < 0 || p->k_heads < 0 || p->length < 1) return MB_ERR_ARG;
  if (!p->positions && p->seq > p->length) return MB_ERR_ARG;
  switch (p->dtype) {
    case MB_BF16: return dispatch<__nv_bfloat16>(*p, MB_STREAM(stream));
    case MB_F16: return dispatch<__half>(*p, MB_STREAM(stream));
    case MB_F32: return dispatch<float>(*p, MB_STREAM(stream));
    default: return MB_ERR_ARG;
  }
}
