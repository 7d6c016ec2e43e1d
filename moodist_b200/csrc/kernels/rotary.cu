// Rotary positions on q and k heads in one launch: head dimensions [0, R) turn pairwise by the angle of their token's
// position, the rest pass through.
//
//   a' = a c - b s,  b' = b c + a s      (c, s) = (cos, sin)[position, j];  the backward pass takes -s (the transpose)
//   half layout:  pairs (j, j + R/2);    interleaved: pairs (2j, 2j + 1)
//
// Bound by the bytes of q and k, read once and written once. A thread moves V elements of both members of V pairs with two
// vector loads and two vector stores, V * sizeof(T) = 16 bytes where sizes, strides and addresses allow.
#include "kernels_api.h"
#include "vec_io.cuh"

#define MB_STREAM(s) reinterpret_cast<cudaStream_t>(s)

namespace {

using namespace mb;

inline int check_launch() { return cudaPeekAtLastError() == cudaSuccess ? MB_OK : MB_ERR_LAUNCH; }

template <typename T, int V>
__global__ void __launch_bounds__(256) rotary_kernel(const mb_rotary_t p) {
  const int half = p.rot / 2;
  const int turns = half / V;                                  // items of a head that turn
  const int copies = (p.dim - p.rot + 2 * V - 1) / (2 * V);    // items that only move (none in place)
  const int per_head = turns + (p.in_place ? 0 : copies);
  const int heads = p.q_heads + p.k_heads;
  const int64_t total = p.batch * p.seq * heads * per_head;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int item = (int)(i % per_head);
    int64_t rest = i / per_head;
    int h = (int)(rest % heads);
    rest /= heads;
    const int64_t s = rest % p.seq, b = rest / p.seq;
    const bool is_k = h >= p.q_heads;
    if (is_k) h -= p.q_heads;
    const mb_rotary_heads_t& x = is_k ? p.k : p.q;
    const T* in = reinterpret_cast<const T*>(x.in) + b * x.in_batch + s * x.in_seq + h * x.in_head;
    T* out = reinterpret_cast<T*>(x.out) + b * x.out_batch + s * x.out_seq + h * x.out_head;
    if (item >= turns) {
      const int c = p.rot + (item - turns) * 2 * V;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (c + k * V < p.dim)
          *reinterpret_cast<Pack<T, V>*>(out + c + k * V) = *reinterpret_cast<const Pack<T, V>*>(in + c + k * V);
      continue;
    }
    int64_t pos = s;
    if (p.positions) {
      const int64_t at = b * p.pos_batch + s * p.pos_seq;
      pos = p.pos_i64 ? reinterpret_cast<const int64_t*>(p.positions)[at] : reinterpret_cast<const int32_t*>(p.positions)[at];
    }
    const int j = item * V;
    const int first = p.interleaved ? 2 * j : j, second = p.interleaved ? 2 * j + V : j + half;
    Pack<T, V> va = *reinterpret_cast<const Pack<T, V>*>(in + first);
    Pack<T, V> vb = *reinterpret_cast<const Pack<T, V>*>(in + second);
    if (pos >= p.length) {
      // a position that the tables do not have shows as NaN
#pragma unroll
      for (int k = 0; k < V; ++k) va.v[k] = vb.v[k] = from_f32<T>(NAN);
    } else if (pos >= 0) {
      float c[V], sn[V];
      load_vec<float, V <= 4 ? V : 4>(p.cos_tab + pos * half + j, c);
      load_vec<float, V <= 4 ? V : 4>(p.sin_tab + pos * half + j, sn);
      if (V == 8) {
        load_vec<float, 4>(p.cos_tab + pos * half + j + 4, c + V / 2);
        load_vec<float, 4>(p.sin_tab + pos * half + j + 4, sn + V / 2);
      }
      float f[2 * V], o[2 * V];
      unpack<T, V>(va, f);
      unpack<T, V>(vb, f + V);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float sk = p.inverse ? -sn[k] : sn[k];
        const float a = p.interleaved ? f[2 * k] : f[k], bb = p.interleaved ? f[2 * k + 1] : f[k + V];
        // spelled out, so that every vector width gives the same bits
        const float oa = fmaf(a, c[k], -__fmul_rn(bb, sk)), ob = fmaf(bb, c[k], __fmul_rn(a, sk));
        if (p.interleaved) {
          o[2 * k] = oa;
          o[2 * k + 1] = ob;
        } else {
          o[k] = oa;
          o[k + V] = ob;
        }
      }
      va = pack<T, V>(o);
      vb = pack<T, V>(o + V);
    }
    *reinterpret_cast<Pack<T, V>*>(out + first) = va;
    *reinterpret_cast<Pack<T, V>*>(out + second) = vb;
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
  const int64_t items = p.batch * p.seq * (p.q_heads + p.k_heads) * per_head;
  if (items == 0) return MB_OK;
  int64_t grid = (items + 255) / 256;
  if (grid > 148 * 16) grid = 148 * 16;
  rotary_kernel<T, V><<<(unsigned)grid, 256, 0, stream>>>(p);
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
