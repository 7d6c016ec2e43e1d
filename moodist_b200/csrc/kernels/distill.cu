// Distillation loss from a teacher's top entries, forward and backward.
//
//   p = softmax(top / tau) over the row's valid entries, q = softmax(z / tau) over the vocabulary
//   row   = (1 - hard) tau^2 sum_k p_k (log p_k - log q_{id_k}) + hard (logsumexp(z) - z_target)
//   dz_j  = (1 - hard) tau (q_j - sum_{k: id_k = j} p_k) + hard (softmax(z)_j - [j = target])
//
// Bound by the bytes of the logits, read once, and of the gradient, written once. The gradient's scale is known in the forward
// pass up to the incoming scalar (which is 1 unless the loss is scaled afterwards), so the forward pass writes it: a CTA walks a
// row twice, first from memory for the maximum and the sum of exponentials, then for the gradient from L2, where the rows in
// work (148 of 256 KB at 128256 words, one CTA of 1024 threads per SM) stay. 4096 x 128256 bf16: 440 us, 4.8 TB/s, held back by
// the exponentials' unit (half of the time busy) and the instructions around it (56 % of the issue slots; every fourth
// exponential as a polynomial on the multiply-add units took 530 us). Two CTAs per SM with a row each read 1.4 times the logits
// from memory, and two that share rows as a cluster pay for their barriers (520 and 474 us when one CTA took 458). Where there
// are fewer rows than SMs, clusters do share them.
// fp16 is the exception: its gradients would underflow before a loss scale reaches them, so there the backward pass reads the
// logits again.
// Sums and row statistics are fp32; sums have a fixed order, so the same inputs give the same bits.
#include "kernels_api.h"
#include "ptx.cuh"
#include "vec_io.cuh"

#define MB_STREAM(s) reinterpret_cast<cudaStream_t>(s)

namespace {

using namespace mb;

inline int check_launch() { return cudaPeekAtLastError() == cudaSuccess ? MB_OK : MB_ERR_LAUNCH; }

constexpr int kSms = 148;
constexpr int kTopThreads = 128;
constexpr int kTopCtas = kSms * 8;
static_assert(kTopCtas + 1 <= MB_DISTILL_COUNTS, "one count per CTA and a ticket");
constexpr int kStaged = 1024;  // teacher entries of a row that are compared in shared memory

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

// One warp per row: the teacher's probabilities over the valid entries, those of a word named several times added up at its first
// place and 0 elsewhere (so that each word of the row is dealt with once), sum p log p, and live: 0 for a row that does not count,
// 1, or 2 if an entry with weight names the target. Per CTA how many rows count. Readies the ticket of the row kernel.
__global__ void __launch_bounds__(kTopThreads) distill_teacher_kernel(const __grid_constant__ mb_distill_t d) {
  constexpr int kWarps = kTopThreads / 32;
  extern __shared__ int4 entries[];  // per warp: the ids (-1: no entry), then exp((t - max) / tau)
  __shared__ int counts[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool staged = d.K <= kStaged;
  const int quads = (d.K + 3) / 4;
  const int4* id_quads = entries + warp * 2 * quads;
  int* ids = reinterpret_cast<int*>(entries + warp * 2 * quads);
  float* ws = reinterpret_cast<float*>(ids + 4 * quads);
  const float inv_tau = 1.f / d.tau;
  int count = 0;
  for (int64_t r = blockIdx.x * (int64_t)kWarps + warp; r < d.rows; r += (int64_t)gridDim.x * kWarps) {
    const int64_t base = r * d.K;
    int64_t target = -1;
    bool counts_too = true;
    if (d.targets) {
      target = d.targets[r];
      counts_too = target != d.ignore_index && target >= 0 && target < d.V;
    }
    float m = -INFINITY, t;
    bool any = false;
    for (int k = lane; k < d.K; k += 32) {
      if (entry(d, base + k, &t)) {
        any = true;
        m = fmaxf(m, t);
      }
    }
    m = warp_reduce_max(m);
    const bool live = counts_too && __any_sync(0xffffffffu, any);
    float s = 0.f, e = 0.f;
    bool hit = false;
    if (live) {
      __syncwarp();
      for (int k = lane; k < d.K; k += 32) {
        float w = 0.f;
        const bool there = entry(d, base + k, &t);
        if (there) {
          t = (t - m) * inv_tau;
          w = expf(t);
          s += w;
          if (!(w <= 0.f)) e += w * t;  // weight 0: t may have overflowed to -inf; NaN goes on
        }
        if (staged) {
          ids[k] = there ? (int)id_at(d, base + k) : -1;
          ws[k] = w;
        }
      }
      if (staged && lane < (4 - d.K % 4) % 4) ids[d.K + lane] = -1;
      s = warp_reduce_sum(s);
      e = warp_reduce_sum(e);
      __syncwarp();
    }
    const float inv = 1.f / s;
    for (int k = lane; k < d.K; k += 32) {
      float p = 0.f;
      if (live && entry(d, base + k, &t)) {
        const int id = (int)id_at(d, base + k);
        bool first = true;
        p = expf((t - m) * inv_tau);
        auto same = [&](int i, float w) {
          if (i < k) first = false;
          if (i > k) p += w;
        };
        if (staged) {
          for (int i = 0; i < d.K; i += 4) {
            const int4 o = id_quads[i / 4];
            if (o.x == id) same(i, ws[i]);
            if (o.y == id) same(i + 1, ws[i + 1]);
            if (o.z == id) same(i + 2, ws[i + 2]);
            if (o.w == id) same(i + 3, ws[i + 3]);
          }
        } else {
          float w;
          for (int i = 0; i < d.K; ++i)
            if (entry(d, base + i, &w) && id_at(d, base + i) == id) same(i, expf((w - m) * inv_tau));
        }
        p = first ? p * inv : 0.f;
        hit |= p != 0.f && id == target;
      }
      d.p[base + k] = p;
    }
    hit = __any_sync(0xffffffffu, hit);
    count += live;
    if (lane == 0) {
      d.live[r] = live ? (hit ? 2 : 1) : 0;
      d.entropy[r] = live ? e * inv - logf(s) : 0.f;
    }
  }
  if (lane == 0) counts[warp] = count;
  __syncthreads();
  grid_release();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) count += counts[w];
    d.counts[blockIdx.x] = count;
    if (blockIdx.x == 0) d.counts[kTopCtas] = 0;
  }
}

inline __host__ __device__ int top_ctas(int64_t rows) {
  const int64_t n = (rows + kTopThreads / 32 - 1) / (kTopThreads / 32);
  return (int)(n < kTopCtas ? n : kTopCtas);
}

// scale, or scale over the number of rows that count; all threads of the CTA get it
template <int kThreads>
__device__ float row_factor(const mb_distill_t& d, int* shared) {
  if (!d.mean) return d.scale;
  if (threadIdx.x == 0) *shared = 0;
  __syncthreads();
  int n = 0;
  for (int i = threadIdx.x; i < top_ctas(d.rows); i += kThreads) n += d.counts[i];
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) atomicAdd(shared, n);
  __syncthreads();
  return d.scale / (float)(*shared > 0 ? *shared : 1);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row as single elements up to the first 16-byte boundary, vectors, and single elements behind the last.
template <typename T>
struct Row {
  static constexpr int kV = 16 / sizeof(T);
  int head, vecs, edge;  // edge: single elements at both ends together
  __device__ __forceinline__ Row(const T* p, int V) {
    head = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
    head = min(head, V);
    vecs = (V - head) / kV;
    edge = V - vecs * kV;
  }
  __device__ __forceinline__ int edge_column(int e) const { return e < head ? e : vecs * kV + e; }
};

// Running maximum and sums of exp((z - max) / tau) and, with kTwo, exp(z - max) over the values a thread has seen; the sums as
// pairs, which are added up at the end
constexpr float kLog2e = 1.4426950409f;
template <bool kTwo>
struct Running {
  float m = -INFINITY;
  F2 st = f2(0.f), s1 = f2(0.f);
  float c;  // log2(e) / tau
  __device__ __forceinline__ explicit Running(float inv_tau) : c(inv_tau * kLog2e) {}
  __device__ __forceinline__ void raise(float to) {
    if (to > m) {
      st = mul2(st, f2(exp2_fast((m - to) * c)));
      if (kTwo) s1 = mul2(s1, f2(exp2_fast((m - to) * kLog2e)));
      m = to;
    }
  }
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }  // -inf - -inf would be NaN
  template <int n>
  __device__ __forceinline__ void add(const float* f) {
    const F2 minus = f2(-base()), cc = f2(c);
#pragma unroll
    for (int i = 0; i < n; i += 2) {
      const F2 x = add2(f2(f[i], f[i + 1]), minus);
      const float2 y = split(mul2(x, cc));
      st = add2(st, f2(exp2_fast(y.x), exp2_fast(y.y)));
      if (kTwo) {
        const float2 y1 = split(mul2(x, f2(kLog2e)));
        s1 = add2(s1, f2(exp2_fast(y1.x), exp2_fast(y1.y)));
      }
    }
  }
  __device__ __forceinline__ void add_one(float z) {
    raise(z);
    st = add2(st, f2(exp2_fast((z - base()) * c), 0.f));
    if (kTwo) s1 = add2(s1, f2(exp2_fast((z - base()) * kLog2e), 0.f));
  }
};

// the largest value of n vectors, NaN left out
template <typename T, int N, int n>
__device__ __forceinline__ float largest(const Pack<T, N> (&p)[n]) {
  if constexpr (sizeof(T) == 2) {
    using P = typename PairOf<T>::type;
    P top = *reinterpret_cast<const P*>(&p[0].w[0]);
#pragma unroll
    for (int i = 1; i < n * N / 2; ++i) top = __hmax2(top, *reinterpret_cast<const P*>(&p[i / (N / 2)].w[i % (N / 2)]));
    const float2 t = pair_to_f32<T>(*reinterpret_cast<const uint32_t*>(&top));
    return fmaxf(t.x, t.y);
  } else {
    float top = __uint_as_float(p[0].w[0]);
#pragma unroll
    for (int i = 1; i < n * N; ++i) top = fmaxf(top, __uint_as_float(p[i / N].w[i % N]));
    return top;
  }
}

// d loss / d z from a value of z: exp((z - m) / tau) * iq + exp(z - m) * i1
template <bool kTwo>
struct Slope {
  float m, c, iq, i1;
  template <int n>
  __device__ __forceinline__ void all(float* f) const {
    const F2 minus = f2(-m), cc = f2(c), q = f2(iq), one = f2(kLog2e), q1 = f2(i1);
#pragma unroll
    for (int k = 0; k < n; k += 2) {
      const F2 x = add2(f2(f[k], f[k + 1]), minus);
      const float2 y = split(mul2(x, cc));
      F2 o = mul2(f2(exp2_fast(y.x), exp2_fast(y.y)), q);
      if (kTwo) {
        const float2 y1 = split(mul2(x, one));
        o = fma2(f2(exp2_fast(y1.x), exp2_fast(y1.y)), q1, o);
      }
      const float2 r = split(o);
      f[k] = r.x;
      f[k + 1] = r.y;
    }
  }
  __device__ __forceinline__ float operator()(float z) const {
    float o = exp2_fast((z - m) * c) * iq;
    if (kTwo) o += exp2_fast((z - m) * kLog2e) * i1;
    return o;
  }
};

// A CTA's part of every row: columns [from, from + count)
struct Part {
  int rank, parts, from, count;
  __device__ __forceinline__ Part(int n, int V) {
    parts = n;
    rank = blockIdx.x % n;
    const int each = ((V + n - 1) / n + 63) / 64 * 64;
    from = min(rank * each, V);
    count = min(each, V - from);
  }
  __device__ __forceinline__ int64_t first_row() const { return blockIdx.x / parts; }
  __device__ __forceinline__ int64_t step() const { return gridDim.x / parts; }
};

// The vectors that a thread is going to read, in order: those of its rows, each row once or, with the gradient, twice. They travel
// kDepth steps of four vectors ahead into the thread's own slots of shared memory, over the ends of walks and rows, so that
// neither the latency of memory nor the barriers between the walks leave the memory idle (four vectors ahead in registers,
// begun anew for each walk: 643 us at 4096 x 128256). Four vectors a step, because the exponentials take 16 of the clocks that a
// warp has per element and row, and everything else has to be issued beside them.
template <typename T, int kThreads, int kDepth>
struct Stream {
  static constexpr int kV = Row<T>::kV, kU = 4;
  static constexpr int kApart = kThreads * kV;  // elements from one of a thread's vectors to the next
  static constexpr int kSlot = kThreads * 16 * kU, kBytes = kDepth * kSlot;
  uint8_t* slots;
  const mb_distill_t* d;
  const Part* part;
  const T* at;     // the next vector to ask for
  const T* end;    // behind the row's last vector
  const T* first;  // this thread's first vector of the row
  int64_t row;     // its row
  int walks;       // walks over the row after this one
  int per_row;     // walks per row, less one
  int slot;        // offset of the slot that comes next
  int live;        // whether `row` counts, known before it is needed

  // the first live row from `row` on that has vectors for this thread
  __device__ __forceinline__ void seek() {
    for (; row < d->rows; row += part->step()) {
      const int now = live;
      if (row + part->step() < d->rows) live = d->live[row + part->step()];
      if (!now) continue;
      const T* z = reinterpret_cast<const T*>(d->logits) + row * d->stride + part->from;
      const Row<T> shape(z, part->count);
      if ((int)threadIdx.x >= shape.vecs) continue;
      end = z + shape.head + shape.vecs * (int64_t)kV;
      first = at = z + shape.head + threadIdx.x * (int64_t)kV;
      walks = per_row;
      return;
    }
    at = end = nullptr;
  }
  __device__ __forceinline__ void begin(uint8_t* smem, const mb_distill_t& args, const Part& mine, bool twice) {
    slots = smem + threadIdx.x * 16;
    d = &args;
    part = &mine;
    row = mine.first_row();
    per_row = twice;
    slot = 0;
    live = row < args.rows ? args.live[row] : 0;
    seek();
#pragma unroll 1
    for (int i = 0; i < kDepth; ++i) ask(i * kSlot);
  }
  __device__ __forceinline__ void ask(int into) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(slots + into);
    if (at + (kU - 1) * kApart < end) {
#pragma unroll
      for (int u = 0; u < kU; ++u)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + u * kThreads * 16), "l"(at + u * kApart) : "memory");
      at += kU * kApart;
    } else if (at < end) {
#pragma unroll 1
      for (int u = 0; u < kU && at < end; ++u, at += kApart)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + u * kThreads * 16), "l"(at) : "memory");
    }
    if (at >= end && at) {
      if (walks > 0) {
        --walks;
        at = first;
      } else {
        row += part->step();
        seek();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // whole(vectors, index of the first) for each full step of one walk over this thread's vectors, single(vector, index) for the
  // vectors of an unfinished last step
  template <typename F, typename G>
  __device__ __forceinline__ void each(int vecs, F whole, G single) {
#pragma unroll 1
    for (int i = threadIdx.x; i < vecs; i += kU * kThreads) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      const Pack<T, kV>* from = reinterpret_cast<const Pack<T, kV>*>(slots + slot);
      if (i + (kU - 1) * kThreads < vecs) {
        Pack<T, kV> v[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) v[u] = from[u * kThreads];
        whole(v, i);
      } else {
#pragma unroll 1
        for (int j = i; j < vecs; j += kThreads) single(from[j - i], j);
      }
      // the vectors' values have been used, so their slot is free
      ask(slot);
      slot += kSlot;
      if (slot == kBytes) slot = 0;
    }
  }
};

// the gradient of one row but for the named places
template <typename T, int kThreads, bool kTwo, typename S>
__device__ __forceinline__ void row_gradient(const Row<T>& row, const T* z, T* g, S& stream, const Slope<kTwo>& slope) {
  constexpr int kV = Row<T>::kV;
  const bool same = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
  for (int e = threadIdx.x; e < row.edge; e += kThreads) {
    const int c = row.edge_column(e);
    g[c] = from_f32<T>(slope(to_f32(z[c])));
  }
  T* out = g + row.head;
  auto put = [&](const Pack<T, kV>& v, int i) {
    float f[kV];
    unpack<T, kV>(v, f);
    slope.template all<kV>(f);
    T* to = out + i * (int64_t)kV;
    if (same) {
      const Pack<T, kV> o = pack<T, kV>(f);
      __stcs(reinterpret_cast<uint4*>(to), *reinterpret_cast<const uint4*>(&o));
    } else {
#pragma unroll
      for (int k = 0; k < kV; ++k) to[k] = from_f32<T>(f[k]);
    }
  };
  stream.each(
      row.vecs,
      [&](const Pack<T, kV>(&v)[S::kU], int i) {
#pragma unroll
        for (int u = 0; u < S::kU; ++u) put(v[u], i + u * kThreads);
      },
      put);
}
template <typename T, int kThreads>
__device__ __forceinline__ void row_zeros(T* g, int V) {
  constexpr int kV = Row<T>::kV;
  const Row<T> row(g, V);
  for (int e = threadIdx.x; e < row.edge; e += kThreads) g[row.edge_column(e)] = from_f32<T>(0.f);
  for (int i = threadIdx.x; i < row.vecs; i += kThreads) *reinterpret_cast<uint4*>(g + row.head + i * (int64_t)kV) = make_uint4(0, 0, 0, 0);
}

// The words that the teacher or the target names. Thread k deals with the teacher's entry k (and kThreads more at a time), whose
// probability the teacher kernel has merged over the row: it subtracts it from the gradient that the walk has written there.
// The target goes with its entry, or alone when the teacher does not name it. Only places of this CTA's part are written, after
// a barrier behind the walk.
template <typename T, int kThreads, bool kTwo>
__device__ __forceinline__ void named_place(const mb_distill_t& d, int64_t r, T* g, const Part& part, const Slope<kTwo>& slope, float a_soft,
                                            float a_hard, int64_t t, int id, float p, float z) {
  if (p != 0.f && id >= part.from && id < part.from + part.count) g[id] = from_f32<T>(slope(z) - p * a_soft - (id == t ? a_hard : 0.f));
}
template <typename T, int kThreads, bool kTwo>
__device__ __forceinline__ void other_places(const mb_distill_t& d, int64_t r, const T* z, T* g, const Part& part, const Slope<kTwo>& slope,
                                             float a_soft, float a_hard, int64_t t, int live) {
  for (int k = threadIdx.x + kThreads; k < d.K; k += kThreads) {
    const float p = d.p[r * d.K + k];
    if (p != 0.f) {
      const int id = (int)id_at(d, r * d.K + k);
      named_place<T, kThreads, kTwo>(d, r, g, part, slope, a_soft, a_hard, t, id, p, to_f32(z[id]));
    }
  }
  if (live == 1 && threadIdx.x == kThreads - 1 && t >= part.from && t < part.from + part.count)
    g[t] = from_f32<T>(slope(to_f32(z[t])) - a_hard);
}

// steps ahead: 192 KB per CTA of 1024 threads, one per SM; 16 KB per CTA of 128, up to eight
constexpr int depth_for(int threads) { return threads > 128 ? 3 : 2; }

__device__ __forceinline__ float ld_cluster(const float* p, int cta) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(cta));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
// every thread of every CTA of the cluster
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// What is left of a row when its walk is over: its named places and its loss wait for the next barrier, which is that of the
// row after. In shared memory, with the threads' teacher entries: in registers it would be spilled inside the walks.
template <bool kTwo>
struct Unfinished {
  int64_t r;
  Slope<kTwo> slope;
  int live;
  float st, s1;
};

// kTwo: the two terms need different exponentials (a hard term, and tau is not 1). The grid is clusters of `parts` CTAs, one row
// at a time per cluster, one barrier per row.
template <typename T, int kThreads, bool kTwo>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
    distill_row_kernel(const __grid_constant__ mb_distill_t d, int parts, T* __restrict__ grad, int64_t grad_stride) {
  constexpr int kV = Row<T>::kV, kWarps = kThreads / 32;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[2][4][kWarps];  // by row parity: a peer may still read the row before's
  __shared__ Unfinished<kTwo> left[2];  // by row parity too
  __shared__ float kept_p[kThreads], kept_z[kThreads];
  __shared__ int kept_id[kThreads];
  __shared__ int shared_count;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float inv_tau = 1.f / d.tau;
  grid_wait();
  const float factor = row_factor<kThreads>(d, &shared_count);
  const float a_soft = (1.f - d.hard) * d.tau * factor, a_hard = d.hard * factor;
  const Part part(parts, d.V);
  using In = Stream<T, kThreads, depth_for(kThreads)>;
  In stream;
  stream.begin(ring, d, part, grad != nullptr);
  int parity = 0;
  bool any = false;
  auto finish = [&](int from) {
    const Unfinished<kTwo> u = left[from];
    const T* z = reinterpret_cast<const T*>(d.logits) + u.r * d.stride;
    const int64_t t = d.hard > 0.f ? d.targets[u.r] : -1;
    if (grad) {
      T* g = grad + u.r * grad_stride;
      named_place<T, kThreads, kTwo>(d, u.r, g, part, u.slope, a_soft, a_hard, t, kept_id[threadIdx.x], kept_p[threadIdx.x], kept_z[threadIdx.x]);
      if (d.K > kThreads || (t >= 0 && u.live == 1)) other_places<T, kThreads, kTwo>(d, u.r, z, g, part, u.slope, a_soft, a_hard, t, u.live);
    }
    if (warp == 0 && part.rank == 0) {
      const float ce = warp_reduce_sum(lane < kWarps ? red[from][3][lane % kWarps] : 0.f);
      if (lane == 0) {
        const float m = u.slope.m;
        d.stats[u.r * 3] = m;
        d.stats[u.r * 3 + 1] = 1.f / u.st;
        d.stats[u.r * 3 + 2] = 1.f / u.s1;
        // the probabilities sum to 1, so log(st) stands outside the sum
        float l = d.hard < 1.f ? (1.f - d.hard) * d.tau * d.tau * (d.entropy[u.r] - ce + logf(u.st)) : 0.f;
        if (d.hard > 0.f) l += d.hard * (logf(u.s1) + m - to_f32(z[t]));
        d.row_loss[u.r] = l;
      }
    }
  };
  // this thread's entry of the next row and whether that row counts, asked for a row ahead
  float next_p = 0.f;
  int next_id = 0, next_live = 0;
  auto peek = [&](int64_t r) {
    if (r >= d.rows) return;
    next_live = d.live[r];
    if (threadIdx.x < d.K) {
      next_p = d.p[r * d.K + threadIdx.x];
      next_id = (int)id_at(d, r * d.K + threadIdx.x);
    }
  };
  peek(part.first_row());
  for (int64_t r = part.first_row(); r < d.rows; r += part.step()) {
    const T* z = reinterpret_cast<const T*>(d.logits) + r * d.stride;
    T* g = grad + r * grad_stride;
    const int live = next_live, my_id = next_id;
    const float my_p = next_p;
    float my_z = 0.f;
    if (live && my_p != 0.f) my_z = to_f32(z[my_id]);
    if (!live) {
      peek(r + part.step());
      if (threadIdx.x == 0 && part.rank == 0) d.row_loss[r] = 0.f;
      if (grad) row_zeros<T, kThreads>(g + part.from, part.count);
      continue;
    }
    const Row<T> row(z + part.from, part.count);
    Running<kTwo> run(inv_tau);
    stream.each(
        row.vecs,
        [&](const Pack<T, kV>(&v)[In::kU], int) {
          run.raise(largest(v));
#pragma unroll
          for (int i = 0; i < In::kU; ++i) {
            float f[kV];
            unpack<T, kV>(v[i], f);
            run.template add<kV>(f);
          }
        },
        [&](const Pack<T, kV>& v, int) {
          const Pack<T, kV> one[1] = {v};
          run.raise(largest(one));
          float f[kV];
          unpack<T, kV>(v, f);
          run.template add<kV>(f);
        });
    for (int e = threadIdx.x; e < row.edge; e += kThreads) run.add_one(to_f32(z[part.from + row.edge_column(e)]));
    // (max, sums) of the warp, then of the cluster: one barrier
    float m = warp_reduce_max(run.m);
    const float2 own = split(run.st), own1 = split(run.s1);
    float st = warp_reduce_sum((own.x + own.y) * exp2_fast((run.m - m) * run.c));
    float s1 = kTwo ? warp_reduce_sum((own1.x + own1.y) * exp2_fast((run.m - m) * kLog2e)) : 0.f;
    // a warp that saw nothing but -inf has NaN here; it counts with nothing, unless it really saw NaN
    if (m == -INFINITY && warp_reduce_sum(own.x + own.y) == 0.f) st = s1 = 0.f;
    if (lane == 0) {
      red[parity][0][warp] = m;
      red[parity][1][warp] = st;
      red[parity][2][warp] = s1;
    }
    if (parts > 1)
      cluster_barrier();
    else
      __syncthreads();
    {
      float wm = -INFINITY, wt = 0.f, w1 = 0.f;
      m = -INFINITY;
      for (int i = lane; i < parts * kWarps; i += 32) {
        const float om = ld_cluster(&red[parity][0][i % kWarps], i / kWarps), ot = ld_cluster(&red[parity][1][i % kWarps], i / kWarps);
        const float o1 = kTwo ? ld_cluster(&red[parity][2][i % kWarps], i / kWarps) : 0.f;
        const float nm = fmaxf(wm, om);
        // (a sum of 0 goes with -inf: nothing of it counts)
        wt = (wt == 0.f ? 0.f : wt * exp2_fast((wm - nm) * run.c)) + (ot == 0.f ? 0.f : ot * exp2_fast((om - nm) * run.c));
        if (kTwo) w1 = (w1 == 0.f ? 0.f : w1 * exp2_fast((wm - nm) * kLog2e)) + (o1 == 0.f ? 0.f : o1 * exp2_fast((om - nm) * kLog2e));
        wm = nm;
      }
      m = warp_reduce_max(wm);
      st = warp_reduce_sum(wt * exp2_fast((wm - m) * run.c));
      s1 = kTwo ? warp_reduce_sum(w1 * exp2_fast((wm - m) * kLog2e)) : st;
    }
    if (any) finish(parity ^ 1);
    any = true;
    const Slope<kTwo> slope{m, run.c, kTwo ? a_soft / st : (a_soft + a_hard) / st, a_hard / s1};
    kept_id[threadIdx.x] = my_id;
    kept_p[threadIdx.x] = my_p;
    kept_z[threadIdx.x] = my_z;
    if (threadIdx.x == 0) left[parity] = Unfinished<kTwo>{r, slope, live, st, s1};
    if (part.rank == 0) {
      // the teacher's entries against q, but for log(st)
      float ce = my_p != 0.f ? my_p * (my_z - m) * inv_tau : 0.f;
      for (int k = threadIdx.x + kThreads; k < d.K; k += kThreads) {
        const float p = d.p[r * d.K + k];
        if (p != 0.f) ce += p * (to_f32(z[id_at(d, r * d.K + k)]) - m) * inv_tau;
      }
      ce = warp_reduce_sum(ce);
      if (lane == 0) red[parity][3][warp] = ce;
    }
    peek(r + part.step());
    if (grad) row_gradient<T, kThreads, kTwo>(row, z + part.from, g + part.from, stream, slope);
    parity ^= 1;
  }
  __syncthreads();
  if (any) finish(parity ^ 1);
  if (parts > 1) cluster_barrier();  // the peers no longer read this CTA's sums
  // the last CTA to get here adds the row losses up, in a fixed order
  __shared__ bool last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(d.counts + kTopCtas, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  float s = 0.f;
  for (int64_t r = threadIdx.x; r < d.rows; r += kThreads) s += __ldcg(d.row_loss + r);
  s = block_reduce_sum<kThreads>(s, red[0][0]);
  if (threadIdx.x == 0) d.loss[0] = s * factor;
}

// the backward pass on its own: the logits once more
template <typename T, int kThreads, bool kTwo>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
    distill_grad_kernel(const __grid_constant__ mb_distill_t d, int parts, const float* __restrict__ gout, T* __restrict__ grad, int64_t grad_stride) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ int shared_count;
  grid_wait();
  const float factor = row_factor<kThreads>(d, &shared_count) * gout[0];
  const float a_soft = (1.f - d.hard) * d.tau * factor, a_hard = d.hard * factor;
  const Part part(parts, d.V);
  Stream<T, kThreads, depth_for(kThreads)> stream;
  stream.begin(ring, d, part, false);
  for (int64_t r = part.first_row(); r < d.rows; r += part.step()) {
    const T* z = reinterpret_cast<const T*>(d.logits) + r * d.stride;
    T* g = grad + r * grad_stride;
    const int live = d.live[r];
    if (!live) {
      row_zeros<T, kThreads>(g + part.from, part.count);
      continue;
    }
    const Row<T> row(z + part.from, part.count);
    float my_p = 0.f, my_z = 0.f;
    int my_id = 0;
    if (threadIdx.x < d.K) {
      my_p = d.p[r * d.K + threadIdx.x];
      my_id = (int)id_at(d, r * d.K + threadIdx.x);
      if (my_p != 0.f) my_z = to_f32(z[my_id]);
    }
    const int64_t t = d.hard > 0.f ? d.targets[r] : -1;
    const float iq = d.stats[r * 3 + 1];
    const Slope<kTwo> slope{d.stats[r * 3], kLog2e / d.tau, kTwo ? a_soft * iq : (a_soft + a_hard) * iq, a_hard * d.stats[r * 3 + 2]};
    row_gradient<T, kThreads, kTwo>(row, z + part.from, g + part.from, stream, slope);
    __syncthreads();
    named_place<T, kThreads, kTwo>(d, r, g, part, slope, a_soft, a_hard, t, my_id, my_p, my_z);
    if (d.K > kThreads || (t >= 0 && live == 1)) other_places<T, kThreads, kTwo>(d, r, z, g, part, slope, a_soft, a_hard, t, live);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) scale_by_kernel(T* __restrict__ x, int64_t n, const float* __restrict__ s) {
  const float f = s[0];
  if (f == 1.f) return;
  constexpr int kV = 16 / sizeof(T);
  const int64_t vecs = n / kV;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < vecs; i += gridDim.x * 256ll) {
    float v[kV];
    load_vec<T, kV>(x + i * kV, v);
#pragma unroll
    for (int k = 0; k < kV; ++k) v[k] *= f;
    store_vec<T, kV>(x + i * kV, v);
  }
  for (int64_t i = vecs * kV + blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) x[i] = from_f32<T>(to_f32(x[i]) * f);
}

// Rows above 8192 words: a CTA of 1024 threads each, one per SM; a cluster of up to eight where the rows are too few to fill the
// GPU otherwise and the parts stay above 4096 words. Shorter rows: a CTA of 128 threads each, many per SM.
constexpr int kLongRow = 8192, kLongThreads = 1024;
inline int row_parts(int64_t rows, int V) {
  int n = 1;
  while (V > kLongRow && n < 8 && rows * n * 2 <= kSms && V / (n * 2) >= 4096) n *= 2;
  return n;
}
inline unsigned row_ctas(int64_t rows, int V) {
  const int parts = row_parts(rows, V);
  const int64_t most = V > kLongRow ? kSms * (1024 / kLongThreads) / parts : kSms * 8;
  return (unsigned)(rows < most ? rows : most) * parts;
}

template <auto kKernel, int kThreads, bool kCluster, typename... Args>
int launch(const mb_distill_t& d, cudaStream_t s, Args... args) {
  constexpr int smem = depth_for(kThreads) * kThreads * 64;
  static bool done[64];  // per kernel and device
  if (smem > 48 * 1024) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= 64) return MB_ERR_DRIVER;
    if (!done[device] && cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return MB_ERR_LAUNCH;
    done[device] = true;
  }
  const int parts = row_parts(d.rows, d.V);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCluster ? parts : 1;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(row_ctas(d.rows, d.V), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kKernel, d, parts, args...) == cudaSuccess ? MB_OK : MB_ERR_LAUNCH;
}

template <typename T, int kThreads, bool kTwo>
int fwd_with(const mb_distill_t& d, void* grad, int64_t grad_stride, cudaStream_t s) {
  return launch<distill_row_kernel<T, kThreads, kTwo>, kThreads, true>(d, s, (T*)grad, grad_stride);
}
template <typename T, int kThreads, bool kTwo>
int bwd_with(const mb_distill_t& d, const float* gout, void* grad, int64_t grad_stride, cudaStream_t s) {
  return launch<distill_grad_kernel<T, kThreads, kTwo>, kThreads, false>(d, s, gout, (T*)grad, grad_stride);
}
template <typename T>
int fwd(const mb_distill_t& d, void* grad, int64_t grad_stride, cudaStream_t s) {
  const bool two = d.hard > 0.f && d.tau != 1.f;
  if (d.V > kLongRow) return two ? fwd_with<T, kLongThreads, true>(d, grad, grad_stride, s) : fwd_with<T, kLongThreads, false>(d, grad, grad_stride, s);
  return two ? fwd_with<T, 128, true>(d, grad, grad_stride, s) : fwd_with<T, 128, false>(d, grad, grad_stride, s);
}
template <typename T>
int bwd(const mb_distill_t& d, const float* gout, void* grad, int64_t grad_stride, cudaStream_t s) {
  const bool two = d.hard > 0.f && d.tau != 1.f;
  if (d.V > kLongRow) return two ? bwd_with<T, kLongThreads, true>(d, gout, grad, grad_stride, s) : bwd_with<T, kLongThreads, false>(d, gout, grad, grad_stride, s);
  return two ? bwd_with<T, 128, true>(d, gout, grad, grad_stride, s) : bwd_with<T, 128, false>(d, gout, grad, grad_stride, s);
}

bool sane(const mb_distill_t& d) {
  return d.rows > 0 && d.V > 0 && d.K > 0 && d.tau > 0.f && d.hard >= 0.f && d.hard <= 1.f && (d.hard == 0.f || d.targets) &&
         (d.top_dtype == MB_F32 || d.top_dtype == MB_BF16 || d.top_dtype == MB_F16);
}

}  // namespace

extern "C" int mb_distill_fwd(const mb_distill_t* d, void* grad, int64_t grad_stride, void* stream) {
  if (!sane(*d)) return MB_ERR_ARG;
  cudaStream_t s = MB_STREAM(stream);
  const int staged = d->K <= kStaged ? kTopThreads / 32 * ((d->K + 3) / 4) * 32 : 0;  // 32 KB at most
  distill_teacher_kernel<<<top_ctas(d->rows), kTopThreads, staged, s>>>(*d);
  if (check_launch()) return MB_ERR_LAUNCH;
  switch (d->dtype) {
    case MB_BF16: return fwd<__nv_bfloat16>(*d, grad, grad_stride, s);
    case MB_F16: return fwd<__half>(*d, grad, grad_stride, s);
    case MB_F32: return fwd<float>(*d, grad, grad_stride, s);
    default: return MB_ERR_ARG;
  }
}

extern "C" int mb_distill_bwd(const mb_distill_t* d, const float* gout, void* grad, int64_t grad_stride, void* stream) {
  if (!sane(*d)) return MB_ERR_ARG;
  switch (d->dtype) {
    case MB_BF16: return bwd<__nv_bfloat16>(*d, gout, grad, grad_stride, MB_STREAM(stream));
    case MB_F16: return bwd<__half>(*d, gout, grad, grad_stride, MB_STREAM(stream));
    case MB_F32: return bwd<float>(*d, gout, grad, grad_stride, MB_STREAM(stream));
    default: return MB_ERR_ARG;
  }
}

extern "C" int mb_scale_by(void* x, int64_t n, int dtype, const float* s, void* stream) {
  if (n <= 0) return MB_OK;
  if (!is_aligned(x, 16)) return MB_ERR_ALIGN;
  int64_t grid = (n / 8 + 255) / 256;
  grid = grid < 1 ? 1 : grid > kSms * 8 ? kSms * 8 : grid;
  switch (dtype) {
    case MB_BF16: scale_by_kernel<__nv_bfloat16><<<(unsigned)grid, 256, 0, MB_STREAM(stream)>>>((__nv_bfloat16*)x, n, s); break;
    case MB_F32: scale_by_kernel<float><<<(unsigned)grid, 256, 0, MB_STREAM(stream)>>>((float*)x, n, s); break;
    default: return MB_ERR_ARG;
  }
  return check_launch();
}
