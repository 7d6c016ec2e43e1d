// Gated projection on tcgen05: h = act(x Wg^T) * (x Wu^T), both products, the activation and their product in one kernel.
//
//   x [T, K], W [2F, K] (gate rows [0, F), up rows [F, 2F)), h [T, F], all bf16, accumulation fp32
//
// A cluster of two CTAs computes 256 rows x 128 columns of h as one 256 x 256 tile of tcgen05.mma.cta_group::2: columns
// [0, 128) of the accumulator are gate columns, [128, 256) the up columns of the same h. The even CTA loads the gate rows of W
// and the odd one the up rows, so each still brings 128 rows of x and 128 rows of W per 64-wide step, as in the plain
// product, and a thread of the epilogue finds both factors of an h in its own TMEM lane. The activation runs on the fp32
// accumulators: h is rounded once. For the backward pass the two projections are kept in 16 bits too (32 would double the
// largest activation of a block): fp16 with one power of two per 8 columns, an eighth of bf16's rounding at 6 % more
// bytes and the range of fp32. In bf16 they alone would add as much error to the gradients as all other roundings together.
//
// Bound by the tensor cores: 4 T F K flops. Against product + activation kernels it saves the write and read of [T, 2F]
// (inference) or the read (training). 8192 rows, 4096 -> 14336, with the projections kept: 1.28 ms (1.50 PFLOP/s) in a burst,
// 1.44 ms under the power cap, which is what the plain product of that size takes.
#pragma once

#include "gemm_pair_tcgen05.cuh"
#include "vec_io.cuh"

namespace mb {
namespace gated {

using namespace gemm;

enum Act : int { kSilu = 0, kGelu = 1, kGeluTanh = 2 };

enum GatedStatus : uint32_t {
  kTimeoutGatedProducer = 0x121,
  kTimeoutGatedMma = 0x122,
  kTimeoutGatedEpilogue = 0x123,
};

constexpr int kHCols = BN / 2;  // h columns of a tile

struct GatedParams {
  int T, F, K;
  __nv_bfloat16* h;
  int64_t ldh;
  // the kept projections, or null: fp16 mantissas [T, 2F] and scales [T, 2 scale_pitch], a byte per 8 columns (gate's, then up's)
  __half* gu;
  uint8_t* scales;
  int scale_pitch;
  int tiles_m, tiles_n, group_m;
  int num_ctas;
  uint32_t* status;
  uint64_t wait_ns;
};

// act(g); the logistic form of the tanh approximation and erfc keep the relative accuracy of the left tail
template <int kAct>
__device__ __forceinline__ float activate(float g) {
  if (kAct == kGelu) return g * 0.5f * erfcf(-g * 0.70710678f);
  const float y = kAct == kSilu ? g : 1.5957691216f * (g + 0.044715f * g * g * g);
  return __fdividef(g, 1.f + __expf(-y));
}
// act(g) and its derivative
template <int kAct>
__device__ __forceinline__ float2 activate_slope(float g) {
  if (kAct == kSilu) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    return make_float2(g * s, s * (1.f + g * (1.f - s)));
  }
  if (kAct == kGelu) {
    const float c = 0.5f * erfcf(-g * 0.70710678f);
    return make_float2(g * c, c + g * __expf(-0.5f * g * g) * 0.39894228f);
  }
  const float y2 = 1.5957691216f * (g + 0.044715f * g * g * g);
  const float s = __fdividef(1.f, 1.f + __expf(-y2));
  return make_float2(g * s, s + g * s * (1.f - s) * 1.5957691216f * (1.f + 0.134145f * g * g));
}

__device__ __forceinline__ void gated_report(const GatedParams& p, uint32_t code) {
  volatile uint32_t* s = p.status;
  if (s && *s == 0) *s = code;
}

// tile index -> (m, n), grouped so that CTAs running together share panels of x and W in L2
__device__ __forceinline__ void gated_tile(const GatedParams& p, int t, int& tm, int& tn) {
  const int per_group = p.group_m * p.tiles_n;
  const int g = t / per_group, first_m = g * p.group_m;
  const int gsz = min(p.group_m, p.tiles_m - first_m);
  const int r = t - g * per_group;
  tm = first_m + r % gsz;
  tn = r / gsz;
}

// 8 values v as fp16 mantissas of v / 2^(e - 127); returns e, which brings the largest finite one to 2^14 .. 2^15
__device__ __forceinline__ uint32_t keep8(const float* v, uint4* to) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
    top = max(top, a < 0x7f800000u ? a : 0u);
  }
  const int e = max((int)(top >> 23) - 14, 1);
  const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i] * inv, v[2 * i + 1] * inv);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *to = make_uint4(w[0], w[1], w[2], w[3]);
  return (uint32_t)e;
}
__device__ __forceinline__ float kept_scale(uint32_t e) { return __uint_as_float(e << 23); }

// The epilogue's patch of shared memory per warp: 32 rows of three 64-byte pieces (32 columns of h, gate and up), padded so
// that 16-byte accesses of eight rows meet no bank twice.
constexpr int kPatchRow = 208;
constexpr int kPatchBytes = 32 * kPatchRow;
constexpr int kGatedPairSmem = kPairStages * kPairStageBytes + 1024 + 256 + 4 * kPatchBytes;

// 16 values of a lane's row -> 32 bytes of its line
__device__ __forceinline__ void patch_put(uint8_t* to, const float* v) {
#pragma unroll
  for (int g = 0; g < 2; ++g)
    reinterpret_cast<uint4*>(to)[g] =
        make_uint4(pack_bf16x2(v[g * 8], v[g * 8 + 1]), pack_bf16x2(v[g * 8 + 2], v[g * 8 + 3]),
                   pack_bf16x2(v[g * 8 + 4], v[g * 8 + 5]), pack_bf16x2(v[g * 8 + 6], v[g * 8 + 7]));
}
// one piece of the patch, 32 rows x 32 columns -> global memory, whole 64-byte runs
template <typename T>
__device__ __forceinline__ void patch_store(const uint8_t* piece, int lane, T* base, int64_t ld, int rows, int cols) {
  const int col = (lane & 3) * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = i * 8 + (lane >> 2);
    const uint4 v = *reinterpret_cast<const uint4*>(piece + rr * kPatchRow + (lane & 3) * 16);
    if (rr < rows && col < cols) *reinterpret_cast<uint4*>(base + (int64_t)rr * ld + col) = v;
  }
}

// The warp's 32 rows x `width` columns of h from the accumulator at `taddr` (gate columns, up columns `up` further on):
// sixteen columns at a time in a rolled loop, because code that is run once per tile from a cold instruction cache costs
// more than the arithmetic (the fully unrolled form took 60 us for one tile).
template <int kAct, bool kSave>
__device__ __forceinline__ void gated_epilogue(const GatedParams& p, uint32_t taddr, int up, int width, uint8_t* patch, int lane,
                                               int row0, int col0) {
  const int rows = p.T - row0;
#pragma unroll 1
  for (int c = 0; c < width; c += 32) {
    const int cols = min(p.F - (col0 + c), width - c);
    uint8_t* line = patch + lane * kPatchRow;
    uint32_t eg = 0, eu = 0;
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      uint32_t rg[16], ru[16];
      tmem_ld_32x16(taddr + c + half * 16, rg);
      tmem_ld_32x16(taddr + up + c + half * 16, ru);
      tmem_ld_wait();
      float g[16], u[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        g[i] = __uint_as_float(rg[i]);
        u[i] = __uint_as_float(ru[i]);
      }
      if (kSave) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int shift = half * 16 + i * 8;
          eg |= keep8(g + i * 8, reinterpret_cast<uint4*>(line + 64 + half * 32) + i) << shift;
          eu |= keep8(u + i * 8, reinterpret_cast<uint4*>(line + 128 + half * 32) + i) << shift;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) g[i] = activate<kAct>(g[i]) * u[i];
      patch_put(line + half * 32, g);
    }
    __syncwarp();
    patch_store(patch, lane, p.h + (int64_t)row0 * p.ldh + col0 + c, p.ldh, rows, cols);
    if (kSave) {
      __half* to = p.gu + (int64_t)row0 * 2 * p.F + col0 + c;
      patch_store(patch + 64, lane, to, 2 * (int64_t)p.F, rows, cols);
      patch_store(patch + 128, lane, to + p.F, 2 * (int64_t)p.F, rows, cols);
      if (lane < rows && cols > 0) {
        // (col0 + c is a multiple of 32 and the pitch one of 16: whole words, the last of which may reach into the padding)
        uint8_t* e = p.scales + (int64_t)(row0 + lane) * 2 * p.scale_pitch + (col0 + c) / 8;
        *reinterpret_cast<uint32_t*>(e) = eg;
        *reinterpret_cast<uint32_t*>(e + p.scale_pitch) = eu;
      }
    }
    __syncwarp();
  }
}

template <int kAct, bool kSave>
__device__ __forceinline__ void gated_pair_body(const GatedParams& p, const CUtensorMap* tmap_x, const CUtensorMap* tmap_w,
                                                uint8_t* smem_raw) {
  uint32_t raw = smem_u32(smem_raw);
  uint8_t* tiles = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(tiles + kPairStages * kPairStageBytes);
  uint64_t* full = bars;                        // [kPairStages]  used in the leader
  uint64_t* empty = bars + kPairStages;         // [kPairStages]  one per CTA
  uint64_t* acc_full = bars + 2 * kPairStages;  // [2]            one per CTA
  uint64_t* acc_empty = acc_full + 2;           // [2]            used in the leader
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile uint32_t* abort_flag = tmem_base_slot + 1;
  uint8_t* epi_patch = reinterpret_cast<uint8_t*>(bars) + 256;

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int cta_rank = (int)cluster_ctarank();  // 0 = leader
  const int num_tiles = p.tiles_m * p.tiles_n;
  const int kblocks = (p.K + BK - 1) / BK;
  const int pair = blockIdx.x >> 1, stride = p.num_ctas >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kPairStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 8);  // 4 epilogue warps in each of the two CTAs
    }
    *abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(tmap_x);
    tma_prefetch_desc(tmap_w);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_base_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  body_sync();
  cluster_sync_all();  // the peer's barriers are initialised before anything signals them
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_base_slot;

  if (warp == 0) {
    if (elect_one()) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += stride) {
        int tm, tn;
        gated_tile(p, t, tm, tn);
        const int row_x = tm * kPairBM + cta_rank * BM;
        const int row_w = tn * kHCols + cta_rank * p.F;  // gate rows in the leader, up rows in its peer
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % kPairStages;
          if (!mbar_wait(&empty[s], ((it / kPairStages) & 1) ^ 1, p.wait_ns)) {
            gated_report(p, kTimeoutGatedProducer);
            ok = false;
            break;
          }
          uint8_t* sa = tiles + s * kPairStageBytes;
          if (cta_rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kPairStageBytes);
          const uint32_t bar = map_to_cta(smem_u32(&full[s]), 0);
          tma_load_2d_pair(sa, tmap_x, bar, kb * BK, row_x);
          tma_load_2d_pair(sa + kATileBytes, tmap_w, bar, kb * BK, row_w);
        }
      }
      if (!ok) *abort_flag = 1;
    }
  } else if (warp == 1) {
    if (cta_rank == 0 && elect_one()) {
      constexpr uint32_t idesc = make_idesc_f16(true, false, false, kPairBM, BN);
      uint32_t it = 0, local_tile = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += stride, ++local_tile) {
        const uint32_t acc = local_tile & 1;
        if (!mbar_wait(&acc_empty[acc], ((local_tile >> 1) & 1) ^ 1, p.wait_ns)) {
          gated_report(p, kTimeoutGatedMma);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * kAccCols;
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % kPairStages;
          if (!mbar_wait(&full[s], (it / kPairStages) & 1, p.wait_ns)) {
            gated_report(p, kTimeoutGatedMma);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t sa = smem_u32(tiles + s * kPairStageBytes), sb = sa + kATileBytes;
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            tc_mma_f16_pair(d_tmem, make_smem_desc(sa + k * 32, 0, 1024), make_smem_desc(sb + k * 32, 0, 1024), idesc, (kb | k) != 0);
          tc_commit_pair(&empty[s], 0x3);
        }
        if (ok) tc_commit_pair(&acc_full[acc], 0x3);
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    const int q = warp & 3;  // TMEM lane quarter this warp may read
    uint8_t* patch = epi_patch + (warp - 2) * kPatchBytes;
    uint32_t local_tile = 0;
    bool ok = true;
    for (int t = pair; t < num_tiles; t += stride, ++local_tile) {
      int tm, tn;
      gated_tile(p, t, tm, tn);
      const uint32_t acc = local_tile & 1;
      if (!mbar_wait(&acc_full[acc], (local_tile >> 1) & 1, p.wait_ns)) {
        if (lane == 0) gated_report(p, kTimeoutGatedEpilogue);
        ok = false;
        break;
      }
      tc_fence_after_sync();
      gated_epilogue<kAct, kSave>(p, tmem_base + acc * kAccCols + ((uint32_t)(q * 32) << 16), kHCols, kHCols, patch, lane,
                                  tm * kPairBM + cta_rank * BM + q * 32, tn * kHCols);
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&acc_empty[acc]), 0));
    }
    if (!ok && lane == 0) *abort_flag = 1;
  }

  body_sync();
  if (*abort_flag) {
    // a wait ran out: give copies that may still be in flight time to land before this shared memory is released
    for (int i = 0; i < 64; ++i) __nanosleep(20000);
  }
  tc_fence_before_sync();
  cluster_sync_all();  // the peer no longer reads this CTA's shared memory or signals its barriers
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

// ---- few rows ------------------------------------------------------------------------------------------------------
// Up to 128 rows the weight's bytes are the bound (4 F K of them: 36 us at F = 14336, K = 4096 and the measured copy rate),
// and a 256-row tile leaves most SMs without one. Here the weight is the M operand: a CTA computes `width` columns of h for
// all rows, the width chosen so that one wave of CTAs covers F, from 128 weight rows by n >= T rows of x per product.
//   width <= 64: gate and up rows are the two halves of one M tile, and the `split` CTAs of a cluster may share the K steps;
//                they join their sums through distributed shared memory, in rank order
//   width <= 128: two products per step, gate and up, which share the step's x
// A stage holds exactly the rows that exist (2 width of the weight, n of x), so nearly all of shared memory is weight in
// flight. The tensor core reads 128 rows from each operand's start all the same: those past the width are whatever the stage
// and its successor hold, in rows of the accumulators that nothing looks at; kRowsSlack keeps the last stage's inside the
// allocation.
// One elected thread issues the copies and one the products (see elect_one): a narrow step is over in 400 clocks, which took
// 830 as "lane 0", and with it the prologue and the launch, which overlap with the kernel before, are what is left beside
// the bytes: T = 1, F = 14336, K = 4096 in 39 us (6.0 TB/s of weight), F = 5632 in 20 us, F = 28672, K = 8192 in 138 us.
enum RowsStatus : uint32_t {
  kTimeoutRowsProducer = 0x131,
  kTimeoutRowsMma = 0x132,
  kTimeoutRowsEpilogue = 0x133,
  kTimeoutRowsDrain = 0x134,
};
constexpr int kRowsMaxStages = 32;
constexpr int kRowsSmem = 227 * 1024;
constexpr int kRowsSlack = (BM - 8) * 128;
constexpr int kRowsBars = (2 * kRowsMaxStages + 1) * 8 + 8;

__host__ __device__ inline int rows_stage_bytes(int width, int n) { return (2 * width + n) * 128; }
__host__ __device__ inline int rows_stages(int width, int n) {
  const int fit = (kRowsSmem - 1024 - kRowsSlack - kRowsBars) / rows_stage_bytes(width, n);
  return fit < kRowsMaxStages ? fit : kRowsMaxStages;
}

// four floats of the shared memory of any CTA of this cluster (a shared::cluster address; a local one is one too)
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

template <int kAct, bool kSave>
__device__ __forceinline__ void gated_rows_body(const GatedParams& p, int width, int n, int split, const CUtensorMap* tmap_x,
                                                const CUtensorMap* tmap_w, uint8_t* smem_raw) {
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* tiles = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const int stages = rows_stages(width, n), stage_bytes = rows_stage_bytes(width, n);
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + stages * stage_bytes + kRowsSlack);  // [stages]
  uint64_t* empty = full + kRowsMaxStages;                                                  // [stages]
  uint64_t* acc_full = empty + kRowsMaxStages;
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(acc_full + 1);

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const bool one_tile = 2 * width <= BM;
  const int rank = blockIdx.x % split, tile = blockIdx.x / split, col0 = tile * width;
  const int all_steps = (p.K + BK - 1) / BK;
  const int step0 = (int)((int64_t)all_steps * rank / split), steps = (int)((int64_t)all_steps * (rank + 1) / split) - step0;
  const int columns = one_tile ? n : 2 * n;
  const uint32_t tmem_cols = columns <= 32 ? 32 : columns <= 64 ? 64 : columns <= 128 ? 128 : 256;

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(acc_full, 1);
    mbar_fence_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(tmap_x);
    tma_prefetch_desc(tmap_w);
  }
  if (warp == 1) {
    tmem_alloc(tmem_base_slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  body_sync();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_base_slot;
  grid_wait();
  grid_release();

  // Stage index, phase and operand addresses are carried along: with one thread issuing copies and one issuing products, the
  // instructions between two of them count.
  if (warp == 0) {
    if (elect_one()) {
      bool ok = true;
      int it = 0, s = 0;
      uint32_t phase = 1;
      uint8_t* sw = tiles;
      for (; it < steps; ++it) {
        if (!mbar_wait(&empty[s], phase, p.wait_ns)) {
          gated_report(p, kTimeoutRowsProducer);
          ok = false;
          break;
        }
        const int k0 = (step0 + it) * BK;
        mbar_arrive_expect_tx(&full[s], stage_bytes);
        tma_load_3d(sw, tmap_w, &full[s], k0, col0, 0);  // gate rows, then up rows
        tma_load_2d(sw + 2 * width * 128, tmap_x, &full[s], k0, 0);
        sw += stage_bytes;
        if (++s == stages) {
          s = 0;
          phase ^= 1;
          sw = tiles;
        }
      }
      if (!ok) {
        // let the copies still in flight land before this CTA's shared memory is given up
        for (int i = it > stages ? it - stages : 0; i < it; ++i)
          if (!mbar_wait(&full[i % stages], (i / stages) & 1, p.wait_ns)) gated_report(p, kTimeoutRowsDrain);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = make_idesc_f16(true, false, false, BM, n);
      const uint64_t first = make_smem_desc(smem_u32(tiles), 0, 1024);
      const uint32_t to_up = (width * 128) >> 4, to_x = 2 * to_up;
      bool ok = true;
      int s = 0;
      uint32_t phase = 0;
      uint64_t dg = first;
      for (int it = 0; it < steps; ++it) {
        if (!mbar_wait(&full[s], phase, p.wait_ns)) {
          gated_report(p, kTimeoutRowsMma);
          ok = false;
          break;
        }
        tc_fence_after_sync();
#pragma unroll
        for (int k = 0; k < BK / UMMA_K; ++k) {
          tc_mma_f16(tmem_base, dg + k * 2, dg + to_x + k * 2, idesc, it | k);
          if (!one_tile) tc_mma_f16(tmem_base + n, dg + to_up + k * 2, dg + to_x + k * 2, idesc, it | k);
        }
        tc_commit(&empty[s]);
        dg += stage_bytes >> 4;
        if (++s == stages) {
          s = 0;
          phase ^= 1;
          dg = first;
        }
      }
      if (ok) tc_commit(acc_full);
    }
  } else {
    // Accumulators to shared memory as sums[row of x][gate columns, up columns] in fp32: every product is done, so the stages
    // are free (2 width x T floats are never more than they hold).
    const int q = warp & 3, r = q * 32 + lane;
    float* sums = reinterpret_cast<float*>(tiles);
    if (mbar_wait(acc_full, 0, p.wait_ns)) {
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16);
      const int held = one_tile ? 2 * width : width;
#pragma unroll 1
      for (int c = 0; c < columns && q * 32 < held; c += 16) {
        uint32_t v[16];
        tmem_ld_32x16(taddr + c, v);
        tmem_ld_wait();
        const int row0 = c < n ? c : c - n;
        float* to = sums + row0 * 2 * width + (c < n ? 0 : width) + r;
        if (r < held) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (row0 + i < p.T) to[i * 2 * width] = __uint_as_float(v[i]);
        }
      }
    } else if (lane == 0) {
      gated_report(p, kTimeoutRowsEpilogue);
    }
    tc_fence_before_sync();
  }
  body_sync();
  if (split > 1) cluster_sync_all();  // every CTA of the cluster has its sums in place
  // each CTA of the cluster finishes its share of the (row, 8 columns) pieces
  {
    const int vecs = width / 8, pieces = p.T * vecs;
    const uint32_t here = smem_u32(tiles);
    for (int i = rank * kNumThreads + (int)threadIdx.x; i < pieces; i += split * kNumThreads) {
      const int t = i / vecs, j = (i - t * vecs) * 8, col = col0 + j;
      if (col >= p.F) continue;
      float g[8], u[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = u[k] = 0.f;
      for (int c = 0; c < split; ++c) {
        const uint32_t from = (split > 1 ? map_to_cta(here, c) : here) + (t * 2 * width + j) * 4;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float4 a = ld_cluster_f4(from + k * 16), b = ld_cluster_f4(from + width * 4 + k * 16);
          g[4 * k] += a.x, g[4 * k + 1] += a.y, g[4 * k + 2] += a.z, g[4 * k + 3] += a.w;
          u[4 * k] += b.x, u[4 * k + 1] += b.y, u[4 * k + 2] += b.z, u[4 * k + 3] += b.w;
        }
      }
      if (kSave) {
        __half* to = p.gu + (int64_t)t * 2 * p.F + col;
        uint8_t* e = p.scales + (int64_t)t * 2 * p.scale_pitch + col / 8;
        e[0] = (uint8_t)keep8(g, reinterpret_cast<uint4*>(to));
        e[p.scale_pitch] = (uint8_t)keep8(u, reinterpret_cast<uint4*>(to + p.F));
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = activate<kAct>(g[k]) * u[k];
      store_vec<__nv_bfloat16, 8>(p.h + t * p.ldh + col, g);
    }
  }
  if (split > 1) cluster_sync_all();  // the peers no longer read this CTA's sums
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, tmem_cols);
  }
}

// ---- input gradient of few rows --------------------------------------------------------------------------------------
// dx[T, K] = dgu[T, 2F] w[2F, K], where 256 x 256 tiles would be too few to fill the GPU and each would walk all of 2F alone
// (301 x 1016 over 5456: 8 tiles, 35 us; 17 us here). As above the weight is the M operand, here as it lies (MN-major): a CTA computes 128
// columns of dx for up to 256 rows, and the `split` CTAs of a cluster share the steps over 2F and join their fp32 sums through
// distributed shared memory, in rank order. Bound by the weight's bytes when T is small.
enum DxStatus : uint32_t {
  kTimeoutDxProducer = 0x141,
  kTimeoutDxMma = 0x142,
  kTimeoutDxEpilogue = 0x143,
  kTimeoutDxDrain = 0x144,
};
struct DxParams {
  int T, K, R;  // R = 2F, the length of the sums
  __nv_bfloat16* dx;
  int64_t lddx;
  int n;      // rows per CTA, a multiple of 16 up to 256
  int split;  // CTAs per cluster
  uint32_t* status;
  uint64_t wait_ns;
};
__host__ __device__ inline int dx_stage_bytes(int n) { return kATileBytes + n * 128; }
__host__ __device__ inline int dx_stages(int n) {
  const int fit = (kRowsSmem - 1024 - kRowsBars) / dx_stage_bytes(n);
  return fit < kRowsMaxStages ? fit : kRowsMaxStages;
}

__device__ __forceinline__ void dx_report(const DxParams& p, uint32_t code) {
  volatile uint32_t* s = p.status;
  if (s && *s == 0) *s = code;
}

__device__ __forceinline__ void gated_dx_body(const DxParams& p, const CUtensorMap* tmap_w, const CUtensorMap* tmap_d, uint8_t* smem_raw) {
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* tiles = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const int n = p.n, split = p.split, stages = dx_stages(n), stage_bytes = dx_stage_bytes(n);
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + stages * stage_bytes);  // [stages]
  uint64_t* empty = full + kRowsMaxStages;                                     // [stages]
  uint64_t* acc_full = empty + kRowsMaxStages;
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(acc_full + 1);

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int rank = blockIdx.x % split, col0 = blockIdx.x / split * BM, row0 = blockIdx.y * n;
  const int all_steps = (p.R + BK - 1) / BK;
  const int step0 = (int)((int64_t)all_steps * rank / split), steps = (int)((int64_t)all_steps * (rank + 1) / split) - step0;
  const uint32_t tmem_cols = n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : 256;

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(acc_full, 1);
    mbar_fence_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(tmap_w);
    tma_prefetch_desc(tmap_d);
  }
  if (warp == 1) {
    tmem_alloc(tmem_base_slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  body_sync();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_base_slot;
  grid_wait();
  grid_release();

  if (warp == 0) {
    if (elect_one()) {
      bool ok = true;
      int it = 0, s = 0;
      uint32_t phase = 1;
      uint8_t* sw = tiles;
      for (; it < steps; ++it) {
        if (!mbar_wait(&empty[s], phase, p.wait_ns)) {
          dx_report(p, kTimeoutDxProducer);
          ok = false;
          break;
        }
        const int r0 = (step0 + it) * BK;
        mbar_arrive_expect_tx(&full[s], stage_bytes);
#pragma unroll
        for (int c = 0; c < BM / 64; ++c) tma_load_2d(sw + c * 8192, tmap_w, &full[s], col0 + c * 64, r0);
        tma_load_2d(sw + kATileBytes, tmap_d, &full[s], r0, row0);
        sw += stage_bytes;
        if (++s == stages) {
          s = 0;
          phase ^= 1;
          sw = tiles;
        }
      }
      if (!ok) {
        // let the copies still in flight land before this CTA's shared memory is given up
        for (int i = it > stages ? it - stages : 0; i < it; ++i)
          if (!mbar_wait(&full[i % stages], (i / stages) & 1, p.wait_ns)) dx_report(p, kTimeoutDxDrain);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = make_idesc_f16(true, true, false, BM, n);
      const uint64_t first_w = make_smem_desc(smem_u32(tiles), 8192, 1024);
      const uint64_t first_d = make_smem_desc(smem_u32(tiles) + kATileBytes, 0, 1024);
      bool ok = true;
      int s = 0;
      uint32_t phase = 0;
      uint64_t dw = first_w, dd = first_d;
      for (int it = 0; it < steps; ++it) {
        if (!mbar_wait(&full[s], phase, p.wait_ns)) {
          dx_report(p, kTimeoutDxMma);
          ok = false;
          break;
        }
        tc_fence_after_sync();
#pragma unroll
        for (int k = 0; k < BK / UMMA_K; ++k) tc_mma_f16(tmem_base, dw + k * (2048 >> 4), dd + k * 2, idesc, it | k);
        tc_commit(&empty[s]);
        dw += stage_bytes >> 4;
        dd += stage_bytes >> 4;
        if (++s == stages) {
          s = 0;
          phase ^= 1;
          dw = first_w;
          dd = first_d;
        }
      }
      if (ok) tc_commit(acc_full);
    }
  } else {
    // accumulators to shared memory as sums[row][128 columns]: every product is done, so the stages are free
    const int q = warp & 3, r = q * 32 + lane;
    float* sums = reinterpret_cast<float*>(tiles);
    if (mbar_wait(acc_full, 0, p.wait_ns)) {
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < n && row0 + c < p.T; c += 16) {
        uint32_t v[16];
        tmem_ld_32x16(taddr + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[(c + i) * BM + r] = __uint_as_float(v[i]);
      }
    } else if (lane == 0) {
      dx_report(p, kTimeoutDxEpilogue);
    }
    tc_fence_before_sync();
  }
  body_sync();
  if (split > 1) cluster_sync_all();  // every CTA of the cluster has its sums in place
  {
    const int rows = min(n, p.T - row0), pieces = rows * (BM / 8);
    const uint32_t here = smem_u32(tiles);
    for (int i = rank * kNumThreads + (int)threadIdx.x; i < pieces; i += split * kNumThreads) {
      const int t = i / (BM / 8), j = i % (BM / 8) * 8, col = col0 + j;
      if (col >= p.K) continue;
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = 0.f;
      for (int c = 0; c < split; ++c) {
        const uint32_t from = (split > 1 ? map_to_cta(here, c) : here) + (t * BM + j) * 4;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float4 a = ld_cluster_f4(from + k * 16);
          f[4 * k] += a.x, f[4 * k + 1] += a.y, f[4 * k + 2] += a.z, f[4 * k + 3] += a.w;
        }
      }
      store_vec<__nv_bfloat16, 8>(p.dx + (row0 + t) * p.lddx + col, f);
    }
  }
  if (split > 1) cluster_sync_all();  // the peers no longer read this CTA's sums
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, tmem_cols);
  }
}

}  // namespace gated
}  // namespace mb
