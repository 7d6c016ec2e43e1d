// Host side of the gated projection and the elementwise half of its backward pass.
#include "gated_tcgen05.cuh"
#include "kernels_api.h"
#include "vec_io.cuh"

#define MB_STREAM(s) reinterpret_cast<cudaStream_t>(s)

namespace mb {
namespace gemm {
int make_tmap_bf16(CUtensorMap* out, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows);
int make_tmap_bf16_stack(CUtensorMap* out, const void* base, uint64_t count, uint64_t apart, uint64_t rows, uint64_t cols, uint64_t ld,
                         uint32_t box_rows);
}
namespace gated {

constexpr int kMaxDevices = 64;

template <int kAct, bool kSave>
__global__ void __launch_bounds__(kNumThreads, 1)
    gated_pair_kernel(const __grid_constant__ GatedParams p, const __grid_constant__ CUtensorMap tmap_x,
                      const __grid_constant__ CUtensorMap tmap_w) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  gated_pair_body<kAct, kSave>(p, &tmap_x, &tmap_w, smem_raw);
}

template <int kAct, bool kSave>
static int launch_pair(GatedParams& p, const CUtensorMap& tx, const CUtensorMap& tw, int device, cudaStream_t stream) {
  auto kern = gated_pair_kernel<kAct, kSave>;
  static int max_clusters[kMaxDevices];  // per instantiation; 0: not asked yet
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(kNumThreads, 1, 1);
  cfg.dynamicSmemBytes = kGatedPairSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (max_clusters[device] == 0) {
    int sms = 0, n = 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kGatedPairSmem) != cudaSuccess)
      return MB_ERR_LAUNCH;
    cfg.gridDim = dim3(sms & ~1, 1, 1);
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = sms / 2;
    }
    max_clusters[device] = n < sms / 2 ? n : sms / 2;
  }
  const int tiles = p.tiles_m * p.tiles_n;
  p.num_ctas = 2 * (tiles < max_clusters[device] ? tiles : max_clusters[device]);
  cfg.gridDim = dim3(p.num_ctas, 1, 1);
  return cudaLaunchKernelEx(&cfg, kern, p, tx, tw) == cudaSuccess ? MB_OK : MB_ERR_LAUNCH;
}

template <int kAct, bool kSave>
__global__ void __launch_bounds__(kNumThreads, 1)
    gated_rows_kernel(const __grid_constant__ GatedParams p, int width, int n, int split, const __grid_constant__ CUtensorMap tmap_x,
                      const __grid_constant__ CUtensorMap tmap_w) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  gated_rows_body<kAct, kSave>(p, width, n, split, &tmap_x, &tmap_w, smem_raw);
}

template <int kAct, bool kSave>
static int launch_rows(const GatedParams& p, int width, int n, int split, const CUtensorMap& tx, const CUtensorMap& tw, int device,
                       cudaStream_t stream) {
  auto kern = gated_rows_kernel<kAct, kSave>;
  static bool configured[kMaxDevices];  // per instantiation
  if (!configured[device]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem) != cudaSuccess) return MB_ERR_LAUNCH;
    configured[device] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((p.F + width - 1) / width * split, 1, 1);
  cfg.blockDim = dim3(kNumThreads, 1, 1);
  cfg.dynamicSmemBytes = kRowsSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, p, width, n, split, tx, tw) == cudaSuccess ? MB_OK : MB_ERR_LAUNCH;
}

static int device_sms(int device) {
  static int sms[kMaxDevices];
  if (sms[device] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) n = 148;
    sms[device] = n;
  }
  return sms[device];
}

// How many clusters of `split` CTAs, one per SM, run at once: the SMs are not a multiple of a cluster in every part of the GPU.
// Asked once per device, for splits of 1, 2, 4 and 8.
template <auto kKernel>
static int active_clusters(int split, int device) {
  static int known[kMaxDevices][4];
  int& n = known[device][split >= 8 ? 3 : split / 2];
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(device_sms(device) / split * split, 1, 1);
    cfg.blockDim = dim3(kNumThreads, 1, 1);
    cfg.dynamicSmemBytes = kRowsSmem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int got = 0;
    if (cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&got, kKernel, &cfg) != cudaSuccess || got <= 0) {
      cudaGetLastError();
      got = device_sms(device) * 3 / 4 / split;
    }
    n = got;
  }
  return n;
}

// Columns of h per CTA and CTAs per K range of the few-rows kernel. One wave of CTAs is to cover F with the narrowest width
// (a multiple of 8) that does; from 128 SMs' worth of columns up it takes more waves. Where F is so small that tiles of 64
// columns leave SMs over, up to 8 CTAs split K, as long as each keeps 8 steps of 64 (F = 1184, K = 4096: 8.5 us in four parts,
// 24 us in one).
static void rows_shape(int F, int K, int device, int& width, int& split) {
  const int sms = device_sms(device);
  for (split = 8; split > 1; split /= 2) {
    const int tiles = active_clusters<gated_rows_kernel<kSilu, false>>(split, device);
    width = ((F + tiles - 1) / tiles + 7) / 8 * 8;
    if (width <= 64 && K >= split * 8 * BK) return;
  }
  const int waves = (F + 128 * sms - 1) / (128 * sms);
  const int ctas = waves * sms;
  width = ((F + ctas - 1) / ctas + 7) / 8 * 8;
}

__global__ void __launch_bounds__(kNumThreads, 1)
    gated_dx_kernel(const __grid_constant__ DxParams p, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_d) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  gated_dx_body(p, &tmap_w, &tmap_d, smem_raw);
}

// dgu[:, :F] = dh * u * act'(g), dgu[:, F:] = dh * act(g): three reads and two writes of [T, F] and a byte per 16 of the kept
// projections, bound by their bytes. The results are rounded to bf16 because the two matrix products that follow take bf16 operands.
// A thread keeps its 8 columns and walks down the rows, so no index is divided. 8192 x 14336: 205 us, 6.1 TB/s.
template <int kAct>
__global__ void __launch_bounds__(256)
    gated_bwd_kernel(const __half* __restrict__ gu, const uint8_t* __restrict__ scales, int scale_pitch,
                     const __nv_bfloat16* __restrict__ dh, __nv_bfloat16* __restrict__ dgu, int64_t T, int F, int64_t lddh) {
  const int v = blockIdx.x * 256 + threadIdx.x, j = v * 8;
  if (j >= F) return;
#pragma unroll 2
  for (int64_t t = blockIdx.y; t < T; t += gridDim.y) {
    const __half* from = gu + t * 2 * F + j;
    const uint8_t* e = scales + t * 2 * scale_pitch + v;
    float g[8], u[8], d[8];
    load_vec<__half, 8>(from, g);
    load_vec<__half, 8>(from + F, u);
    load_vec<__nv_bfloat16, 8>(dh + t * lddh + j, d);
    const float sg = kept_scale(e[0]), su = kept_scale(e[scale_pitch]);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float2 a = activate_slope<kAct>(g[k] * sg);
      g[k] = d[k] * (u[k] * su) * a.y;
      u[k] = d[k] * a.x;
    }
    __nv_bfloat16* to = dgu + t * 2 * F + j;
    store_vec<__nv_bfloat16, 8>(to, g);
    store_vec<__nv_bfloat16, 8>(to + F, u);
  }
}

}  // namespace gated
}  // namespace mb

using namespace mb;
using namespace mb::gated;

extern "C" int mb_gated_scale_pitch(int F) { return (F / 8 + 15) / 16 * 16; }

extern "C" int mb_gated_fwd_bf16(const void* x, const void* w, void* h, void* gu, void* scales, int64_t T, int F, int K, int64_t ldx,
                                 int64_t ldw, int64_t ldh, int act, uint32_t* status, uint64_t wait_ns, void* stream) {
  if (T <= 0) return MB_OK;
  if (F <= 0 || K <= 0 || T > (1 << 30) || F > (1 << 29) || act < 0 || act > 2 || !gu != !scales) return MB_ERR_ARG;
  if (F % 8 || K % 8 || ldx % 8 || ldw % 8 || ldh % 8) return MB_ERR_ALIGN;
  if (!is_aligned(x, 16) || !is_aligned(w, 16) || !is_aligned(h, 16) || !is_aligned(gu, 16) || !is_aligned(scales, 16)) return MB_ERR_ALIGN;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= kMaxDevices) return MB_ERR_DRIVER;
  // Few rows: the weight's bytes bound the time and a 256-row tile would leave SMs idle (F = 14336, K = 4096, one row: 39 us,
  // 65 us in pair tiles; 128 rows: 46 us; from 129 rows pair tiles, 55 us).
  const bool few = T <= BM;
  int width = kHCols, split = 1;
  if (few) rows_shape(F, K, device, width, split);
  const int x_rows = few ? (int)(T + 15) / 16 * 16 : BM;
  CUtensorMap tx, tw;
  int rc = gemm::make_tmap_bf16(&tx, x, T, K, ldx, x_rows);
  if (rc) return rc;
  rc = few ? gemm::make_tmap_bf16_stack(&tw, w, 2, F * (uint64_t)ldw, F, K, ldw, width)
           : gemm::make_tmap_bf16(&tw, w, 2 * (uint64_t)F, K, ldw, width);
  if (rc) return rc;
  GatedParams p{};
  p.T = (int)T;
  p.F = F;
  p.K = K;
  p.h = (__nv_bfloat16*)h;
  p.ldh = ldh;
  p.gu = (__half*)gu;
  p.scales = (uint8_t*)scales;
  p.scale_pitch = mb_gated_scale_pitch(F);
  p.tiles_m = (int)((T + kPairBM - 1) / kPairBM);
  p.tiles_n = (F + kHCols - 1) / kHCols;
  p.group_m = 4;
  p.status = status;
  p.wait_ns = wait_ns ? wait_ns : kDefaultWaitNs;
  cudaStream_t s = MB_STREAM(stream);
  switch (act * 2 + (gu ? 1 : 0)) {
    case 0: return few ? launch_rows<kSilu, false>(p, width, x_rows, split, tx, tw, device, s) : launch_pair<kSilu, false>(p, tx, tw, device, s);
    case 1: return few ? launch_rows<kSilu, true>(p, width, x_rows, split, tx, tw, device, s) : launch_pair<kSilu, true>(p, tx, tw, device, s);
    case 2: return few ? launch_rows<kGelu, false>(p, width, x_rows, split, tx, tw, device, s) : launch_pair<kGelu, false>(p, tx, tw, device, s);
    case 3: return few ? launch_rows<kGelu, true>(p, width, x_rows, split, tx, tw, device, s) : launch_pair<kGelu, true>(p, tx, tw, device, s);
    case 4: return few ? launch_rows<kGeluTanh, false>(p, width, x_rows, split, tx, tw, device, s) : launch_pair<kGeluTanh, false>(p, tx, tw, device, s);
    default: return few ? launch_rows<kGeluTanh, true>(p, width, x_rows, split, tx, tw, device, s) : launch_pair<kGeluTanh, true>(p, tx, tw, device, s);
  }
}

extern "C" int mb_gated_bwd_bf16(const void* gu, const void* scales, const void* dh, void* dgu, int64_t T, int F, int64_t lddh, int act,
                                 void* stream) {
  if (T <= 0) return MB_OK;
  if (F <= 0 || act < 0 || act > 2) return MB_ERR_ARG;
  if (F % 8 || lddh % 8 || !is_aligned(gu, 16) || !is_aligned(dh, 16) || !is_aligned(dgu, 16)) return MB_ERR_ALIGN;
  const int across = (F / 8 + 255) / 256;
  const int64_t down = (148 * 16 + across - 1) / across;
  const dim3 grid(across, (unsigned)(T < down ? T : down));
  auto k = act == kSilu ? gated_bwd_kernel<kSilu> : act == kGelu ? gated_bwd_kernel<kGelu> : gated_bwd_kernel<kGeluTanh>;
  k<<<grid, 256, 0, MB_STREAM(stream)>>>((const __half*)gu, (const uint8_t*)scales, mb_gated_scale_pitch(F),
                                                   (const __nv_bfloat16*)dh, (__nv_bfloat16*)dgu, T, F, lddh);
  return cudaPeekAtLastError() == cudaSuccess ? MB_OK : MB_ERR_LAUNCH;
}

extern "C" int mb_gated_dx_bf16(const void* dgu, const void* w, void* dx, int64_t T, int F, int K, int64_t lddgu, int64_t ldw,
                                int64_t lddx, uint32_t* status, uint64_t wait_ns, void* stream) {
  if (T <= 0) return MB_OK;
  if (F <= 0 || K <= 0 || T > (1 << 30) || F > (1 << 29)) return MB_ERR_ARG;
  if (F % 8 || K % 8 || lddgu % 8 || ldw % 8 || lddx % 8 || !is_aligned(dgu, 16) || !is_aligned(w, 16) || !is_aligned(dx, 16))
    return MB_ERR_ALIGN;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= kMaxDevices) return MB_ERR_DRIVER;
  const int sms = device_sms(device);
  // Up to a quarter of the SMs' worth of 256 x 256 tiles the split kernel is ahead (us, split and tiles): 1 row, 14336 -> 4096
  // 38 and 161; 256, 11008 -> 4096 51 and 106; 1024, 1408 -> 2048 18 and 20, which is where it ends.
  const int64_t pair_tiles = (T + kPairBM - 1) / kPairBM * ((K + BN - 1) / BN);
  if (pair_tiles * 4 > sms)
    return mb_gemm_bf16(dgu, w, dx, (int)T, K, 2 * F, lddgu, ldw, lddx, 0, 1, 0, 0, status, wait_ns, stream);
  DxParams p{};
  p.T = (int)T;
  p.K = K;
  p.R = 2 * F;
  p.dx = (__nv_bfloat16*)dx;
  p.lddx = lddx;
  const int row_tiles = (int)((T + 255) / 256);
  p.n = (int)((T + row_tiles - 1) / row_tiles + 15) / 16 * 16;
  const int tiles = (K + BM - 1) / BM;
  p.split = 8;
  while (p.split > 1 && (tiles * row_tiles > active_clusters<gated_dx_kernel>(p.split, device) || p.R < p.split * 4 * BK)) p.split /= 2;
  p.status = status;
  p.wait_ns = wait_ns ? wait_ns : kDefaultWaitNs;
  CUtensorMap tw, td;
  int rc = gemm::make_tmap_bf16(&tw, w, 2 * (uint64_t)F, K, ldw, BK);
  if (rc) return rc;
  rc = gemm::make_tmap_bf16(&td, dgu, T, 2 * (uint64_t)F, lddgu, p.n);
  if (rc) return rc;
  static bool configured[kMaxDevices];
  if (!configured[device]) {
    if (cudaFuncSetAttribute(gated_dx_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem) != cudaSuccess) return MB_ERR_LAUNCH;
    configured[device] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(tiles * p.split, row_tiles, 1);
  cfg.blockDim = dim3(kNumThreads, 1, 1);
  cfg.dynamicSmemBytes = kRowsSmem;
  cfg.stream = MB_STREAM(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, gated_dx_kernel, p, tw, td) == cudaSuccess ? MB_OK : MB_ERR_LAUNCH;
}
