// The gated feed-forward product for few tokens (M <= 128): both weights are
// read once, whatever M is, so their bytes are what bounds it.
//
// The weights stand on the tensor cores' M side: a tile is 128 features, its
// gate rows and its up rows are two accumulators D[f, m] of as many columns as
// there are tokens (in sixteens), and an MMA takes time in proportion to them.
// kN, the smallest of 16, 32, 64, 128 that holds them, is the accumulators'
// place in TMEM and the room for the tokens in a stage. A feature's gate and up values meet in one TMEM lane, and
// a warp stores 32 consecutive features of a token at once.
//
// With 74 tiles or more one SM takes a tile whole: that many SMs ask for more
// than the memory gives. Fewer tiles are cut along K among the CTAs of a
// cluster (up to 8), and joined through distributed shared memory: each CTA
// owns a share of the tokens, every CTA stores its sums of those tokens into
// the owner's shared memory, and the owner adds the parts in their order along
// K. No workspace, no atomics, and the same result every time. (Joining
// through global memory by whichever CTA came last took 9 us for one token and
// 70 for 77, against a floor of 7 to 23.)
//
// Measured on B200: one token at 3072 x 12288 (151 MB) 28.5 us, 5.3 TB/s (6.3
// at four times the features: what is left is a launch's start and end); 77
// tokens at 2056 x 5640 (47.6 MB) 17.5 us. Past some 30 tokens the tokens' own
// re-reads by every tile take the load path into the SMs, which gives 43 bytes
// a cycle: 128 tokens at 3072 x 12288 take 43 us.
//
// Warp 4 loads (TMA; gate and up tiles of 16 KB and the tokens per
// stage), warp 5 issues tcgen05.mma, warps 0-3 own the 128 lanes.
#include <string.h>

#include <type_traits>

#include "common.cuh"
#include "gated.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace gfx {

GFX_DEFINE_STATUS_READER(gated_few_device_status)

namespace gated {

constexpr int kFewTile = 128, kFewK = 64, kFewThreads = 192;
constexpr int kFewWeightBytes = kFewTile * kFewK * 2;

template <int kN>
struct FewRing {
  static constexpr int kStageBytes = 2 * kFewWeightBytes + kN * kFewK * 2;
  static constexpr int kStages = (232448 - 1024 - 256) / kStageBytes;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + 256;
};

struct FewArgs {
  CUtensorMap wg, wu, x;
  int M, F, steps, tiles;  // steps: K stages of a tile
  int columns;             // tokens in sixteens: the MMA's N and the rows of x per stage
  const void* bg;
  const void* bu;
  void* h;
  float* save;
  int* status_host;
};

// One feature of one token: biases, activation, product, and what a backward wants kept.
template <typename T, int kAct>
__device__ __forceinline__ void finish(const FewArgs& a, long long m, int f, float g, float u) {
  if (a.bg != nullptr) g += to_f32<T>(static_cast<const T*>(a.bg)[f]);
  if (a.bu != nullptr) u += to_f32<T>(static_cast<const T*>(a.bu)[f]);
  if (a.save != nullptr) {
    a.save[m * a.F + f] = g;
    a.save[((long long)a.M + m) * a.F + f] = u;
  }
  static_cast<T*>(a.h)[m * a.F + f] = from_f32<T>(activation<kAct>(g) * u);
}

template <typename T, int kAct, int kN>
__global__ void __launch_bounds__(kFewThreads, 1) few_kernel(const __grid_constant__ FewArgs a) {
  constexpr int kStages = FewRing<kN>::kStages, kStageBytes = FewRing<kN>::kStageBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(base + kStages * kStageBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_base = reinterpret_cast<uint32_t*>(drain + 1);
  static_assert((2 * kStages + 5) * 8 + 4 <= 256, "barrier area");
  static_assert((kN + 32) * 1024 <= kStages * kStageBytes, "the join's memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int parts = (int)cluster_nctarank(), part = (int)cluster_ctarank();
  const int k0 = a.steps * part / parts, k1 = a.steps * (part + 1) / parts;
  const int first = blockIdx.x / parts, stride = gridDim.x / parts;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 4);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == 5) tc::tmem_alloc<1>(tmem_base, 4 * kN);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_base;
  pdl_trigger();

  bool ok = true;
  if (warp == 4) {
    if (lane == 0) {
      tma_prefetch_desc(&a.wg);
      tma_prefetch_desc(&a.wu);
      tma_prefetch_desc(&a.x);
      // the first stages' weights come into L2 while the stream's previous kernel ends
      for (int k = k0; k < k1 && k < k0 + kStages; ++k) {
        tma_prefetch_l2_2d(&a.wg, k * kFewK, first * kFewTile);
        tma_prefetch_l2_2d(&a.wu, k * kFewK, first * kFewTile);
      }
      pdl_wait();
      uint32_t it = 0;
      for (int t = first; t < a.tiles && ok; t += stride) {
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % kStages;
          if (!mbar_wait(&empty[s], ((it / kStages) & 1) ^ 1, kDevErrEmptyBarrierTimeout)) {
            ok = false;
            break;
          }
          uint8_t* st = base + s * kStageBytes;
          mbar_arrive_expect_tx(&full[s], 2 * kFewWeightBytes + a.columns * kFewK * 2);
          tma_load_2d(st, &a.wg, &full[s], k * kFewK, t * kFewTile);
          tma_load_2d(st + kFewWeightBytes, &a.wu, &full[s], k * kFewK, t * kFewTile);
          tma_load_2d(st + 2 * kFewWeightBytes, &a.x, &full[s], k * kFewK, 0);
        }
      }
      if (!ok) {  // a wait gave up: let the copies in flight land before the memory is given back
        const unsigned long long t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    pdl_wait();  // its waits are limited, and the stream's previous kernel is not
    constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t id = (1u << 4) | (kType << 7) | (kType << 10) | ((uint32_t)(a.columns >> 3) << 17) |
                        ((uint32_t)(kFewTile >> 4) << 24);
    uint32_t it = 0;
    int n = 0;
    for (int t = first; t < a.tiles && ok; t += stride, ++n) {
      const int acc = n & 1;
      if (!mbar_wait(&acc_empty[acc], ((n >> 1) & 1) ^ 1, kDevErrMmaBarrierTimeout)) {
        ok = false;
        break;
      }
      tc::tc_fence_after();
      for (int k = k0; k < k1; ++k, ++it) {
        const int s = it % kStages;
        if (!mbar_wait(&full[s], (it / kStages) & 1, kDevErrFullBarrierTimeout)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        if (lane == 0) {
          const uint32_t sg = smem_u32(base + s * kStageBytes);
          const uint64_t dg = tc::sw128_desc(sg), du = tc::sw128_desc(sg + kFewWeightBytes);
          const uint64_t dx = tc::sw128_desc(sg + 2 * kFewWeightBytes);
#pragma unroll
          for (int q = 0; q < kFewK / 16; ++q) {
            const uint32_t more = k != k0 || q != 0;
            tc::umma_f16<1>(tmem + acc * 2 * kN, dg + 2 * q, dx + 2 * q, id, more);
            tc::umma_f16<1>(tmem + acc * 2 * kN + kN, du + 2 * q, dx + 2 * q, id, more);
          }
          tc::umma_commit<1>(&empty[s]);
          if (k == k1 - 1) tc::umma_commit<1>(&acc_full[acc]);
        }
        __syncwarp();
      }
    }
    if (lane == 0) tc::umma_commit<1>(drain);
    __syncwarp();
    if (!mbar_wait(drain, 0, kDevErrMmaBarrierTimeout)) ok = false;
  } else if (parts == 1) {
    pdl_wait();
    int n = 0;
    for (int t = first; t < a.tiles; t += stride, ++n) {
      const int acc = n & 1;
      if (!mbar_wait(&acc_full[acc], (n >> 1) & 1, kDevErrEpilogueBarrierTimeout)) {
        ok = false;
        break;
      }
      tc::tc_fence_after();
      const int f = t * kFewTile + warp * 32 + lane;
      const uint32_t d = tmem + ((uint32_t)(warp * 32) << 16) + acc * 2 * kN;
      for (int c = 0; c < a.M; c += 16) {
        uint32_t g[16], u[16];
        tc::tmem_ld16_nowait(d + c, g);
        tc::tmem_ld16_nowait(d + kN + c, u);
        tc::tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          asm volatile("" : "+r"(g[e]), "+r"(u[e]));
          if (f < a.F && c + e < a.M) finish<T, kAct>(a, c + e, f, __uint_as_float(g[e]), __uint_as_float(u[e]));
        }
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
    }
  }

  if (parts > 1) {
    // one tile a cluster; owner o finishes tokens [o share, (o + 1) share)
    const int share = (a.M + 4 * parts - 1) / (4 * parts) * 4;
    cluster_sync_all();  // every CTA's loads and MMAs are done: the stages' memory is free
    if (warp < 4) {
      pdl_wait();
      if (!mbar_wait(&acc_full[0], 0, kDevErrEpilogueBarrierTimeout)) ok = false;
      tc::tc_fence_after();
      const uint32_t d = tmem + ((uint32_t)(warp * 32) << 16);
      // [part][four tokens of the owner][gate, up][128 features][4]: a warp stores 512 bytes in a row
      const uint32_t spot = smem_u32(base) + (uint32_t)(part * share * 1024 + (warp * 32 + lane) * 16);
      for (int o = 0; o * share < a.M; ++o) {
        const uint32_t to = mapa_shared(spot, o);
        for (int c = 0; c < share && o * share + c < a.M; c += 4) {
          uint32_t g[4], u[4];
          tc::tmem_ld4_nowait(d + o * share + c, g);
          tc::tmem_ld4_nowait(d + kN + o * share + c, u);
          tc::tmem_wait_ld();
          asm volatile("" : "+r"(g[0]), "+r"(g[1]), "+r"(g[2]), "+r"(g[3]));
          asm volatile("" : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]));
          st_shared_cluster_v4(to + c * 1024, g);
          st_shared_cluster_v4(to + c * 1024 + 2048, u);
        }
      }
      tc::tc_fence_before();
    }
    cluster_sync_all();
    const int mine = min(share, a.M - part * share);
    for (int i = threadIdx.x; ok && i < (mine + 3) / 4 * kFewTile; i += kFewThreads) {
      const int m = i / kFewTile * 4, c = i % kFewTile, f = first * kFewTile + c;
      float g[4] = {0.0f, 0.0f, 0.0f, 0.0f}, u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int p = 0; p < parts; ++p) {
        const uint32_t at = smem_u32(base) + (uint32_t)((p * share + m) * 1024 + c * 16);
        const uint4 x = lds128(at), y = lds128(at + 2048);
        g[0] += __uint_as_float(x.x), g[1] += __uint_as_float(x.y);
        g[2] += __uint_as_float(x.z), g[3] += __uint_as_float(x.w);
        u[0] += __uint_as_float(y.x), u[1] += __uint_as_float(y.y);
        u[2] += __uint_as_float(y.z), u[3] += __uint_as_float(y.w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (f < a.F && m + e < mine) finish<T, kAct>(a, part * share + m + e, f, g[e], u[e]);
    }
  }
  if (!ok) mirror_device_error(a.status_host);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 5) tc::tmem_dealloc<1>(tmem, 4 * kN);
}

template <typename T, int kAct, int kN>
static int launch_few(FewArgs& a, int parts, cudaStream_t st, int sms) {
  auto kern = few_kernel<T, kAct, kN>;
  static bool ready[64] = {false};
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return set_error(GFX_ERR_CUDA, "gated few_kernel: no current device");
  if (!ready[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FewRing<kN>::kSmemBytes);
    if (e != cudaSuccess)
      return set_error(GFX_ERR_CUDA, "gated few_kernel: cannot set %d bytes of shared memory: %s",
                       FewRing<kN>::kSmemBytes, cudaGetErrorString(e));
    ready[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = parts, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(parts > 1 ? a.tiles * parts : (a.tiles < sms ? a.tiles : sms));
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = FewRing<kN>::kSmemBytes;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  a.status_host = host_status_word(dev);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) return set_error(GFX_ERR_CUDA, "gated few_kernel launch: %s", cudaGetErrorString(e));
  return check_launch("gated few_kernel");
}

template <typename T, int kAct>
static int launch_few_n(FewArgs& a, int parts, cudaStream_t st, int sms) {
  if (a.M <= 16) return launch_few<T, kAct, 16>(a, parts, st, sms);
  if (a.M <= 32) return launch_few<T, kAct, 32>(a, parts, st, sms);
  if (a.M <= 64) return launch_few<T, kAct, 64>(a, parts, st, sms);
  return launch_few<T, kAct, 128>(a, parts, st, sms);
}

// CTAs a tile: as many as leave every SM at most one, at least four stages each.
static int few_parts(int tiles, int steps, int sms) {
  int parts = sms / tiles;
  if (parts > steps / 4) parts = steps / 4;
  return parts < 1 ? 1 : (parts > 8 ? 8 : parts);
}

template <typename T>
static int few_t(const GatedArgs& g, int act, void* h, float* save, cudaStream_t st, int sms) {
  FewArgs a;
  memset(&a, 0, sizeof(a));
  constexpr CUtensorMapDataType kType =
      std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  a.columns = (g.M + 15) / 16 * 16;
  int rc;
  if ((rc = make_tmap_2d(&a.wg, kType, g.w_gate, g.K, g.F, (uint64_t)g.ldg * 2, kFewK, kFewTile,
                         CU_TENSOR_MAP_SWIZZLE_128B)) ||
      (rc = make_tmap_2d(&a.wu, kType, g.w_up, g.K, g.F, (uint64_t)g.ldu * 2, kFewK, kFewTile,
                         CU_TENSOR_MAP_SWIZZLE_128B)) ||
      (rc = make_tmap_2d(&a.x, kType, g.x, g.K, g.M, (uint64_t)g.ldx * 2, kFewK, a.columns,
                         CU_TENSOR_MAP_SWIZZLE_128B)))
    return rc;
  a.M = g.M, a.F = g.F, a.steps = (g.K + kFewK - 1) / kFewK;
  a.tiles = (g.F + kFewTile - 1) / kFewTile;
  a.bg = g.b_gate, a.bu = g.b_up, a.h = h, a.save = save;
  const int parts = few_parts(a.tiles, a.steps, sms);
  if (act == kSilu) return launch_few_n<T, kSilu>(a, parts, st, sms);
  if (act == kGelu) return launch_few_n<T, kGelu>(a, parts, st, sms);
  return launch_few_n<T, kGeluTanh>(a, parts, st, sms);
}

}  // namespace gated

int launch_gated_forward_few(const GatedArgs& a, int dtype, int act, void* h, float* save, cudaStream_t st, int sms) {
  return dtype == GFX_DTYPE_F16 ? gated::few_t<__half>(a, act, h, save, st, sms)
                                : gated::few_t<__nv_bfloat16>(a, act, h, save, st, sms);
}

}  // namespace gfx
