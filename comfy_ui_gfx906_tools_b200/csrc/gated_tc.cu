// The matrix products of the gated feed-forward block on the 5th-generation
// tensor cores: forward (two projections, activation and product in one
// kernel), input gradient and weight gradients.
//
//   forward  D[m, c] = sum_k x[m, k] W[c, k], c < 128 of the gate's rows, the
//            other 128 of the up projection's same rows; the epilogue adds the
//            biases and writes h = a(g) u (and g, u in float32 for a backward)
//   dx       D[m, n] = sum_f dg[m, f] Wg[f, n] + sum_f du[m, f] Wu[f, n]
//   dW       D[f, n] = sum_m dg[m, f] x[m, n]   (du for the up projection)
//
// One kernel with three roles. A cluster of two CTAs computes a tile of 512
// rows x 256 columns as two row blocks of 256 with tcgen05.mma.cta_group::2
// (M = 256, N = 256, K = 16): each CTA loads its own 128 rows of either block
// of A and its own 128 of the 256 columns of B. In the forward CTA 0's half of
// B is the gate's weights and CTA 1's the up projection's, so both projections
// of a feature land in the same thread's TMEM lane. The operands that a
// gradient needs transposed (Wg as [F, n], dg as [m, F], x as [m, n]) are read
// where they lie: TMA brings 64 x 64 boxes and the descriptor names them
// MN-major.
//
// What bounds it is the load path into an SM: 256 x 256 tiles ask 64 bytes a
// cycle of it at the tensor cores' full rate, which is the path's peak, and
// ran them 66% of the cycles (4608 x 3072 x 4096, 1.77 GHz); the second row
// block asks 48. A product with too few 512-row tiles to fill the GPU takes
// one block a tile (kBlocks = 1, 7 stages instead of 4).
//
// Per CTA: warp 8 loads (TMA), warp 9 of CTA 0 issues the MMAs of the pair,
// warps 0-7 write tiles out: a thread owns one row and half of the columns,
// takes its 128 accumulators into registers at once and gives the TMEM back
// before it computes and stores (32 bytes at a time, whole sectors). TMEM holds
// two 256-column accumulators. With one block they alternate between tiles.
// With two, a new tile starts on the first block's share of the stages that are
// loaded while the second block's accumulator is still read. A stage's barrier
// lives in CTA 0 and counts both CTAs' bytes. Persistent: one pair per two
// SMs; tiles are walked in panels whose reused operand stays in L2.
//
// Tiles that do not fill a last wave are cut along the contraction, so that
// all pairs work on them at once (dx of 4608 x 3072 is 108 tiles for 74 pairs:
// 74 whole ones, then 34 in two halves each). The pairs of a wave move along
// the contraction side by side, which keeps the shared operands in L2; ranges
// that start anywhere would not. Each epilogue warp leaves its sums of a cut
// tile in the workspace and counts itself in; the last one of a tile adds all
// parts in their order, so the result does not depend on who came last.
//
// Measured on B200 at 4608 x 3072 x 12288 in bfloat16 (696 GFLOP each): forward
// 430 us (1.62 PFLOP/s), 508 with g and u kept (453 MB more to write), weight
// gradients 410 us (1.70), input gradient 431 us (1.61; 510 before the cut); a
// library product of the same shape takes 465 to 480. Under the power cap, one
// after the other for seconds, 488 / 590 / 505 / 523 us.
#include <string.h>

#include <type_traits>

#include "common.cuh"
#include "gated.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace gfx {

GFX_DEFINE_STATUS_READER(gated_tc_device_status)

namespace gated {

enum : int { kForward = 0, kInputGrad = 1, kWeightGrad = 2 };

constexpr int kBlockRows = 256, kTileCols = 256;  // of a pair; a CTA owns 128 rows of a block
constexpr int kStageK = 64;
constexpr int kOperandBytes = 128 * kStageK * 2;  // a CTA's share of a block of A, or of B, per stage
constexpr int kEpilogueWarps = 8, kLoadWarp = 8, kMmaWarp = 9, kThreads = 320;

template <int kBlocks>
struct Ring {
  static constexpr int kStages = kBlocks == 2 ? 4 : 7;
  static constexpr int kStageBytes = (kBlocks + 1) * kOperandBytes;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + 256;
  static_assert(kSmemBytes <= 232448, "shared memory");
};

struct TcArgs {
  CUtensorMap a0, a1, b0, b1;
  int rows, cols;       // of the output (forward: M, F; dx: M, K; dW: F, K)
  int depth;            // of the contraction, per segment (K; F; M)
  int tiles_i, tiles_j; // row tiles and column tiles
  int tiles_half;       // dW: row tiles of one weight; the second's follow
  int whole, cut, parts;// tiles taken whole, and those cut in `parts` along the contraction
  float* partial;       // sums of cut tiles, [cut * parts][2 CTAs][blocks][8 warps][128][32]
  int* counters;        // [cut][2][blocks][8], zero between calls
  int panel;            // tiles of the fast direction that are walked before the slow one moves
  int i_fast;
  void* out0;           // h; dx; dWg
  void* out1;           // dWu
  long long ld;         // row stride of the outputs
  const void* bias0;    // forward: bg, bu
  const void* bias1;
  float* save;          // forward: g, u
  int wide;             // rows of every output are 32-byte aligned
  int overlap;          // the stream's next kernel may start while this one ends
  unsigned long long wait_ns;  // limit of the waits for a whole contraction, and for the kernel's last MMA
  int* status_host;
};

// TMA load of one box into this CTA, counted on the barrier at `bar`, which may be the other CTA's.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, "
      "%4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}

// Shared-memory descriptor of an MN-major operand in 64 (MN) x 64 (K) boxes with the 128-byte swizzle: 64 elements of
// MN are 8 KB apart, 8 steps of K 1 KB.
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

template <typename T, int kRole>
constexpr uint32_t instruction_desc() {
  const uint32_t type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  const uint32_t a_mn = kRole == kWeightGrad ? 1u : 0u, b_mn = kRole == kForward ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) | (a_mn << 15) | (b_mn << 16) | ((uint32_t)(kTileCols >> 3) << 17) |
         ((uint32_t)(kBlockRows >> 4) << 24);
}

__device__ __forceinline__ void st_global_v8(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

__device__ __forceinline__ void st_global_v4(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// 32 consecutive values of one row (float bits) from column c on; columns past `cols` (a multiple of 8) are left out.
template <typename T>
__device__ __forceinline__ void store_row(T* row, int c, int cols, bool wide, const uint32_t (&f)[32]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int q = 0; q < 32; q += 8) {
      if (c + q >= cols) break;
      if (wide) {
        const uint32_t v[8] = {f[q], f[q + 1], f[q + 2], f[q + 3], f[q + 4], f[q + 5], f[q + 6], f[q + 7]};
        st_global_v8(row + c + q, v);
      } else {
        st_global_v4(row + c + q, f[q], f[q + 1], f[q + 2], f[q + 3]);
        st_global_v4(row + c + q + 4, f[q + 4], f[q + 5], f[q + 6], f[q + 7]);
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < 32; q += 16) {
      uint32_t v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = pack2<T>(__uint_as_float(f[q + 2 * j]), __uint_as_float(f[q + 2 * j + 1]));
      if (wide && c + q + 16 <= cols) {
        st_global_v8(row + c + q, v);
      } else {
        if (c + q < cols) st_global_v4(row + c + q, v[0], v[1], v[2], v[3]);
        if (c + q + 8 < cols) st_global_v4(row + c + q + 8, v[4], v[5], v[6], v[7]);
      }
    }
  }
}

__device__ __forceinline__ void tile_at(const TcArgs& a, int t, int& i, int& j) {
  const int nf = a.i_fast ? a.tiles_i : a.tiles_j, ns = a.i_fast ? a.tiles_j : a.tiles_i;
  const int p = t / (a.panel * ns), rest = t - p * a.panel * ns;
  const int width = min(a.panel, nf - p * a.panel);
  const int f = p * a.panel + rest % width, s = rest / width;
  i = a.i_fast ? f : s;
  j = a.i_fast ? s : f;
}

// What a pair does at once: a tile, or one part of a cut tile.
struct Unit {
  int tile, part, k0, k1;  // part -1: the whole tile
};

__device__ __forceinline__ Unit unit_at(const TcArgs& a, int u, int total) {
  Unit w{u, -1, 0, total};
  if (u >= a.whole) {
    const int v = u - a.whole;
    w.tile = a.whole + v % a.cut;
    if (a.parts > 1) {
      w.part = v / a.cut;
      w.k0 = (int)((long long)total * w.part / a.parts);
      w.k1 = (int)((long long)total * (w.part + 1) / a.parts);
    }
  }
  return w;
}

template <typename T, int kRole, int kAct, int kBlocks>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) pair_kernel(const __grid_constant__ TcArgs a) {
  constexpr int kStages = Ring<kBlocks>::kStages, kStageBytes = Ring<kBlocks>::kStageBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(base + kStages * kStageBytes);  // CTA 0's: both CTAs' loads landed
  uint64_t* empty = full + kStages;      // each CTA's: the MMAs have read the stage
  uint64_t* acc_full = empty + kStages;  // each CTA's [2]: the accumulator is complete
  uint64_t* acc_empty = acc_full + 2;    // CTA 0's [2]: both CTAs' epilogues are done with it
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_base = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cr = cluster_ctarank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int units = a.whole + a.cut * a.parts;
  const int steps = (a.depth + kStageK - 1) / kStageK;  // per segment
  const int stages = kRole == kInputGrad ? 2 * steps : steps;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 2 * kEpilogueWarps);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == kMmaWarp) tc::tmem_alloc<2>(tmem_base, 512);
  tc::tc_fence_before();
  cluster_sync_all();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_base;
  if (a.overlap) pdl_trigger();

  bool ok = true;
  if (warp == kLoadWarp) {
    if (lane == 0) {
      tma_prefetch_desc(&a.a0);
      tma_prefetch_desc(&a.b0);
      pdl_wait();
      uint32_t it = 0;
      for (int u = pair; u < units && ok; u += pairs) {
        const Unit w = unit_at(a, u, stages);
        int i, j;
        tile_at(a, w.tile, i, j);
        const int half = kRole == kWeightGrad && i >= a.tiles_half;
        const int r0 = (half ? i - a.tiles_half : i) * (kBlocks * kBlockRows) + (int)cr * 128;
        const int c0 = kRole == kForward ? j * 128 : j * kTileCols + (int)cr * 128;
        for (int k = w.k0; k < w.k1; ++k, ++it) {
          const int seg = k >= steps ? 1 : 0;
          const CUtensorMap* am = (kRole == kWeightGrad ? half : seg) ? &a.a1 : &a.a0;
          const CUtensorMap* bm = (kRole == kForward ? (int)cr : kRole == kInputGrad ? seg : 0) ? &a.b1 : &a.b0;
          const int s = it % kStages;
          if (!mbar_wait(&empty[s], ((it / kStages) & 1) ^ 1, kDevErrEmptyBarrierTimeout)) {
            ok = false;
            break;
          }
          if (cr == 0) mbar_arrive_expect_tx(&full[s], 2 * kStageBytes);
          const uint32_t bar = mapa_shared(smem_u32(&full[s]), 0);
          const uint32_t sb = smem_u32(base + s * kStageBytes), sa = sb + kOperandBytes;
          const int kk = (k - seg * steps) * kStageK;
          if constexpr (kRole == kForward) {
            load_box(sb, bm, bar, kk, c0);
          } else {
            load_box(sb, bm, bar, c0, kk);
            load_box(sb + 8192, bm, bar, c0 + 64, kk);
          }
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            const uint32_t sab = sa + b * kOperandBytes;
            const int r = r0 + b * kBlockRows;
            if constexpr (kRole == kWeightGrad) {
              load_box(sab, am, bar, r, kk);
              load_box(sab + 8192, am, bar, r + 64, kk);
            } else {
              load_box(sab, am, bar, kk, r);
            }
          }
        }
      }
      if (!ok) {  // a wait gave up: let the copies in flight land before the memory is given back
        const unsigned long long t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) {
        }
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    pdl_wait();  // its waits are limited, and the stream's previous kernel is not
    if (cr == 0) {
      constexpr uint32_t kId = instruction_desc<T, kRole>();
      constexpr uint64_t kStepA = kRole == kWeightGrad ? 128 : 2, kStepB = kRole == kForward ? 2 : 128;  // 16 of K
      // block b's share of a stage; k = 0 starts its accumulator
      auto multiply = [&](int s, int b, int acc, int k) {
        const uint32_t sb = smem_u32(base + s * kStageBytes), sa = sb + (1 + b) * kOperandBytes;
        const uint64_t ad = kRole == kWeightGrad ? mn_desc(sa) : tc::sw128_desc(sa);
        const uint64_t bd = kRole == kForward ? tc::sw128_desc(sb) : mn_desc(sb);
#pragma unroll
        for (int q = 0; q < kStageK / 16; ++q)
          tc::umma_f16<2>(tmem + acc * kTileCols, ad + q * kStepA, bd + q * kStepB, kId, (k | q) != 0);
      };
      auto commit = [&](uint64_t* bar) {
        tc::umma_commit<2>(bar, 0);
        tc::umma_commit<2>(bar, 1);
      };
      auto loaded = [&](uint32_t it) {
        if (!mbar_wait(&full[it % kStages], (it / kStages) & 1, kDevErrFullBarrierTimeout)) return false;
        tc::tc_fence_after();
        return true;
      };
      uint32_t it = 0;
      int n = 0;
      for (int u = pair; u < units && ok; u += pairs, ++n) {
        const Unit w = unit_at(a, u, stages);
        const int total = w.k1 - w.k0;
        int k = 0;
        if constexpr (kBlocks == 2) {
          // the first stages: the first block as soon as its accumulator is free, then the second
          const int ahead = total < kStages ? total : kStages;
          ok = mbar_wait(&acc_empty[0], (n & 1) ^ 1, kDevErrMmaBarrierTimeout);
          tc::tc_fence_after();
          for (int q = 0; q < ahead && ok; ++q) {
            ok = loaded(it + q);
            if (ok && lane == 0) {
              multiply((it + q) % kStages, 0, 0, q);
              if (q == total - 1) commit(&acc_full[0]);
            }
            __syncwarp();
          }
          ok = ok && mbar_wait(&acc_empty[1], (n & 1) ^ 1, kDevErrMmaBarrierTimeout);
          if (!ok) break;
          tc::tc_fence_after();
          for (; k < ahead; ++k, ++it) {
            if (lane == 0) {
              multiply(it % kStages, 1, 1, k);
              commit(&empty[it % kStages]);
              if (k == total - 1) commit(&acc_full[1]);
            }
            __syncwarp();
          }
        } else if (!mbar_wait(&acc_empty[n & 1], ((n >> 1) & 1) ^ 1, kDevErrMmaBarrierTimeout)) {
          ok = false;
          break;
        } else {
          tc::tc_fence_after();
        }
        for (; k < total; ++k, ++it) {
          if (!loaded(it)) {
            ok = false;
            break;
          }
          if (lane == 0) {
            const int s = it % kStages;
            const bool last = k == total - 1;
            multiply(s, 0, kBlocks == 2 ? 0 : n & 1, k);
            if (last) commit(&acc_full[kBlocks == 2 ? 0 : n & 1]);
            if constexpr (kBlocks == 2) {
              multiply(s, 1, 1, k);
              if (last) commit(&acc_full[1]);
            }
            commit(&empty[s]);
          }
          __syncwarp();
        }
      }
      if (lane == 0) commit(drain);
      __syncwarp();
    }
    // CTA 1's warp comes here at once and waits as long as the kernel runs
    if (!mbar_wait_for(drain, 0, kDevErrMmaBarrierTimeout, a.wait_ns)) ok = false;
  } else {
    const int quadrant = warp & 3, side = warp >> 2;  // 32 TMEM lanes; which half of the columns
    pdl_wait();
    int n = 0;
    for (int u = pair; u < units && ok; u += pairs, ++n) {
      const Unit w = unit_at(a, u, stages);
      int i, j;
      tile_at(a, w.tile, i, j);
      const int half = kRole == kWeightGrad && i >= a.tiles_half;
      const int row0 = (half ? i - a.tiles_half : i) * (kBlocks * kBlockRows) + (int)cr * 128 + quadrant * 32 + lane;
#pragma unroll 1
      for (int b = 0; b < kBlocks; ++b) {
        const int acc = kBlocks == 2 ? b : n & 1;
        const int row = row0 + b * kBlockRows;
        if (!mbar_wait_for(&acc_full[acc], (kBlocks == 2 ? n : n >> 1) & 1, kDevErrEpilogueBarrierTimeout, a.wait_ns)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        // this thread's columns: forward, 64 features of the gate and the same of the up projection
        const uint32_t d = tmem + ((uint32_t)(quadrant * 32) << 16) + acc * kTileCols;
        constexpr int kSide = kRole == kForward ? 64 : 128, kThird = kRole == kForward ? 128 : 64;
        uint32_t v[4][32];
        tc::tmem_ld32_nowait(d + side * kSide, v[0]);
        tc::tmem_ld32_nowait(d + side * kSide + 32, v[1]);
        tc::tmem_ld32_nowait(d + side * kSide + kThird, v[2]);
        tc::tmem_ld32_nowait(d + side * kSide + kThird + 32, v[3]);
        tc::tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 4; ++q) tc::tmem_landed(v[q]);
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(&acc_empty[acc], 0);
        if (w.part >= 0) {
          // this warp's values of part p of the tile: 32 groups of four per lane
          const int place = ((w.tile - a.whole) * 2 + (int)cr) * kBlocks * 8 + b * 8 + warp;
          const long long part_size = (long long)a.cut * 2 * kBlocks * 8 * 4096;
          float* region = a.partial + (long long)place * 4096 + lane * 4;
          float* mine = region + w.part * part_size;
#pragma unroll
          for (int g = 0; g < 32; ++g) {
            const uint32_t* x = &v[g / 8][g % 8 * 4];
            st_global_v4(mine + g * 128, x[0], x[1], x[2], x[3]);
          }
          __threadfence();
          __syncwarp();
          int before = 0;
          if (lane == 0) before = atomicAdd(&a.counters[place], 1);
          if (__shfl_sync(0xFFFFFFFFu, before, 0) != a.parts - 1) continue;
          __threadfence();
          if (lane == 0) a.counters[place] = 0;
          // The parts come through this warp's 16 KB of the stages' memory, which is free: a pair's cut tile is the
          // last thing it does, and its loads and MMAs (the second block's too) are done. Two parts: the other one is
          // added to the registers (a sum of two has no order). More: all of them, from the first on.
          if (kBlocks == 2 && b == 0 &&
              !mbar_wait_for(&acc_full[1], n & 1, kDevErrEpilogueBarrierTimeout, a.wait_ns)) {
            ok = false;
            break;
          }
          const bool two = a.parts == 2;
          uint8_t* buf = base + warp * 16384 + lane * 16;
          if (!two) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int e = 0; e < 32; ++e) v[q][e] = 0u;
          }
#pragma unroll 1
          for (int p = two ? 1 - w.part : 0; p < (two ? 2 - w.part : a.parts); ++p) {
            const float* theirs = region + p * part_size;
#pragma unroll
            for (int g = 0; g < 32; ++g) cp_async_16(buf + g * 512, theirs + g * 128, 16);
            asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
            for (int g = 0; g < 32; ++g) {
              const uint4 x = lds128(smem_u32(buf) + g * 512);
              uint32_t* to = &v[g / 8][g % 8 * 4];
              to[0] = __float_as_uint(__uint_as_float(to[0]) + __uint_as_float(x.x));
              to[1] = __float_as_uint(__uint_as_float(to[1]) + __uint_as_float(x.y));
              to[2] = __float_as_uint(__uint_as_float(to[2]) + __uint_as_float(x.z));
              to[3] = __float_as_uint(__uint_as_float(to[3]) + __uint_as_float(x.w));
            }
          }
        }
        if constexpr (kRole == kForward) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int col = j * 128 + side * 64 + 32 * q;
            if (col >= a.cols) break;
            if (a.bias0 != nullptr || a.bias1 != nullptr) {
              float bg = 0.0f, bu = 0.0f;
              if (a.bias0 != nullptr && col + lane < a.cols) bg = to_f32<T>(static_cast<const T*>(a.bias0)[col + lane]);
              if (a.bias1 != nullptr && col + lane < a.cols) bu = to_f32<T>(static_cast<const T*>(a.bias1)[col + lane]);
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                v[q][e] = __float_as_uint(__uint_as_float(v[q][e]) + __shfl_sync(0xFFFFFFFFu, bg, e));
                v[q + 2][e] = __float_as_uint(__uint_as_float(v[q + 2][e]) + __shfl_sync(0xFFFFFFFFu, bu, e));
              }
            }
            if (row < a.rows) {
              if (a.save != nullptr) {
                store_row<float>(a.save + (long long)row * a.cols, col, a.cols, a.wide, v[q]);
                store_row<float>(a.save + ((long long)a.rows + row) * a.cols, col, a.cols, a.wide, v[q + 2]);
              }
#pragma unroll
              for (int e = 0; e < 32; ++e)
                v[q][e] = __float_as_uint(activation<kAct>(__uint_as_float(v[q][e])) * __uint_as_float(v[q + 2][e]));
              store_row<T>(static_cast<T*>(a.out0) + row * a.ld, col, a.cols, a.wide, v[q]);
            }
          }
        } else if (row < a.rows) {
          T* out = static_cast<T*>(half ? a.out1 : a.out0) + row * a.ld;
#pragma unroll
          for (int q = 0; q < 4; ++q) store_row<T>(out, j * kTileCols + side * 128 + 32 * q, a.cols, a.wide, v[q]);
        }
      }
    }
  }
  if (!ok) mirror_device_error(a.status_host);
  tc::tc_fence_before();
  cluster_sync_all();  // no CTA leaves while its peer may still signal its barriers
  tc::tc_fence_after();
  if (warp == kMmaWarp) tc::tmem_dealloc<2>(tmem, 512);
}

// Limits of a launch whose pairs take `units` tiles each of `stages` along the contraction. A wait for one stage has the
// usual limit. A wait for a whole contraction, or for the kernel's last MMA, may rightly take longer: it has 4 us a stage
// (one takes 0.4 to 1 us) and 0.1 ms a tile besides. A pipeline that is stuck ends earlier all the same, by the stage's
// limit: every wait ends once one of them has given up. A launch of more than some 25 ms does not let the stream's next
// kernel in early, whose own waits would count the rest of this one.
static void set_limits(TcArgs& a, long long units, long long stages) {
  const unsigned long long longest = (unsigned long long)units * (4000ull * (unsigned long long)stages + 100000ull);
  a.wait_ns = kWaitTimeoutNs + longest;
  a.overlap = longest < 100000000ull;
}

template <typename T, int kRole, int kAct, int kBlocks>
static int launch_pair_blocks(TcArgs& a, cudaStream_t st, int sms) {
  constexpr int kSmemBytes = Ring<kBlocks>::kSmemBytes;
  auto kern = pair_kernel<T, kRole, kAct, kBlocks>;
  static int pairs_at_once[64] = {0};  // per device; every thread writes the same value
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return set_error(GFX_ERR_CUDA, "gated pair_kernel: no current device");
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (pairs_at_once[dev] == 0) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    int n = 0;
    cfg.gridDim = dim3(sms / 2 * 2);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
    if (e != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      return set_error(GFX_ERR_CUDA, "gated pair_kernel: no CTA pair fits the GPU: %s", cudaGetErrorString(e));
    }
    pairs_at_once[dev] = n < sms / 2 ? n : sms / 2;
  }
  // a pair takes at most one part of a cut tile (it uses the stages' memory to join them)
  if (a.cut * a.parts > pairs_at_once[dev]) a.parts = 1;
  const int units = a.whole + a.cut * a.parts;
  const int pairs = units < pairs_at_once[dev] ? units : pairs_at_once[dev];
  const long long steps = (a.depth + kStageK - 1) / kStageK;
  set_limits(a, (units + pairs - 1) / pairs, kRole == kInputGrad ? 2 * steps : steps);
  cfg.gridDim = dim3(2 * pairs);
  a.status_host = host_status_word(dev);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) return set_error(GFX_ERR_CUDA, "gated pair_kernel launch: %s", cudaGetErrorString(e));
  return check_launch("gated pair_kernel");
}

struct Plan {
  int blocks, tiles_half, whole, cut, parts;
  size_t partial_bytes() const { return parts > 1 ? (size_t)cut * parts * 2 * blocks * 8 * 4096 * sizeof(float) : 0; }
};

// Row blocks a tile, and the cut of the last wave, by the cycles that they take: a stage of 64 along the contraction
// is 780 cycles with one row block and 1150 with two (measured: 66% and 89% of the tensor cores' rate); joining the
// parts of a tile takes some 6000 a block for the exchange and 3000 for each part that is read. `rows` in `halves` (dW: both weights'), `stages` along the contraction.
static Plan make_plan(long long rows, int halves, int tiles_j, int stages, bool may_cut, int sms) {
  const int pairs = sms / 2;
  Plan best{};
  double least = 0.0;
  for (int blocks = 1; blocks <= 2; ++blocks) {
    const int half = (int)((rows + blocks * kBlockRows - 1) / (blocks * kBlockRows));
    const int tiles = half * halves * tiles_j, rest = tiles % pairs;
    const double wave = (double)stages * (blocks == 1 ? 780 : 1150);
    for (int parts = 1; parts <= 8; ++parts) {
      if (parts > 1 && (!may_cut || rest == 0 || rest * parts > pairs || stages / parts < 4)) break;
      const double t = tiles / pairs * wave + (rest ? wave / parts : 0.0) + (parts > 1 ? (6000.0 + 3000.0 * (parts == 2 ? 1 : parts)) * blocks : 0.0);
      if (best.blocks == 0 || t < least) {
        least = t;
        best = Plan{blocks, half, tiles - rest, rest, parts};
      }
    }
  }
  return best;
}

// workspace: the counters' region and then plan.partial_bytes(); null: no tile is cut.
template <typename T, int kRole, int kAct>
static int launch_pair(TcArgs& a, int halves, int stages, void* workspace, cudaStream_t st, int sms) {
  const Plan p = make_plan(a.rows, halves, a.tiles_j, stages, workspace != nullptr, sms);
  a.tiles_half = p.tiles_half;
  a.tiles_i = p.tiles_half * halves;
  a.whole = p.whole, a.cut = p.cut, a.parts = p.parts;
  a.counters = static_cast<int*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + kSplitKCounterBytes);
  return p.blocks == 2 ? launch_pair_blocks<T, kRole, kAct, 2>(a, st, sms)
                       : launch_pair_blocks<T, kRole, kAct, 1>(a, st, sms);
}

static int stages_of(int depth) { return (depth + kStageK - 1) / kStageK; }

template <typename T>
constexpr CUtensorMapDataType map_type() {
  return std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// Boxes of 64 (inner) x `outer_box`, 128-byte swizzle.
template <typename T>
static int box_map(CUtensorMap* m, const void* p, long long inner, long long outer, long long ld, int outer_box) {
  return make_tmap_2d(m, map_type<T>(), p, (uint64_t)inner, (uint64_t)outer, (uint64_t)ld * 2, 64, outer_box,
                      CU_TENSOR_MAP_SWIZZLE_128B);
}

static bool rows32(const void* p, long long ld) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0 && ld % 16 == 0; }

template <typename T>
static int forward_tc(const GatedArgs& g, int act, void* h, float* save, void* workspace, cudaStream_t st,
                      int sms) {
  TcArgs a;
  memset(&a, 0, sizeof(a));
  int rc;
  if ((rc = box_map<T>(&a.a0, g.x, g.K, g.M, g.ldx, 128)) || (rc = box_map<T>(&a.b0, g.w_gate, g.K, g.F, g.ldg, 128)) ||
      (rc = box_map<T>(&a.b1, g.w_up, g.K, g.F, g.ldu, 128)))
    return rc;
  a.rows = g.M, a.cols = g.F, a.depth = g.K;
  a.tiles_j = (g.F + 127) / 128;
  a.panel = 16, a.i_fast = 1;
  a.out0 = h, a.ld = g.F, a.bias0 = g.b_gate, a.bias1 = g.b_up, a.save = save;
  a.wide = rows32(h, g.F) && (reinterpret_cast<uintptr_t>(save) & 31) == 0;
  if (act == kSilu) return launch_pair<T, kForward, kSilu>(a, 1, stages_of(g.K), workspace, st, sms);
  if (act == kGelu) return launch_pair<T, kForward, kGelu>(a, 1, stages_of(g.K), workspace, st, sms);
  return launch_pair<T, kForward, kGeluTanh>(a, 1, stages_of(g.K), workspace, st, sms);
}

// dx [M, K] from dgu [M, 2F]
template <typename T>
static int input_grad_tc(const GatedArgs& g, const void* dgu, void* dx, void* workspace, cudaStream_t st, int sms) {
  TcArgs a;
  memset(&a, 0, sizeof(a));
  const T* d = static_cast<const T*>(dgu);
  int rc;
  if ((rc = box_map<T>(&a.a0, d, g.F, g.M, 2ll * g.F, 128)) || (rc = box_map<T>(&a.a1, d + g.F, g.F, g.M, 2ll * g.F, 128)) ||
      (rc = box_map<T>(&a.b0, g.w_gate, g.K, g.F, g.ldg, 64)) || (rc = box_map<T>(&a.b1, g.w_up, g.K, g.F, g.ldu, 64)))
    return rc;
  a.rows = g.M, a.cols = g.K, a.depth = g.F;
  a.tiles_j = (g.K + 255) / 256;
  a.panel = 16, a.i_fast = 1;
  a.out0 = dx, a.ld = g.K;
  a.wide = rows32(dx, g.K);
  return launch_pair<T, kInputGrad, kSilu>(a, 1, 2 * stages_of(g.F), workspace, st, sms);
}

// dWg, dWu [F, K]: both, or one of them
template <typename T>
static int weight_grad_tc(const GatedArgs& g, const void* dgu, void* dwg, void* dwu, void* workspace,
                          cudaStream_t st, int sms) {
  TcArgs a;
  memset(&a, 0, sizeof(a));
  const T* d = static_cast<const T*>(dgu);
  const T* d0 = dwg ? d : d + g.F;  // one weight wanted alone is the first half, and there is no second
  int rc;
  if ((rc = box_map<T>(&a.a0, d0, g.F, g.M, 2ll * g.F, 64)) || (rc = box_map<T>(&a.a1, d + g.F, g.F, g.M, 2ll * g.F, 64)) ||
      (rc = box_map<T>(&a.b0, g.x, g.K, g.M, g.ldx, 64)))
    return rc;
  a.rows = g.F, a.cols = g.K, a.depth = g.M;
  a.tiles_j = (g.K + 255) / 256;
  a.panel = 16, a.i_fast = 0;
  a.out0 = dwg ? dwg : dwu, a.out1 = dwu, a.ld = g.K;
  a.wide = rows32(a.out0, g.K) && rows32(a.out1, g.K);
  return launch_pair<T, kWeightGrad, kSilu>(a, dwg && dwu ? 2 : 1, stages_of(g.M), workspace, st, sms);
}

}  // namespace gated

size_t gated_forward_tc_workspace(int M, int K, int F, int sms) {
  const size_t n = gated::make_plan(M, 1, (F + 127) / 128, gated::stages_of(K), true, sms).partial_bytes();
  return n ? kSplitKCounterBytes + n : 0;
}

size_t gated_backward_tc_workspace(int M, int K, int F, int sms) {
  using namespace gated;
  const int tiles_j = (K + 255) / 256;
  size_t n = make_plan(M, 1, tiles_j, 2 * stages_of(F), true, sms).partial_bytes();
  for (int halves = 1; halves <= 2; ++halves) {
    const size_t w = make_plan(F, halves, tiles_j, stages_of(M), true, sms).partial_bytes();
    n = w > n ? w : n;
  }
  return kSplitKCounterBytes + n;
}

int launch_gated_forward_tc(const GatedArgs& a, int dtype, int act, void* h, float* save, void* workspace,
                            cudaStream_t st, int sms) {
  return dtype == GFX_DTYPE_F16 ? gated::forward_tc<__half>(a, act, h, save, workspace, st, sms)
                                : gated::forward_tc<__nv_bfloat16>(a, act, h, save, workspace, st, sms);
}

int launch_gated_input_grad(const GatedArgs& a, int dtype, const void* dgu, void* dx, void* workspace, cudaStream_t st,
                            int sms) {
  return dtype == GFX_DTYPE_F16 ? gated::input_grad_tc<__half>(a, dgu, dx, workspace, st, sms)
                                : gated::input_grad_tc<__nv_bfloat16>(a, dgu, dx, workspace, st, sms);
}

int launch_gated_weight_grad(const GatedArgs& a, int dtype, const void* dgu, void* dwg, void* dwu, void* workspace,
                             cudaStream_t st, int sms) {
  return dtype == GFX_DTYPE_F16 ? gated::weight_grad_tc<__half>(a, dgu, dwg, dwu, workspace, st, sms)
                                : gated::weight_grad_tc<__nv_bfloat16>(a, dgu, dwg, dwu, workspace, st, sms);
}

}  // namespace gfx
