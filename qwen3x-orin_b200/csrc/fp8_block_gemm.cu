// The projection of E4M3 activations with E4M3 weights, both with one FP32 scale per block of 128:
//   out[t, n] = bf16( sum over blocks b of sa[b, t] * sw[n / 128, b] * (sum over k in b of a[t, k] * w[n, k]) )
// sa [ceil(K / 128), T] as the quantisers of fp8_block.cu write it, sw [ceil(N / 128), ceil(K / 128)].  A block's products
// are summed in FP32 by the tensor cores, multiplied by the two scales and added to the running FP32 sum; the one rounding
// is to bf16.  The scales are multiplied with each other first, once per token and block, so that an output costs one fused
// multiply and add per block (the additions set the pace of some tiles, see below); the price is that a product of
// scales outside FP32's range is lost even where the sum would have brought it back.
//
// Three kernels on tcgen05 (kind::f8f6f4: E4M3 x E4M3 -> FP32 in tensor memory), operands fetched by bulk tensor copies
// into rings of 128-byte-swizzled stages, one stage per block of 128 columns of K:
//   * strip: 128 outputs are the MMA's rows, 16 to 128 tokens its columns, K is split over a cluster; for few tokens,
//     bound by reading the weights;
//   * panel: 128 tokens are the rows, 128 outputs the columns, one CTA per tile; bound by how evenly the tiles fill the SMs;
//   * pair:  256 tokens x 256 (or 160) outputs on two SMs at once; for many tokens, bound by the tensor cores and their power.
// The hardware's accumulator cannot be scaled between two blocks of K, so every block starts a fresh accumulator and the
// scaled sum lives in registers: accumulators take turns, and while the tensor cores fill the others, the adding warps read
// one and add it, times its scales, to their FP32 sums.  (A thread's sums stay with one warp for the whole of K: no order of
// additions depends on timing.)
//
// Waits are bounded; one that runs out raises a sticky word (q3x_b200_fp8_block_gemm_error), and the CTA drains its
// copies, frees its tensor memory and returns.
#include <cuda.h>

#include "device_utils.cuh"
#include "host_checks.hpp"
#include "q3x_b200.h"
#include "tcgen05.cuh"

namespace q3x {
namespace {

using namespace tcgen05;

constexpr int kBlockK = Q3X_B200_FP8_BLOCK;  // 128 codes = one swizzled row of 128 bytes
constexpr int kRowBytes = kBlockK;

__device__ unsigned int g_error;

// One block's product: D[128, n] = A[128, 128] B[n, 128]^T, four instructions of 32 columns of K.
__device__ __forceinline__ void block_product(uint32_t accumulator, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
  for (int step = 0; step < kBlockK / 32; ++step)
    mma_e4m3(accumulator, operand_descriptor(a + step * 32), operand_descriptor(b + step * 32), idesc, step > 0 ? 1u : 0u);
}

// The cluster: a barrier of all its threads in two parts, a rank's copy of an address, and an arrival on a rank's copy of a
// barrier.  They do not publish memory to the cluster, which would cost a fence of a thousand cycles: they hand on barriers
// and tensor memory, which have fences of their own, or say that values have been read.  (Both instructions want the whole
// warp at once, and are reached from branches that one lane takes.)
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(uint32_t address, int rank) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(address), "r"(rank));
  return there;
}
__device__ __forceinline__ void arrive_remote(uint32_t there) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(there) : "memory");
}
// Four floats into another CTA's shared memory; their bytes complete on a barrier of that CTA.
__device__ __forceinline__ void push(uint32_t there, const float4& v, uint32_t barrier_there) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(there),
               "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(barrier_there)
               : "memory");
}
__device__ __forceinline__ float4 add4(const float4& a, const float4& b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
// One FP32 from global to shared memory; the lane's copies so far arrive on the barrier, which counts on that arrival,
// when they have landed; and the wait for them at the end.
__device__ __forceinline__ void copy_scale(uint32_t to, const float* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint32_t barrier) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(barrier) : "memory");
}
__device__ __forceinline__ float load_shared(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// A bounded wait of a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool wait_warp(uint32_t barrier, uint32_t parity) {
  return __all_sync(kFullMask, barrier_try(barrier, parity)) || __all_sync(kFullMask, wait_bounded(barrier, parity));
}
__device__ __forceinline__ void block_product_pair(uint32_t accumulator, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
  for (int step = 0; step < kBlockK / 32; ++step)
    mma_e4m3_pair(accumulator, operand_descriptor(a + step * 32), operand_descriptor(b + step * 32), idesc, step > 0 ? 1u : 0u);
}

__device__ __forceinline__ uint32_t shared_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ------------------------------------------------------------------------------------------------------------- panel
namespace panel {

// Tiles of 128 tokens x 128 outputs, one CTA each: for products with too few tiles of 256 x 256 to give every pair of SMs
// one.  A block's product takes 256 cycles of the tensor cores, but its 32 KB come at 64 bytes per cycle at most, in 512:
// that bounds it (4096 x 10240 x 5120: 65 bytes per cycle and SM leave L2, the tensor pipe is active for 51 % of the time), and
// is why pairs take over as soon as they fill the GPU.  200 x 5120 x 17408: 40.0 us (pairs 45.7), 777 x 5120 x 6144: 32.2 us
// (34.9).
constexpr int kRows = 128;                  // tokens of a tile
constexpr int kCols = 128;                  // outputs of a tile
constexpr int kThreads = 384;               // warp 0 fetches codes, 2 scales, 1 and 3 issue, 4 to 11 add up
constexpr int kAdders = 8;                  // warps: 4 lane quarters x 2 halves of the outputs
constexpr int kMine = kCols / 2;            // outputs of one adding warp
constexpr int kLaunchRegisters = 168;       // 65536 / 384, rounded down to 8
constexpr int kBand = 16;                   // token tiles walked together
constexpr int kBuffers = 4;                 // accumulators, one block of K after the other
constexpr int kStageBytes = (kRows + kCols) * kRowBytes;
constexpr int kStages = 6;
constexpr int kSlots = 16;                  // of scales, one per block in flight
constexpr int kSlotFloats = kRows + 4;      // the tokens', the weight block's, 3 unused
constexpr int kStore = kStages * kStageBytes;                  // [adder][32 rows][32 outputs] bf16
constexpr int kScales = kStore + kAdders * 32 * 64;
constexpr int kBarriers = kScales + kSlots * kSlotFloats * 4;
constexpr int kTmemSlot = kBarriers + 8 * (2 * kStages + 2 * kBuffers);
constexpr int kShared = kTmemSlot + 16;
static_assert(kStages + kBuffers <= kSlots, "see the warp that fetches scales");
static_assert(kShared <= 232448, "shared memory of one CTA");

__global__ void __launch_bounds__(kThreads, 1)
    block_gemm_panel_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                            const float* __restrict__ sa, const float* __restrict__ sw, int tokens, int out_features,
                            int blocks, int row_tiles, int col_tiles, uint16_t* __restrict__ out) {
  extern __shared__ __align__(1024) uint8_t shared[];
  const uint32_t base = shared_address(shared);
  const uint32_t full = base + kBarriers, empty = full + 8 * kStages, filled = empty + 8 * kStages,
                 drained = filled + 8 * kBuffers;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(shared + kTmemSlot);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = row_tiles * col_tiles;

  if (threadIdx.x == 0) {
    prefetch_map(&map_a);
    prefetch_map(&map_w);
    for (int s = 0; s < kStages; ++s) {
      barrier_init(full + 8 * s, 1 + 32);  // the codes' fetcher and every lane of the scales'
      barrier_init(empty + 8 * s, 1);
    }
    for (int i = 0; i < kBuffers; ++i) {
      barrier_init(filled + 8 * i, 1);
      barrier_init(drained + 8 * i, kAdders);
    }
    barrier_init_fence();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + kTmemSlot), "r"(kBuffers * kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  // only now: a successor that took this SM's tensor memory first would wait for this kernel and this kernel for it
  release_next_kernel();
  wait_for_prior_kernels();

  // tile -> (token tile, output tile): bands of kBand token tiles, output tiles one after the other within a band, so that
  // the tiles in flight share their operands in L2
  auto tile_at = [&](int tile, int& row_tile, int& col_tile) {
    const int band = tile / (kBand * col_tiles), first = band * kBand;
    const int height = min(kBand, row_tiles - first), rest = tile - first * col_tiles;
    col_tile = rest / height;
    row_tile = first + rest % height;
  };

  bool healthy = true;
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      int step = 0;
      for (int tile = blockIdx.x; tile < tiles && healthy; tile += gridDim.x) {
        int row_tile, col_tile;
        tile_at(tile, row_tile, col_tile);
        for (int b = 0; b < blocks; ++b, ++step) {
          const int s = step % kStages;
          if (step >= kStages && !(healthy = wait_warp(empty + 8 * s, (step / kStages - 1) & 1))) break;
          const uint32_t at = base + s * kStageBytes;
          if (elect_one()) {
            barrier_expect(full + 8 * s, kStageBytes);
            load_box(at, &map_a, b * kBlockK, row_tile * kRows, full + 8 * s);
            load_box(at + kRows * kRowBytes, &map_w, b * kBlockK, col_tile * kCols, full + 8 * s);
          }
        }
      }
      // no copy is in flight when the CTA ends, whatever became of its readers
      for (int last = max(0, step - kStages); last < step; ++last)
        if (!wait_warp(full + 8 * (last % kStages), (last / kStages) & 1)) healthy = false;
    } else if (warp == 2) {
      // The scales of a block, copied without passing through registers (a load held in one for two blocks was measured to
      // hold up the whole warp wherever the compiler moved it).  A slot is free again: when step
      // t - kStages has left its stage, its accumulator had come round, so step t - kStages - kBuffers was drained, its scales
      // and all older ones read; slot t % kSlots holds a step at least that old.
      int step = 0;
      for (int tile = blockIdx.x; tile < tiles && healthy; tile += gridDim.x) {
        int row_tile, col_tile;
        tile_at(tile, row_tile, col_tile);
        const float* rows = sa + row_tile * kRows;
        const int visible = min(kRows, tokens - row_tile * kRows);
        const float* weight = sw + static_cast<size_t>(col_tile) * blocks;
        for (int b = 0; b < blocks; ++b, ++step) {
          const int s = step % kStages;
          if (step >= kStages && !(healthy = wait_warp(empty + 8 * s, (step / kStages - 1) & 1))) break;
          const uint32_t slot = base + kScales + (step % kSlots) * kSlotFloats * 4;
#pragma unroll
          for (int i = 0; i < kRows; i += 32) copy_scale(slot + (i + lane) * 4, rows + min(i + lane, visible - 1));
          if (lane == 0) copy_scale(slot + kRows * 4, weight + b);
          copies_arrive(full + 8 * s);
          rows += tokens;
        }
      }
      copies_wait();
    } else {
      // Warp 1 issues the even steps, warp 3 the odd ones.  A warp's instructions wait in line behind its own products, so
      // one warp alone would test the next barriers only once its products are in the pipe, and the pipe would run dry
      // for the time of those tests.
      const int steps = (tiles - static_cast<int>(blockIdx.x) + gridDim.x - 1) / gridDim.x * blocks;
      int step = warp >> 1;
      for (; step < steps; step += 2) {
        const int s = step % kStages, buffer = step % kBuffers, round = step / kBuffers;
        if (!(healthy = wait_warp(full + 8 * s, (step / kStages) & 1))) break;
        if (round > 0 && !(healthy = wait_warp(drained + 8 * buffer, (round - 1) & 1))) break;
        fence_after_sync();
        const uint32_t at = base + s * kStageBytes;
        if (elect_one()) {
          block_product(tmem + buffer * kCols, at, at + kRows * kRowBytes, instruction_descriptor_e4m3(kCols));
          commit(filled + 8 * buffer);
          commit(empty + 8 * s);
        }
        __syncwarp();
      }
      // (products complete in order: after this warp's last one none of them is reading shared memory)
      if (step >= 2 && !wait_warp(filled + 8 * ((step - 2) % kBuffers), ((step - 2) / kBuffers) & 1)) healthy = false;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int quarter = warp & 3, half_cols = (warp - 4) >> 2;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half_cols * kMine;
    uint8_t* store = shared + kStore + (warp - 4) * 32 * 64;
    const uint32_t row_scale = base + kScales + (quarter * 32 + lane) * 4, col_scale = base + kScales + kRows * 4;
    int step = 0;
    for (int tile = blockIdx.x; tile < tiles && healthy; tile += gridDim.x) {
      float sum[kMine];
#pragma unroll
      for (int i = 0; i < kMine; ++i) sum[i] = 0.0f;
      for (int b = 0; b < blocks; ++b, ++step) {
        if (!(healthy = wait_warp(filled + 8 * (step % kBuffers), (step / kBuffers) & 1))) break;
        fence_after_sync();
        // the block's accumulator, 32 columns at a time and the next 32 on their way meanwhile, times its scales
        const uint32_t columns = lane_base + step % kBuffers * kCols;
        uint32_t d[2][32];
        load32(columns, d[0]);
        const float scale = __fmul_rn(load_shared(row_scale + step % kSlots * (kSlotFloats * 4)),
                                      load_shared(col_scale + step % kSlots * (kSlotFloats * 4)));
#pragma unroll
        for (int g = 0; g < kMine / 32; ++g) {
          wait_loads(d[g & 1]);
          if (g + 1 < kMine / 32) {
            load32(columns + (g + 1) * 32, d[(g + 1) & 1]);
          } else {
            fence_before_sync();
            __syncwarp();
            if (lane == 0) barrier_arrive(drained + 8 * (step % kBuffers));
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 r = fma2(make_float2(scale, scale),
                                  make_float2(__uint_as_float(d[g & 1][i]), __uint_as_float(d[g & 1][i + 1])),
                                  make_float2(sum[g * 32 + i], sum[g * 32 + i + 1]));
            sum[g * 32 + i] = r.x;
            sum[g * 32 + i + 1] = r.y;
          }
        }
      }
      if (!healthy) break;
      int row_tile, col_tile;
      tile_at(tile, row_tile, col_tile);
      const int row0 = row_tile * kRows + quarter * 32, col0 = col_tile * kCols + half_cols * kMine;
      // 32 rows x 32 outputs at a time through the warp's own 2 KB, so that a store covers whole 64-byte pieces of eight
      // rows (16-byte parts permuted by the row: free of bank conflicts both ways)
#pragma unroll
      for (int g = 0; g < kMine / 32; ++g) {
#pragma unroll
        for (int part = 0; part < 4; ++part) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = sum[g * 32 + part * 8 + e];
          st_vec(store + lane * 64 + ((part ^ ((lane >> 1) & 3)) << 4), pack8(v));
        }
        __syncwarp();
        const int col = col0 + g * 32 + (lane & 3) * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 8 + (lane >> 2), t = row0 + r;
          const uint4 v = ld_vec(store + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
          if (t < tokens && col < out_features) st_vec(out + static_cast<size_t>(t) * out_features + col, v);
        }
        __syncwarp();
      }
    }
  }
  if (!healthy) atomicExch(&g_error, 1u);
  __syncwarp();
  fence_before_sync();
  __syncthreads();
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kBuffers * kCols) : "memory");
}

}  // namespace panel

// -------------------------------------------------------------------------------------------------------------- pair
namespace pair {

// Two CTAs share one tile of 256 tokens x 256 outputs: each holds its 128 tokens' codes and accumulators and HALF of the
// weights' codes, and one tensor instruction runs on both SMs (cta_group::2).  Against two tiles of 128 x 256 every SM
// fetches 32 KB instead of 48 KB per block of K, and an instruction of 128 columns reads 6 KB of shared memory instead
// of 8 in its 64 cycles, which is what lets the accumulators be four of 128 columns: each half of the outputs has two, and
// a half is read while three other products run.  8192 x 34816 x 5120: 1.12 to 1.16 ms from a cool start (2.5 to 2.6 PFLOP/s
// of the 3.3 that twice the measured bf16 rate makes), 1.31 to 1.35 ms in a long run, where the GPU holds its clocks down for
// power.
//
// Tiles of 256 tokens x 160 outputs are for products whose tiles of 256 x 256 would leave many SMs idle in their last (or
// only) round.  Their block is one product of all outputs, with three accumulators; their border between two weight blocks
// can lie anywhere.  256 x 10240 x 5120: 17.6 us (256 outputs 20.3, panels 25.4), 512 x 10240 x 5120: 31.7 us (33.5, 36.4).
// A block takes 0.31 us with few SMs at work; with the additions left out 0.24, with three of four products left out too the
// same.  So fetching it, 26 KB per SM at 64 bytes per cycle, is the floor of 0.24 us, and the adding warps, which read an
// accumulator in three loads with a wait each before they give it back, cost the other 0.07.  (Tiles of 96 or 128 outputs:
// 0.28 us.)
constexpr int kRows = 128;                  // tokens of a CTA
constexpr int kThreads = 384;               // warp 0 fetches codes, 2 scales, 1 and 3 issue (leader), 4 to 11 add up
constexpr int kAdders = 8;                  // warps: 4 lane quarters x 2 halves of the outputs
constexpr int kLaunchRegisters = 168;       // 65536 / 384, rounded down to 8; the compiler spills a little all the same: 24 bytes
                                            // stored and 64 loaded with 256 outputs, 20 and 64 with 160
constexpr size_t kBandBytes = 36u << 20;    // of activations, see band_tiles_of
constexpr int kMostShared = 232448;         // shared memory of one CTA

template <int COLS>  // outputs of a tile
struct Shape {
  static constexpr int kProducts = COLS == 256 ? 2 : 1;          // per block; each has a range of the outputs
  static constexpr int kWide = COLS / kProducts;                 // outputs of a product
  static constexpr int kDepth = 512 / COLS;                      // accumulators per range of outputs
  static constexpr int kBuffers = kProducts * kDepth;
  static constexpr int kMine = COLS / 2;                         // outputs of one adding warp
  static constexpr int kBox = kMine % 64 == 0 ? 64 : 16;   // outputs of one store
  static constexpr bool kAligned = 128 % kMine == 0;             // a warp's outputs lie in one weight block
  static constexpr int kStageBytes = (kRows + COLS / 2) * kRowBytes;
  static constexpr int kSlots = COLS == 256 ? 5 : 7;             // of scales, one per block in flight
  static constexpr int kSlotBytes = (kRows + 4) * 4;             // the tokens', two weight blocks' for each half of the outputs
  static constexpr int kStoreBytes = kAdders * 32 * kMine * 2;   // [adder][box][32 rows][kBox outputs] bf16
  static constexpr int kStages = (kMostShared - kStoreBytes - kSlots * kSlotBytes - 384) / kStageBytes;
  static constexpr int kStore = kStages * kStageBytes;
  static constexpr int kScales = kStore + kStoreBytes;
  static constexpr int kBarriers = (kScales + kSlots * kSlotBytes + 31) / 32 * 32;  // (accumulators' first: see next_block)
  static constexpr int kTmemSlot = kBarriers + 8 * (2 * kStages + 2 * kBuffers + 2 * kSlots);
  static constexpr int kShared = kTmemSlot + 16;
  static_assert(COLS % 32 == 0 && kMine % kBox == 0 && kWide <= 256 && kBuffers * kWide <= 512 && kStageBytes % 1024 == 0);
  static_assert(kShared <= kMostShared);
  // (scales arrive on their stage's barrier: those of a block must not come before the stage's last block was complete)
  static_assert(kSlots <= kStages);
};

// Columns first to first + 31 of an adding warp's kMine (or the 16 that are left) into registers.
template <int kMine>
__device__ __forceinline__ void load_columns(uint32_t columns, int first, uint32_t (&d)[32]) {
  if (kMine % 32 == 0 || first + 32 <= kMine) load32(columns + first, d);
  else load16(columns + first, reinterpret_cast<uint32_t (&)[16]>(d));
}

template <int COLS>
__global__ void __launch_bounds__(kThreads, 1)
    block_gemm_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                           const __grid_constant__ CUtensorMap map_out, const float* __restrict__ sa,
                           const float* __restrict__ sw, int tokens, int out_features, int blocks, int row_tiles,
                           int col_tiles, int band_tiles) {
  using S = Shape<COLS>;
  constexpr int kStages = S::kStages, kBuffers = S::kBuffers, kSlots = S::kSlots, kProducts = S::kProducts, kWide = S::kWide;
  extern __shared__ __align__(1024) uint8_t shared[];
  const uint32_t base = shared_address(shared);
  const uint32_t filled = base + S::kBarriers, drained = filled + 8 * kBuffers, full = drained + 8 * kBuffers,
                 empty = full + 8 * kStages, scaled = empty + 8 * kStages, taken = scaled + 8 * kSlots;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(shared + S::kTmemSlot);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, tiles = row_tiles * col_tiles;

  if (threadIdx.x == 0) {
    prefetch_map(&map_a);
    prefetch_map(&map_w);
    prefetch_map(&map_out);
    for (int s = 0; s < kStages; ++s) {
      // (the leader's: both CTAs' codes complete on it; its own scales' lanes arrive, and the peer's warp 1 for its scales)
      barrier_init(full + 8 * s, 1 + 32 + 1);
      barrier_init(empty + 8 * s, kProducts);
    }
    for (int i = 0; i < kBuffers; ++i) {
      barrier_init(filled + 8 * i, 1);
      barrier_init(drained + 8 * i, 2 * kAdders / kProducts);  // (the leader's: the warps of both CTAs that read it)
    }
    for (int i = 0; i < kSlots; ++i) {
      barrier_init(scaled + 8 * i, 32);
      barrier_init(taken + 8 * i, kAdders);
    }
    barrier_init_fence();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + S::kTmemSlot), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  // only now: a successor that took this SM's tensor memory first would wait for this kernel and this kernel for it
  release_next_kernel();
  wait_for_prior_kernels();

  // tile -> (token tile, output tile): bands of band_tiles token tiles, output tiles one after the other within a band, so
  // that the tiles in flight share their operands in L2
  auto tile_at = [&](int tile, int& row_tile, int& col_tile) {
    const int band = tile / (band_tiles * col_tiles), first = band * band_tiles;
    const int height = min(band_tiles, row_tiles - first), rest = tile - first * col_tiles;
    col_tile = rest / height;
    row_tile = first + rest % height;
  };

  bool healthy = true;
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      const uint32_t leader_full = at_rank(full, 0);
      int step = 0;
      for (int tile = pair; tile < tiles && healthy; tile += pairs) {
        int row_tile, col_tile;
        tile_at(tile, row_tile, col_tile);
        const int row0 = (row_tile * 2 + rank) * kRows, col0 = col_tile * COLS + rank * (kWide / 2);
        for (int b = 0; b < blocks; ++b, ++step) {
          const int s = step % kStages;
          if (step >= kStages && !(healthy = wait_warp(empty + 8 * s, (step / kStages - 1) & 1))) break;
          const uint32_t at = base + s * S::kStageBytes;
          if (elect_one()) {
            if (rank == 0) barrier_expect(full + 8 * s, 2 * S::kStageBytes);
            load_box_pair(at, &map_a, b * kBlockK, row0, leader_full + 8 * s);
#pragma unroll
            for (int i = 0; i < kProducts; ++i)
              load_box_pair(at + (kRows + i * (kWide / 2)) * kRowBytes, &map_w, b * kBlockK, col0 + i * kWide, leader_full + 8 * s);
          }
        }
      }
      // No copy is in flight when the CTA ends: the leader sees its own and its peer's land.  (The peer ends when its adders
      // have their last product, which needs its copies, or after a wait of 200 ms that ran out long after its last copy.)
      if (rank == 0)
        for (int last = max(0, step - kStages); last < step; ++last)
          if (!wait_warp(full + 8 * (last % kStages), (last / kStages) & 1)) healthy = false;
    } else if (warp == 2) {
      // The scales of a block, copied without passing through registers (a load held in one for two blocks was measured to
      // hold up the whole warp wherever the compiler moved it).  Products wait for them, so that the adding warps need not.
      // A slot is free again when this CTA's adding warps have read it.  (Asking instead for the product that must have
      // followed that came two blocks later, and three blocks ahead left 690 cycles per block, whatever the tile.)
      const int weight_rows = (out_features + kBlockK - 1) / kBlockK;
      int step = 0;
      for (int tile = pair; tile < tiles && healthy; tile += pairs) {
        int row_tile, col_tile;
        tile_at(tile, row_tile, col_tile);
        // (a token or weight block past the end takes the last one's scale: its sums are not stored)
        const int row0 = (row_tile * 2 + rank) * kRows;
        const int weight_row = (col_tile * COLS + (lane >> 1 & 1) * S::kMine) / kBlockK + (lane & 1);
        const float* weight = sw + static_cast<size_t>(min(weight_row, weight_rows - 1)) * blocks;
        for (int b = 0; b < blocks; ++b, ++step) {
          const int slot = step % kSlots;
          if (step >= kSlots && !(healthy = wait_warp(taken + 8 * slot, (step / kSlots - 1) & 1))) break;
          const uint32_t at = base + S::kScales + slot * S::kSlotBytes;
          const float* rows = sa + static_cast<size_t>(b) * tokens;
#pragma unroll
          for (int i = 0; i < kRows; i += 32) copy_scale(at + (i + lane) * 4, rows + min(row0 + i + lane, tokens - 1));
          if (lane < 4) copy_scale(at + (kRows + lane) * 4, weight + b);
          copies_arrive(rank == 0 ? full + 8 * (step % kStages) : scaled + 8 * slot);
        }
      }
      copies_wait();
    } else if (rank == 1) {
      // The peer's warp 1 tells the leader that the peer's scales are there.
      const uint32_t leader_full = at_rank(full, 0);
      const int steps = (tiles - pair + pairs - 1) / pairs * blocks;
      for (int step = 0; warp == 1 && step < steps; ++step) {
        if (!(healthy = wait_warp(scaled + 8 * (step % kSlots), (step / kSlots) & 1))) break;
        if (lane == 0) arrive_remote(leader_full + 8 * (step % kStages));
      }
    } else {
      // Two warps of the leader issue, a product each in turn.  A warp's instructions wait in line behind its own products, so
      // one warp alone would test the next barriers only once its products are in the pipe, and the pipe would run dry
      // for the time of those tests.
      const int products = (tiles - pair + pairs - 1) / pairs * blocks * kProducts;
      int product = warp >> 1;
      for (; product < products; product += 2) {
        const int step = product / kProducts, s = step % kStages, buffer = product % kBuffers, round = product / kBuffers;
        if (!(healthy = wait_warp(full + 8 * s, (step / kStages) & 1))) break;
        if (round > 0 && !(healthy = wait_warp(drained + 8 * buffer, (round - 1) & 1))) break;
        fence_after_sync();
        const uint32_t at = base + s * S::kStageBytes;
        if (elect_one()) {
          block_product_pair(tmem + buffer * kWide, at, at + (kRows + product % kProducts * (kWide / 2)) * kRowBytes,
                             instruction_descriptor_e4m3(kWide, 256));
          commit_pair(filled + 8 * buffer);
          commit_pair(empty + 8 * s);
        }
        __syncwarp();
      }
      // (products complete in order: after this warp's last one none of them is reading shared memory)
      const int last = product - 2;
      if (last >= 0 && !wait_warp(filled + 8 * (last % kBuffers), (last / kBuffers) & 1)) healthy = false;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    // State of the block at hand, carried along because this loop is bound by its instructions: its accumulator, the
    // barriers of that and their phase, its scales.  (With two accumulators per half, columns and barriers differ in one bit.)
    const int mine = kProducts == 2 ? half * kWide : half * S::kMine, own = kProducts == 2 ? half : 0;
    uint32_t columns = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + mine;
    uint32_t ready = filled + 8 * own, free = at_rank(drained, 0) + 8 * own, phase = 0, scales = base + S::kScales, read = taken;
    auto next_block = [&] {
      if constexpr (kProducts == 2) {
        columns ^= 2 * kWide;
        ready ^= 16;
        free ^= 16;
        phase ^= (ready & 16) == 0 ? 1u : 0u;
      } else {
        const bool last = ready == filled + 8 * (kBuffers - 1);
        columns = last ? columns - (kBuffers - 1) * kWide : columns + kWide;
        ready = last ? filled : ready + 8;
        free = last ? free - 8 * (kBuffers - 1) : free + 8;
        phase ^= last ? 1u : 0u;
      }
      const bool last = read == taken + 8 * (kSlots - 1);
      scales = last ? base + S::kScales : scales + S::kSlotBytes;
      read = last ? taken : read + 8;
    };
    constexpr int kMine = S::kMine, kBoxBytes = 32 * S::kBox * 2, kPieces = S::kBox / 8;
    uint8_t* store = shared + S::kStore + (warp - 4) * (kMine / S::kBox) * kBoxBytes;
    for (int tile = pair; tile < tiles && healthy; tile += pairs) {
      float sum[kMine];
#pragma unroll
      for (int i = 0; i < kMine; ++i) sum[i] = 0.0f;
      int row_tile, col_tile;
      tile_at(tile, row_tile, col_tile);
      const int x = col_tile * COLS + half * kMine, y = (row_tile * 2 + rank) * kRows + quarter * 32;
      const int border = kBlockK - x % kBlockK;  // this warp's outputs before it lie in one weight block, the others in the next
      for (int b = 0; b < blocks; ++b) {
        if (!(healthy = wait_warp(ready, phase))) break;
        fence_after_sync();
        // the block's accumulator, 32 columns at a time and the next 32 on their way meanwhile, times its scales
        uint32_t d[2][32];
        load_columns<kMine>(columns, 0, d[0]);
        const float row_scale = load_shared(scales + (quarter * 32 + lane) * 4);
        const float scale = __fmul_rn(row_scale, load_shared(scales + (kRows + half * 2) * 4));
        const float scale_beyond = S::kAligned ? scale : __fmul_rn(row_scale, load_shared(scales + (kRows + half * 2 + 1) * 4));
#pragma unroll
        for (int g = 0; g < kMine; g += 32) {
          wait_loads(d[g / 32 & 1]);
          if (g + 32 < kMine) {
            load_columns<kMine>(columns, g + 32, d[(g / 32 + 1) & 1]);
          } else {
            fence_before_sync();
            __syncwarp();
            if (lane == 0) {
              arrive_remote(free);
              barrier_arrive(read);
            }
            next_block();
          }
#pragma unroll
          for (int i = 0; i < 32 && g + i < kMine; i += 2) {
            const float by = S::kAligned || g + i / 16 * 16 < border ? scale : scale_beyond;
            const float2 r = fma2(make_float2(by, by),
                                  make_float2(__uint_as_float(d[g / 32 & 1][i]), __uint_as_float(d[g / 32 & 1][i + 1])),
                                  make_float2(sum[g + i], sum[g + i + 1]));
            sum[g + i] = r.x;
            sum[g + i + 1] = r.y;
          }
        }
      }
      if (!healthy) break;
      // The warp's 32 rows leave through its own part of shared memory (swizzled as the copy reads them), so that the next
      // tile's additions start at once: all SMs end a tile together, and plain stores held them up for 3000 cycles.
      if (lane == 0) store_wait_read<0>();
      __syncwarp();
#pragma unroll
      for (int piece = 0; piece < kMine / 8; ++piece) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = sum[piece * 8 + e];
        // (the swizzle exchanges 16-byte pieces by bits 7 and up of the address: by the row, or by fours of rows)
        const int place = piece % kPieces ^ (lane / (8 / kPieces) & (kPieces - 1));
        st_vec(store + piece / kPieces * kBoxBytes + lane * (S::kBox * 2) + place * 16, pack8(v));
      }
      fence_async_proxy();
      __syncwarp();
      if (lane == 0 && y < tokens) {
#pragma unroll
        for (int i = 0; i < kMine / S::kBox; ++i)
          if (x + i * S::kBox < out_features) store_box(&map_out, x + i * S::kBox, y, shared_address(store) + i * kBoxBytes);
        store_commit();
      }
    }
    if (lane == 0) store_wait<0>();
  }
  if (!healthy) atomicExch(&g_error, 1u);
  __syncwarp();
  fence_before_sync();
  __syncthreads();
  cluster_arrive();
  cluster_wait();  // no CTA's memory is in use by another any more
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  cluster_arrive();
  cluster_wait();
}

}  // namespace pair

// ------------------------------------------------------------------------------------------------------------- strip
namespace strip {

// Outputs are the rows of the product, so that one token costs 16 columns and not a tile of 128 rows.  All that counts is to
// keep the weights coming: 131 to 202 KB of them are in flight per SM, and K is split until every SM has a share.  One token,
// 34816 x 5120: 29.9 us, 6.0 TB/s (0.91 of what a copy reaches); 5120 x 17408: 17.1 us (0.80); 48 tokens: 19.2 us.  What is left
// is the fixed part, some 3 us of launch, first fetch and joining of sums, and the SMs that clusters of this size leave idle.
constexpr int kRows = 128;     // outputs of a tile
constexpr int kMaxSplits = 8;  // CTAs of a cluster, one share of K each
constexpr int kBuffers = 4;    // accumulators, one block of K after the other (with two, 32 x 34816 x 5120 takes 33.2 us, not
                               // 32.7, and 128 x 5120 x 17408 28.1, not 26.9; one token does not mind)

// Warp 0 fetches codes, 2 scales, 1 and 3 issue; the others add up: four for the four quarters of the lanes, and from 64
// tokens on four more for the upper half of the tokens (128 tokens in one thread's registers: 57 us for 34816 x 5120,
// bound by the additions; with 64 each 12 bytes are still spilled).
template <int COLS>
struct Shape {
  static constexpr int kAdders = COLS >= 64 ? 8 : 4;
  static constexpr int kMine = COLS / (kAdders / 4);              // tokens of one adding warp
  static constexpr int kThreads = 128 + 32 * kAdders;
  static constexpr int kStageBytes = (kRows + COLS) * kRowBytes;
  static constexpr int kStages = COLS == 16 ? 11 : COLS == 32 ? 9 : COLS == 64 ? 7 : 4;
  static constexpr int kSlots = COLS == 128 ? 8 : 16;             // of scales, one per block in flight
  static constexpr int kSlotFloats = COLS + 4;                    // the tokens' scales, the weight block's, 3 unused
  static constexpr int kPartial = kStages * kStageBytes;          // [from][own group][output row] of four tokens' FP32 sums
  static constexpr int kScales = kPartial + (COLS / 4 + kMaxSplits) * kRows * 16;
  static constexpr int kBarriers = kScales + kSlots * kSlotFloats * 4;
  static constexpr int kShared = 1024 + kBarriers + 320;
  static constexpr int kColumns = kBuffers * COLS;                       // of tensor memory
  static_assert(kStages + kBuffers <= kSlots, "a slot is free when the step a ring of stages earlier has left its stage");
  static_assert(16 * kStages + 16 * kBuffers + 20 <= 320 && kShared <= 232448, "shared memory of one CTA");
};

// The cluster's CTAs share the blocks of K of one tile.  The sums of tokens 4 g to 4 g + 3 belong to rank g % splits:
// everybody pushes them into that CTA's shared memory, the pushes complete on its barrier, and it adds them in rank order.
// (Sums left in place and read by the others took two fences at cluster scope for each tile, a microsecond each.)
template <int COLS>
__global__ void __launch_bounds__(Shape<COLS>::kThreads, 1)
    block_gemm_strip_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                            const float* __restrict__ sa, const float* __restrict__ sw, int tokens, int out_features, int blocks,
                            int token_tiles, int tiles, int splits, uint16_t* __restrict__ out) {
  using S = Shape<COLS>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t raw[];
  uint8_t* shared = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t base = shared_address(shared);
  const uint32_t full = base + S::kBarriers, empty = full + 8 * kStages, filled = empty + 8 * kStages,
                 drained = filled + 8 * kBuffers, ready = drained + 8 * kBuffers, released = ready + 8;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(shared + S::kBarriers + 16 * kStages + 16 * kBuffers + 16);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % splits, cluster = blockIdx.x / splits, clusters = gridDim.x / splits;
  const int first = static_cast<int>(static_cast<long long>(blocks) * rank / splits);
  const int count = static_cast<int>(static_cast<long long>(blocks) * (rank + 1) / splits) - first;

  if (threadIdx.x == 0) {
    prefetch_map(&map_a);
    prefetch_map(&map_w);
    for (int s = 0; s < kStages; ++s) {
      barrier_init(full + 8 * s, 1 + 32);  // the codes' fetcher and every lane of the scales'
      barrier_init(empty + 8 * s, 1);
    }
    for (int i = 0; i < kBuffers; ++i) {
      barrier_init(filled + 8 * i, 1);
      barrier_init(drained + 8 * i, S::kAdders);
    }
    barrier_init(ready, 1);
    barrier_init(released, S::kAdders * splits);
    barrier_init_fence();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     shared_address(const_cast<uint32_t*>(tmem_slot))),
                 "r"(S::kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  cluster_arrive();  // (waited for where the first push is made)
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  // only now: a successor that took this SM's tensor memory first would wait for this kernel and this kernel for it
  release_next_kernel();
  wait_for_prior_kernels();

  bool healthy = true;
  if (warp == 0) {
    int step = 0;
    for (int tile = cluster; tile < tiles && healthy; tile += clusters) {
      const int row0 = tile / token_tiles * kRows, token0 = tile % token_tiles * COLS;
      for (int b = first; b < first + count; ++b, ++step) {
        const int s = step % kStages;
        if (step >= kStages && !(healthy = wait_warp(empty + 8 * s, (step / kStages - 1) & 1))) break;
        const uint32_t at = base + s * S::kStageBytes;
        if (elect_one()) {
          barrier_expect(full + 8 * s, S::kStageBytes);
          load_box(at, &map_w, b * kBlockK, row0, full + 8 * s);
          load_box(at + kRows * kRowBytes, &map_a, b * kBlockK, token0, full + 8 * s);
        }
      }
    }
    // no copy is in flight when the CTA ends, whatever became of its readers
    for (int last = max(0, step - kStages); last < step; ++last)
      if (!wait_warp(full + 8 * (last % kStages), (last / kStages) & 1)) healthy = false;
  } else if (warp == 1 || warp == 3) {  // even and odd steps, as in the panel kernel
    const int steps = (tiles - cluster + clusters - 1) / clusters * count;
    int step = warp >> 1;
    for (; step < steps; step += 2) {
      const int s = step % kStages, buffer = step % kBuffers, round = step / kBuffers;
      if (!(healthy = wait_warp(full + 8 * s, (step / kStages) & 1))) break;
      if (round > 0 && !(healthy = wait_warp(drained + 8 * buffer, (round - 1) & 1))) break;
      fence_after_sync();
      const uint32_t at = base + s * S::kStageBytes;
      if (elect_one()) {
        block_product(tmem + buffer * COLS, at, at + kRows * kRowBytes, instruction_descriptor_e4m3(COLS));
        commit(empty + 8 * s);
        commit(filled + 8 * buffer);
      }
      __syncwarp();
    }
    if (step >= 2 && !wait_warp(filled + 8 * ((step - 2) % kBuffers), ((step - 2) / kBuffers) & 1)) healthy = false;
  } else if (warp == 2) {
    // (slots as in the panel kernel; a token past the end takes the last one's scale, its sums are not stored)
    int step = 0;
    for (int tile = cluster; tile < tiles && healthy; tile += clusters) {
      const int token0 = tile % token_tiles * COLS, visible = min(COLS, tokens - token0);
      const float* tokens_at = sa + static_cast<size_t>(first) * tokens + token0;
      const float* weight = sw + static_cast<size_t>(tile / token_tiles) * blocks + first;
      for (int b = 0; b < count; ++b, ++step) {
        const int s = step % kStages;
        if (step >= kStages && !(healthy = wait_warp(empty + 8 * s, (step / kStages - 1) & 1))) break;
        const uint32_t slot = base + S::kScales + (step % S::kSlots) * (S::kSlotFloats * 4);
#pragma unroll
        for (int i = 0; i < COLS; i += 32)
          if (i + lane < COLS) copy_scale(slot + (i + lane) * 4, tokens_at + min(i + lane, visible - 1));
        if (lane == 0) copy_scale(slot + COLS * 4, weight + b);
        copies_arrive(full + 8 * s);
        tokens_at += tokens;
      }
    }
    copies_wait();
  } else {
    constexpr int kMine = S::kMine, kGroup = kMine < 32 ? kMine : 32, kAdding = S::kThreads - 128;
    const int quarter = warp & 3, row = quarter * 32 + lane, col0 = ((warp - 4) >> 2) * kMine;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + col0;
    const float* scales = reinterpret_cast<const float*>(shared + S::kScales);
    const float4* partial = reinterpret_cast<const float4*>(shared + S::kPartial);
    int step = 0, done = 0;
    bool entered = false;  // into the cluster: its barriers exist
    for (int tile = cluster; tile < tiles; tile += clusters, ++done) {
      float sum[kMine];  // this thread's output row, this warp's tokens
#pragma unroll
      for (int i = 0; i < kMine; ++i) sum[i] = 0.0f;
      for (int b = 0; b < count; ++b, ++step) {
        const int buffer = step % kBuffers;
        if (!(healthy = wait_warp(filled + 8 * buffer, (step / kBuffers) & 1))) break;
        fence_after_sync();
        const float* slot = scales + (step % S::kSlots) * S::kSlotFloats;
        const float2 weight = make_float2(slot[COLS], slot[COLS]);
#pragma unroll
        for (int g = 0; g < kMine; g += kGroup) {
          uint32_t d[kGroup];
          if constexpr (kGroup == 16) load16(lane_base + buffer * COLS + g, d);
          else load32(lane_base + buffer * COLS + g, d);
          float4 f[kGroup / 4];
#pragma unroll
          for (int i = 0; i < kGroup / 4; ++i) f[i] = reinterpret_cast<const float4*>(slot + col0 + g)[i];
          wait_loads(d);
          if (g + kGroup == kMine) {
            fence_before_sync();
            __syncwarp();
            if (lane == 0) barrier_arrive(drained + 8 * buffer);
          }
#pragma unroll
          for (int i = 0; i < kGroup; i += 2) {
            const float2 scale =
                mul2(i % 4 == 0 ? make_float2(f[i / 4].x, f[i / 4].y) : make_float2(f[i / 4].z, f[i / 4].w), weight);
            const float2 r = fma2(scale, make_float2(__uint_as_float(d[i]), __uint_as_float(d[i + 1])),
                                  make_float2(sum[g + i], sum[g + i + 1]));
            sum[g + i] = r.x;
            sum[g + i + 1] = r.y;
          }
        }
      }
      if (!healthy) break;
      const int row0 = tile / token_tiles * kRows, token0 = tile % token_tiles * COLS, visible = min(COLS, tokens - token0);
      const int groups = (visible + 3) / 4, per = (COLS / 4 + splits - 1) / splits;
      const int own = (groups + splits - 1 - rank) / splits;  // groups of this rank
      // (the first pushes wait until every CTA of the cluster has its barriers, the others until the last sums were read)
      if (!entered) cluster_wait();
      entered = true;
      if (done > 0 && !(healthy = wait_warp(released, (done - 1) & 1))) break;
      // Only behind that wait: it says that this CTA's other adding warps have seen the last tile's phase of `ready`.  A rank
      // without tokens completes a phase by this arrival alone, and a warp that two phases overtook would wait for good.
      // (Sums that come before it drive the count of bytes below zero; the phase still lacks this arrival.)
      if (warp == 4 && lane == 0) barrier_expect(ready, static_cast<uint32_t>(splits * own * kRows * 16));
      int owner = col0 / 4 % splits, place = rank * per + col0 / 4 / splits;
#pragma unroll
      for (int i = 0; i < kMine; i += 4) {
        if (col0 + i < visible)
          push(at_rank(base + S::kPartial + (place * kRows + row) * 16, owner),
               make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]), at_rank(ready, owner));
        if (++owner == splits) {
          owner = 0;
          ++place;
        }
      }
      __syncwarp();
      if (!(healthy = wait_warp(ready, done & 1))) break;
      for (int item = threadIdx.x - 128; item < own * (kRows / 2); item += kAdding) {  // (own group, two outputs)
        const int group = item / (kRows / 2), r = item % (kRows / 2) * 2;
        float4 even = make_float4(0.0f, 0.0f, 0.0f, 0.0f), odd = even;
        for (int from = 0; from < splits; ++from) {
          const float4* at = partial + (from * per + group) * kRows + r;
          even = add4(even, at[0]);
          odd = add4(odd, at[1]);
        }
        const int t = (group * splits + rank) * 4;
        const uint32_t two[4] = {pack_bf16x2(even.x, odd.x), pack_bf16x2(even.y, odd.y), pack_bf16x2(even.z, odd.z),
                                 pack_bf16x2(even.w, odd.w)};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t + i < visible && row0 + r < out_features)
            st_u32(out + static_cast<size_t>(token0 + t + i) * out_features + row0 + r, two[i]);
      }
      __syncwarp();
      if (lane < splits) arrive_remote(at_rank(released, lane));
    }
    if (!entered) cluster_wait();
  }
  if (warp < 4) cluster_wait();
  if (!healthy) atomicExch(&g_error, 1u);
  __syncwarp();
  fence_before_sync();
  __syncthreads();
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns) : "memory");
  cluster_arrive();
  cluster_wait();  // no CTA leaves while another may still push into it
}

}  // namespace strip

// ------------------------------------------------------------------------------------------------------------- host

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// [rows, cols] in boxes of box_cols x box_rows, whose rows of 32 or 128 bytes are swizzled; past the edges it reads as zero
// and is not written.
bool encode_map(CUtensorMap* map, CUtensorMapDataType type, int element, const void* p, size_t rows, size_t cols, int box_cols,
                int box_rows) {
  const EncodeTiled encode = encoder();
  if (encode == nullptr) return false;
  const cuuint64_t sizes[2] = {cols, rows}, strides[1] = {cols * element};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)}, steps[2] = {1, 1};
  const CUtensorMapSwizzle swizzle = box_cols * element == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_32B;
  auto attempt = [&] {
    return encode(map, type, 2, const_cast<void*>(p), sizes, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (attempt()) return true;
  // A host thread whose first CUDA call this is has no context yet, which this one (of the driver's) wants and does not
  // make; selecting the thread's own device does, under stream capture too.
  int device = 0;
  return cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess && attempt();
}
bool encode_codes(CUtensorMap* map, const uint8_t* codes, size_t rows, size_t cols, int box_rows) {
  return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, rows, cols, kBlockK, box_rows);
}

// Opts a kernel in to its shared memory, once per device; `registers` (when not 0) is what the kernel's register split
// was written for.
template <auto kKernel>
int prepare_kernel(int shared, int registers) {
  static std::atomic<unsigned long long> ready{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return static_cast<int>(e);
  const unsigned long long bit = 1ull << (device & 63);
  if (ready.load(std::memory_order_acquire) & bit) return host::kOk;
  if (registers != 0) {
    cudaFuncAttributes attributes;
    if ((e = cudaFuncGetAttributes(&attributes, kKernel)) != cudaSuccess) return static_cast<int>(e);
    if (attributes.numRegs != registers) return host::kNotSupported;  // the split would wait for registers it never gets
  }
  if ((e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared)) != cudaSuccess)
    return static_cast<int>(e);
  ready.fetch_or(bit, std::memory_order_release);
  return host::kOk;
}

struct Problem {
  const uint8_t *weights, *activations;
  const float *weight_scales, *activation_scales;
  int tokens, out_features, in_features, blocks;
  uint16_t* out;
  cudaStream_t stream;
};

int launch_panel(const Problem& p) {
  constexpr auto kernel = panel::block_gemm_panel_kernel;
  const int status = prepare_kernel<kernel>(panel::kShared, panel::kLaunchRegisters);
  if (status != host::kOk) return status;
  CUtensorMap a, w;
  if (!encode_codes(&a, p.activations, p.tokens, p.in_features, panel::kRows) ||
      !encode_codes(&w, p.weights, p.out_features, p.in_features, panel::kCols))
    return host::kNotSupported;
  const int row_tiles = (p.tokens + panel::kRows - 1) / panel::kRows;
  const int col_tiles = (p.out_features + panel::kCols - 1) / panel::kCols;
  const int tiles = row_tiles * col_tiles, sms = host::current_device_sm_count();
  host::launch_kernel(kernel, dim3(tiles < sms ? tiles : sms), dim3(panel::kThreads), panel::kShared, p.stream, true, a, w,
                      p.activation_scales, p.weight_scales, p.tokens, p.out_features, p.blocks, row_tiles, col_tiles, p.out);
  return host::launch_status();
}

// Clusters of `splits` CTAs of a prepared kernel that are resident at once (one CTA per SM; a cluster lives inside one
// group of SMs, so that sizes that do not divide the groups leave SMs idle: 74 of two, 45 of three, 33 of four, 26 of five,
// 22 of six, 15 of seven or eight).
template <auto kKernel, int kThreads>
int resident_clusters(int splits, int shared) {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> cache[kMaxDevices][strip::kMaxSplits + 1] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxDevices) return 1;
  int n = cache[device][splits].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(splits);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = shared;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = splits;
    attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kKernel, &config) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      n = 1;
    }
    cache[device][splits].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <auto kKernel, typename... Args>
int launch_clusters(const Problem& p, int size, int clusters, int threads, int shared, Args... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(clusters * size);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = shared;
  config.stream = p.stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = size;
  attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attributes;
  config.numAttrs = host::overlap_allowed() ? 2 : 1;
  (void)cudaLaunchKernelEx(&config, kKernel, args...);
  return host::launch_status();
}

// Token tiles that are walked together: as many as have their activations, which every output tile reads again, in L2 beside
// the weights that pass through; the weights are read from memory once per band.  8192 x 34816 x 5120 in a long run: bands of
// 8 tiles 1340 us, 16 1309, 32 1316; 8192 x 5120 x 17408, whose tiles are 3.4 times as long: 4 tiles 692 us, 8 677, 16 696.
int band_tiles_of(const Problem& p, int row_tiles) {
  const size_t tile_bytes = 2 * static_cast<size_t>(pair::kRows) * p.in_features;
  const int most = static_cast<int>(pair::kBandBytes / tile_bytes), bands = most < 1 ? row_tiles : (row_tiles + most - 1) / most;
  return (row_tiles + bands - 1) / bands;
}

template <int COLS>
int launch_pair(const Problem& p) {
  using S = pair::Shape<COLS>;
  constexpr auto kernel = pair::block_gemm_pair_kernel<COLS>;
  const int status = prepare_kernel<kernel>(S::kShared, pair::kLaunchRegisters);
  if (status != host::kOk) return status;
  CUtensorMap a, w, o;
  if (!encode_codes(&a, p.activations, p.tokens, p.in_features, pair::kRows) ||
      !encode_codes(&w, p.weights, p.out_features, p.in_features, S::kWide / 2) ||
      !encode_map(&o, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.out, p.tokens, p.out_features, S::kBox, 32))
    return host::kNotSupported;
  const int row_tiles = (p.tokens + 2 * pair::kRows - 1) / (2 * pair::kRows), col_tiles = (p.out_features + COLS - 1) / COLS;
  const int tiles = row_tiles * col_tiles, resident = resident_clusters<kernel, pair::kThreads>(2, S::kShared);
  return launch_clusters<kernel>(p, 2, tiles < resident ? tiles : resident, pair::kThreads, S::kShared, a, w, o,
                                 p.activation_scales, p.weight_scales, p.tokens, p.out_features, p.blocks, row_tiles, col_tiles,
                                 band_tiles_of(p, row_tiles));
}

// How a strip's tiles are shared out: the number of CTAs per tile with the fewest blocks on the busiest one, a tile's end
// (pushing and adding the sums, the more tokens the longer) counted as kEnd blocks.
struct StripPlan {
  int tiles, token_tiles, splits, clusters;
  long long rounds, blocks;  // tiles one after the other on the busiest CTA, and the blocks of one of them
};
template <int COLS>
StripPlan plan_strip(const Problem& p) {
  using S = strip::Shape<COLS>;
  constexpr auto kernel = strip::block_gemm_strip_kernel<COLS>;
  constexpr int kEnd = 2 + COLS / 32;
  StripPlan best{};
  const int token_tiles = (p.tokens + COLS - 1) / COLS, tiles = (p.out_features + strip::kRows - 1) / strip::kRows * token_tiles;
  for (int splits = 1; splits <= strip::kMaxSplits && splits <= p.blocks; ++splits) {
    const int resident = resident_clusters<kernel, S::kThreads>(splits, S::kShared);
    const long long rounds = (tiles + resident - 1) / resident, blocks = (p.blocks + splits - 1) / splits;
    if (best.splits == 0 || rounds * (blocks + kEnd) < best.rounds * (best.blocks + kEnd))
      best = StripPlan{tiles, token_tiles, splits, tiles < resident ? tiles : resident, rounds, blocks};
  }
  return best;
}

template <int COLS>
int launch_strip(const Problem& p) {
  using S = strip::Shape<COLS>;
  constexpr auto kernel = strip::block_gemm_strip_kernel<COLS>;
  const int status = prepare_kernel<kernel>(S::kShared, 0);
  if (status != host::kOk) return status;
  CUtensorMap a, w;
  if (!encode_codes(&a, p.activations, p.tokens, p.in_features, COLS) ||
      !encode_codes(&w, p.weights, p.out_features, p.in_features, strip::kRows))
    return host::kNotSupported;
  const StripPlan plan = plan_strip<COLS>(p);
  return launch_clusters<kernel>(p, plan.splits, plan.clusters, S::kThreads, S::kShared, a, w, p.activation_scales,
                                 p.weight_scales, p.tokens, p.out_features, p.blocks, plan.token_tiles, plan.tiles, plan.splits, p.out);
}

// More than 64 tokens: the kernel with the least time by what each was measured to take, in hundredths of a microsecond:
// a fixed part, then for every round of tiles on the busiest CTA so much per block of K -- panels 3 + 0.30 us
// (200 x 5120 x 17408: 40.0 us, pairs of 256 outputs 50.2, of 160 45.6), pairs of 256
// outputs 4.5 + 0.42 us (2048 x 10240 x 5120: 92.9 us, of 160 outputs 108.5, panels 118.5; 1337 x 5120 x 6144: 43.4, 51.9, 48.7), of
// 160 outputs 4.5 + 0.35 us (512 x 10240 x 5120: 31.7 us, of 256 outputs 33.5, panels 36.4), strips of 128 tokens 3.6 + 0.48 us and
// 3.5 us for the sums of a tile (128 x 5120 x 17408: 26.6 us, panels 38.3; 128 x 10240 x 5120: 23.2 us, panels 15.7).
// The times are those of full rounds.  A round with few tiles is shorter than the model has it (200 x 5120 x 17408 on pairs of
// 256 outputs 61.6 us against 50.2, 512 x 10240 x 5120 38.1 against 33.5) and long runs of rounds are longer (4096 x 10240 x 5120 156
// against 174): the errors of the kernels go the same way, and at each of these sizes the least time was the chosen one's.
int launch_many(const Problem& p) {
  const long long sms = host::current_device_sm_count(), pairs = sms / 2 > 0 ? sms / 2 : 1;
  auto tiles = [&](long long rows, long long cols) {
    return (p.tokens + rows - 1) / rows * ((p.out_features + cols - 1) / cols);
  };
  const long long panel_time = 300 + (tiles(panel::kRows, panel::kCols) + sms - 1) / sms * p.blocks * 30;
  const long long wide_time = 450 + (tiles(2 * pair::kRows, 256) + pairs - 1) / pairs * p.blocks * 42;
  const long long narrow_time = 450 + (tiles(2 * pair::kRows, 160) + pairs - 1) / pairs * p.blocks * 35;
  if (p.tokens <= 128) {
    const int status = prepare_kernel<strip::block_gemm_strip_kernel<128>>(strip::Shape<128>::kShared, 0);
    if (status != host::kOk) return status;
    const StripPlan plan = plan_strip<128>(p);
    const long long strip_time = 360 + plan.rounds * (plan.blocks * 48 + 350);
    if (strip_time < panel_time && strip_time < wide_time && strip_time < narrow_time) return launch_strip<128>(p);
  }
  if (panel_time <= wide_time && panel_time <= narrow_time) return launch_panel(p);
  return wide_time <= narrow_time ? launch_pair<256>(p) : launch_pair<160>(p);
}

}  // namespace
}  // namespace q3x

using namespace q3x;
using namespace q3x::host;

extern "C" int q3x_b200_fp8_block_gemm_bf16(const uint8_t* weights, const float* weight_scales, const uint8_t* activations,
                                            const float* activation_scales, size_t tokens, size_t out_features,
                                            size_t in_features, uint16_t* out, void* stream) {
  if (tokens == 0 || out_features == 0) return kOk;
  if (in_features == 0 || in_features % 16 != 0 || out_features % 8 != 0) return kInvalid;
  // (a tile's coordinates, one tile past the end included, are 32-bit integers)
  constexpr size_t kMost = 0x7fffffffu - 256;
  if (tokens > kMost || out_features > kMost || in_features > kMost) return kInvalid;
  if (weights == nullptr || weight_scales == nullptr || activations == nullptr || activation_scales == nullptr || out == nullptr)
    return kInvalid;
  const size_t blocks = (in_features + kBlockK - 1) / kBlockK;
  const Span so = span(out, tokens * out_features * 2);
  const Span inputs[] = {span(weights, out_features * in_features), span(activations, tokens * in_features),
                         span(weight_scales, (out_features + kBlockK - 1) / kBlockK * blocks * sizeof(float)),
                         span(activation_scales, blocks * tokens * sizeof(float))};
  if (wraps(so)) return kInvalid;
  for (const Span& i : inputs)
    if (wraps(i) || overlap(so, i)) return kInvalid;
  if (!aligned16(weights) || !aligned16(activations) || !aligned16(out) ||
      (reinterpret_cast<uintptr_t>(weight_scales) & 3u) != 0 || (reinterpret_cast<uintptr_t>(activation_scales) & 3u) != 0)
    return kNotSupported;
  // (tiles are counted in 32 bits)
  if (((tokens + 15) / 16) * ((out_features + 127) / 128) > 0x7fffffffu / 2) return kNotSupported;
  clear_stale_error();
  const Problem p{weights, activations, weight_scales, activation_scales, static_cast<int>(tokens), static_cast<int>(out_features),
                  static_cast<int>(in_features), static_cast<int>(blocks), out, as_stream(stream)};
  if (tokens <= 16) return launch_strip<16>(p);
  if (tokens <= 32) return launch_strip<32>(p);
  if (tokens <= 64) return launch_strip<64>(p);
  return launch_many(p);
}

extern "C" int q3x_b200_fp8_block_gemm_error(void) {
  unsigned int word = 0;
  // (the copy alone waits for the blocking streams only; a product on a non-blocking one may still be running)
  if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(&word, g_error, sizeof(word)) != cudaSuccess) {
    clear_stale_error();
    return -1;
  }
  return static_cast<int>(word);
}
