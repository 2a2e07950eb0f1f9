// The projection of E4M3 activations with E4M3 weights, both with one FP32 scale per block of 128:
//   out[t, n] = bf16( sum over blocks b of sa[b, t] * sw[n / 128, b] * (sum over k in b of a[t, k] * w[n, k]) )
// sa [ceil(K / 128), T] as the quantisers of fp8_block.cu write it, sw [ceil(N / 128), ceil(K / 128)].  A block's products
// are summed in FP32 by the tensor cores, multiplied by the two scales and added to the running FP32 sum; the one rounding
// is to bf16.
//
// Two kernels on tcgen05 (kind::f8f6f4: E4M3 x E4M3 -> FP32 in tensor memory), operands fetched by bulk tensor copies
// into rings of 128-byte-swizzled stages, one stage per block of 128 columns of K:
//   * panel: 128 tokens are the MMA's rows, 256 (or 128) outputs its columns; bound by the tensor cores;
//   * strip: 128 outputs are the rows, 16 to 128 tokens the columns; bound by reading the weights.
// The hardware's accumulator cannot be scaled between two blocks of K, so every block starts a fresh accumulator and the
// scaled sum lives in registers: two accumulators alternate, and while the tensor cores fill one, the epilogue warps read
// the other and add it, times its scale, to their FP32 sums.
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

// The cluster: a barrier of all its threads, an arrival on a rank's copy of a barrier, a rank's copy of four floats, and the
// bounded wait for arrivals from other CTAs.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same in two parts, without publishing memory (barriers are published by their own fence).
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t at_rank(uint32_t address, int rank) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(address), "r"(rank));
  return there;
}
__device__ __forceinline__ void arrive_cluster(uint32_t there) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(there) : "memory");
}
// The same without publishing memory to the cluster, which costs a fence of a thousand cycles: for arrivals that hand on
// tensor memory, whose accesses have fences of their own.
__device__ __forceinline__ void arrive_remote(uint32_t there) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(there) : "memory");
}
// A float into another CTA's shared memory; completes its four bytes on a barrier of that CTA.
__device__ __forceinline__ void push(uint32_t there, float value, uint32_t barrier_there) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(there), "f"(value),
               "r"(barrier_there)
               : "memory");
}
__device__ __forceinline__ float4 add4(const float4& a, const float4& b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
__device__ __forceinline__ float4 load_from(uint32_t address, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at_rank(address, rank))
               : "memory");
  return v;
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
__device__ __forceinline__ bool wait_cluster(uint32_t barrier, uint32_t parity) {
  const bool done = wait_warp(barrier, parity);
  asm volatile("fence.acq_rel.cluster;" ::: "memory");
  return done;
}
__device__ __forceinline__ void block_product_pair(uint32_t accumulator, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
  for (int step = 0; step < kBlockK / 32; ++step)
    mma_e4m3_pair(accumulator, operand_descriptor(a + step * 32), operand_descriptor(b + step * 32), idesc, step > 0 ? 1u : 0u);
}

__device__ __forceinline__ uint32_t shared_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ------------------------------------------------------------------------------------------------------------- panel
namespace panel {

constexpr int kRows = 128;                  // tokens of a tile
constexpr int kThreads = 384;               // warp 0 fetches codes, 2 scales, 1 and 3 issue, 4 to 11 add up
constexpr int kAdders = 8;                  // warps: 4 lane quarters x 2 column halves
constexpr int kLaunchRegisters = 168;       // 65536 / 384, rounded down to 8
constexpr int kSlotFloats = kRows + 4;
constexpr int kBand = 16;                   // token tiles walked together

// Four accumulators of 128 columns.  256 outputs: one for each half of the outputs and parity of the block of K, each half
// added up by four warps; 128 outputs: one for each block of K modulo four, half of its columns for four warps.
constexpr int kBuffers = 4, kBufferCols = 128;

template <int COLS>
struct Shape {
  static constexpr int kHalves = COLS / kBufferCols;              // products per block
  static constexpr int kMine = COLS / 2;                          // outputs of one adding warp
  static constexpr int kReaders = kAdders / kHalves;              // warps that read one accumulator
  static constexpr int kTurn = kBuffers / kHalves;                // blocks until an accumulator comes round again
  static constexpr int kStageBytes = (kRows + COLS) * kRowBytes;
  static constexpr int kStages = COLS == 256 ? 4 : 6;
  static constexpr int kSlots = COLS == 256 ? 8 : 16;             // of scales, one per block in flight
  static constexpr int kStore = kStages * kStageBytes;          // [adder][32 rows][32 outputs] bf16
  static constexpr int kScales = kStore + kAdders * 32 * 64;    // [slot][128 tokens, 2 column halves, 2 unused] FP32
  static constexpr int kBarriers = kScales + kSlots * kSlotFloats * 4;
  static constexpr int kShared = 1024 + kBarriers + 256;  // (1024: the stages start on a 1024-byte boundary)
  static_assert(kStages + kTurn <= kSlots, "see the warp that fetches scales");
  static_assert(16 * kStages + 16 * kBuffers + 4 <= 256 && kShared <= 232448, "shared memory of one CTA");
};

template <int COLS>
__global__ void __launch_bounds__(kThreads, 1)
    block_gemm_panel_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                            const float* __restrict__ sa, const float* __restrict__ sw, int tokens, int out_features,
                            int blocks, int row_tiles, int col_tiles, uint16_t* __restrict__ out) {
  using S = Shape<COLS>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t raw[];
  uint8_t* shared = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t base = shared_address(shared);
  const uint32_t full = base + S::kBarriers, empty = full + 8 * kStages, filled = empty + 8 * kStages,
                 drained = filled + 8 * kBuffers;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(shared + S::kBarriers + 16 * kStages + 16 * kBuffers);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = row_tiles * col_tiles;

  if (threadIdx.x == 0) {
    prefetch_map(&map_a);
    prefetch_map(&map_w);
    for (int s = 0; s < kStages; ++s) {
      barrier_init(full + 8 * s, 1 + 32);  // the codes' fetcher and every lane of the scales'
      barrier_init(empty + 8 * s, S::kHalves);
    }
    for (int i = 0; i < kBuffers; ++i) {
      barrier_init(filled + 8 * i, 1);
      barrier_init(drained + 8 * i, S::kReaders);
    }
    barrier_init_fence();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(const_cast<uint32_t*>(tmem_slot))),
                 "r"(kBuffers * kBufferCols)
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
          const uint32_t at = base + s * S::kStageBytes;
          if (elect_one()) {
            barrier_expect(full + 8 * s, S::kStageBytes);
            load_box(at, &map_a, b * kBlockK, row_tile * kRows, full + 8 * s);
            load_box(at + kRows * kRowBytes, &map_w, b * kBlockK, col_tile * COLS, full + 8 * s);
          }
        }
      }
      // no copy is in flight when the CTA ends, whatever became of its readers
      for (int last = max(0, step - kStages); last < step; ++last)
        if (!wait_warp(full + 8 * (last % kStages), (last / kStages) & 1)) healthy = false;
    } else if (warp == 2) {
      // The scales of a block, copied without passing through registers (a load held in one for two blocks was measured to
      // hold up the whole warp wherever the compiler moved it).  A slot is free again: when step
      // t - kStages has left its stage, its accumulator had come round, so step t - kStages - kTurn was drained, its scales
      // and all older ones read; slot t % kSlots holds a step at least that old.
      const int weight_rows = (out_features + kBlockK - 1) / kBlockK;
      int step = 0;
      for (int tile = blockIdx.x; tile < tiles && healthy; tile += gridDim.x) {
        int row_tile, col_tile;
        tile_at(tile, row_tile, col_tile);
        const float* rows = sa + row_tile * kRows;
        const int visible = min(kRows, tokens - row_tile * kRows);
        // (a weight block past the end reads the last one's scale: its sums are not stored)
        const int weight_row = min((col_tile * COLS + (lane & 1) * (COLS / 2)) / kBlockK, weight_rows - 1);
        const float* weight = sw + static_cast<size_t>(weight_row) * blocks;
        for (int b = 0; b < blocks; ++b, ++step) {
          const int s = step % kStages;
          if (step >= kStages && !(healthy = wait_warp(empty + 8 * s, (step / kStages - 1) & 1))) break;
          const uint32_t slot = base + S::kScales + (step % S::kSlots) * kSlotFloats * 4;
#pragma unroll
          for (int i = 0; i < kRows; i += 32) copy_scale(slot + (i + lane) * 4, rows + min(i + lane, visible - 1));
          if (lane < 2) copy_scale(slot + (kRows + lane) * 4, weight + b);
          copies_arrive(full + 8 * s);
          rows += tokens;
        }
      }
      copies_wait();
    } else {
      // Two warps issue in turn: the halves of the outputs, or the even and the odd blocks.  A warp's instructions wait in
      // line behind its own products, so one warp alone would test the next barriers only once its products are in the
      // pipe, and the pipe would run dry for the time of those tests (measured: 900 cycles per block instead of 512).
      const int turn = warp >> 1, steps = (tiles - static_cast<int>(blockIdx.x) + gridDim.x - 1) / gridDim.x * blocks;
      int step = S::kHalves == 2 ? 0 : turn, last = -1;
      for (; step < steps; step += S::kHalves == 2 ? 1 : 2) {
        const int s = step % kStages, round = step / S::kTurn;
        const int buffer = S::kHalves == 2 ? (step & 1) * 2 + turn : step % kBuffers;
        if (!(healthy = wait_warp(full + 8 * s, (step / kStages) & 1))) break;
        if (round > 0 && !(healthy = wait_warp(drained + 8 * buffer, (round - 1) & 1))) break;
        fence_after_sync();
        const uint32_t at = base + s * S::kStageBytes;
        if (elect_one()) {
          block_product(tmem + buffer * kBufferCols, at, at + kRows * kRowBytes + (S::kHalves == 2 ? turn * kBufferCols * kRowBytes : 0),
                        instruction_descriptor_e4m3(kBufferCols));
          commit(empty + 8 * s);
          commit(filled + 8 * buffer);
        }
        __syncwarp();
        last = step;
      }
      // (products complete in order: after this warp's last one none of them is reading shared memory)
      if (last >= 0) {
        const int buffer = S::kHalves == 2 ? (last & 1) * 2 + turn : last % kBuffers;
        if (!wait_warp(filled + 8 * buffer, (last / S::kTurn) & 1)) healthy = false;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    constexpr int kMine = S::kMine, kTurn = S::kTurn;
    const int quarter = warp & 3, half_cols = (warp - 4) >> 2;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (S::kHalves == 2 ? 0 : half_cols * kMine);
    auto buffer_of = [&](int at) { return S::kHalves == 2 ? (at & 1) * 2 + half_cols : at % kBuffers; };
    uint8_t* store = shared + S::kStore + (warp - 4) * 32 * 64;
    const uint32_t row_scale = base + S::kScales + (quarter * 32 + lane) * 4, col_scale = base + S::kScales + (kRows + half_cols) * 4;
    int step = 0;
    for (int tile = blockIdx.x; tile < tiles && healthy; tile += gridDim.x) {
      float sum[kMine];
#pragma unroll
      for (int i = 0; i < kMine; ++i) sum[i] = 0.0f;
      // One block: 32 columns of its accumulator at a time, times its scales, onto the sums; the next 32 columns, which may
      // be the next block's first, are on their way meanwhile.
      // Whether its products are complete is asked before the last columns but one are added and answered after.
      uint32_t d[2][32];
      float2 factors;
      auto begin = [&](int at) {  // a block whose products are complete
        fence_after_sync();
        load32(lane_base + buffer_of(at) * kBufferCols, d[0]);
        factors = make_float2(load_shared(row_scale + at % S::kSlots * (kSlotFloats * 4)),
                              load_shared(col_scale + at % S::kSlots * (kSlotFloats * 4)));
      };
      bool begun = false;
      for (int b = 0; b < blocks; ++b) {
        if (!begun) {
          if (!(healthy = wait_warp(filled + 8 * buffer_of(step), (step / kTurn) & 1))) break;
          begin(step);
        }
        const uint32_t columns = lane_base + buffer_of(step) * kBufferCols;
        const float scale = __fmul_rn(factors.x, factors.y);
        bool complete = false;
#pragma unroll
        for (int g = 0; g < kMine / 32; ++g) {
          wait_loads(d[g & 1]);
          if (g + 1 < kMine / 32) {
            load32(columns + (g + 1) * 32, d[(g + 1) & 1]);
            if (g + 2 == kMine / 32) complete = barrier_try(filled + 8 * buffer_of(step + 1), ((step + 1) / kTurn) & 1);
          } else {
            fence_before_sync();
            __syncwarp();
            if (lane == 0) barrier_arrive(drained + 8 * buffer_of(step));
            ++step;
            begun = b + 1 < blocks && __all_sync(kFullMask, complete);
            if (begun) begin(step);
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
      const int row0 = row_tile * kRows + quarter * 32, col0 = col_tile * COLS + half_cols * kMine;
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
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kBuffers * kBufferCols) : "memory");
}

}  // namespace panel

// -------------------------------------------------------------------------------------------------------------- pair
namespace pair {

// Two CTAs share one tile of 256 tokens x 256 outputs: each holds its 128 tokens' codes and accumulators and HALF of the
// weights' codes, and one tensor instruction runs on both SMs (cta_group::2).  Against two tiles of 128 x 256 every SM
// fetches 32 KB instead of 48 KB per block of K, and an instruction of 128 columns reads 6 KB of shared memory instead
// of 8 in its 64 cycles, which is what lets the accumulators be four of 128 columns: each half of the outputs has two, and
// a half is read while three other products run.
//
// Few tiles leave SMs idle, so with kSplit a cluster of `splits` pairs shares the blocks of K of a tile: each pair adds up
// its share, and the pairs exchange their FP32 sums through the staging area, one half of the outputs after the other:
// everybody's warps of that half write, everybody adds the rows whose index is its pair's modulo `splits`, in pair order.
constexpr int kRows = 128;                  // tokens of a CTA
constexpr int kCols = 256;                  // outputs of a tile
constexpr int kHalf = 128;                  // outputs of one product
constexpr int kThreads = 384;               // warp 0 fetches codes, 2 scales, 1 and 3 issue (leader), 4 to 11 add up
constexpr int kAdders = 8;                  // warps: 4 lane quarters x 2 halves
constexpr int kLaunchRegisters = 168;       // 65536 / 384, rounded down to 8
constexpr int kBand = 8;                    // token tiles walked together
constexpr int kBuffers = 4;                 // accumulators: parity of the block x half
constexpr int kStageBytes = (kRows + kCols / 2) * kRowBytes;
constexpr int kStages = 5;
constexpr int kSlots = 4;                   // of scales
constexpr int kSlotFloats = kRows + 4;      // the tokens', the two halves' weight blocks', 2 unused
constexpr int kStore = kStages * kStageBytes;                  // [adder][2][32 rows][64 outputs] bf16
constexpr int kScales = kStore + kAdders * 2 * 32 * 128;
constexpr int kBarriers = kScales + kSlots * kSlotFloats * 4;
constexpr int kTmemSlot = kBarriers + 8 * (2 * kStages + 2 * kBuffers + 2 * kSlots + 2);
constexpr int kMaxSplits = 4;
static_assert(kScales - kStore == kRows * kHalf * 4, "the staging area holds one half's FP32 sums");
constexpr int kShared = kTmemSlot + 16;
static_assert(kShared <= 232448, "shared memory of one CTA");

// The exchange of kSplit.  A row of a half is 512 bytes, its 16-byte pieces permuted by the row: a warp writes 32 rows of
// one column and reads one row without bank conflicts.
template <typename Store>
__device__ __forceinline__ bool join_halves(const float (&sum)[kHalf], int half, int quarter, int adder, int lane, int rank,
                                            int share, int splits, int& rounds, uint8_t* staging, uint32_t staging_at,
                                            uint32_t ready, uint32_t released, Store&& store) {
  for (int h = 0; h < 2; ++h, ++rounds) {
    if (half == h) {
      if (rounds > 0 && !wait_cluster(released, (rounds - 1) & 1)) return false;
      const int row = quarter * 32 + lane;
#pragma unroll
      for (int piece = 0; piece < kHalf / 4; ++piece)
        *reinterpret_cast<float4*>(staging + row * (kHalf * 4) + ((piece ^ (row & 31)) << 4)) =
            make_float4(sum[piece * 4], sum[piece * 4 + 1], sum[piece * 4 + 2], sum[piece * 4 + 3]);
      __syncwarp();
      if (lane < splits) arrive_cluster(at_rank(ready, lane * 2 + rank));
    }
    if (!wait_cluster(ready, rounds & 1)) return false;
    // four rows' loads are in flight together: one after the other they took 7 us per half
    constexpr int kBatch = 4;
    for (int row0 = share + adder * splits; row0 < kRows; row0 += kBatch * kAdders * splits) {
      float4 p[kBatch][kMaxSplits];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int row = row0 + i * kAdders * splits;
        const uint32_t at = staging_at + row * (kHalf * 4) + ((lane ^ (row & 31)) << 4);
#pragma unroll
        for (int from = 0; from < kMaxSplits; ++from)
          p[i][from] = from < splits && row < kRows ? load_from(at, from * 2 + rank) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        float4 total = p[i][0];
#pragma unroll
        for (int from = 1; from < kMaxSplits; ++from)
          if (from < splits) total = add4(total, p[i][from]);
        if (row0 + i * kAdders * splits < kRows) store(row0 + i * kAdders * splits, h * kHalf + lane * 4, total);
      }
    }
    __syncwarp();
    if (lane < splits) arrive_cluster(at_rank(released, lane * 2 + rank));
  }
  return true;
}

template <bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    block_gemm_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                           const __grid_constant__ CUtensorMap map_out, const float* __restrict__ sa,
                           const float* __restrict__ sw, int tokens, int out_features, int blocks, int row_tiles,
                           int col_tiles, int splits, uint16_t* __restrict__ out) {
  extern __shared__ __align__(1024) uint8_t shared[];
  const uint32_t base = shared_address(shared);
  const uint32_t full = base + kBarriers, empty = full + 8 * kStages, filled = empty + 8 * kStages,
                 drained = filled + 8 * kBuffers, scaled = drained + 8 * kBuffers, taken = scaled + 8 * kSlots,
                 ready = taken + 8 * kSlots, released = ready + 8;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(shared + kTmemSlot);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1, tiles = row_tiles * col_tiles;
  const int share = kSplit ? (blockIdx.x >> 1) % splits : 0;  // of the blocks of K; the pair's place in the cluster
  const int leader = share * 2;                               // the cluster rank of the pair's leader
  const int cluster = kSplit ? (blockIdx.x >> 1) / splits : blockIdx.x >> 1;
  const int clusters = kSplit ? (gridDim.x >> 1) / splits : gridDim.x >> 1;
  const int first = kSplit ? static_cast<int>(static_cast<long long>(blocks) * share / splits) : 0;
  const int count = kSplit ? static_cast<int>(static_cast<long long>(blocks) * (share + 1) / splits) - first : blocks;

  if (threadIdx.x == 0) {
    prefetch_map(&map_a);
    prefetch_map(&map_w);
    prefetch_map(&map_out);
    for (int s = 0; s < kStages; ++s) {
      barrier_init(full + 8 * s, 1);    // (the leader's: both CTAs' copies complete on it)
      barrier_init(empty + 8 * s, 2);   // both halves' products
    }
    for (int i = 0; i < kBuffers; ++i) {
      barrier_init(filled + 8 * i, 1);
      barrier_init(drained + 8 * i, kAdders);  // (the leader's: four warps of each CTA)
    }
    for (int i = 0; i < kSlots; ++i) {
      barrier_init(scaled + 8 * i, 32);
      barrier_init(taken + 8 * i, kAdders);
    }
    if (kSplit) {
      barrier_init(ready, kAdders / 2 * splits);
      barrier_init(released, kAdders * splits);
    }
    barrier_init_fence();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + kTmemSlot), "r"(kBuffers * kHalf)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  cluster_sync();
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
      const uint32_t leader_full = at_rank(full, leader);
      int step = 0;
      for (int tile = cluster; tile < tiles && healthy; tile += clusters) {
        int row_tile, col_tile;
        tile_at(tile, row_tile, col_tile);
        const int row0 = (row_tile * 2 + rank) * kRows, col0 = col_tile * kCols + rank * (kHalf / 2);
        for (int b = first; b < first + count; ++b, ++step) {
          const int s = step % kStages;
          if (step >= kStages && !(healthy = wait_warp(empty + 8 * s, (step / kStages - 1) & 1))) break;
          const uint32_t at = base + s * kStageBytes;
          if (elect_one()) {
            if (rank == 0) barrier_expect(full + 8 * s, 2 * kStageBytes);
            load_box_pair(at, &map_a, b * kBlockK, row0, leader_full + 8 * s);
            load_box_pair(at + kRows * kRowBytes, &map_w, b * kBlockK, col0, leader_full + 8 * s);
            load_box_pair(at + (kRows + kHalf / 2) * kRowBytes, &map_w, b * kBlockK, col0 + kHalf, leader_full + 8 * s);
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
      // hold up the whole warp wherever the compiler moved it).
      const int weight_rows = (out_features + kBlockK - 1) / kBlockK;
      int step = 0;
      for (int tile = cluster; tile < tiles && healthy; tile += clusters) {
        int row_tile, col_tile;
        tile_at(tile, row_tile, col_tile);
        // (a token or weight block past the end takes the last one's scale: its sums are not stored)
        const int row0 = (row_tile * 2 + rank) * kRows;
        const float* weight = sw + static_cast<size_t>(min(col_tile * 2 + (lane & 1), weight_rows - 1)) * blocks;
        for (int b = first; b < first + count; ++b, ++step) {
          const int slot = step % kSlots;
          if (step >= kSlots && !(healthy = wait_warp(taken + 8 * slot, (step / kSlots - 1) & 1))) break;
          const uint32_t at = base + kScales + slot * (kSlotFloats * 4);
          const float* rows = sa + static_cast<size_t>(b) * tokens;
#pragma unroll
          for (int i = 0; i < kRows; i += 32) copy_scale(at + (i + lane) * 4, rows + min(row0 + i + lane, tokens - 1));
          if (lane < 2) copy_scale(at + (kRows + lane) * 4, weight + b);
          copies_arrive(scaled + 8 * slot);
        }
      }
      copies_wait();
    } else if (rank == 0) {
      // Two warps issue, one for each half of the outputs.  A warp's instructions wait in line behind its own products, so
      // one warp alone would test the next barriers only once its products are in the pipe, and the pipe would run dry
      // for the time of those tests.
      const int half = warp >> 1, steps = (tiles - cluster + clusters - 1) / clusters * count;
      int step = 0;
      for (; step < steps; ++step) {
        const int s = step % kStages, buffer = (step & 1) * 2 + half;
        if (!(healthy = wait_warp(full + 8 * s, (step / kStages) & 1))) break;
        if (step >= 2 && !(healthy = wait_warp(drained + 8 * buffer, (step / 2 - 1) & 1))) break;
        fence_after_sync();
        const uint32_t at = base + s * kStageBytes;
        if (elect_one()) {
          block_product_pair(tmem + buffer * kHalf, at, at + (kRows + half * (kHalf / 2)) * kRowBytes,
                             instruction_descriptor_e4m3(kHalf, 256));
          commit_pair(filled + 8 * buffer, leader);
          commit_pair(empty + 8 * s, leader);
        }
        __syncwarp();
      }
      // (products complete in order: after this warp's last one none of them is reading shared memory)
      if (step > 0 && !wait_warp(filled + 8 * (((step - 1) & 1) * 2 + half), ((step - 1) / 2) & 1)) healthy = false;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * kHalf;
    const uint32_t leader_drained = at_rank(drained, leader) + 8 * half;
    const uint32_t row_scale = base + kScales + (quarter * 32 + lane) * 4, col_scale = base + kScales + (kRows + half) * 4;
    uint8_t* store = shared + kStore + (warp - 4) * 2 * 32 * 128;
    const uint32_t mine = filled + 8 * half;
    int step = 0, rounds = 0;
    for (int tile = cluster; tile < tiles && healthy; tile += clusters) {
      float sum[kHalf];
#pragma unroll
      for (int i = 0; i < kHalf; ++i) sum[i] = 0.0f;
      // One block: 32 columns of its accumulator at a time, times its scales, onto the sums; the next 32 columns, which may
      // be the next block's first, are on their way meanwhile.  Whether that block's products are complete is asked
      // before the last columns but one are added and answered after.
      uint32_t d[2][32];
      float2 factors;
      auto begin = [&](int at) {  // a block whose products and scales are there
        fence_after_sync();
        load32(lane_base + (at & 1) * (2 * kHalf), d[0]);
        factors = make_float2(load_shared(row_scale + at % kSlots * (kSlotFloats * 4)),
                              load_shared(col_scale + at % kSlots * (kSlotFloats * 4)));
      };
      bool begun = false;
      for (int b = 0; b < count; ++b) {
        if (!begun) {
          if (!(healthy = wait_warp(mine + 16 * (step & 1), (step / 2) & 1) &&
                          wait_warp(scaled + 8 * (step % kSlots), (step / kSlots) & 1)))
            break;
          begin(step);
        }
        const uint32_t columns = lane_base + (step & 1) * (2 * kHalf);
        const float scale = __fmul_rn(factors.x, factors.y);
        bool complete = false;
#pragma unroll
        for (int g = 0; g < kHalf / 32; ++g) {
          wait_loads(d[g & 1]);
          if (g + 1 < kHalf / 32) {
            load32(columns + (g + 1) * 32, d[(g + 1) & 1]);
            if (g + 2 == kHalf / 32) {  // (both asked, without a branch: the warp stays together)
              const bool products = barrier_try(mine + 16 * (~step & 1), ((step + 1) / 2) & 1);
              const bool scales = barrier_try(scaled + 8 * ((step + 1) % kSlots), ((step + 1) / kSlots) & 1);
              complete = products & scales;
            }
          } else {
            fence_before_sync();
            __syncwarp();
            if (lane == 0) {
              arrive_remote(leader_drained + 16 * (step & 1));
              barrier_arrive(taken + 8 * (step % kSlots));
            }
            ++step;
            begun = b + 1 < count && __all_sync(kFullMask, complete);
            if (begun) begin(step);
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
      if constexpr (kSplit) {
        healthy = join_halves(sum, half, quarter, warp - 4, lane, rank, share, splits, rounds, shared + kStore, base + kStore, ready,
                              released, [&](int row, int col, const float4& total) {
                                int row_tile, col_tile;
                                tile_at(tile, row_tile, col_tile);
                                const int t = (row_tile * 2 + rank) * kRows + row, o = col_tile * kCols + col;
                                if (t < tokens && o < out_features)
                                  *reinterpret_cast<uint2*>(out + static_cast<size_t>(t) * out_features + o) =
                                      make_uint2(pack_bf16x2(total.x, total.y), pack_bf16x2(total.z, total.w));
                              });
        continue;
      }
      // The warp's 32 rows x 128 outputs leave through its own 8 KB (swizzled as the copy reads them), so that the next
      // tile's additions start at once: all SMs end a tile together, and plain stores held them up for 3000 cycles.
      int row_tile, col_tile;
      tile_at(tile, row_tile, col_tile);
      const int x = col_tile * kCols + half * kHalf, y = (row_tile * 2 + rank) * kRows + quarter * 32;
      if (lane == 0) store_wait_read<0>();
      __syncwarp();
#pragma unroll
      for (int piece = 0; piece < 16; ++piece) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = sum[piece * 8 + e];
        st_vec(store + piece / 8 * (32 * 128) + lane * 128 + ((piece % 8 ^ (lane & 7)) << 4), pack8(v));
      }
      fence_async_proxy();
      __syncwarp();
      if (lane == 0 && y < tokens) {
        if (x < out_features) store_box(&map_out, x, y, shared_address(store));
        if (x + 64 < out_features) store_box(&map_out, x + 64, y, shared_address(store) + 32 * 128);
        store_commit();
      }
    }
    if (lane == 0) store_wait<0>();
  }
  if (!healthy) atomicExch(&g_error, 1u);
  __syncwarp();
  fence_before_sync();
  __syncthreads();
  cluster_sync();  // neither CTA's memory is in use by the other any more
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kBuffers * kHalf) : "memory");
  __syncwarp();
  cluster_sync();
}

}  // namespace pair

// ------------------------------------------------------------------------------------------------------------- strip
namespace strip {

constexpr int kRows = 128;     // outputs of a tile
constexpr int kMaxSplits = 8;  // CTAs of a cluster, one share of K each

// Warp 0 fetches codes, 2 scales, 1 and 3 issue; the others add up: four for the four quarters of the lanes, and from 64
// tokens on four more for the upper half of the tokens (128 tokens in one thread's registers: 57 us for 34816 x 5120,
// bound by the additions).
template <int COLS>
struct Shape {
  static constexpr int kAdders = COLS >= 64 ? 8 : 4;
  static constexpr int kMine = COLS / (kAdders / 4);              // tokens of one adding warp
  static constexpr int kThreads = 128 + 32 * kAdders;
  static constexpr int kStageBytes = (kRows + COLS) * kRowBytes;
  static constexpr int kStages = COLS == 16 ? 11 : COLS == 32 ? 10 : COLS == 64 ? 7 : 4;
  static constexpr int kSlots = COLS == 128 ? 8 : 16;             // of scales, one per block in flight
  static constexpr int kSlotFloats = COLS + 4;                    // the tokens' scales, the weight block's, 3 unused
  static constexpr int kPartial = kStages * kStageBytes;          // [from][own token][output row] FP32, pushed by the cluster
  static constexpr int kScales = kPartial + (COLS + kMaxSplits) * kRows * 4;
  static constexpr int kBarriers = kScales + kSlots * kSlotFloats * 4;
  static constexpr int kShared = 1024 + kBarriers + 256;
  static constexpr int kColumns = 2 * COLS;                       // of tensor memory
  static_assert(kStages + 2 <= kSlots, "a slot is free when the step a ring of stages earlier has left its stage");
  static_assert(16 * kStages + 52 <= 256 && kShared <= 232448, "shared memory of one CTA");
};

// The cluster's CTAs share the blocks of K of one tile.  Token t's sums belong to rank t % splits: everybody pushes them into
// that CTA's shared memory, the pushes complete on its barrier, and it adds them in rank order.  (Sums left in place and
// read by the others took two fences at cluster scope for each tile, a microsecond each.)
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
  const uint32_t full = base + S::kBarriers, empty = full + 8 * kStages, filled = empty + 8 * kStages, drained = filled + 16,
                 ready = drained + 16, released = ready + 8;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(shared + S::kBarriers + 16 * kStages + 48);
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
    for (int i = 0; i < 2; ++i) {
      barrier_init(filled + 8 * i, 1);
      barrier_init(drained + 8 * i, S::kAdders);
    }
    barrier_init(ready, 1);
    barrier_init(released, S::kAdders * splits);
    barrier_init_fence();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(const_cast<uint32_t*>(tmem_slot))),
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
    const int half = warp >> 1, steps = (tiles - cluster + clusters - 1) / clusters * count;
    int step = half;
    for (; step < steps; step += 2) {
      const int s = step % kStages;
      if (!(healthy = wait_warp(full + 8 * s, (step / kStages) & 1))) break;
      if (step >= 2 && !(healthy = wait_warp(drained + 8 * half, (step / 2 - 1) & 1))) break;
      fence_after_sync();
      const uint32_t at = base + s * S::kStageBytes;
      if (elect_one()) {
        block_product(tmem + half * COLS, at, at + kRows * kRowBytes, instruction_descriptor_e4m3(COLS));
        commit(empty + 8 * s);
        commit(filled + 8 * half);
      }
      __syncwarp();
    }
    if (step >= 2 && !wait_warp(filled + 8 * half, (step / 2 - 1) & 1)) healthy = false;
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
    float* partial = reinterpret_cast<float*>(shared + S::kPartial);
    int step = 0, done = 0;
    bool entered = false;  // into the cluster: its barriers exist
    for (int tile = cluster; tile < tiles; tile += clusters, ++done) {
      float sum[kMine];  // this thread's output row, this warp's tokens
#pragma unroll
      for (int i = 0; i < kMine; ++i) sum[i] = 0.0f;
      for (int b = 0; b < count; ++b, ++step) {
        const int half = step & 1;
        if (!(healthy = wait_warp(filled + 8 * half, (step / 2) & 1))) break;
        fence_after_sync();
        const float* slot = scales + (step % S::kSlots) * S::kSlotFloats;
        const float2 weight = make_float2(slot[COLS], slot[COLS]);
#pragma unroll
        for (int g = 0; g < kMine; g += kGroup) {
          uint32_t d[kGroup];
          if constexpr (kGroup == 16) load16(lane_base + half * COLS + g, d);
          else load32(lane_base + half * COLS + g, d);
          float4 f[kGroup / 4];
#pragma unroll
          for (int i = 0; i < kGroup / 4; ++i) f[i] = reinterpret_cast<const float4*>(slot + col0 + g)[i];
          wait_loads(d);
          if (g + kGroup == kMine) {
            fence_before_sync();
            __syncwarp();
            if (lane == 0) barrier_arrive(drained + 8 * half);
          }
#pragma unroll
          for (int i = 0; i < kGroup; i += 2) {
            const float2 scale = mul2(i % 4 == 0 ? make_float2(f[i / 4].x, f[i / 4].y) : make_float2(f[i / 4].z, f[i / 4].w), weight);
            const float2 r = fma2(scale, make_float2(__uint_as_float(d[i]), __uint_as_float(d[i + 1])),
                                  make_float2(sum[g + i], sum[g + i + 1]));
            sum[g + i] = r.x;
            sum[g + i + 1] = r.y;
          }
        }
      }
      if (!healthy) break;
      const int row0 = tile / token_tiles * kRows, token0 = tile % token_tiles * COLS, visible = min(COLS, tokens - token0);
      const int per = (COLS + splits - 1) / splits, own = (visible + splits - 1 - rank) / splits;  // tokens of a rank; of this one here
      if (warp == 4 && lane == 0) barrier_expect(ready, static_cast<uint32_t>(splits * own * kRows * 4));
      // (the first pushes wait until every CTA of the cluster has its barriers, the others until the last sums were read)
      if (!entered) cluster_wait();
      entered = true;
      if (done > 0 && !(healthy = wait_warp(released, (done - 1) & 1))) break;
      int owner = col0 % splits, place = rank * per + col0 / splits;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        if (col0 + i < visible) push(at_rank(base + S::kPartial + (place * kRows + row) * 4, owner), sum[i], at_rank(ready, owner));
        if (++owner == splits) {
          owner = 0;
          ++place;
        }
      }
      __syncwarp();
      if (!(healthy = wait_warp(ready, done & 1))) break;
      for (int item = threadIdx.x - 128; item < own * (kRows / 4); item += kAdding) {  // (own token, four outputs)
        const int t = item / (kRows / 4), r = item % (kRows / 4) * 4;
        float4 total = *reinterpret_cast<const float4*>(partial + t * kRows + r);
        for (int from = 1; from < splits; ++from)
          total = add4(total, *reinterpret_cast<const float4*>(partial + (from * per + t) * kRows + r));
        if (row0 + r < out_features)
          *reinterpret_cast<uint2*>(out + static_cast<size_t>(token0 + t * splits + rank) * out_features + row0 + r) =
              make_uint2(pack_bf16x2(total.x, total.y), pack_bf16x2(total.z, total.w));
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
  __syncwarp();
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

// [rows, cols] in boxes of box_rows rows of 128 bytes, swizzled; past the edges it reads as zero.
bool encode_map(CUtensorMap* map, CUtensorMapDataType type, int element, const void* p, size_t rows, size_t cols, int box_rows) {
  const EncodeTiled encode = encoder();
  if (encode == nullptr) return false;
  const cuuint64_t sizes[2] = {cols, rows}, strides[1] = {cols * element};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / element), static_cast<cuuint32_t>(box_rows)}, steps[2] = {1, 1};
  return encode(map, type, 2, const_cast<void*>(p), sizes, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool encode_codes(CUtensorMap* map, const uint8_t* codes, size_t rows, size_t cols, int box_rows) {
  return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, rows, cols, box_rows);
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

template <int COLS>
int launch_panel(const Problem& p) {
  using S = panel::Shape<COLS>;
  constexpr auto kernel = panel::block_gemm_panel_kernel<COLS>;
  const int status = prepare_kernel<kernel>(S::kShared, panel::kLaunchRegisters);
  if (status != host::kOk) return status;
  CUtensorMap a, w;
  if (!encode_codes(&a, p.activations, p.tokens, p.in_features, panel::kRows) ||
      !encode_codes(&w, p.weights, p.out_features, p.in_features, COLS))
    return host::kNotSupported;
  const int row_tiles = (p.tokens + panel::kRows - 1) / panel::kRows, col_tiles = (p.out_features + COLS - 1) / COLS;
  if (static_cast<long long>(row_tiles) * col_tiles > 0x7fffffff / 2) return host::kNotSupported;
  const int tiles = row_tiles * col_tiles, sms = host::current_device_sm_count();
  host::launch_kernel(kernel, dim3(tiles < sms ? tiles : sms), dim3(panel::kThreads), S::kShared, p.stream, true, a, w,
                      p.activation_scales, p.weight_scales, p.tokens, p.out_features, p.blocks, row_tiles, col_tiles, p.out);
  return host::launch_status();
}

// Clusters of `splits` CTAs that are resident at once (one CTA per SM; a cluster lives inside one group of SMs, so that
// sizes that do not divide the groups leave SMs idle: 74 of two, 45 of three, 33 of four, 15 of seven or eight).
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

template <bool kSplit>
int launch_pair(const Problem& p, int splits) {
  constexpr auto kernel = pair::block_gemm_pair_kernel<kSplit>;
  const int status = prepare_kernel<kernel>(pair::kShared, pair::kLaunchRegisters);
  if (status != host::kOk) return status;
  CUtensorMap a, w, o;
  if (!encode_codes(&a, p.activations, p.tokens, p.in_features, pair::kRows) ||
      !encode_codes(&w, p.weights, p.out_features, p.in_features, pair::kHalf / 2) ||
      !encode_map(&o, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.out, p.tokens, p.out_features, 32))
    return host::kNotSupported;
  const int row_tiles = (p.tokens + 2 * pair::kRows - 1) / (2 * pair::kRows), col_tiles = (p.out_features + pair::kCols - 1) / pair::kCols;
  if (static_cast<long long>(row_tiles) * col_tiles > 0x7fffffff / 2) return host::kNotSupported;
  const int tiles = row_tiles * col_tiles, resident = resident_clusters<kernel, pair::kThreads>(2 * splits, pair::kShared);
  return launch_clusters<kernel>(p, 2 * splits, tiles < resident ? tiles : resident, pair::kThreads, pair::kShared, a, w, o,
                                 p.activation_scales, p.weight_scales, p.tokens, p.out_features, p.blocks, row_tiles, col_tiles,
                                 splits, p.out);
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
  const int out_tiles = (p.out_features + strip::kRows - 1) / strip::kRows, token_tiles = (p.tokens + COLS - 1) / COLS;
  if (static_cast<long long>(out_tiles) * token_tiles > 0x7fffffff / 2) return host::kNotSupported;
  const int tiles = out_tiles * token_tiles;
  // CTAs that share a tile's blocks of K: the count with the fewest blocks on the busiest CTA, joining the sums counted
  // as kJoin blocks
  constexpr double kJoin = 3.0;
  int splits = 1, clusters = 1;
  double least = 1e300;
  for (int s = 1; s <= strip::kMaxSplits && s <= p.blocks; ++s) {
    const int resident = resident_clusters<kernel, S::kThreads>(s, S::kShared);
    const double time = static_cast<double>((tiles + resident - 1) / resident) * ((p.blocks + s - 1) / s) + (s > 1 ? kJoin : 0.0);
    if (time < least) {
      least = time;
      splits = s;
      clusters = tiles < resident ? tiles : resident;
    }
  }
  return launch_clusters<kernel>(p, splits, clusters, S::kThreads, S::kShared, a, w, p.activation_scales, p.weight_scales, p.tokens,
                                 p.out_features, p.blocks, token_tiles, tiles, splits, p.out);
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
  clear_stale_error();
  const Problem p{weights, activations, weight_scales, activation_scales, static_cast<int>(tokens), static_cast<int>(out_features),
                  static_cast<int>(in_features), static_cast<int>(blocks), out, as_stream(stream)};
  if (tokens <= 16) return launch_strip<16>(p);
  if (tokens <= 32) return launch_strip<32>(p);
  if (tokens <= 64) return launch_strip<64>(p);
  if (tokens <= 128) return launch_strip<128>(p);
  // 256 outputs per tile where that still gives every SM a tile
  const size_t wide_tiles = (tokens + 127) / 128 * ((out_features + 255) / 256);
  return wide_tiles >= static_cast<size_t>(current_device_sm_count()) ? launch_pair<false>(p, 1) : launch_panel<128>(p);
}

extern "C" int q3x_b200_fp8_block_gemm_error(void) {
  unsigned int word = 0;
  if (cudaMemcpyFromSymbol(&word, g_error, sizeof(word)) != cudaSuccess) return -1;
  return static_cast<int>(word);
}
