// The few tcgen05 (fifth-generation tensor core) building blocks the hand-written kernels here share: shared-memory
// matrix descriptors for 128-byte-swizzled operands, the instruction descriptor of a bf16 x bf16 -> FP32 product with
// M = 128, issue / commit, a BOUNDED wait on the completion barrier, tensor-memory loads and stores of a thread's own
// lane, the fences between the proxies, and (for E4M3 operands fetched by bulk tensor copies) the matching instruction,
// barriers and copies.  Operand tiles are rows of 64 bf16 (128 bytes) whose 16-byte pieces are
// permuted by the row's low three bits -- the 128-byte swizzle -- in blocks whose base is 1024-byte aligned.
#pragma once
#include <cstdint>

#include "bounded_wait.hpp"

namespace q3x {
namespace tcgen05 {

constexpr uint32_t kWaitLimit = 1u << 20;  // polls (and 50 ms, whichever comes first)

// K-major operand ([rows][k], k contiguous) of 64-element rows; groups of eight rows 1024 bytes apart
__device__ __forceinline__ uint64_t operand_descriptor(uint32_t shared_address) {
  return static_cast<uint64_t>((shared_address & 0x3ffffu) >> 4) | (static_cast<uint64_t>(1) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// bf16 x bf16 -> FP32, M = 128, N = n, both operands K-major
__host__ __device__ constexpr uint32_t instruction_descriptor(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
}
__device__ __forceinline__ void mma(uint32_t accumulator, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(accumulator),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[128, n] (+)= A[128, k] B[n, k]^T: 16 elements of k per instruction; 64 per block of either operand
__device__ __forceinline__ void product(uint32_t accumulator, uint32_t a_base, uint32_t a_block_bytes, uint32_t b_base,
                                        uint32_t b_block_bytes, int k, uint32_t idesc, bool accumulate) {
  for (int step = 0; step < k / 16; ++step) {
    const uint32_t block = step >> 2, inside = (step & 3) * 32;
    mma(accumulator, operand_descriptor(a_base + block * a_block_bytes + inside),
        operand_descriptor(b_base + block * b_block_bytes + inside), idesc, (accumulate || step > 0) ? 1u : 0u);
  }
}
__device__ __forceinline__ void commit(uint32_t barrier) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(barrier) : "memory");
}
// Whether the phase is complete; one that is not may hold the warp, until it is or for some microseconds.
__device__ __forceinline__ bool barrier_try(uint32_t barrier, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done)
               : "r"(barrier), "r"(parity)
               : "memory");
  return done != 0;
}
__device__ __forceinline__ uint64_t wall_clock() {
  uint64_t now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
  return now;
}
// A wait on the completion barrier that is bounded in TIME (50 ms on the global timer; a product here completes in
// microseconds): false means it ran out.  (The first poll, which mostly ends it, comes before the timer is read.)
__device__ __forceinline__ bool wait(uint32_t barrier, uint32_t parity) {
  return barrier_try(barrier, parity) ||
         wait_in_time([=] { return barrier_try(barrier, parity); }, [] { return wall_clock(); }, 50000000ull, kWaitLimit);
}
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }


// n consecutive columns of this thread's lane (the loads are waited for by the caller, so that several can be in flight)
__device__ __forceinline__ void load16(uint32_t address, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(address)
               : "memory");
}
__device__ __forceinline__ void load32(uint32_t address, uint32_t (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(address)
               : "memory");
}
__device__ __forceinline__ void store32(uint32_t address, const uint32_t (&r)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(address), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }


// MN-major operand ([k][rows], the row index contiguous: e.g. a value cache [key][dimension] as the B operand of P V):
// blocks of [k][64 rows]; eight k-lines of a block are 1024 bytes apart, the next 64 rows `block_bytes` further
__device__ __forceinline__ uint64_t operand_descriptor_mn(uint32_t shared_address, uint32_t block_bytes) {
  return static_cast<uint64_t>((shared_address & 0x3ffffu) >> 4) | (static_cast<uint64_t>((block_bytes >> 4) & 0x3fffu) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
constexpr uint32_t kBOperandMnMajor = 1u << 16;  // or-ed into an instruction descriptor

// ---- E4M3 x E4M3 -> FP32 (32 elements of k per instruction; rows of 128 codes are the same 128 bytes as 64 bf16)
__host__ __device__ constexpr uint32_t instruction_descriptor_e4m3(int n, int m = 128) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void mma_e4m3(uint32_t accumulator, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(accumulator),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The same on a pair of CTAs: M = 256, each CTA holds 128 rows of A and of the accumulator and n / 2 rows of B, at the
// same offsets; the leader (rank 0 of the cluster) issues, and a commit arrives on both CTAs' copies of the barrier.
__device__ __forceinline__ void mma_e4m3_pair(uint32_t accumulator, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(accumulator),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_pair(uint32_t barrier) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(barrier),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}
// One lane of a converged warp, always the same one.  A warp that issues walks its loop with all lanes and lets this one
// issue: addresses and descriptors then stay warp-uniform, which is what the tensor instructions take (a loop entered by
// one lane alone moves every one of them into uniform registers again, a hundred cycles per instruction).
__device__ __forceinline__ bool elect_one() {
  uint32_t elected;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected)::"memory");
  return elected != 0;
}

// ---- barriers and bulk tensor copies
__device__ __forceinline__ void barrier_init(uint32_t barrier, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(barrier), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void barrier_expect(uint32_t barrier, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier), "r"(bytes) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t barrier) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(barrier) : "memory");
}
// The bounded wait for kernels that wait once per tile of a long loop: the timer is only read after a thousand polls
// (it costs more than a completed wait), and the bound is 200 ms.
__device__ __forceinline__ bool wait_bounded(uint32_t barrier, uint32_t parity) {
  for (int spin = 0; spin < 1024; ++spin)
    if (barrier_try(barrier, parity)) return true;
  return wait_in_time([=] { return barrier_try(barrier, parity); }, [] { return wall_clock(); }, 200000000ull, 1u << 28);
}
// Box of a two-dimensional tensor map at (x, y) into this CTA's shared memory; completes `bytes` on the barrier.
__device__ __forceinline__ void load_box(uint32_t shared_address, const void* map, int x, int y, uint32_t barrier) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                   shared_address),
               "l"(map), "r"(x), "r"(y), "r"(barrier)
               : "memory");
}
// The same into this CTA of a pair, completing on a barrier of either CTA of it (a cluster address).
__device__ __forceinline__ void load_box_pair(uint32_t shared_address, const void* map, int x, int y, uint32_t barrier) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                   shared_address),
               "l"(map), "r"(x), "r"(y), "r"(barrier)
               : "memory");
}
__device__ __forceinline__ void store_box(const void* map, int x, int y, uint32_t shared_address) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
               "r"(shared_address)
               : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// all but the newest N stores have read their shared memory / have completed
template <int N>
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
template <int N>
__device__ __forceinline__ void store_wait() { asm volatile("cp.async.bulk.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void prefetch_map(const void* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// wait_loads() that also names the registers waited for, so that no use of them can be scheduled in front of it
__device__ __forceinline__ void wait_loads(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void wait_loads(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}

}  // namespace tcgen05
}  // namespace q3x
