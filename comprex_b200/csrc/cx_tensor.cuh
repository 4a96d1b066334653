// The fifth-generation tensor cores: tensor memory, matrix instructions, tile copies, and the barriers between them.
// Every wait is bounded: one that runs out says so to its caller.
#pragma once
#include <cuda.h>

#include "cx_device.cuh"

namespace cxt {

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// True in one lane of the warp.  What one thread issues here takes its operands from the warp's uniform registers, which
// the compiler fills where the whole warp comes by: the loops around are the warp's, only the instructions themselves are
// behind this.  (Behind a test of the lane's number a tile copy took 250 cycles.)
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes != 0;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of the same shared variable in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}

// ---- barriers ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void fence_barrier_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Waits for a phase of a barrier: at most 2^21 tries of about a microsecond each, then false.  Acquire at the scope of the
// CTA: what the barriers here guard comes by tile copies, matrix instructions and loads of tensor memory, which their own
// completion and fences order.  (At the scope of the cluster a wait took 500 cycles; as a loop in C++ with a vote 220; so,
// where the phase is there already, 40.)
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, 2097152;\n"
      "again:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
      "@p bra there;\n\t"
      "sub.u32 n, n, 1;\n\tsetp.ne.u32 q, n, 0;\n\t@q bra again;\n"
      "there:\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// One look at it.  The answer takes 200 cycles: ask for the next phase before the work on this one.
__device__ __forceinline__ bool look(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// the same answer in all lanes of the warp
__device__ __forceinline__ bool wait_together(uint32_t bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, wait(bar, parity)); }

// ---- tile copies (global -> shared, 128-byte swizzle; the inner coordinate is a multiple of 64 elements) ----------
// CG == 2: the barrier may be the one of the other CTA of the pair.
template <int CG>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if (CG == 1)
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// ---- tensor memory -------------------------------------------------------------------------------------------------
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t where, uint32_t columns) {
  if (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {
  if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of the warp's 32 lanes: lane i gets row i
__device__ __forceinline__ void tmem_load32(uint32_t tmem, uint32_t (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(tmem));
}
// Until all of the warp's loads are there.  `r`, which one of them fills, is an operand: no use of it may move up.
__device__ __forceinline__ void tmem_load_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :: "memory");
}

// ---- matrix instructions -------------------------------------------------------------------------------------------
// An operand tile in shared memory with the 128-byte swizzle (atoms of 8 rows of 128 bytes, 1024-byte aligned).
//   consecutive along k:       rows are the operand's rows, an atom is 8 rows of 64 elements of k, atoms 1024 bytes apart
//   consecutive along m or n:  rows are k, an atom is 8 of k by 64 elements, the next 8 of k 1024 bytes on, the next 64
//                              elements `chunk` bytes on
// The lower word holds the address and `chunk`, in 16 bytes: adding to it moves the tile (shared memory ends below 2^18).
__device__ __forceinline__ uint32_t operand_at(uint32_t addr, uint32_t chunk) { return addr >> 4 | (chunk >> 4) << 16; }
constexpr uint32_t kOperandHigh = 1024u >> 4 | 1u << 14 | 2u << 29;
// kind::f16, sums in 32 bits; both operands bf16, or both f16
__host__ __device__ constexpr uint32_t instruction(bool bf16, bool a_along_m, bool b_along_n, int m, int n) {
  return 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (a_along_m ? 1u : 0u) << 15 | (b_along_n ? 1u : 0u) << 16 |
         (uint32_t)(n / 8) << 17 | (uint32_t)(m / 16) << 24;
}
template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t instr, bool add) {
  if (CG == 1)
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(instr), "r"((uint32_t)add), "r"(kOperandHigh) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], x, y, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(instr), "r"((uint32_t)add), "r"(kOperandHigh) : "memory");
}
// the barrier (CG == 2: of both CTAs of the pair) gets an arrival when all matrix instructions so far are complete
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
}

}  // namespace cxt
