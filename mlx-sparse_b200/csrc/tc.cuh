// Thin wrappers of the PTX that feeds the sm_100a tensor cores: mbarriers, TMA
// tile loads, tensor memory, and tcgen05.mma with operands in shared or tensor
// memory. All for cta_group::1.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace msx {
namespace tc {

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---- mbarriers -----------------------------------------------------------------
__device__ __forceinline__ void bar_init(uint64_t *bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(ok)
               : "r"(smem_addr(bar)), "r"(parity)
               : "memory");
  return ok != 0;
}

__device__ __forceinline__ bool bar_test(uint64_t *bar, uint32_t parity) {  // does not wait
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(ok)
               : "r"(smem_addr(bar)), "r"(parity)
               : "memory");
  return ok != 0;
}

// What a wait goes by: `polls` tries at once, then until `limit_ns` have passed,
// far beyond any run of these kernels. A wait that gives up sets the device's
// error flag and the CTA's `stop`, which makes every other wait of the CTA give up
// too, so that all warps reach the kernel's end. A limit of 0 (for tests) gives up
// wherever a barrier is not passed already.
struct Watch {
  int *error;
  unsigned long long limit_ns;
  int polls;
};
constexpr long long kWaitNs = 20ll * 1000 * 1000 * 1000;
constexpr unsigned long long kSettleNs = 1000ull * 1000 * 1000;
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
static __device__ __noinline__ bool bar_wait_slow(uint64_t *bar, uint32_t parity, volatile int *stop, const Watch *w) {
  const unsigned long long begin = now_ns(), limit = w->limit_ns;
  while (!(limit ? bar_try(bar, parity) : bar_test(bar, parity))) {
    if (*stop) return false;
    if (now_ns() - begin >= limit) {
      *stop = 1;
      *w->error = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, volatile int *stop, const Watch *w) {
  if (bar_test(bar, parity)) return true;
#pragma unroll 1
  for (int i = 0; i < w->polls; ++i)
    if (bar_try(bar, parity)) return true;
  return bar_wait_slow(bar, parity, stop, w);
}

// The same by a whole warp, which goes on or gives up as one.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *stop, const Watch *w) {
  return __all_sync(~0u, bar_wait(bar, parity, stop, w));
}

// After a wait gave up: copies and products that were issued end by themselves,
// and must have ended before the CTA's memory goes away. Waits, whatever `stop`
// says and a second at most, until the barrier has passed the phase `parity`. Of a
// barrier that copies arrive at, that is the phase armed last: a bit that starts as
// 1, which a new barrier has passed, and turns with each arming.
static __device__ __noinline__ void bar_settle(uint64_t *bar, uint32_t parity) {
  const unsigned long long begin = now_ns();
  while (!bar_try(bar, parity) && now_ns() - begin < kSettleNs) {
  }
}

// ---- TMA -----------------------------------------------------------------------
__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          smem_addr(dst)),
      "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// Untiled: both addresses 16-byte aligned, a multiple of 16 bytes.
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_addr(dst)),
               "l"(src), "r"(bytes), "r"(smem_addr(bar))
               : "memory");
}

// ---- tensor memory -------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t *dst, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this warp's 32 lanes, a register for each column.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
// Keeps the compiler from using loaded registers before the wait above it.
__device__ __forceinline__ void tie32(uint32_t *r) {
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tie16(uint32_t *r) {
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// ---- matrix products -------------------------------------------------------------
// Shared-memory operand tiles come from TMA boxes of 64 16-bit elements (128
// bytes, 128-byte swizzle) by some rows: row r of a box is at r * 128 bytes, 8
// rows make the 1024-byte swizzle atom.
//  K-major  (the box's 64 elements run along K): atoms along M/N every 1024
//           bytes; 16 elements of K are 32 bytes further on.
//  MN-major (the box's 64 elements run along M/N): atoms along K every 1024
//           bytes, the next 64 of M/N `box_bytes` further; 16 rows of K are
//           2048 bytes further on.
// A descriptor's upper word is the same for all (atoms 1024 bytes apart); the
// lower holds the address and the distance of M/N boxes, and steps along K add
// to it.
constexpr uint32_t kDescHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_k_major(uint32_t addr) { return addr >> 4 | 1u << 16; }
__device__ __forceinline__ uint32_t desc_mn_major(uint32_t addr, uint32_t box_bytes) {
  return addr >> 4 | (box_bytes >> 4) << 16;
}

// Instruction descriptor of kind::f16 with fp32 accumulation; both operands are
// of one type. `a_mn` / `b_mn`: that operand is MN-major.
__host__ __device__ constexpr uint32_t mma_desc(bool bf16, int m, int n, bool a_mn, bool b_mn) {
  return 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (a_mn ? 1u : 0u) << 15 | (b_mn ? 1u : 0u) << 16 |
         (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
// a, b: lower descriptor words; mma_ts: a is an address in tensor memory. The
// whole warp runs these with the same operands, which keeps them in uniform
// registers; the one lane with `leader` issues.
__device__ __forceinline__ void mma_ss(bool leader, uint32_t d, uint32_t a, uint32_t b, uint32_t desc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 x, y;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %6, 0;\n"
      " mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(desc), "r"((uint32_t)accumulate), "r"(kDescHigh), "r"((uint32_t)leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts(bool leader, uint32_t d, uint32_t a, uint32_t b, uint32_t desc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 y;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %6, 0;\n"
      " mov.b64 y, {%2, %5};\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(desc), "r"((uint32_t)accumulate), "r"(kDescHigh), "r"((uint32_t)leader)
      : "memory");
}
// Arrives at `bar` when every product issued so far by this thread is done.
__device__ __forceinline__ void mma_commit(bool leader, uint64_t *bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_addr(bar)),
      "r"((uint32_t)leader)
      : "memory");
}

}  // namespace tc
}  // namespace msx
