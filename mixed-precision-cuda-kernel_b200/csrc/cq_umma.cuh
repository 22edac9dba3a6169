// tcgen05 and TMA instructions of the attention kernels for prompts, and bounded waits.
#pragma once

#include <cuda.h>

#include "cq_common.cuh"

namespace umma {

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity), "r"(20000u) : "memory");
  return ok != 0;
}
// Bounded wait: after two seconds of the device's clock (or at once where another wait of the CTA ran out) it gives up, notes
// that in *gone and in the status word, and returns false; the CTA then runs on to its end.
__device__ __forceinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, volatile int* gone, uint32_t* status) {
  unsigned long long t0 = 0;
  for (uint32_t it = 0; it < (1u << 26); ++it) {
    if (bar_try(bar, parity)) return true;
    if (*gone) return false;
    if ((it & 15u) == 15u) {
      unsigned long long t1;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1));
      if (t0 == 0) t0 = t1;
      else if (t1 - t0 > 2000000000ull) break;
    }
  }
  *gone = 1;
  if (status) atomicOr(status, (uint32_t)CQ_ERR_DEVICE_TIMEOUT);
  return false;
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* gone, uint32_t* status) {
  if (bar_try(bar, parity)) return true;
  return bar_wait_slow(bar, parity, gone, status);
}
// the same by a whole warp: all of its lanes go the same way
__device__ __forceinline__ bool bar_wait_warp(uint32_t bar, uint32_t parity, volatile int* gone, uint32_t* status) {
  return __all_sync(0xffffffffu, bar_wait(bar, parity, gone, status));
}
// one lane of a converged warp; what it alone does with values that are the same in all lanes stays on the uniform datapath
__device__ __forceinline__ bool elected() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void alloc(uint32_t* to, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_at(to)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc(uint32_t at, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols) : "memory");
}
// arrives on the barrier when the MMAs that this thread has issued are done
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// D (tensor memory, 128 lanes) (+)= A . B, fp16 in, fp32 out: A from shared or from tensor memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, uint32_t add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"(add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t shape, uint32_t add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(shape), "r"(add) : "memory");
}
// instruction descriptor: fp16 operands, fp32 sums, m x n; b_rows: B's rows (the sums' direction) lie one behind the other
__host__ __device__ constexpr uint32_t shape_of(int m, int n, bool b_rows) {
  return (1u << 4) | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Operand in shared memory with the 128-byte swizzle: rows of 64 halves, eight of them 1024 bytes; wide: bytes between
// stretches of 64 columns where the operand's columns lie along the rows (0 for the other orientation).
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t wide) {
  return (uint64_t)((at >> 4) & 0x3FFFu) | ((uint64_t)((wide >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
#define CQ_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define CQ_I8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
#define CQ_B8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
// 32 columns of this warp's lanes
__device__ __forceinline__ void load32(uint32_t at, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : CQ_R8(r, 0), CQ_R8(r, 8), CQ_R8(r, 16), CQ_R8(r, 24) : "r"(at) : "memory");
}
__device__ __forceinline__ void load16(uint32_t at, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : CQ_R8(r, 0), CQ_R8(r, 8) : "r"(at) : "memory");
}
__device__ __forceinline__ void store32(uint32_t at, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
               ::"r"(at), CQ_I8(r, 0), CQ_I8(r, 8), CQ_I8(r, 16), CQ_I8(r, 24) : "memory");
}
__device__ __forceinline__ void store16(uint32_t at, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               ::"r"(at), CQ_I8(r, 0), CQ_I8(r, 8) : "memory");
}
// Results of load32 may be used from here on: waits for them, and keeps the compiler from using them before.
template <int N> __device__ __forceinline__ void wait_load(uint32_t* r) {
  static_assert(N == 16 || N == 32, "");
  if constexpr (N == 16) asm volatile("tcgen05.wait::ld.sync.aligned;" : CQ_B8(r, 0), CQ_B8(r, 8)::"memory");
  else asm volatile("tcgen05.wait::ld.sync.aligned;" : CQ_B8(r, 0), CQ_B8(r, 8), CQ_B8(r, 16), CQ_B8(r, 24)::"memory");
}
__device__ __forceinline__ void wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// a box of a tensor map to shared memory
__device__ __forceinline__ void tma(uint32_t to, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               ::"r"(to), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}

}  // namespace umma
