// The tcgen05 tensor cores, tensor memory and mbarriers, as the attention kernels use them (one CTA, 128 rows a product).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace pf {

__device__ __forceinline__ uint32_t shared_of(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t *bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_of(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_of(bar)) : "memory");
}
// Waits for the phase of `parity`; false after about two seconds, or as soon as another thread has given up.
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, int *stalled) {
  uint64_t start = 0;
  for (uint32_t i = 1;; ++i) {
    uint32_t done;
    asm volatile("{.reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p;}"
                 : "=r"(done)
                 : "r"(shared_of(bar)), "r"(parity)
                 : "memory");
    if (done) return true;
    if ((i & 255) == 0) {
      uint64_t now;
      asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
      if (start == 0) start = now;
      if (*(volatile int *)stalled || now - start > 2000000000ull) {
        *(volatile int *)stalled = 1;
        return false;
      }
    }
  }
}
// The same for a warp whose next instructions need all of its lanes.
__device__ __forceinline__ bool bar_wait_warp(uint64_t *bar, uint32_t parity, int *stalled) {
  return __all_sync(0xffffffffu, bar_wait(bar, parity, stalled));
}

__device__ __forceinline__ void fence_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_of(bar)) : "memory");
}
// An operand in shared memory.  Contracted along its rows: `stride` bytes between groups of eight rows.  Contracted down its
// rows: `stride` between groups of eight rows and `lead` between panels of a swizzle's width; without a swizzle (16-byte
// chunks, eight of them 128 bytes) the two change places.
constexpr uint32_t kNoSwizzle = 0, kSwizzle128 = 2, kSwizzle64 = 4;
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead, uint32_t stride, uint32_t swizzle) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((lead >> 4) & 0x3fff) << 16 | (uint64_t)((stride >> 4) & 0x3fff) << 32 |
         (uint64_t)1 << 46 | (uint64_t)swizzle << 61;
}
// 128 rows, n columns, fp32 sums; f16 operands or (the same codes) e4m3 ones.  `down`: contracted down its rows.
__host__ __device__ constexpr uint32_t shape_of(int n, bool a_down, bool b_down) {
  return 1u << 4 | (a_down ? 1u << 15 : 0u) | (b_down ? 1u << 16 : 0u) | (uint32_t)(n / 8) << 17 | (uint32_t)(128 / 16) << 24;
}
__host__ __device__ constexpr uint32_t shape_f16(int n, bool b_down) { return shape_of(n, false, b_down); }
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t shape_, bool add) {
  asm volatile(
      "{.reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;}" ::"r"(d), "l"(a),
      "l"(b), "r"(shape_), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t shape_, bool add) {
  asm volatile(
      "{.reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;}" ::"r"(d), "r"(a),
      "l"(b), "r"(shape_), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_e4m3_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t shape_, bool add) {
  asm volatile(
      "{.reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;}" ::"r"(d), "l"(a),
      "l"(b), "r"(shape_), "r"((uint32_t)add)
      : "memory");
}
#define PF_R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define PF_R16(r, i) PF_R4(r, i), PF_R4(r, i + 4), PF_R4(r, i + 8), PF_R4(r, i + 12)
#define PF_I4(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
#define PF_I16(r, i) PF_I4(r, i), PF_I4(r, i + 4), PF_I4(r, i + 8), PF_I4(r, i + 12)
__device__ __forceinline__ void load32(uint32_t (&r)[32], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : PF_R16(r, 0), PF_R16(r, 16)
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void load16(uint32_t (&r)[16], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : PF_R16(r, 0)
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void store16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      PF_I16(r, 0)
      : "memory");
}

// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpair(uint64_t x, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

}  // namespace pf
