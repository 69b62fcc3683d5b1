// What the paged cache's attention kernels share: wrappers of instructions, bounded waits, operands in shared memory.
#pragma once
#include "mz_paged.cuh"

namespace mzp {
constexpr float LOG2E = 1.4426950408889634f;
constexpr int SPIN_LIMIT = 1000000;              // looks of a wait before it gives up

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(s));
  return d;
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t warp_max_u32(uint32_t v) { uint32_t r; asm("redux.sync.max.u32 %0, %1, 0xffffffff;" : "=r"(r) : "r"(v)); return r; }
__device__ __forceinline__ float warp_max(float v) { float r; asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 book128(uint32_t a) {      // constant after the set-up
  uint4 v;
  asm("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
// the 64 codes of a row: a whole sector by one thread, read once
__device__ __forceinline__ void ldg256(uint32_t (&v)[8], const void* p) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "l"(p));
}
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void fence_operands() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(n) : "memory"); }
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}\n"
               : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
// Waits for the phase of this parity.  Who gives up says so before it goes on; the others notice.
__device__ __forceinline__ void bar_wait(uint32_t bar, uint32_t parity, volatile int* s_failed) {
#ifdef MZ_BOUNDS
  if (*s_failed) return;                         // a test makes every wait run out
#endif
  for (int it = 0; it < SPIN_LIMIT; ++it) {
    if (bar_test(bar, parity)) return;
    if ((it & 63) == 63 && *s_failed) return;
  }
  *s_failed = 1;
}
// shared-memory operand, not swizzled, major along the kept dimension: cores of 8 rows x 16 bytes, 128 bytes apart along the reduction,
// `chunk` bytes apart along the kept dimension
__device__ __forceinline__ uint64_t descriptor(uint32_t sa, uint32_t chunk) {
  return (uint64_t)((sa >> 4) & 0x3FFF) | (128ull >> 4) << 16 | (uint64_t)(chunk >> 4) << 32 | 1ull << 46;
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }      // -126 <= e <= 127

// pairs of fp32 operations
__device__ __forceinline__ void add2(float& a0, float& a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void fma2(float& c0, float& c1, float a0, float a1, float f) {      // c += a * f
  asm("{\n\t.reg .b64 a, c, f;\n\tmov.b64 c, {%0, %1};\n\tmov.b64 a, {%2, %3};\n\tmov.b64 f, {%4, %4};\n\tfma.rn.f32x2 c, a, f, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "+f"(c0), "+f"(c1) : "f"(a0), "f"(a1), "f"(f));
}
}  // namespace mzp
