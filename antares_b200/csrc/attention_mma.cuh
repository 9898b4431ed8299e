// What the prompt attention kernels use of the 5th-generation tensor cores: descriptors, bounded waits, MMAs issued by one
// elected thread, tensor memory loads and stores.
#pragma once
#include "common.cuh"

namespace ab200 {

constexpr unsigned AP_WAIT_POLLS = 1u << 22;

__device__ __forceinline__ uint32_t ap_smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 128-byte-swizzled operand (rows of 128 B, atoms of 8 rows = 1024 B, stride between atoms 1024 B).  lead: bytes
// between blocks of 64 elements along MN for an MN-major operand (unused, 1 unit, for a K-major one).
__device__ __forceinline__ uint64_t ap_desc(uint32_t addr, uint32_t lead_bytes) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)((lead_bytes >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

__device__ __forceinline__ bool ap_wait(uint32_t bar, unsigned parity, unsigned polls = AP_WAIT_POLLS) {
  for (unsigned i = 0; i < polls; ++i) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}
__device__ __forceinline__ void ap_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// The whole warp runs the issuing loop and only these instructions are one thread's: in a divergent branch every
// descriptor would have to be moved into uniform registers on its own.
__device__ __forceinline__ void ap_commit(uint32_t bar) {
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar) : "memory");
}
// D (+)= A.B, A in shared memory (ss) or tensor memory (ts)
__device__ __forceinline__ void ap_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b),
      "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void ap_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b),
      "r"(idesc), "r"(accumulate)
      : "memory");
}
#define AP_R16(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7]), \
    "=r"(r[o + 8]), "=r"(r[o + 9]), "=r"(r[o + 10]), "=r"(r[o + 11]), "=r"(r[o + 12]), "=r"(r[o + 13]), "=r"(r[o + 14]), "=r"(r[o + 15])
#define AP_I16(r) "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), \
    "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
// 32 columns of this warp's 32 lanes; the caller waits
__device__ __forceinline__ void ap_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : AP_R16(r, 0), AP_R16(r, 16)
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void ap_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];" : AP_R16(r, 0) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void ap_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::AP_I16(r), "r"(taddr) : "memory");
}
__device__ __forceinline__ void ap_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ap_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ap_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace ab200
