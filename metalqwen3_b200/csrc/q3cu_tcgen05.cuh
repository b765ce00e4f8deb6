// q3cu_tcgen05.cuh -- the tensor-core instructions (tcgen05) the kernels share.
#pragma once

#include "q3cu_device.cuh"

namespace q3 {

// Shared-memory matrix descriptor of a K-major, 128-byte-swizzled operand:
// start address / 16, leading offset 1 (unused with the swizzle), stride 1024 B
// between 8-row groups (/16), descriptor version 1, layout SWIZZLE_128B (2).
__device__ __forceinline__ uint64_t tc_sdesc(uint32_t smem_addr) {
    return uint64_t((smem_addr & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 :: "r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// All 512 tensor-memory columns, for a kernel with one CTA per SM (one whole warp calls each).
__device__ __forceinline__ void tc_alloc512(uint32_t *smem_base) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_addr(smem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_free512(uint32_t base) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(base), "r"(512) : "memory");
}

// Shared-memory matrix descriptor of an MN-major, 128-byte-swizzled operand of
// bf16: rows of 64 M/N elements (128 B), one row per K index; stride 1024 B
// between groups of 8 rows along K, `mn_stride` bytes between 64-element blocks
// along M/N.
__device__ __forceinline__ uint64_t tc_sdesc_mn(uint32_t smem_addr, uint32_t mn_stride) {
    return uint64_t((smem_addr & 0x3FFFFu) >> 4) | (uint64_t(mn_stride >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

// One lane of a converged warp, always the same, known to the compiler as such: what it issues keeps its operands in
// uniform registers (under a plain `lane == 0` every operand is moved there first, about 100 cycles per product).
__device__ __forceinline__ bool tc_elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// D (tensor memory, f32) (+)= A * B, bf16 operands, K = 16.  A from shared
// memory or, packed two to a column, from tensor memory; B from shared memory.
__device__ __forceinline__ void tc_mma_bf16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_mma_bf16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr) : "memory");
}
// The wait, with the loaded registers as operands: nothing that reads them can
// be scheduled before it.
__device__ __forceinline__ void tc_wait_ld16(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :: "memory");
}
// 32 columns of this warp's 32 lanes to or from registers (thread = lane).  A load's registers hold the values only
// after tc_wait_ld32.
#define TC_R32(v, o) \
    o(v[0]), o(v[1]), o(v[2]), o(v[3]), o(v[4]), o(v[5]), o(v[6]), o(v[7]), o(v[8]), o(v[9]), o(v[10]), o(v[11]), \
    o(v[12]), o(v[13]), o(v[14]), o(v[15]), o(v[16]), o(v[17]), o(v[18]), o(v[19]), o(v[20]), o(v[21]), o(v[22]), \
    o(v[23]), o(v[24]), o(v[25]), o(v[26]), o(v[27]), o(v[28]), o(v[29]), o(v[30]), o(v[31])
#define TC_LIST32 \
    "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28," \
    "%29,%30,%31}"
__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 " TC_LIST32 ", [%32];"
                 : TC_R32(v, "=r") : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_wait_ld32(uint32_t *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : TC_R32(v, "+r") :: "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], " TC_LIST32 ";" :: TC_R32(v, "r"), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 :: "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
                    "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tc_st8(uint32_t taddr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
                 :: "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(taddr)
                 : "memory");
}

}  // namespace q3
