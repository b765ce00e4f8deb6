// q3cu_mma.cuh -- warp-wide matrix products of a few rows (mma.sync) and their operands.
#pragma once

#include "q3cu_paged.cuh"

namespace q3 {

// d += a b.  The tensor cores cut the sum where binary32 would round it, so a long chain into one accumulator drifts
// towards zero (2e-6 of the result after some hundred products); what is summed over many goes through a fresh
// accumulator for a few products and is added by an ordinary addition (add_to).
__device__ __forceinline__ void add_to(float (&sum)[4], const float (&part)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += part[i];
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// An 8 x 8 block of 16-bit values, a lane (g, t) holding columns 2 t and 2 t + 1 of row g, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ float4 lds4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
// Two floats as PARTS bf16 each, every one the nearest to what the ones before leave: 8 bits of mantissa a part, so
// two parts are within 2^-17 of the float and three within 2^-25.
template <int PARTS>
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t (&part)[PARTS]) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        part[i] = pack_bf16(x, y);
        x -= __uint_as_float(part[i] << 16);
        y -= __uint_as_float(part[i] & 0xffff0000u);
    }
}

// A float as its nearest tf32 (11 bits) and the rest, which is exact and below half a step of the first; the tensor
// cores cut the rest to 11 bits of its own: 2^-22 of the float.  (A NaN may leave `hi`, not `lo`.)
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}

}  // namespace q3
