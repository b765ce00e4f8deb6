// q3cu_f16.cuh -- Q8_0 codes and lifted operands as f16, for products whose operands have more than bf16's 8 bits.
#pragma once

#include "q3cu_device.cuh"

namespace q3 {

// Two bytes of `codes` (already with the top bits flipped: code + 128), by a selector that puts 0x64 above each, as f16.
__device__ __forceinline__ uint32_t codes_f16(uint32_t codes, uint32_t pick) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(__byte_perm(codes, 0x64646464u, pick)), "r"(0x64806480u));  // - 1152
    return r;
}
// Two bytes of `codes`, in the lower halves of the 16-bit words of b, as f16 over 128: 8 + (code + 128) / 128, whose sign bit
// a logical operation flips and whose upper byte it puts there, less 9.
__device__ __forceinline__ uint32_t codes_f16_128th(uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"((b & 0x00ff00ffu) ^ 0x48804880u), "r"(0x48804880u));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 f16_pair(uint32_t x) {
    float2 v;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(v.x), "=f"(v.y) : "r"(x));
    return v;
}
// x and y as PARTS f16 each, every one the nearest to what the ones before leave.
template <int PARTS>
__device__ __forceinline__ void split_f16(float x, float y, uint32_t (&part)[PARTS]) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        part[i] = pack_f16(x, y);
        if (i + 1 < PARTS) {
            const float2 v = f16_pair(part[i]);
            x -= v.x;
            y -= v.y;
        }
    }
}
// a * b, each half rounded.
__device__ __forceinline__ uint32_t mul_f16(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// The power of two that brings a magnitude (as binary32's bits) to [2^14, 2^15), no more than 2^126, and its inverse.
__device__ __forceinline__ float lift(uint32_t bits) { return __uint_as_float(uint32_t(min(268 - int(bits >> 23), 253)) << 23); }
__device__ __forceinline__ float lift_back(uint32_t bits) {
    return __uint_as_float(uint32_t(254 - min(268 - int(bits >> 23), 253)) << 23);
}

}  // namespace q3
