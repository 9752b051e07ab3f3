// kv4_codes.cuh -- 4-bit codes as f16 numbers.
#pragma once

#include <cstdint>
#include <cuda_fp16.h>

namespace b200 {

// (x & mask) | bits in one instruction (written with operators it takes two).
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
    return r;
}

// Nibbles k and k + 4 of w (k = 0 .. 3) as f16 pairs of code - LESS, exactly: 0x640u is 1024 + u, 0x54u0 is 64 + u.
template <int LESS = 8>
__device__ __forceinline__ void codes4(uint32_t w, uint32_t (&p)[4]) {
    const __half2 far = __half2half2(__ushort_as_half(0x6400 + LESS)), near = __half2half2(__ushort_as_half(0x5400 + 16 * LESS));
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t x = k ? w >> 8 : w;
        const uint32_t lo = and_or(x, 0x000f000fu, 0x64006400u), hi = and_or(x, 0x00f000f0u, 0x54005400u);
        const __half2 a = __hsub2(*reinterpret_cast<const __half2 *>(&lo), far), b = __hsub2(*reinterpret_cast<const __half2 *>(&hi), near);
        p[2 * k] = *reinterpret_cast<const uint32_t *>(&a);
        p[2 * k + 1] = *reinterpret_cast<const uint32_t *>(&b);
    }
}

}  // namespace b200
