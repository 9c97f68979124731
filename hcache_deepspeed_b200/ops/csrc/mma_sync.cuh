// Warp-level matrix instructions for kernels whose tensor work is a small part of their time.
#pragma once
#include <stdint.h>

namespace hds {

// c (16 x 8, fp32) += a (16 x 16) b (16 x 8), 16-bit operands. Lane = 4 * g + t: a0 row g, a1 row g + 8 at k 2t, 2t + 1; a2, a3 the same rows
// at k 2t + 8, 2t + 9; b0, b1 column g at those k; c[0], c[1] row g, columns 2t, 2t + 1; c[2], c[3] row g + 8.
template <bool kBf16>
__device__ __forceinline__ void mma_m16n8k16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (kBf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace hds
