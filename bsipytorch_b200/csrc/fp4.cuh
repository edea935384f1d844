// Values of the 4-bit formats, shared by their packer and their product.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace bsi {
namespace {

// The value of an e4m3 byte (exact; the NaN byte does not occur in scales that the packer writes).
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
    uint32_t h;
    const uint16_t pair = static_cast<uint16_t>(byte);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(pair));
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xFFFFu)));
}

// The values of eight codes, the lowest nibble first.
__device__ __forceinline__ void e2m1_values(uint32_t codes, float* v) {
    uint32_t h[4];
    asm("{\n.reg .b8 b0, b1, b2, b3;\n"
        "mov.b32 {b0, b1, b2, b3}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

}  // namespace
}  // namespace bsi
