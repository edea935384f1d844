// Values of the 4-bit formats, shared by their packer and their product.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp4.h>

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

// The values of the two codes of a byte, the lower nibble first. A byte by itself, through CUDA's own conversion: with a word taken apart
// into four bytes in one asm block the assembler of CUDA 12.9 gave zeros for its lower bytes when the word was a widened half word.
__device__ __forceinline__ float2 e2m1_values(uint32_t byte) {
    return __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(byte), __NV_E2M1)));
}

}  // namespace
}  // namespace bsi
