// Microscaled 4-bit floating point: matrices rounded to e2m1 elements under block scales, and back.
//
//   mxfp4   blocks of 32 along a row, scale 2^(floor(log2 amax) - 2) held as e8m0; larger quotients saturate at 6
//   nvfp4   blocks of 16, scale e4m3(amax / (6 g)) held as e4m3, under a power of two g per row, the smallest with
//           448 * 6 * g >= the row's largest magnitude (at least 2^-100; 1 for a row of zeros)
//
// An element is the e2m1 value nearest to x / scale, ties to the even code, saturating. g is a power of two per row, not one float32
// per tensor, so that a row's values depend on that row alone and one pass over it is enough; scale * g is exact in float32, and so
// is every comparison behind the rounding: the quotient is IEEE's (a product with the rounded reciprocal and one residual step), and
// where it is a border between two codes it is exactly that border.
//
// Layout. Codes: two to a byte, the lower nibble first, rows `ld` bytes apart (a multiple of 16 >= K / 2 rounded up to 16 bytes),
// zero behind column K. Scales: as the tensor cores take them, 512 bytes for 128 rows x 4 scales: byte
// (r % 32) * 16 + (r % 128) / 32 * 4 + j of tile (r / 128, group), groups of 4 consecutive blocks; as many groups as ceil(K / 256) * 256
// columns have, those behind K zero.
#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fp4.cuh"

namespace bsi {
namespace {

constexpr int kUnit = 16;            // elements of a thread at a time
constexpr int kHeld = 2;             // units that a thread keeps between the search for the row's maximum and the rounding
constexpr int kMaxThreads = 512;

__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// 16 elements as they lie in memory, zero behind column K.
template <typename T>
struct Unit {
    static constexpr int kVecs = kUnit * sizeof(T) / 16;
    uint4 u[kVecs];

    __device__ __forceinline__ void load(const T* row, int64_t c, int64_t K, bool vector) {
        if (vector && c + kUnit <= K) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) u[i] = *reinterpret_cast<const uint4*>(row + c + i * (16 / sizeof(T)));
        } else {
            T* e = reinterpret_cast<T*>(u);
#pragma unroll
            for (int i = 0; i < kUnit; ++i) e[i] = c + i < K ? row[c + i] : static_cast<T>(0.0f);
        }
    }
    // Largest magnitude as a float32's bits: the order of non-negative floats, infinities and NaN above all.
    __device__ __forceinline__ uint32_t magnitude() const {
        if constexpr (sizeof(T) == 4) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) m = max(max(m, max(u[i].x & 0x7FFFFFFFu, u[i].y & 0x7FFFFFFFu)), max(u[i].z & 0x7FFFFFFFu, u[i].w & 0x7FFFFFFFu));
            return m;
        } else {
            // both halves of a word at once: a sign bit less, 16-bit patterns are in the order of their magnitudes
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                m = __vmaxu2(m, __vmaxu2(u[i].x & 0x7FFF7FFFu, u[i].y & 0x7FFF7FFFu));
                m = __vmaxu2(m, __vmaxu2(u[i].z & 0x7FFF7FFFu, u[i].w & 0x7FFF7FFFu));
            }
            const unsigned short top = static_cast<unsigned short>(max(m & 0xFFFFu, m >> 16));
            return __float_as_uint(widen(*reinterpret_cast<const T*>(&top)));
        }
    }
    __device__ __forceinline__ void values(float (&x)[kUnit]) const {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const uint32_t word[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 4) {
                    x[i * 4 + j] = __uint_as_float(word[j]);
                } else {
                    const T* p = reinterpret_cast<const T*>(&word[j]);
                    x[i * 8 + j * 2] = widen(p[0]);
                    x[i * 8 + j * 2 + 1] = widen(p[1]);
                }
            }
        }
    }
};

// Two e2m1 codes, lo in the lower nibble; four such bytes.
__device__ __forceinline__ uint32_t codes8(const float* v) {
    uint32_t r;
    asm("{\n.reg .b8 b0, b1, b2, b3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
        "mov.b32 %0, {b0, b1, b2, b3};\n}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// x / scale correctly rounded where the quotient is no smaller than 2^-100 (a smaller one is no border's neighbour), two at a time: the
// residual of the first guess is exact in a fused multiply-add, and one step with a correctly rounded reciprocal ends at the rounded
// quotient (Markstein's theorem; the scale's significand has four bits).
__device__ __forceinline__ void quotients(float& x, float& y, float scale, float inv) {
    unsigned long long v, s, i, q, r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    asm("mov.b64 %0, {%1, %1};" : "=l"(s) : "f"(-scale));
    asm("mov.b64 %0, {%1, %1};" : "=l"(i) : "f"(inv));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q) : "l"(v), "l"(i));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(q), "l"(s), "l"(v));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(q) : "l"(r), "l"(i), "l"(q));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(q));
}

__device__ __forceinline__ uint32_t e4m3_byte(float v) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
    return r & 0xFFu;
}

// A power of two as a float32, exponents of -149 and more.
__device__ __forceinline__ float power_of_two(int e) {
    return e >= -126 ? __uint_as_float(static_cast<uint32_t>(e + 127) << 23) : __uint_as_float(1u << (e + 149));
}

// One row a CTA. What bounds it is the matrix's bytes; a row's maximum has to be known before its first code, so a thread keeps up to
// two units as they came (beyond 16384 columns the rest is read again), and what fills the wait are other rows: 64 bytes of a unit's
// row, not 16 float32 values, keep the registers low enough for it (8192 x 4096 bfloat16 nvfp4: 71 us with 92 registers).
template <typename T, bool MX>
__global__ void __launch_bounds__(kMaxThreads, sizeof(T) == 4 ? 2 : 3)
    fp4_quantize_kernel(const T* __restrict__ x, int64_t K, int64_t ldx, int vector, uint8_t* __restrict__ codes, int64_t ld, uint8_t* __restrict__ scales,
                        float* __restrict__ row_scale) {
    __shared__ uint32_t part[kMaxThreads / 32];
    const uint32_t r = blockIdx.x;
    const T* row = x + r * ldx;
    const int units = static_cast<int>((K + 255) / 256 * 16);       // also those whose scales are there without elements
    const int groups = units / (MX ? 8 : 4);
    const int threads = static_cast<int>(blockDim.x);
    float g = 1.0f;
    bool finite = true;
    Unit<T> held[kHeld];
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
        const int u = static_cast<int>(threadIdx.x) + h * threads;
        if (u < units) held[h].load(row, static_cast<int64_t>(u) * kUnit, K, vector != 0);
    }
    if constexpr (!MX) {
        uint32_t top = 0;
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
            if (static_cast<int>(threadIdx.x) + h * threads < units) top = max(top, held[h].magnitude());
        for (int u = static_cast<int>(threadIdx.x) + kHeld * threads; u < units; u += threads) {
            Unit<T> v;
            v.load(row, static_cast<int64_t>(u) * kUnit, K, vector != 0);
            top = max(top, v.magnitude());
        }
        top = __reduce_max_sync(0xFFFFFFFFu, top);
        if (threads > 32) {
            if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
            __syncthreads();
            for (int w = 0; w < threads / 32; ++w) top = max(top, part[w]);
        }
        finite = top < 0x7F800000u;
        if (finite && top != 0) {
            // the smallest e with top <= 2688 * 2^e = 1.3125 * 2^(11 + e)
            const int e = static_cast<int>(top >> 23) - 127 - 11 + ((top & 0x7FFFFFu) > 0x280000u ? 1 : 0);
            g = power_of_two(max(e, -100));
        }
        if (threadIdx.x == 0) row_scale[r] = finite ? g : __uint_as_float(0x7FC00000u);
    }
    uint8_t* crow = codes + r * ld;
    uint8_t* stile = scales + static_cast<int64_t>(r / 128) * groups * 512 + (r % 32) * 16 + (r % 128) / 32 * 4;
    const float six_g = 6.0f * g;
    auto pack = [&](const Unit<T>& unit, int u, bool live) {
        uint32_t m = live ? unit.magnitude() : 0u;
        float scale, inv;
        uint32_t byte;
        if constexpr (MX) {
            m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));            // the block's other half
            // e8m0: the exponent of amax less 2 under the bias of 127; not finite: NaN
            byte = m >= 0x7F800000u ? 255u : static_cast<uint32_t>(max(static_cast<int>(m >> 23) - 2, 0));
            scale = 0.0f;
            inv = byte == 255u ? 0.0f : power_of_two(127 - static_cast<int>(byte));
        } else {
            byte = finite ? e4m3_byte(__fdiv_rn(__uint_as_float(m), six_g)) : 0u;
            scale = e4m3_value(byte) * g;
            inv = byte != 0u ? __frcp_rn(scale) : 0.0f;
        }
        if (!live) return;
        float q[kUnit];
        unit.values(q);
#pragma unroll
        for (int e = 0; e < kUnit; e += 2) {
            if constexpr (MX) {
                q[e] *= inv;
                q[e + 1] *= inv;
            } else {
                quotients(q[e], q[e + 1], scale, inv);
            }
        }
        const uint2 packed = inv != 0.0f ? make_uint2(codes8(q), codes8(q + 8)) : make_uint2(0u, 0u);
        if (static_cast<int64_t>(u) * 8 < ld) *reinterpret_cast<uint2*>(crow + static_cast<int64_t>(u) * 8) = packed;
        if (MX) {
            if ((u & 1) == 0) stile[static_cast<int64_t>(u >> 3) * 512 + ((u >> 1) & 3)] = static_cast<uint8_t>(byte);
        } else {
            stile[static_cast<int64_t>(u >> 2) * 512 + (u & 3)] = static_cast<uint8_t>(byte);
        }
    };
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
        const int u = static_cast<int>(threadIdx.x) + h * threads;
        if (h * threads < units) pack(held[h], u, u < units);
    }
    for (int u0 = kHeld * threads; u0 < units; u0 += threads) {
        const int u = u0 + static_cast<int>(threadIdx.x);
        Unit<T> v;
        if (u < units) v.load(row, static_cast<int64_t>(u) * kUnit, K, vector != 0);
        pack(v, u, u < units);
    }
}

// A thread writes 16 bytes at a time, a warp 512 in a row; a row a CTA. What bounds it is the output's bytes.
template <typename T, bool MX>
__global__ void __launch_bounds__(256) fp4_dequantize_kernel(const uint8_t* __restrict__ codes, int64_t ld, const uint8_t* __restrict__ scales,
                                                             const float* __restrict__ row_scale, int64_t K, T* __restrict__ out, int64_t ldo, int vector) {
    constexpr int kVec = 16 / sizeof(T);         // 4 or 8 elements, 2 or 4 bytes of codes, all of one block
    const uint32_t r = blockIdx.x;
    const int64_t groups = (K + 255) / 256 * (MX ? 2 : 4);
    const uint8_t* crow = codes + r * ld;
    const uint8_t* stile = scales + (r / 128) * groups * 512 + (r % 32) * 16 + (r % 128) / 32 * 4;
    const float g = MX ? 1.0f : row_scale[r];
    T* dst = out + r * ldo;
    const int pieces = static_cast<int>((K + kVec - 1) / kVec);
    for (int i = threadIdx.x; i < pieces; i += 256) {
        const int block = i * kVec / (MX ? 32 : 16);
        const uint32_t byte = stile[static_cast<int64_t>(block >> 2) * 512 + (block & 3)];
        const float scale = MX ? (byte == 255u ? __uint_as_float(0x7FC00000u) : power_of_two(static_cast<int>(byte) - 127)) : e4m3_value(byte) * g;
        using Codes = std::conditional_t<kVec == 4, uint16_t, uint32_t>;
        const uint32_t word = reinterpret_cast<const Codes*>(crow)[i];
        alignas(16) T y[kVec];
#pragma unroll
        for (int e = 0; e < kVec; e += 2) {
            const float2 v = e2m1_values(word >> (4 * e) & 255u);
            y[e] = static_cast<T>(v.x * scale);
            y[e + 1] = static_cast<T>(v.y * scale);
        }
        const int64_t c = static_cast<int64_t>(i) * kVec;
        if (vector && c + kVec <= K) {
            *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(y);
        } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (c + e < K) dst[c + e] = y[e];
        }
    }
}

int check_matrix(const char* what, int format, int dtype, int64_t rows, int64_t K, int64_t ld, const void* codes, const void* scales, const void* row_scale) {
    if (format != BSI_FP4_MX && format != BSI_FP4_NV) {
        set_error("%s: format must be BSI_FP4_MX or BSI_FP4_NV, got %d", what, format);
        return BSI_ERR_INVALID;
    }
    if (dtype != BSI_DTYPE_F32 && dtype != BSI_DTYPE_F16 && dtype != BSI_DTYPE_BF16) {
        set_error("%s: dtype must be a BSI_DTYPE_* code, got %d", what, dtype);
        return BSI_ERR_INVALID;
    }
    if (rows < 0 || K < 1 || rows > 0x7FFFFFFFll || K > (1ll << 30) || ld % 16 != 0 || ld < (K + 31) / 32 * 16) {
        set_error("%s: %lld rows of %lld, codes %lld bytes apart", what, static_cast<long long>(rows), static_cast<long long>(K), static_cast<long long>(ld));
        return BSI_ERR_INVALID;
    }
    if (rows > 0 && (codes == nullptr || scales == nullptr || (format == BSI_FP4_NV && row_scale == nullptr) ||
                     (reinterpret_cast<uintptr_t>(codes) & 15u) || (reinterpret_cast<uintptr_t>(scales) & 15u) || (reinterpret_cast<uintptr_t>(row_scale) & 3u))) {
        set_error("%s: null or misaligned codes, scales or row scales", what);
        return BSI_ERR_INVALID;
    }
    return BSI_OK;
}

template <typename T>
int launch_quantize(const void* x, int64_t rows, int64_t K, int64_t ldx, int format, uint8_t* codes, int64_t ld, uint8_t* scales, float* row_scale,
                    cudaStream_t stream) {
    const int vector = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (rows == 1 || ldx * sizeof(T) % 16 == 0);
    const int64_t units = (K + 255) / 256 * 16;
    // two units a thread, or one where the rows do not fill the GPU
    const int64_t wanted = rows > 4 * sm_count() ? (units + 1) / 2 : units;
    const int threads = static_cast<int>(std::min<int64_t>(kMaxThreads, (wanted + 31) / 32 * 32));
    const T* p = static_cast<const T*>(x);
    if (format == BSI_FP4_MX)
        fp4_quantize_kernel<T, true><<<static_cast<unsigned>(rows), threads, 0, stream>>>(p, K, ldx, vector, codes, ld, scales, row_scale);
    else
        fp4_quantize_kernel<T, false><<<static_cast<unsigned>(rows), threads, 0, stream>>>(p, K, ldx, vector, codes, ld, scales, row_scale);
    return check_launch("fp4_quantize launch");
}

template <typename T>
int launch_dequantize(const uint8_t* codes, int64_t ld, const uint8_t* scales, const float* row_scale, int64_t rows, int64_t K, int format, void* out,
                      int64_t ldo, cudaStream_t stream) {
    const int vector = (reinterpret_cast<uintptr_t>(out) & 15u) == 0 && (rows == 1 || ldo * sizeof(T) % 16 == 0);
    const unsigned grid = static_cast<unsigned>(rows);
    T* p = static_cast<T*>(out);
    if (format == BSI_FP4_MX)
        fp4_dequantize_kernel<T, true><<<grid, 256, 0, stream>>>(codes, ld, scales, row_scale, K, p, ldo, vector);
    else
        fp4_dequantize_kernel<T, false><<<grid, 256, 0, stream>>>(codes, ld, scales, row_scale, K, p, ldo, vector);
    return check_launch("fp4_dequantize launch");
}

}  // namespace
}  // namespace bsi

extern "C" int64_t bsi_b200_fp4_scale_bytes(int64_t rows, int64_t K, int format) {
    if (rows < 0 || K < 1 || (format != BSI_FP4_MX && format != BSI_FP4_NV)) return -1;
    return (rows + 127) / 128 * ((K + 255) / 256 * (format == BSI_FP4_MX ? 2 : 4)) * 512;
}

extern "C" int bsi_b200_fp4_quantize(const void* x, int dtype, int64_t rows, int64_t K, int64_t ldx, int format, uint8_t* codes, int64_t ld,
                                     uint8_t* scales, float* row_scale, bsi_stream_t stream) {
    using namespace bsi;
    int rc = check_matrix("fp4_quantize", format, dtype, rows, K, ld, codes, scales, row_scale);
    if (rc != BSI_OK) return rc;
    if (rows == 0) return BSI_OK;
    if (x == nullptr || reinterpret_cast<uintptr_t>(x) % (dtype == BSI_DTYPE_F32 ? 4 : 2) != 0) return fail(BSI_ERR_INVALID, "fp4_quantize: null or misaligned x");
    rc = require_sm100();
    if (rc != BSI_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == BSI_DTYPE_F32 ? launch_quantize<float>(x, rows, K, ldx, format, codes, ld, scales, row_scale, s)
           : dtype == BSI_DTYPE_F16 ? launch_quantize<__half>(x, rows, K, ldx, format, codes, ld, scales, row_scale, s)
                                    : launch_quantize<__nv_bfloat16>(x, rows, K, ldx, format, codes, ld, scales, row_scale, s);
}

extern "C" int bsi_b200_fp4_dequantize(const uint8_t* codes, int64_t ld, const uint8_t* scales, const float* row_scale, int64_t rows, int64_t K,
                                       int format, void* out, int dtype, int64_t ldo, bsi_stream_t stream) {
    using namespace bsi;
    int rc = check_matrix("fp4_dequantize", format, dtype, rows, K, ld, codes, scales, row_scale);
    if (rc != BSI_OK) return rc;
    if (rows == 0) return BSI_OK;
    if (out == nullptr || ldo < K || reinterpret_cast<uintptr_t>(out) % (dtype == BSI_DTYPE_F32 ? 4 : 2) != 0)
        return fail(BSI_ERR_INVALID, "fp4_dequantize: null or misaligned output, or rows that overlap");
    rc = require_sm100();
    if (rc != BSI_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == BSI_DTYPE_F32 ? launch_dequantize<float>(codes, ld, scales, row_scale, rows, K, format, out, ldo, s)
           : dtype == BSI_DTYPE_F16 ? launch_dequantize<__half>(codes, ld, scales, row_scale, rows, K, format, out, ldo, s)
                                    : launch_dequantize<__nv_bfloat16>(codes, ld, scales, row_scale, rows, K, format, out, ldo, s);
}
