// What the kernels over rows of logits share: how a row is cut and read, running softmax statistics, reductions.
//
// A row of V logits starts on any element, so it is seen as 16-byte pieces of the memory that it lies in: piece v holds the
// elements v * kVec - shift .. + kVec - 1, where shift is the row's offset from a 16-byte boundary in elements. Only the first and
// the last piece can hold elements of a neighbour; those are read one by one and read as -inf where they are not the row's.
// A cluster of CTAs shares a row; CTA c owns the pieces [n c / C, n (c + 1) / C).
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"

namespace bsi {
namespace vocab {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Rows of a 2-D or 3-D tensor: row r lies at (r / per) * block + (r % per) * row elements.
struct RowPlan {
    int64_t per, block, row;
    __host__ __device__ int64_t at(int64_t r) const {
        return per == 0 ? r * row : (r / per) * block + (r % per) * row;
    }
};

template <typename T>
struct Piece;
template <>
struct Piece<float> {
    static constexpr int kVec = 4;
    static __device__ __forceinline__ float one(float v) { return v; }
    static __device__ __forceinline__ void unpack(const uint4& u, float* z) {
        z[0] = __uint_as_float(u.x); z[1] = __uint_as_float(u.y); z[2] = __uint_as_float(u.z); z[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* z) {
        return make_uint4(__float_as_uint(z[0]), __float_as_uint(z[1]), __float_as_uint(z[2]), __float_as_uint(z[3]));
    }
    static __device__ __forceinline__ float narrow(float v) { return v; }
};
template <>
struct Piece<__half> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
    static __device__ __forceinline__ void unpack(const uint4& u, float* z) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            z[2 * i] = f.x;
            z[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* z) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(z[2 * i], z[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
};
template <>
struct Piece<__nv_bfloat16> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ void unpack(const uint4& u, float* z) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {      // a bfloat16 is a float32's upper half
            z[2 * i] = __uint_as_float(w[i] << 16);
            z[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* z) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(z[2 * i], z[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
};

// max that keeps a NaN: a NaN among the logits has to reach the result.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Piece range of one CTA over one row.
template <typename T>
struct Span {
    static constexpr int kVec = Piece<T>::kVec;
    const T* row;        // element 0 of the row
    const uint4* grid;   // piece 0
    int shift;           // elements of piece 0 that lie before the row
    int64_t V;
    int64_t first, last;      // this CTA's pieces
    int64_t lo, hi;           // pieces in [lo, hi) lie wholly inside the row

    __device__ Span(const T* r, int64_t v, int part, int parts) : row(r), V(v) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(r);
        shift = static_cast<int>((a & 15u) / sizeof(T));
        grid = reinterpret_cast<const uint4*>(a & ~uintptr_t(15));
        const int64_t n = (V + shift + kVec - 1) / kVec;
        first = n * part / parts;
        last = n * (part + 1) / parts;
        lo = shift == 0 ? 0 : 1;
        hi = (V + shift) / kVec;
    }
    __device__ __forceinline__ int64_t element(int64_t v) const { return v * kVec - shift; }
    // The values of any piece, -inf where it has none.
    __device__ __forceinline__ void load_edge(int64_t v, float* z) const {
        const int64_t e0 = element(v);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const int64_t i = e0 + e;
            z[e] = i >= 0 && i < V ? Piece<T>::one(row[i]) : -CUDART_INF_F;
        }
    }
    __device__ __forceinline__ bool whole(int64_t v) const { return v >= lo && v < hi; }
    __device__ __forceinline__ void load(int64_t v, float* z) const {
        if (whole(v)) Piece<T>::unpack(grid[v], z);
        else load_edge(v, z);
    }
    // The elements this CTA owns are [begin(), end()).
    __device__ __forceinline__ int64_t begin() const { const int64_t e = element(first); return e < 0 ? 0 : e; }
    __device__ __forceinline__ int64_t end() const { const int64_t e = element(last); return e > V ? V : e; }
};

// Running maximum m and sum s of exp(scale (z - m)); where W, also w, the sum of exp(scale (z - m)) * scale (z - m) / ln 2, from
// which the entropy follows. m stays -inf until a value above it is seen; with s and w zero until then nothing is divided by it.
struct Stats {
    float m, s, w;
};

// Two sets of statistics as one. c: scale * log2(e).
__device__ __forceinline__ Stats merge(const Stats& a, const Stats& b, float c) {
    Stats r;
    r.m = max_nan(a.m, b.m);
    if (r.m == -CUDART_INF_F) return Stats{-CUDART_INF_F, 0.0f, 0.0f};
    const float da = a.m == -CUDART_INF_F ? 0.0f : (a.m - r.m) * c, db = b.m == -CUDART_INF_F ? 0.0f : (b.m - r.m) * c;
    const float fa = exp2_fast(da), fb = exp2_fast(db);
    // a side without any mass adds nothing, however far below it lies
    r.s = (a.s != 0.0f ? a.s * fa : 0.0f) + (b.s != 0.0f ? b.s * fb : 0.0f);
    r.w = (a.s != 0.0f && fa != 0.0f ? fa * (a.w + da * a.s) : 0.0f) + (b.s != 0.0f && fb != 0.0f ? fb * (b.w + db * b.s) : 0.0f);
    return r;
}

__device__ __forceinline__ Stats warp_merge(Stats v, float c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Stats u;
        u.m = __shfl_xor_sync(0xFFFFFFFFu, v.m, o);
        u.s = __shfl_xor_sync(0xFFFFFFFFu, v.s, o);
        u.w = __shfl_xor_sync(0xFFFFFFFFu, v.w, o);
        v = merge(v, u, c);
    }
    return v;
}

// Takes n values (kVec at a time) into the statistics: one maximum for the batch, a new reference only where it rises.
template <int N, bool W>
__device__ __forceinline__ void take(Stats& st, const float (&z)[N], float c) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = max_nan(top, z[i]);
    if (!(top <= st.m)) {                  // higher, or a NaN
        const float d = (st.m - top) * c;
        const float f = exp2_fast(d);      // 0 at the first batch, whose s and w are 0
        if (W) st.w = st.s != 0.0f && f != 0.0f ? f * (st.w + d * st.s) : 0.0f;
        st.s *= f;
        st.m = top;
    }
    if (st.m == -CUDART_INF_F) return;     // nothing but -inf so far
    float s = 0.0f, w = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        // Below -200 the power of two is 0 in float32 whatever the product, -inf included: 0 * -200 adds nothing to w
        const float d = W ? max_nan((z[i] - st.m) * c, -200.0f) : (z[i] - st.m) * c;
        const float e = exp2_fast(d);
        s += e;
        if (W) w = fmaf(e, d, w);
    }
    st.s += s;
    if (W) st.w += w;
}

// One whole number per float32, larger for a larger value; -0 as +0, every NaN as one number above all others.
__device__ __forceinline__ uint32_t ordered(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

}  // namespace vocab
}  // namespace bsi
