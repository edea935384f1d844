// What the kernels over rows of logits share: how a row is cut and read, running softmax statistics, reductions.
//
// A row of V logits starts on any element, so it is seen as 16-byte pieces of the memory that it lies in: piece v holds the
// elements v * kVec - shift .. + kVec - 1, where shift is the row's offset from a 16-byte boundary in elements. Only the first and
// the last piece can hold elements of a neighbour; those are read one by one and read as -inf where they are not the row's.
// A cluster of CTAs shares a row; CTA c owns the pieces [n c / C, n (c + 1) / C).
//
// 256 threads a CTA: a row's phases (stream, reduce, look for the largest, write) follow one another with barriers between them, so
// what keeps an SM busy are several CTAs in different phases (score_kernel of 1024 x 50272 float16: 512 threads, 2 CTAs an SM 111 us).
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <type_traits>

#include "common.cuh"

namespace bsi {
namespace vocab {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBatch = 4;               // 16-byte pieces that a thread has under way
constexpr float kLn2 = 0.6931471805599453f;

// Rows of a 2-D or 3-D tensor: row r lies at (r / per) * block + (r % per) * row elements.
struct RowPlan {
    int64_t per, block, row;
    __device__ __forceinline__ int64_t at(uint32_t r) const {      // rows are fewer than 2^31; a 64-bit division costs 100 instructions
        if (per == 0) return static_cast<int64_t>(r) * row;
        const uint32_t n = static_cast<uint32_t>(per), b = r / n;
        return b * block + (r - b * n) * row;
    }
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

// Two float32 in one instruction: a third of the statistics' instructions are additions and products of float32.
struct Two {
    unsigned long long v;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ void split(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Two fma2(const Two& a, const Two& b, const Two& c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ Two add2(const Two& a, const Two& b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two mul2(const Two& a, const Two& b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

// 16 bytes of logits. top: the largest value, a NaN if there is one. finite_floor: values below -1e30 (float16: the lowest) as that,
// so that a masked place times its weight of 0 is 0. Thresholds are passed as word(): a value in every lane of a 32-bit word.
template <typename T>
struct Piece;
template <>
struct Piece<float> {
    using Raw = float;
    static constexpr int kVec = 4;
    static constexpr uint32_t kNone = 0xFF800000u;      // -inf
    static constexpr float kFar = 4194304.0f;
    static __device__ __forceinline__ float one(float v) { return v; }
    static __device__ __forceinline__ void unpack(const uint4& u, float* z) {
        z[0] = __uint_as_float(u.x); z[1] = __uint_as_float(u.y); z[2] = __uint_as_float(u.z); z[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* z) {
        return make_uint4(__float_as_uint(z[0]), __float_as_uint(z[1]), __float_as_uint(z[2]), __float_as_uint(z[3]));
    }
    static __device__ __forceinline__ float narrow(float v) { return v; }
    template <int B>
    static __device__ __forceinline__ float top(const uint4 (&u)[B]) {
        float m = __uint_as_float(u[0].x);
#pragma unroll
        for (int b = 0; b < B; ++b) m = max_nan(max_nan(m, __uint_as_float(u[b].x)), max_nan(__uint_as_float(u[b].y), max_nan(__uint_as_float(u[b].z), __uint_as_float(u[b].w))));
        return m;
    }
    static __device__ __forceinline__ uint4 finite_floor(const uint4& u) {
        const float lo = -1e30f;
        return make_uint4(__float_as_uint(max_nan(__uint_as_float(u.x), lo)), __float_as_uint(max_nan(__uint_as_float(u.y), lo)),
                          __float_as_uint(max_nan(__uint_as_float(u.z), lo)), __float_as_uint(max_nan(__uint_as_float(u.w), lo)));
    }
    struct Count {
        Two n;      // ones as float32, two lanes
        __device__ __forceinline__ Count() : n(0.0f, 0.0f) {}
        static __device__ __forceinline__ float ge(uint32_t v, float t) {
            float r;
            asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(v)), "f"(t));
            return r;
        }
        __device__ __forceinline__ void add(const uint4& u, uint32_t thr) {
            const float t = __uint_as_float(thr);
            n = add2(n, add2(Two(ge(u.x, t), ge(u.y, t)), Two(ge(u.z, t), ge(u.w, t))));
        }
        __device__ __forceinline__ int total() const {
            float a, b;
            n.split(a, b);
            return static_cast<int>(a + b);
        }
    };
    static __device__ __forceinline__ uint32_t word(float v) { return __float_as_uint(v); }
    // One bit for each value that is not below thr (a NaN is not).
    static __device__ __forceinline__ uint32_t reach(const uint4& u, uint32_t thr) {
        const float t = __uint_as_float(thr);
        return (__uint_as_float(u.x) < t ? 0u : 1u) | (__uint_as_float(u.y) < t ? 0u : 2u) | (__uint_as_float(u.z) < t ? 0u : 4u) | (__uint_as_float(u.w) < t ? 0u : 8u);
    }
    // 16 bits of a value's place in the order, and the smallest value of a place. kFloor: the first one above -inf.
    static constexpr uint32_t kFloor = 0x0080u;
    static __device__ __forceinline__ uint32_t place(float v) {
        if (v != v) return 0xFFFFu;
        const uint32_t u = __float_as_uint(v + 0.0f);
        return ((u & 0x80000000u) ? ~u : (u | 0x80000000u)) >> 16;
    }
    static __device__ __forceinline__ float smallest(uint32_t place) {
        const uint32_t k = place << 16;
        return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
    }
    static __device__ __forceinline__ float next_up(float v) {
        const uint32_t b = __float_as_uint(v);
        if ((b << 1) == 0u) return __uint_as_float(1u);
        return __uint_as_float((b & 0x80000000u) ? b - 1u : b + 1u);
    }
    static __device__ __forceinline__ float nan() { return __uint_as_float(0x7FC00000u); }
};

template <typename T>
__device__ __forceinline__ T from_bits16(unsigned short b) { return *reinterpret_cast<const T*>(&b); }

template <typename T, typename T2>
struct Piece16 {
    using Raw = T;
    static constexpr int kVec = 8;
    static __device__ __forceinline__ T2 as2(uint32_t w) { return *reinterpret_cast<const T2*>(&w); }
    static __device__ __forceinline__ uint32_t bits(const T2& h) { return *reinterpret_cast<const uint32_t*>(&h); }
    static __device__ __forceinline__ T2 top2(const uint4& u) {
        return __hmax2_nan(__hmax2_nan(as2(u.x), as2(u.y)), __hmax2_nan(as2(u.z), as2(u.w)));
    }
    template <int B>
    static __device__ __forceinline__ float top(const uint4 (&u)[B]) {
        T2 m = top2(u[0]);
#pragma unroll
        for (int b = 1; b < B; ++b) m = __hmax2_nan(m, top2(u[b]));
        return static_cast<float>(__hmax_nan(m.x, m.y));
    }
    // Counts are exact in the 16-bit type: at most 4 kBatch of them a half, 256 is bfloat16's limit.
    struct Count {
        T2 n;
        __device__ __forceinline__ Count() { const uint32_t zero = 0u; n = as2(zero); }
        __device__ __forceinline__ void add(const uint4& u, uint32_t thr) {
            const T2 t = as2(thr);
            n = __hadd2(n, __hadd2(__hadd2(__hge2(as2(u.x), t), __hge2(as2(u.y), t)), __hadd2(__hge2(as2(u.z), t), __hge2(as2(u.w), t))));
        }
        __device__ __forceinline__ int total() const { return static_cast<int>(static_cast<float>(n.x) + static_cast<float>(n.y)); }
    };
    static __device__ __forceinline__ uint32_t word(T v) { return *reinterpret_cast<const unsigned short*>(&v) * 0x10001u; }
    static __device__ __forceinline__ uint32_t reach2(uint32_t w, const T2& t) {
        const uint32_t below = __hlt2_mask(as2(w), t);
        return (~below & 1u) | (~below >> 30 & 2u);
    }
    static __device__ __forceinline__ uint32_t reach(const uint4& u, uint32_t thr) {
        const T2 t = as2(thr);
        return reach2(u.x, t) | reach2(u.y, t) << 2 | reach2(u.z, t) << 4 | reach2(u.w, t) << 6;
    }
    static __device__ __forceinline__ uint32_t place(float v) {
        if (v != v) return 0xFFFFu;
        const T h = static_cast<T>(v + 0.0f);       // exact: v is one of T's values
        const uint32_t b = *reinterpret_cast<const unsigned short*>(&h);
        return (b & 0x8000u) ? ~b & 0xFFFFu : b | 0x8000u;
    }
    static constexpr uint32_t kFloor = std::is_same<T, __half>::value ? 0x0400u : 0x0080u;
    static __device__ __forceinline__ T smallest(uint32_t place) {
        return from_bits16<T>(static_cast<unsigned short>((place & 0x8000u) ? place & 0x7FFFu : ~place));
    }
    static __device__ __forceinline__ T next_up(T v) {
        const unsigned short b = *reinterpret_cast<const unsigned short*>(&v);
        if ((b & 0x7FFFu) == 0u) return from_bits16<T>(1);
        return from_bits16<T>(static_cast<unsigned short>((b & 0x8000u) ? b - 1u : b + 1u));
    }
    static __device__ __forceinline__ T nan() { return from_bits16<T>(0x7FFF); }
};
template <>
struct Piece<__half> : Piece16<__half, __half2> {
    static constexpr uint32_t kNone = 0xFC00FC00u;
    static constexpr float kFar = 60000.0f;
    static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
    static __device__ __forceinline__ void unpack(const uint4& u, float* z) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(as2(w[i]));
            z[2 * i] = f.x;
            z[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* z) {
        return make_uint4(bits(__floats2half2_rn(z[0], z[1])), bits(__floats2half2_rn(z[2], z[3])), bits(__floats2half2_rn(z[4], z[5])),
                          bits(__floats2half2_rn(z[6], z[7])));
    }
    static __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ uint4 finite_floor(const uint4& u) {
        const __half2 lo = as2(0xFBFFFBFFu);
        return make_uint4(bits(__hmax2_nan(as2(u.x), lo)), bits(__hmax2_nan(as2(u.y), lo)), bits(__hmax2_nan(as2(u.z), lo)), bits(__hmax2_nan(as2(u.w), lo)));
    }
};
template <>
struct Piece<__nv_bfloat16> : Piece16<__nv_bfloat16, __nv_bfloat162> {
    static constexpr uint32_t kNone = 0xFF80FF80u;
    static constexpr float kFar = 4194304.0f;
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
        return make_uint4(bits(__floats2bfloat162_rn(z[0], z[1])), bits(__floats2bfloat162_rn(z[2], z[3])), bits(__floats2bfloat162_rn(z[4], z[5])),
                          bits(__floats2bfloat162_rn(z[6], z[7])));
    }
    static __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ uint4 finite_floor(const uint4& u) {
        const __nv_bfloat162 lo = as2(0xF149F149u);      // -0.99e30
        return make_uint4(bits(__hmax2_nan(as2(u.x), lo)), bits(__hmax2_nan(as2(u.y), lo)), bits(__hmax2_nan(as2(u.z), lo)), bits(__hmax2_nan(as2(u.w), lo)));
    }
};

// Piece range of one CTA over one row.
template <typename T>
struct Span {
    static constexpr int kVec = Piece<T>::kVec;
    const T* row;        // element 0 of the row
    const uint4* grid;   // piece 0
    int shift;           // elements of piece 0 that lie before the row
    int V;
    int first, last;     // this CTA's pieces
    int lo, hi;          // pieces in [lo, hi) lie wholly inside the row

    __device__ __forceinline__ Span(const T* r, int v, int part, int parts) : row(r), V(v) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(r);
        shift = static_cast<int>((a & 15u) / sizeof(T));
        grid = reinterpret_cast<const uint4*>(a & ~uintptr_t(15));
        const int64_t n = (static_cast<int64_t>(V) + shift + kVec - 1) / kVec;
        const int lg = 31 - __clz(parts);          // parts is a power of two
        first = static_cast<int>((n * part) >> lg);
        last = static_cast<int>((n * (part + 1)) >> lg);
        lo = shift == 0 ? 0 : 1;
        hi = static_cast<int>((static_cast<int64_t>(V) + shift) / kVec);
    }
    __device__ __forceinline__ int element(int v) const { return v * kVec - shift; }
    __device__ __forceinline__ bool whole(int v) const { return v >= lo && v < hi; }
    // A piece that is not whole, -inf where it has no value of the row.
    __device__ __noinline__ uint4 load_edge(int v) const {
        float z[kVec];
        const int e0 = element(v);
#pragma unroll
        for (int e = 0; e < kVec; ++e) z[e] = e0 + e >= 0 && e0 + e < V ? Piece<T>::one(row[e0 + e]) : -CUDART_INF_F;
        return Piece<T>::pack(z);       // exact: the values are T's
    }
    // A part's whole pieces, and the row's ends.
    __device__ __forceinline__ int whole_first() const { return max(first, lo); }
    __device__ __forceinline__ int whole_last() const { return max(whole_first(), min(last, hi)); }
    __device__ __forceinline__ bool has_left() const { return first < lo && first < last; }
    __device__ __forceinline__ bool has_right() const { return last > hi && last > first && (last - 1 >= lo || lo == 0); }
    // The elements this CTA owns are [begin(), end()).
    __device__ __forceinline__ int begin() const { return max(element(first), 0); }
    __device__ __forceinline__ int end() const { return static_cast<int>(min(static_cast<int64_t>(last) * kVec - shift, static_cast<int64_t>(V))); }
};

// Softmax statistics: maximum m, s = sum exp(scale (z - m)); where wanted w = sum e * d with e = exp(scale (z - m)) = 2^d, from which
// the entropy follows. Nothing seen but -inf: m = -inf, s = w = 0.
struct Stats {
    float m, s, w;
};

// scale * log2(e) in two parts, both above 0: a rounded factor alone would be off by 2^-25 of itself, which exponents of 30 turn into 1e-6 of a weight.
struct Factor {
    float hi, lo;
    __device__ __forceinline__ float times(float x) const { return fmaf(x, lo, x * hi); }
};

// The warp's statistics as one: their maximum first, then sums against it.
__device__ __forceinline__ Stats warp_merge(const Stats& v, const Factor& c) {
    float m = v.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (m == -CUDART_INF_F) return Stats{m, 0.0f, 0.0f};
    const float d = v.s != 0.0f ? c.times(v.m - m) : 0.0f;
    const float f = exp2_fast(d);
    // a side without any mass adds nothing, however far below it lies
    float s = v.s != 0.0f && f != 0.0f ? v.s * f : 0.0f, w = v.s != 0.0f && f != 0.0f ? f * fmaf(d, v.s, v.w) : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
    }
    return Stats{m, s, w};
}

// The whole pieces of a CTA's rows (row, row + step, ... below end; with weights, those whose weight is not 0) on their way through
// shared memory: chunks of kBatch pieces per thread, copied in bulk by one thread and waited for by all, one row's behind the other's.
// What is under way depends neither on what the threads hold in registers nor on where in a row they are: a row's first chunks come
// while the row before it is being finished. As many chunks as there are stages are under way; a stage is filled again when every warp
// is done with it. Every wait is bounded: one that gives up says so in the status word and to the block, which then waits for nothing any
// more, gives NaN for the row and the rows behind it (gave_up(), behind a barrier of the block), and at the end for what is still under way
// to land, bounded again: a copy must not arrive in shared memory that has become another CTA's.
#ifndef BSI_ROWS_WAIT_CYCLES
#define BSI_ROWS_WAIT_CYCLES 500000000ll       // about 0.25 s; real waits are microseconds
#define BSI_ROWS_WAIT_HINT 20000u              // ns that a wait may sleep before it looks at the clock; 0: it does not
#endif
constexpr int kChunk = kBatch * kThreads;      // pieces
constexpr long long kWaitCycles = BSI_ROWS_WAIT_CYCLES;

__device__ __forceinline__ uint32_t shared_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// What thread 0 has still to issue; in shared memory, as no other thread needs it.
struct Feed {
    const void* logits;
    const float* weights;
    RowPlan rows;
    int V, part, parts;
    uint32_t row, step, end, stage, round;      // round: how often the stages have been through
    int chunk, pieces;
    const uint4* source;
    int broken;        // by any thread
};

// The next row that has pieces, from r on.
template <typename T>
__device__ __noinline__ void open_row(Feed* f, uint32_t r) {
    for (; r < f->end; r += f->step) {
        if (f->weights != nullptr && f->weights[r] == 0.0f) continue;
        const Span<T> span(static_cast<const T*>(f->logits) + f->rows.at(r), f->V, f->part, f->parts);
        f->pieces = span.whole_last() - span.whole_first();
        f->source = span.grid + span.whole_first();
        if (f->pieces > 0) break;
    }
    f->row = r;
    f->chunk = 0;
}

template <typename T>
struct Ring {
    uint4* data;
    uint32_t full, empty;      // barriers of stage 0
    uint32_t stages;
    Feed* feed;
    int* status;
    bool broken;

    // By all threads; a barrier of the block stands between this and the first chunk. bars: 2 * stages of them.
    __device__ __forceinline__ Ring(uint4* d, uint64_t* bars, int n, Feed* f, const void* z, const RowPlan& plan, int v, int p, int ps, const float* w,
                                    uint32_t first_row, uint32_t stride, uint32_t last_row, int* st)
        : data(d), full(shared_address(bars)), empty(full + 8u * n), stages(n), feed(f), status(st), broken(false) {
        if (threadIdx.x == 0) {
            for (int i = 0; i < n; ++i) {
                asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full + 8u * i));
                asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(empty + 8u * i), "r"(kWarps));
            }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            f->logits = z;
            f->weights = w;
            f->rows = plan;
            f->V = v;
            f->part = p;
            f->parts = ps;
            f->step = stride;
            f->end = last_row;
            f->stage = f->round = 0;
            f->broken = 0;
            open_row<T>(f, first_row);
            for (int i = 0; i < n; ++i) issue();
        }
    }
    __device__ __forceinline__ void issue() {
        if (feed->row >= feed->end) return;
        const uint32_t s = feed->stage;
        const int at = feed->chunk * kChunk;
        const uint32_t bytes = static_cast<uint32_t>(min(kChunk, feed->pieces - at)) * 16u;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full + 8u * s), "r"(bytes) : "memory");
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(shared_address(data + s * kChunk)), "l"(__cvta_generic_to_global(feed->source + at)), "r"(bytes), "r"(full + 8u * s)
                     : "memory");
        feed->stage = s + 1 == stages ? 0u : s + 1;
        if (s + 1 == stages) ++feed->round;
        ++feed->chunk;
        if (feed->chunk * kChunk >= feed->pieces) open_row<T>(feed, feed->row + feed->step);
    }
    static __device__ __forceinline__ bool landed(uint32_t bar, uint32_t parity) {
        uint32_t ok;
        if constexpr (BSI_ROWS_WAIT_HINT == 0u)
            asm volatile("{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                         : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        else
            asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}\n"
                         : "=r"(ok) : "r"(bar), "r"(parity), "r"(BSI_ROWS_WAIT_HINT) : "memory");
        return ok != 0u;
    }
    __device__ __forceinline__ bool gave_up() const { return *static_cast<volatile int*>(&feed->broken) != 0; }
    __device__ __forceinline__ void wait(uint32_t bar, uint32_t parity) {
        if (!broken && !landed(bar, parity)) broken = !waited(feed, bar, parity, status);
    }
    static __device__ __noinline__ bool waited(Feed* feed, uint32_t bar, uint32_t parity, int* status) {
        const long long t0 = clock64();
        while (!landed(bar, parity)) {
            volatile int* gave_up = &feed->broken;
            if (clock64() - t0 > kWaitCycles) {
                *gave_up = 1;
                atomicCAS(status, 0, 144);
            }
            if (*gave_up != 0) return false;
        }
        return true;
    }
    // Behind the last row.
    __device__ __forceinline__ void finish() const {
        if (threadIdx.x == 0 && gave_up()) {
            for (uint32_t s = 0; s < stages; ++s) {
                const uint32_t times = feed->round + (s < feed->stage ? 1u : 0u);      // how often it has been filled
                const long long t0 = clock64();
                while (times != 0u && !landed(full + 8u * s, (times - 1u) & 1u) && clock64() - t0 < 30000000ll) {}
            }
        }
    }
    // A chunk's stage and how often that had been filled before, odd or even. (Counted along: a remainder by a number of stages that is
    // not known at compile time costs 20 instructions, and five of them were a third of a chunk's.)
    struct Place {
        uint32_t stage, phase;
    };
    __device__ __forceinline__ void advance(Place& p) const {
        if (++p.stage == stages) {
            p.stage = 0;
            p.phase ^= 1u;
        }
    }
    __device__ __forceinline__ const uint4* at(const Place& p) const { return data + p.stage * kChunk; }
    // The chunk there, behind its arrival.
    __device__ __forceinline__ const uint4* arrive(const Place& p) {
        wait(full + 8u * p.stage, p.phase);
        return at(p);
    }
    // The warp is done with the chunk there. (Chunks are released in order, so its stage is the one that is filled next.)
    __device__ __forceinline__ void release(const Place& p) {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(empty + 8u * p.stage) : "memory");
        if (threadIdx.x == 0 && feed->row < feed->end) {
            wait(empty + 8u * p.stage, p.phase);
            if (!broken) issue();
        }
        __syncwarp();
    }
};

// One thread's running statistics. The reference that the exponents are taken against is a whole number `base` near m * c in powers
// of two: d = z * c - base is then one fused multiply-add with one rounding (of d, not of z * c), and moving the reference
// multiplies s by an exact power of two. It is moved only when a value passes it by 2^32, which float32 sums have room for: moving it
// with every new maximum, as some lane of a warp has one in nearly every batch, took 60 instructions of 300. Where |m * c| passes kFar
// (2^22, where whole numbers grow sparse; float16: 60000, so that the floor stays far below; logits of a mask's size and nothing else)
// the reference is m itself and d = (z - m) * c.
template <typename T, bool W>
struct Running {
    float m, base, s, w;
    bool far;

    __device__ __forceinline__ Running() : m(-INFINITY), base(NAN), s(0.0f), w(0.0f), far(false) {}      // no value passes a NaN: the first batch sets base

    // A new reference at a new maximum.
    __device__ __forceinline__ void raise(float top, const Factor& factor) {
        const float c = factor.hi;
        const float old_m = m, old_base = base;
        const bool old_far = far;
        base = rintf(top * c);
        far = !(fabsf(base) < Piece<T>::kFar);    // also a NaN, +inf
        if (s == 0.0f) return;                    // nothing counts yet
        float d;
        if (!far && !old_far) d = old_base - base;
        else if (far && old_far) d = (old_m - top) * c;
        else if (far) d = old_base - top * c;     // upwards out of range: what was is nothing
        else d = old_m * c - base;
        const float f = exp2_fast(d);
        if (W) w = f != 0.0f ? f * (w + d * s) : 0.0f;
        s = f != 0.0f ? s * f : 0.0f;
    }

    // Returns the largest of the values.
    template <int B>
    __device__ __forceinline__ float take(const uint4 (&u)[B], const Factor& factor) {
        constexpr int kVec = Piece<T>::kVec;
        const float c = factor.hi;
        const float top = Piece<T>::top(u);
        if (far ? !(top <= m) : !(fmaf(top, c, -32.0f) <= base)) raise(top, factor);      // far higher, or a NaN
        m = max_nan(m, top);
        if (m == -CUDART_INF_F) return top;       // nothing but -inf so far
        float s0 = 0.0f, s1 = 0.0f, w0 = 0.0f, w1 = 0.0f;
        if (!far) {
            const Two cc(c, c), ll(factor.lo, factor.lo), bb(-base, -base);
            Two ss(0.0f, 0.0f), ww(0.0f, 0.0f);
#pragma unroll
            for (int b = 0; b < B; ++b) {
                float z[kVec];
                Piece<T>::unpack(W ? Piece<T>::finite_floor(u[b]) : u[b], z);
#pragma unroll
                for (int e = 0; e < kVec; e += 2) {
                    const Two x01(z[e], z[e + 1]);
                    Two d = fma2(x01, cc, bb);
                    if (!W) d = fma2(x01, ll, d);      // the entropy's statistics have the factor log2(e), whose float32 is good to 2^-26
                    float d0, d1;
                    d.split(d0, d1);
                    const Two x(exp2_fast(d0), exp2_fast(d1));
                    ss = add2(ss, x);
                    if (W) ww = fma2(x, d, ww);
                }
            }
            ss.split(s0, s1);
            ww.split(w0, w1);
        } else {
#pragma unroll 1
            for (int b = 0; b < B; ++b) {
                float z[kVec];
                const uint4 p = b == 0 ? u[0] : b == 1 ? u[B > 1 ? 1 : 0] : b == 2 ? u[B > 2 ? 2 : 0] : u[B - 1];
                Piece<T>::unpack(p, z);
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    const float d = max_nan((z[e] - m) * c, -200.0f);       // 2^-200 is 0 here
                    const float x = exp2_fast(d);
                    s0 += x;
                    if (W) w0 = fmaf(x, d, w0);
                }
            }
        }
        s += s0 + s1;
        if (W) w += w0 + w1;
        return top;
    }

    // Against m, as warp_merge() takes them.
    __device__ __forceinline__ Stats stats(const Factor& c) const {
        if (m == -CUDART_INF_F) return Stats{m, 0.0f, 0.0f};
        if (far) return Stats{m, s, w};
        const float d = -fmaf(m, W ? 0.0f : c.lo, fmaf(m, c.hi, -base));       // base - m * c, down to -32
        const float f = exp2_fast(d);
        return Stats{m, s * f, W ? f * fmaf(d, s, w) : 0.0f};
    }
};
static_assert(kBatch <= 4, "take()'s rare branch names the pieces");

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
