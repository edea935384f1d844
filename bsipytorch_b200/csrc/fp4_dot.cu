// Product of two 4-bit matrices on the 5th-generation tensor cores:
//     y[m][n] = act( (sum_k x[m][k] w[n][k]) * gx[m] * gw[n] + bias[n] ),   x, w: e2m1 values times their block scales
//
// tcgen05.mma.kind::mxf4 / mxf4nvf4 multiplies the codes and both block scales itself (K = 64 per instruction) and accumulates in
// float32 in TMEM; what is left for the epilogue are the per-row factors of the nvfp4 format, the bias, ReLU and one rounding.
//
// The weights' rows are the instruction's M (TMEM lanes), the tokens its N, so that one token takes the same way as a prompt, and a
// warp of the epilogue stores 32 neighbouring outputs of a token. Up to 128 tokens, a CTA by itself with all of them (fp4_linear_kernel):
//
//   warp 0     TMA producer: per k-block of 256 elements one box of weights (128 x 128 B), one of tokens (BN x 128 B), both 128-byte
//              swizzled, and their scales as they lie in memory (512 bytes for 128 rows x 4 scales, whole tiles)
//   warp 1     MMA issuer: 4 MMAs of K = 64
//   warps 2-5  epilogue
//   warps 6-9  the block's scales from shared memory into TMEM, a set of columns for every stage of the operand ring
// Where the tiles leave SMs idle, a cluster of 2, 4 or 8 CTAs shares a tile, each with a part of K; the parts' float32 sums meet in
// shared memory and are added in the parts' order, each CTA for its share of the tokens.
// Every wait is bounded: on a timeout the role records its site in the status word, raises the CTA's abort flag, what is under way is
// waited for (bounded again), TMEM is freed and the kernel returns.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>

#include "fp4.cuh"
#include "tcgen05.cuh"

namespace bsi {

__device__ int g_fp4_status = 0;

int take_fp4_status(int* v) {
    int s = 0;
    BSI_CUDA_TRY(cudaMemcpyFromSymbol(&s, g_fp4_status, sizeof(int)));
    if (s != 0) {
        const int zero = 0;
        BSI_CUDA_TRY(cudaMemcpyToSymbol(g_fp4_status, &zero, sizeof(int)));
    }
    *v = s;
    return BSI_OK;
}

namespace {

constexpr int kRowBytes = 128;         // bytes of a k-block in a row: 256 elements
constexpr int kTileM = 128;
constexpr int kThreads = 320;
constexpr int kScaleTile = 512;        // 128 rows x 4 scales
constexpr long long kWaitCycles = 500000000ll;    // about 0.25 s; real waits are microseconds
constexpr int kSiteBase = 128;         // of the status word: sites 129 and up are this kernel's

template <int BN, bool MX>
struct Cfg {
    static constexpr int kGroups = MX ? 2 : 4;                   // scale tiles of a k-block per 128 rows
    static constexpr int kWBytes = kTileM * kRowBytes;
    static constexpr int kXBytes = BN * kRowBytes;
    static constexpr int kWScale = kGroups * kScaleTile;
    static constexpr int kXScale = kGroups * kScaleTile;
    static constexpr int kStageBytes = kWBytes + kXBytes + kWScale + kXScale;      // a multiple of 1 KB
    // two CTAs per SM for the narrow tiles, whose MMAs are short beside their loads
    static constexpr int kPerSm = BN <= 64 ? 2 : 1;
    static constexpr int kBudget = (kPerSm == 2 ? 113 : 226) * 1024 - 2048;
    static constexpr int kStages = kBudget / kStageBytes > 8 ? 8 : kBudget / kStageBytes;
    static constexpr int kSmem = kStages * kStageBytes + (3 * kStages + 2) * 8 + 32 + BN * 4 + 1024;
    // TMEM: the accumulator, then a set of scales for each stage (4 columns for each tile of 512 bytes)
    static constexpr int kScaleCols = 4 * kGroups * 2;
    static constexpr int kScale0 = BN < 32 ? 32 : BN;
    static constexpr int kNeed = kScale0 + kStages * kScaleCols;
    static constexpr int kTmemCols = kNeed <= 128 ? 128 : (kNeed <= 256 ? 256 : 512);
    static_assert(kStageBytes % 1024 == 0 && kStages >= 3 && kNeed <= 512 && kPerSm * kTmemCols <= 512, "does not fit");
    static_assert(BN * kTileM * 4 <= kStages * kStageBytes, "the parts' sums meet in the operand ring");
};

struct Args {
    const uint8_t* w_scales;
    const uint8_t* x_scales;
    const float* w_row;      // null: 1
    const float* x_row;
    const float* bias;       // null: none
    void* y;
    int64_t ldy;
    int M, N;                // tokens, outputs
    int blocks;              // k-blocks
    int relu;
    int dependent;           // launched behind the packer as its dependent: what it writes is read behind griddepcontrol.wait
};

__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort_flag, int site) {
    if (mbar_try(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
        if (mbar_try_parked(bar, parity, 20000u)) return true;
        if (*abort_flag) return false;
        if (clock64() - t0 > kWaitCycles) {
            *abort_flag = 1;
            atomicCAS(&g_fp4_status, 0, kSiteBase + site);
            return false;
        }
    }
}

__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!mbar_try(bar, parity) && clock64() - t0 < kWaitCycles / 16) {}
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(__cvta_generic_to_global(src)), "r"(bytes), "r"(bar)
                 : "memory");
}

template <int N>
__device__ __forceinline__ void tmem_store(uint32_t taddr, const uint32_t* r) {
    if constexpr (N >= 32) {
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
            "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
            ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
              "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
              "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
            : "memory");
        if constexpr (N > 32) tmem_store<N - 32>(taddr + 32, r + 32);
    } else if constexpr (N >= 16) {
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
            ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
              "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
            : "memory");
        if constexpr (N > 16) tmem_store<N - 16>(taddr + 16, r + 16);
    } else {
        static_assert(N == 8, "columns in multiples of 8");
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
    }
}

// One warp's share of a k-block's scales into TMEM: GROUPS tiles of 512 bytes of the weights, then GROUPS x NT of the tokens, group by
// group. A tile is 32 lanes of 16 bytes, four columns; every quarter of TMEM's lanes holds the same, so each of four warps writes all.
// (tcgen05.cp, which copies a tile into all quarters by itself, stands between the MMAs: 60 to 100 cycles for each tile, and 12 of them
// beside the 512 cycles of a k-block's MMAs held 8192 x 4096 -> 16384 nvfp4 at 3.0 PFLOP/s where without them it ran at 5.0.)
template <int GROUPS, int NT>
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, const uint8_t* tiles) {
    constexpr int kTiles = GROUPS * (1 + NT);
    const int lane = threadIdx.x & 31;
    uint32_t r[4 * kTiles];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
        const int b = j - GROUPS;
        const int tile = j < GROUPS ? j : GROUPS + (b % NT) * GROUPS + b / NT;      // tokens' tiles lie row tile by row tile
        const uint4 u = *reinterpret_cast<const uint4*>(tiles + tile * kScaleTile + lane * 16);
        r[4 * j] = u.x;
        r[4 * j + 1] = u.y;
        r[4 * j + 2] = u.z;
        r[4 * j + 3] = u.w;
    }
    tmem_store<4 * kTiles>(tmem, r);
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// e2m1 (1) at bits 7 and 10, N >> 3 at 17, e8m0 scales (1) at 23, M >> 7 at 27; which of a word's scales: bits 4 and 29.
template <bool MX>
__host__ __device__ constexpr uint32_t instruction(int n, int pair) {
    return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | ((MX ? 1u : 0u) << 23) | (1u << 27) |
           (static_cast<uint32_t>(pair) << 4) | (static_cast<uint32_t>(pair) << 29);
}

template <bool MX>
__device__ __forceinline__ void umma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (MX) {
        asm volatile(
            "{\n.reg .pred p;\n"
            "setp.ne.b32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
    } else {
        asm volatile(
            "{\n.reg .pred p;\n"
            "setp.ne.b32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
    }
}

template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// One rounding, to the output's type.
template <typename T>
__device__ __forceinline__ T finished(float sum, float factor, float bias, int relu) {
    const float v = __fmaf_rn(sum, factor, bias);
    return narrow<T>(relu && v < 0.0f ? 0.0f : v);
}

// The same with the two row factors one after the other, the smaller one first: their product may be infinite where the sum times both
// is 0 or in range (a token near 3e38 against a weight row near 1e8 that is zero where the token is not: 2^117 * 2^16). With the packer's
// factors, powers of two from 2^-100 on, and a sum, a multiple of 2^-20, the first step is exact or overflows as the whole does.
template <typename T>
__device__ __forceinline__ T finished_apart(float sum, float a, float b, float bias, int relu) {
    const bool less = fabsf(a) < fabsf(b);
    return finished<T>(sum * (less ? a : b), less ? b : a, bias, relu);
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float remote_float(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("{\n.reg .b32 a;\nmapa.shared::cluster.u32 a, %1, %2;\nld.shared::cluster.f32 %0, [a];\n}" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

template <int BN, bool MX, typename OutT>
__global__ void __launch_bounds__(kThreads) fp4_linear_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Args a) {
    using C = Cfg<BN, MX>;
    constexpr int kStages = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * C::kStageBytes);      // full[], empty[], scaled[], done, drained
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * kStages + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* token_scale = reinterpret_cast<float*>(tmem_slot + 4);      // BN
    const uint32_t base = smem_u32(smem), bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
    auto scaled = [&](int s) { return bar0 + 8u * (2 * kStages + s); };
    const uint32_t done = bar0 + 8u * (3 * kStages), drained = done + 8u;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = static_cast<int>(cluster_size()), part = static_cast<int>(cluster_rank());
    const int n0 = static_cast<int>(blockIdx.x) / parts * kTileM;      // first output (row of the weights)
    const int kb0 = static_cast<int>(static_cast<int64_t>(a.blocks) * part / parts);
    const int kb1 = static_cast<int>(static_cast<int64_t>(a.blocks) * (part + 1) / parts);
    const int count = kb1 - kb0;

    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
            mbar_init(scaled(s), 4);
        }
        mbar_init(done, 1);
        mbar_init(drained, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"(static_cast<uint32_t>(C::kTmemCols)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            const int64_t groups = static_cast<int64_t>(a.blocks) * C::kGroups;
            const uint8_t* ws = a.w_scales + (n0 / 128) * groups * kScaleTile;
            const uint8_t* xs = a.x_scales;        // of the one row tile
            auto load_w = [&](int i) {
                const int s = i % kStages;
                const uint32_t dst = base + s * C::kStageBytes;
                mbar_expect_tx(full(s), C::kStageBytes);
                tma_load_2d(dst, &map_w, (kb0 + i) * kRowBytes, n0, full(s));
                bulk_load(dst + C::kWBytes + C::kXBytes, ws + static_cast<int64_t>(kb0 + i) * C::kWScale, C::kWScale, full(s));
            };
            auto load_x = [&](int i) {
                const int s = i % kStages;
                const uint32_t dst = base + s * C::kStageBytes;
                tma_load_2d(dst + C::kWBytes, &map_x, (kb0 + i) * kRowBytes, 0, full(s));
                bulk_load(dst + C::kWBytes + C::kXBytes + C::kWScale, xs + static_cast<int64_t>(kb0 + i) * C::kXScale, C::kXScale, full(s));
            };
            // the weights come from before the packer: a ring of them ahead of the wait for it. (The packer lets nothing start before
            // its CTAs have exited, so this is ahead of its writes becoming visible, not beside the packing.)
            const int ahead = a.dependent ? min(kStages, count) : 0;
            for (int i = 0; i < ahead; ++i) load_w(i);
            if (a.dependent) asm volatile("griddepcontrol.wait;" ::: "memory");
            int issued = 0;
            for (int i = 0; i < count; ++i) {
                if (i >= ahead) {
                    if (i >= kStages && !wait_for(empty(i % kStages), (static_cast<uint32_t>(i / kStages) & 1u) ^ 1u, abort_flag, 1)) break;
                    load_w(i);
                }
                load_x(i);
                issued = i + 1;
            }
            if (*abort_flag) {
                for (int i = max(0, issued - kStages); i < issued; ++i) drain(full(i % kStages), static_cast<uint32_t>(i / kStages) & 1u);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            bool ok = true;
            for (int i = 0; i < count; ++i) {
                const int s = i % kStages;
                // the warps that write the scales have waited for the block
                if (!wait_for(scaled(s), static_cast<uint32_t>(i / kStages) & 1u, abort_flag, 2)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t wa = base + s * C::kStageBytes, xa = wa + C::kWBytes;
                const uint32_t ca = tmem + C::kScale0 + s * C::kScaleCols, cb = ca + 4 * C::kGroups;
                const uint64_t da = umma_desc(wa), db = umma_desc(xa);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int g = MX ? k >> 1 : k;
                    umma_fp4<MX>(tmem, da + 2u * k, db + 2u * k, instruction<MX>(BN, MX ? (k & 1) * 2 : 0), ca + 4 * g, cb + 4 * g,
                                 (i | k) != 0 ? 1u : 0u);
                }
                umma_commit(empty(s));
            }
            if (ok) {
                umma_commit(done);
            } else {
                umma_commit(drained);
                drain(drained, 0);
            }
        }
    } else if (warp >= 6) {
        // A stage was loaded again only behind the MMAs that read its last scales, so its columns are free when it is full
        const uint32_t cols = tmem + C::kScale0 + (static_cast<uint32_t>(warp & 3) << 21);      // its quarter: 32 lanes, at bit 16
        for (int i = 0; i < count; ++i) {
            const int s = i % kStages;
            if (!__all_sync(0xFFFFFFFFu, wait_for(full(s), static_cast<uint32_t>(i / kStages) & 1u, abort_flag, 3))) break;
            tc_fence_after();
            scales_to_tmem<C::kGroups, 1>(cols + s * C::kScaleCols, smem + s * C::kStageBytes + C::kWBytes + C::kXBytes);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(scaled(s));
        }
    }
    __syncwarp();

    // epilogue: TMEM lane = output, column = token
    const int quad = warp & 3;
    const int feature = quad * 32 + lane;
    const int n = n0 + feature;
    const bool epi = warp >= 2 && warp < 6;
    bool ok = true;
    float* sums = reinterpret_cast<float*>(smem);
    OutT* y = static_cast<OutT*>(a.y);
    float gw = 1.0f, bias = 0.0f;
    if (epi) {
        if (n < a.N) {
            if (a.w_row != nullptr) gw = a.w_row[n];
            if (a.bias != nullptr) bias = a.bias[n];
        }
        if (a.dependent) asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int c = threadIdx.x - 64; c < BN; c += 128) token_scale[c] = a.x_row != nullptr && c < a.M ? *behind_wait(a.x_row + c) : 1.0f;
        asm volatile("bar.sync 1, 128;" ::: "memory");       // the four epilogue warps
        ok = __all_sync(0xFFFFFFFFu, wait_for(done, 0, abort_flag, 4));
        tc_fence_after();
    }
    auto store = [&](float v, int c) {
        if (c < a.M && n < a.N) y[c * a.ldy + n] = finished_apart<OutT>(v, gw, token_scale[c], bias, a.relu);
    };
    if (epi && ok) {
        const uint32_t at = tmem + (static_cast<uint32_t>(quad * 32) << 16);
        constexpr int kPiece = BN < 32 ? 16 : 32;
        for (int c = 0; c < BN && c < a.M; c += kPiece) {
            int32_t v[32];
            if constexpr (BN < 32) tmem_ld16(at + c, v);
            else tmem_ld32(at + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                if (parts == 1) store(__int_as_float(v[e]), c + e);
                else sums[(c + e) * kTileM + feature] = __int_as_float(v[e]);
            }
        }
    }
    if (parts > 1) {
        cluster_sync();
        if (epi && ok) {
            // tokens beyond M have no sums; an aborted part leaves its ring's contents, and the status word tells
            const int lo = BN * part / parts, hi = BN * (part + 1) / parts;
            for (int c = lo; c < hi && c < a.M; ++c) {
                float v = 0.0f;
                for (int p = 0; p < parts; ++p) v += remote_float(smem_u32(sums + c * kTileM + feature), static_cast<uint32_t>(p));
                store(v, c);
            }
        }
        cluster_sync();      // the others read this CTA's sums
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(static_cast<uint32_t>(C::kTmemCols)) : "memory");
    }
}

// ---- more than 128 tokens: paired CTAs ------------------------------------------------------------------------------------------
//
// A pair of CTAs (tcgen05 cta_group::2) works on 256 outputs x BN tokens: each CTA loads its own 128 rows of the weights, half of the
// tokens and the scales that its tensor core reads, its own weights' and all the tokens'. 38 KB a k-block and CTA for 512 cycles of
// MMAs at BN = 256; a CTA by itself with a tile of 128 x 256 would load 54 KB, and the way from L2 to an SM carries about 64 bytes a cycle.
// Persistent: pairs walk over the tiles, loads run ahead into the next one, and the epilogue takes a finished accumulator into registers
// in one go (8 warps, BN / 2 columns each), hands TMEM back and stores while the next tile's MMAs run.
//   warp 0      TMA producer (both CTAs; operands signal the leader's barrier, a CTA's scales one of its own)
//   warp 1      TMEM; MMA issuer (leader)
//   warps 4-11  epilogue (both CTAs)
//   warps 12-15 each block's scales into TMEM, a set of columns for every stage (both CTAs)
// (Loads and MMAs issued by the scales' warps between blocks: the loads go out late, 3.4 PFLOP/s.)
constexpr int kPairThreads = 512;
constexpr int kPairRegsLow = 72, kPairRegsHigh = 184;       // an epilogue thread holds 128 sums
// setmaxnreg.inc draws only on what the CTA was launched with
static_assert(2 * 128 * kPairRegsLow + 2 * 128 * kPairRegsHigh <= kPairThreads * (65536 / kPairThreads / 8 * 8), "more registers than the CTA has");

template <int BN, bool MX>
struct PairCfg {
    static constexpr int kGroups = MX ? 2 : 4;
    static constexpr int kNTiles = BN / 128;
    static constexpr int kWBytes = kTileM * kRowBytes;
    static constexpr int kXBytes = BN / 2 * kRowBytes;
    static constexpr int kWScale = kGroups * kScaleTile;
    static constexpr int kXScale = kNTiles * kGroups * kScaleTile;
    static constexpr int kStageBytes = kWBytes + kXBytes + kWScale + kXScale;
    static constexpr int kFixed = 8 * (BN / 2) * 4 + 512 + 1024;      // token factors of the 8 epilogue warps, barriers and slots, alignment
    static constexpr int kFit = (232448 - kFixed) / kStageBytes;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    static constexpr int kSmem = kStages * kStageBytes + kFixed;
    static constexpr int kScaleCols = 4 * kGroups * (1 + kNTiles);
    static constexpr int kTmemCols = 512;
    static constexpr int kOperandBytes = kWBytes + kXBytes, kScaleBytes = kWScale + kXScale;
    static_assert(kStageBytes % 1024 == 0 && kStages >= 4 && BN + kStages * kScaleCols <= kTmemCols && (4 * kStages + 3) * 8 + 16 <= 512, "does not fit");
};

__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t leader_bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(leader_bar)
                 : "memory");
}
template <bool MX>
__device__ __forceinline__ void umma_fp4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (MX) {
        asm volatile(
            "{\n.reg .pred p;\n"
            "setp.ne.b32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
    } else {
        asm volatile(
            "{\n.reg .pred p;\n"
            "setp.ne.b32 p, %6, 0;\n"
            "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
    }
}
// Arrives on the barrier at this offset in both CTAs once all earlier MMAs are done.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
// M = 256 over the pair.
template <bool MX>
__host__ __device__ constexpr uint32_t instruction_pair(int n, int pair) {
    return (instruction<MX>(n, pair) & ~(3u << 27)) | (2u << 27);
}

struct PairArgs {
    const float* w_row;
    const float* x_row;
    const float* bias;
    void* y;
    int64_t ldy;
    int M, N, blocks, relu, dependent;
    int tiles_n, tiles;      // tiles along the outputs, in all
};

// A wait that, when it gives up, ends both CTAs' work.
struct PairWait {
    volatile int* flag;
    uint32_t peer_flag;
    __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity, int site) const {
        if (mbar_try(bar, parity)) return true;
        const long long t0 = clock64();
        for (;;) {
            if (mbar_try_parked(bar, parity, 20000u)) return true;
            if (*flag) return false;
            if (clock64() - t0 > kWaitCycles) {
                *flag = 1;
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_flag), "r"(1) : "memory");
                atomicCAS(&g_fp4_status, 0, kSiteBase + site);
                return false;
            }
        }
    }
};

template <int BN, bool MX, typename OutT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    fp4_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_ws,
                    const __grid_constant__ CUtensorMap map_xs, const PairArgs a) {
    using C = PairCfg<BN, MX>;
    constexpr int kStages = C::kStages;
    constexpr int kCols = BN / 2;        // columns of an epilogue warp
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * C::kStageBytes);      // full[], empty[], loaded[], scaled[], tfull, tempty, drained
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 4 * kStages + 3);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* token_scale = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 512);      // [8][kCols]
    const uint32_t base = smem_u32(smem), bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
    auto loaded = [&](int s) { return bar0 + 8u * (2 * kStages + s); };      // a CTA's own scales
    auto scaled = [&](int s) { return bar0 + 8u * (3 * kStages + s); };      // the leader's: both CTAs' scales are in TMEM
    const uint32_t tfull = bar0 + 8u * (4 * kStages), tempty = tfull + 8u, drained = tfull + 16u;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int first = static_cast<int>(blockIdx.x) / 2, step = static_cast<int>(gridDim.x) / 2;
    const PairWait wait{abort_flag, in_cta(smem_u32(const_cast<int*>(abort_flag)), rank ^ 1u)};

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
            mbar_init(loaded(s), 1);
            mbar_init(scaled(s), 8);
        }
        mbar_init(tfull, 1);
        mbar_init(tempty, 16);       // the epilogue warps of both CTAs, at the leader's
        mbar_init(drained, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"(static_cast<uint32_t>(C::kTmemCols)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    const int64_t total = first < a.tiles ? static_cast<int64_t>((a.tiles - 1 - first) / step + 1) * a.blocks : 0;
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairRegsLow));
        if (warp == 0 && lane == 0) {
            if (a.dependent) asm volatile("griddepcontrol.wait;" ::: "memory");
            int64_t issued = 0;
            int s = 0, kb = 0, tile = first;
            uint32_t phase = 0;
            while (issued < total && wait(empty(s), phase ^ 1u, 1)) {
                const int n0 = tile % a.tiles_n * 256, m0 = tile / a.tiles_n * BN;
                const uint32_t dst = base + s * C::kStageBytes, bar = in_cta(full(s), 0), own = loaded(s);
                if (rank == 0) mbar_expect_tx(full(s), 2 * C::kOperandBytes);
                mbar_expect_tx(own, C::kScaleBytes);
                // tiles of 512 bytes are the rows of the scales' maps; a row tile beyond the last reads as zeros
                const uint32_t sc = dst + C::kOperandBytes;
                tma_load_2d(sc, &map_ws, 0, ((n0 >> 7) + static_cast<int>(rank)) * a.blocks * C::kGroups + kb * C::kGroups, own);
#pragma unroll
                for (int q = 0; q < C::kNTiles; ++q)
                    tma_load_2d(sc + C::kWScale + q * C::kGroups * kScaleTile, &map_xs, 0, ((m0 >> 7) + q) * a.blocks * C::kGroups + kb * C::kGroups, own);
                tma_load_pair(dst, &map_w, kb * kRowBytes, n0 + static_cast<int>(rank) * 128, bar);
                tma_load_pair(dst + C::kWBytes, &map_x, kb * kRowBytes, m0 + static_cast<int>(rank) * (BN / 2), bar);
                ++issued;
                if (++kb == a.blocks) {
                    kb = 0;
                    tile += step;
                }
                if (++s == kStages) {
                    s = 0;
                    phase ^= 1u;
                }
            }
            if (issued < total) {
                // let what was issued land (bounded); the operands' barriers that count are the leader's
                for (int64_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i) {
                    const int q = static_cast<int>(i % kStages);
                    const uint32_t p = static_cast<uint32_t>(i / kStages) & 1u;
                    if (rank == 0) drain(full(q), p);
                    drain(loaded(q), p);
                }
            }
        } else if (warp == 1 && lane == 0 && rank == 0) {
            int s = 0, kb = 0;
            uint32_t phase = 0, tphase = 0;
            int64_t i = 0;
            for (; i < total; ++i) {
                if (!((kb != 0 || wait(tempty, tphase ^ 1u, 2)) && wait(full(s), phase, 3) && wait(scaled(s), phase, 4))) break;
                tc_fence_after();
                const uint32_t wa = base + s * C::kStageBytes, xa = wa + C::kWBytes;
                const uint32_t ca = tmem + BN + s * C::kScaleCols, cb = ca + 4 * C::kGroups;
                const uint64_t da = umma_desc(wa), db = umma_desc(xa);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int g = MX ? k >> 1 : k;
                    umma_fp4_pair<MX>(tmem, da + 2u * k, db + 2u * k, instruction_pair<MX>(BN, MX ? (k & 1) * 2 : 0), ca + 4 * g, cb + 4 * g * C::kNTiles,
                                      (kb | k) != 0 ? 1u : 0u);
                }
                commit_pair(empty(s));
                if (++kb == a.blocks) {
                    commit_pair(tfull);
                    kb = 0;
                    tphase ^= 1u;
                }
                if (++s == kStages) {
                    s = 0;
                    phase ^= 1u;
                }
            }
            if (i < total) {
                commit_pair(drained);
                drain(drained, 0);
            }
        }
    } else if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairRegsLow));
        const uint32_t cols = tmem + BN + (static_cast<uint32_t>(warp & 3) << 21);      // the warp's quarter of the lanes, at bit 16
        int s = 0;
        uint32_t phase = 0;
        for (int64_t i = 0; i < total; ++i) {
            // A stage was loaded again only behind the MMAs that read its last scales, so its columns are free when it is full
            if (!__all_sync(0xFFFFFFFFu, wait(loaded(s), phase, 5))) break;
            tc_fence_after();
            scales_to_tmem<C::kGroups, C::kNTiles>(cols + s * C::kScaleCols, smem + s * C::kStageBytes + C::kOperandBytes);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(in_cta(scaled(s), 0)) : "memory");
            if (++s == kStages) {
                s = 0;
                phase ^= 1u;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPairRegsHigh));
        const int quad = warp & 3, half = (warp - 4) >> 2;
        if (a.dependent) asm volatile("griddepcontrol.wait;" ::: "memory");
        const uint32_t leader_tempty = in_cta(tempty, 0);
        uint32_t phase = 0;
        float* scale = token_scale + (warp - 4) * kCols;
        for (int t = first; t < a.tiles; t += step) {
            const int n = t % a.tiles_n * 256 + static_cast<int>(rank) * 128 + quad * 32 + lane, m0 = t / a.tiles_n * BN;
            // what the tile needs beside its sums, while the MMAs run
            const int m = m0 + half * kCols;
            __syncwarp();
            for (int c = lane; c < kCols; c += 32) scale[c] = a.x_row != nullptr && m + c < a.M ? *behind_wait(a.x_row + m + c) : 1.0f;
            const float gw = a.w_row != nullptr && n < a.N ? a.w_row[n] : 1.0f, bias = a.bias != nullptr && n < a.N ? a.bias[n] : 0.0f;
            __syncwarp();
            // The product of two row factors is one instruction less an output than one factor after the other; a warp whose factors could
            // leave float32's normal numbers together (also a NaN: the largest as a whole number) takes them apart.
            bool apart = false;
            if constexpr (!MX) {
                uint32_t high = 0u, low = 0xFFFFFFFFu;
                for (int c = lane; c < kCols; c += 32) {
                    const uint32_t bits = __float_as_uint(fabsf(scale[c]));
                    high = max(high, bits);
                    low = min(low, bits);
                }
                const uint32_t w = __float_as_uint(fabsf(gw));
                const float most = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, high)) * __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, w));
                const float least = __uint_as_float(__reduce_min_sync(0xFFFFFFFFu, low)) * __uint_as_float(__reduce_min_sync(0xFFFFFFFFu, w));
                apart = !(most < CUDART_INF_F && least >= 1.17549435e-38f);
            }
            if (!__all_sync(0xFFFFFFFFu, wait(tfull, phase, 6))) break;
            phase ^= 1u;
            tc_fence_after();
            int32_t v[kCols / 32][32];
            const uint32_t at = tmem + (static_cast<uint32_t>(quad * 32) << 16) + half * kCols;
#pragma unroll
            for (int q = 0; q < kCols / 32; ++q) tmem_ld32(at + q * 32, v[q]);
#pragma unroll
            for (int q = 0; q < kCols / 32; ++q) tmem_ld_wait_for(v[q]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(leader_tempty) : "memory");
            const int tokens = min(kCols, a.M - m);
            if (n < a.N) {
                OutT* y = static_cast<OutT*>(a.y) + static_cast<int64_t>(m) * a.ldy + n;
                if (apart) {
                    // seldom: a small loop over a copy in local memory, so that the code around it stays as short as without
                    float sums[kCols];
#pragma unroll
                    for (int c = 0; c < kCols; ++c) sums[c] = __int_as_float(v[c / 32][c % 32]);
#pragma unroll 1
                    for (int c = 0; c < tokens; ++c, y += a.ldy) *y = finished_apart<OutT>(sums[c], gw, scale[c], bias, a.relu);
                } else if (tokens == kCols) {
#pragma unroll
                    for (int c = 0; c < kCols; ++c, y += a.ldy) *y = finished<OutT>(__int_as_float(v[c / 32][c % 32]), gw * scale[c], bias, a.relu);
                } else {
#pragma unroll
                    for (int c = 0; c < kCols; ++c, y += a.ldy)
                        if (c < tokens) *y = finished<OutT>(__int_as_float(v[c / 32][c % 32]), gw * scale[c], bias, a.relu);
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();      // the other CTA's MMAs read this one's shared memory, its warps signal this one's barriers
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(static_cast<uint32_t>(C::kTmemCols)) : "memory");
    }
}

int make_codes_map(CUtensorMap* map, const uint8_t* codes, int64_t rows, int64_t bytes, int64_t ld, int box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return fail(BSI_ERR_CUDA, "fp4_linear: cuTensorMapEncodeTiled entry point not found");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(bytes), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(kRowBytes), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("fp4_linear: cuTensorMapEncodeTiled failed with CUresult %d", static_cast<int>(r));
        return BSI_ERR_CUDA;
    }
    return BSI_OK;
}

struct Operands {
    const uint8_t *w, *x;
    int64_t ldw, ldx, K;
};

template <int BN, bool MX, typename OutT>
int launch(const Operands& o, const Args& a, cudaStream_t stream) {
    using C = Cfg<BN, MX>;
    static bool attr_set[64] = {false};
    int dev = 0;
    BSI_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        BSI_CUDA_TRY(cudaFuncSetAttribute(fp4_linear_kernel<BN, MX, OutT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    CUtensorMap mw, mx;
    const int64_t bytes = (o.K + 31) / 32 * 16;
    int rc = make_codes_map(&mw, o.w, a.N, bytes, o.ldw, kTileM);
    if (rc == BSI_OK) rc = make_codes_map(&mx, o.x, a.M, bytes, o.ldx, BN);
    if (rc != BSI_OK) return rc;
    const int tiles_n = (a.N + kTileM - 1) / kTileM;
    const int64_t slots = static_cast<int64_t>(C::kPerSm) * sm_count();
    int parts = 1;
    while (parts < 8 && static_cast<int64_t>(tiles_n) * parts * 2 <= slots && a.blocks >= parts * 4) parts *= 2;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(parts);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(tiles_n * parts), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = a.dependent ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, fp4_linear_kernel<BN, MX, OutT>, mw, mx, a);
    if (e != cudaSuccess) {
        set_error("fp4_linear launch: %s", cudaGetErrorString(e));
        return BSI_ERR_CUDA;
    }
    return BSI_OK;
}

// The scales as rows of 512 bytes, `groups` of them a box.
int make_scales_map(CUtensorMap* map, const uint8_t* scales, int64_t tiles, int groups) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return fail(BSI_ERR_CUDA, "fp4_linear: cuTensorMapEncodeTiled entry point not found");
    const cuuint64_t dims[2] = {kScaleTile / 4, static_cast<cuuint64_t>(tiles)};
    const cuuint64_t strides[1] = {kScaleTile};
    const cuuint32_t box[2] = {kScaleTile / 4, static_cast<cuuint32_t>(groups)};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<uint8_t*>(scales), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("fp4_linear: cuTensorMapEncodeTiled failed with CUresult %d", static_cast<int>(r));
        return BSI_ERR_CUDA;
    }
    return BSI_OK;
}

template <int BN, bool MX, typename OutT>
int launch_pair(const Operands& o, const Args& a, cudaStream_t stream) {
    using C = PairCfg<BN, MX>;
    static bool attr_set[64] = {false};
    int dev = 0;
    BSI_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        BSI_CUDA_TRY(cudaFuncSetAttribute(fp4_pair_kernel<BN, MX, OutT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    CUtensorMap mw, mx, mws, mxs;
    const int64_t bytes = (o.K + 31) / 32 * 16, per_row_tile = static_cast<int64_t>(a.blocks) * C::kGroups;
    int rc = make_codes_map(&mw, o.w, a.N, bytes, o.ldw, kTileM);
    if (rc == BSI_OK) rc = make_codes_map(&mx, o.x, a.M, bytes, o.ldx, BN / 2);
    if (rc == BSI_OK) rc = make_scales_map(&mws, a.w_scales, (a.N + 127ll) / 128 * per_row_tile, C::kGroups);
    if (rc == BSI_OK) rc = make_scales_map(&mxs, a.x_scales, (a.M + 127ll) / 128 * per_row_tile, C::kGroups);
    if (rc != BSI_OK) return rc;
    PairArgs p{a.w_row, a.x_row, a.bias, a.y, a.ldy, a.M, a.N, a.blocks, a.relu, a.dependent, (a.N + 255) / 256, 0};
    p.tiles = p.tiles_n * ((a.M + BN - 1) / BN);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min(p.tiles, sm_count() / 2)), 1, 1);
    cfg.blockDim = dim3(kPairThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = a.dependent ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, fp4_pair_kernel<BN, MX, OutT>, mw, mx, mws, mxs, p);
    if (e != cudaSuccess) {
        set_error("fp4_linear launch: %s", cudaGetErrorString(e));
        return BSI_ERR_CUDA;
    }
    return BSI_OK;
}

template <bool MX, typename OutT>
int launch_width(const Operands& o, const Args& a, cudaStream_t stream) {
    if (a.M <= 16) return launch<16, MX, OutT>(o, a, stream);
    if (a.M <= 32) return launch<32, MX, OutT>(o, a, stream);
    if (a.M <= 64) return launch<64, MX, OutT>(o, a, stream);
    if (a.M <= 128) return launch<128, MX, OutT>(o, a, stream);
    // rounds of the GPU's pairs over tiles of 256 or 128 tokens; a narrow tile's MMAs are half as long, its loads three quarters
    const int64_t pairs = sm_count() / 2, outputs = (a.N + 255) / 256;
    const int64_t wide = (outputs * ((a.M + 255) / 256) + pairs - 1) / pairs, narrow_ = (outputs * ((a.M + 127) / 128) + pairs - 1) / pairs;
    if (wide * 4 <= narrow_ * 3) return launch_pair<256, MX, OutT>(o, a, stream);
    return launch_pair<128, MX, OutT>(o, a, stream);
}

template <bool MX>
int launch_type(const Operands& o, const Args& a, int dtype, cudaStream_t stream) {
    switch (dtype) {
        case BSI_DTYPE_F32: return launch_width<MX, float>(o, a, stream);
        case BSI_DTYPE_F16: return launch_width<MX, __half>(o, a, stream);
        default: return launch_width<MX, __nv_bfloat16>(o, a, stream);
    }
}

}  // namespace
}  // namespace bsi

extern "C" int bsi_b200_fp4_linear(const uint8_t* x_codes, int64_t ldx, const uint8_t* x_scales, const float* x_row_scale,
                                   const uint8_t* w_codes, int64_t ldw, const uint8_t* w_scales, const float* w_row_scale, const float* bias,
                                   int64_t M, int64_t N, int64_t K, int format, void* y, int64_t ldy, int y_dtype, int activation, int behind_packer,
                                   bsi_stream_t stream) {
    using namespace bsi;
    if (format != BSI_FP4_MX && format != BSI_FP4_NV) {
        set_error("fp4_linear: format must be BSI_FP4_MX or BSI_FP4_NV, got %d", format);
        return BSI_ERR_INVALID;
    }
    if (y_dtype != BSI_DTYPE_F32 && y_dtype != BSI_DTYPE_F16 && y_dtype != BSI_DTYPE_BF16) {
        set_error("fp4_linear: y_dtype must be a BSI_DTYPE_* code, got %d", y_dtype);
        return BSI_ERR_INVALID;
    }
    if (activation != BSI_ACT_NONE && activation != BSI_ACT_RELU) return fail(BSI_ERR_INVALID, "fp4_linear: activation must be BSI_ACT_NONE or BSI_ACT_RELU");
    const int64_t least = (K + 31) / 32 * 16;
    if (M < 0 || N < 0 || K < 1 || M > (1ll << 23) || N > (1ll << 24) || K > (1ll << 30) || ldx % 16 != 0 || ldw % 16 != 0 || ldx < least || ldw < least || ldy < N) {
        set_error("fp4_linear: %lld x %lld x %lld, codes %lld and %lld bytes apart, outputs %lld", static_cast<long long>(M), static_cast<long long>(N),
                  static_cast<long long>(K), static_cast<long long>(ldx), static_cast<long long>(ldw), static_cast<long long>(ldy));
        return BSI_ERR_INVALID;
    }
    if (M == 0 || N == 0) return BSI_OK;
    if (x_codes == nullptr || x_scales == nullptr || w_codes == nullptr || w_scales == nullptr || y == nullptr) return fail(BSI_ERR_INVALID, "fp4_linear: null operand");
    if (format == BSI_FP4_NV && (x_row_scale == nullptr || w_row_scale == nullptr)) return fail(BSI_ERR_INVALID, "fp4_linear: nvfp4 operands need row scales");
    if ((reinterpret_cast<uintptr_t>(x_codes) | reinterpret_cast<uintptr_t>(w_codes) | reinterpret_cast<uintptr_t>(x_scales) | reinterpret_cast<uintptr_t>(w_scales)) & 15u)
        return fail(BSI_ERR_INVALID, "fp4_linear: codes and scales must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(x_row_scale) | reinterpret_cast<uintptr_t>(w_row_scale) | reinterpret_cast<uintptr_t>(bias)) & 3u)
        return fail(BSI_ERR_INVALID, "fp4_linear: misaligned row scales or bias");
    if (reinterpret_cast<uintptr_t>(y) % (y_dtype == BSI_DTYPE_F32 ? 4 : 2) != 0) return fail(BSI_ERR_INVALID, "fp4_linear: misaligned output");
    const int rc = require_sm100();
    if (rc != BSI_OK) return rc;
    Args a{w_scales, x_scales, format == BSI_FP4_NV ? w_row_scale : nullptr, format == BSI_FP4_NV ? x_row_scale : nullptr, bias, y, ldy,
           static_cast<int>(M), static_cast<int>(N), static_cast<int>((K + 255) / 256), activation == BSI_ACT_RELU ? 1 : 0,
           behind_packer != 0 && pdl_enabled() ? 1 : 0};
    const Operands o{w_codes, x_codes, ldw, ldx, K};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return format == BSI_FP4_MX ? launch_type<true>(o, a, y_dtype, s) : launch_type<false>(o, a, y_dtype, s);
}
