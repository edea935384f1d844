// Product of two 4-bit matrices on the 5th-generation tensor cores:
//     y[m][n] = act( (sum_k x[m][k] w[n][k]) * gx[m] * gw[n] + bias[n] ),   x, w: e2m1 values times their block scales
//
// tcgen05.mma.kind::mxf4 / mxf4nvf4 multiplies the codes and both block scales itself (K = 64 per instruction) and accumulates in
// float32 in TMEM; what is left for the epilogue are the per-row factors of the nvfp4 format, the bias, ReLU and one rounding.
//
// The weights' rows are the instruction's M (128 TMEM lanes), the tokens its N: one form serves one token (N = 16) and a prompt
// (N = 256), and a warp of the epilogue stores 32 neighbouring outputs of a token.
//
//   warp 0     TMA producer: per k-block of 256 elements one box of weights (128 x 128 B), one of tokens (BN x 128 B), both 128-byte
//              swizzled, and their scales as they lie in memory (512 bytes for 128 rows x 4 scales, whole tiles)
//   warp 1     MMA issuer: tcgen05.cp of the block's scales into TMEM (two sets in turn), 4 MMAs of K = 64
//   warps 2-5  epilogue
// Where the tiles leave SMs idle, a cluster of 2, 4 or 8 CTAs shares a tile, each with a part of K; the parts' float32 sums meet in
// shared memory and are added in the parts' order, each CTA for its share of the tokens.
// Every wait is bounded: on a timeout the role records its site in the status word, raises the CTA's abort flag, what is under way is
// waited for (bounded again), TMEM is freed and the kernel returns.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
constexpr int kThreads = 192;
constexpr int kScaleTile = 512;        // 128 rows x 4 scales
constexpr long long kWaitCycles = 500000000ll;    // about 0.25 s; real waits are microseconds
constexpr int kSiteBase = 128;         // of the status word: sites 129 and up are this kernel's

template <int BN, bool MX>
struct Cfg {
    static constexpr int kGroups = MX ? 2 : 4;                   // scale tiles of a k-block per 128 rows
    static constexpr int kNTiles = BN > 128 ? 2 : 1;             // scale row tiles that BN tokens lie in
    static constexpr int kWBytes = kTileM * kRowBytes;
    static constexpr int kXBytes = BN * kRowBytes;
    static constexpr int kWScale = kGroups * kScaleTile;
    static constexpr int kXScale = kNTiles * kGroups * kScaleTile;
    static constexpr int kStageBytes = kWBytes + kXBytes + kWScale + kXScale;      // a multiple of 1 KB
    // two CTAs per SM for the narrow tiles, whose MMAs are short beside their loads
    static constexpr int kPerSm = BN <= 64 ? 2 : 1;
    static constexpr int kBudget = (kPerSm == 2 ? 113 : 226) * 1024 - 2048;
    static constexpr int kStages = kBudget / kStageBytes > 8 ? 8 : kBudget / kStageBytes;
    static constexpr int kSmem = kStages * kStageBytes + (2 * kStages + 2) * 8 + 32 + 1024;
    // TMEM: the accumulator, then two sets of scales (4 columns for each tile of 512 bytes)
    static constexpr int kScaleCols = 4 * kGroups * (1 + kNTiles);
    static constexpr int kScale0 = BN < 32 ? 32 : BN;
    static constexpr int kNeed = kScale0 + 2 * kScaleCols;
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
    int dependent;           // the packer in front may still be running: what it writes is read behind griddepcontrol.wait
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

// 512 bytes of scales: 32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
    return static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(128u >> 4) << 32) | (1ull << 46);
}

__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
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
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * C::kStageBytes);      // full[], empty[], done, drain
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t base = smem_u32(smem), bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
    const uint32_t done = bar0 + 8u * (2 * kStages), drained = done + 8u;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = static_cast<int>(cluster_size()), part = static_cast<int>(cluster_rank());
    const int n0 = static_cast<int>(blockIdx.x) / parts * kTileM;      // first output (row of the weights)
    const int m0 = static_cast<int>(blockIdx.y) * BN;                  // first token
    const int kb0 = static_cast<int>(static_cast<int64_t>(a.blocks) * part / parts);
    const int kb1 = static_cast<int>(static_cast<int64_t>(a.blocks) * (part + 1) / parts);
    const int count = kb1 - kb0;

    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
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
            // the tokens' scale tiles that are there (the last column tile may end in the first)
            const int x_tiles = C::kNTiles == 2 && m0 + 128 < a.M ? 2 : 1;
            const uint32_t bytes = static_cast<uint32_t>(C::kWBytes + C::kXBytes + C::kWScale + x_tiles * C::kGroups * kScaleTile);
            const int64_t groups = static_cast<int64_t>(a.blocks) * C::kGroups;
            const uint8_t* ws = a.w_scales + (n0 / 128) * groups * kScaleTile;
            const uint8_t* xs = a.x_scales + (m0 / 128) * groups * kScaleTile;
            auto load_w = [&](int i) {
                const int s = i % kStages;
                const uint32_t dst = base + s * C::kStageBytes;
                mbar_expect_tx(full(s), bytes);
                tma_load_2d(dst, &map_w, (kb0 + i) * kRowBytes, n0, full(s));
                bulk_load(dst + C::kWBytes + C::kXBytes, ws + static_cast<int64_t>(kb0 + i) * C::kWScale, C::kWScale, full(s));
            };
            auto load_x = [&](int i) {
                const int s = i % kStages;
                const uint32_t dst = base + s * C::kStageBytes;
                tma_load_2d(dst + C::kWBytes, &map_x, (kb0 + i) * kRowBytes, m0, full(s));
                for (int t = 0; t < x_tiles; ++t)
                    bulk_load(dst + C::kWBytes + C::kXBytes + C::kWScale + t * C::kGroups * kScaleTile,
                              xs + (t * groups + static_cast<int64_t>(kb0 + i) * C::kGroups) * kScaleTile, C::kGroups * kScaleTile, full(s));
            };
            // the weights come from before the packer: a ring of them ahead of the wait for it
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
                if (!wait_for(full(s), static_cast<uint32_t>(i / kStages) & 1u, abort_flag, 2)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t wa = base + s * C::kStageBytes, xa = wa + C::kWBytes;
                const uint32_t sa = xa + C::kXBytes, sb = sa + C::kWScale;
                // a set of columns is written again only two blocks later; copies and MMAs of one thread run in order
                const uint32_t cols = tmem + C::kScale0 + (i & 1) * C::kScaleCols;
                const uint32_t ca = cols, cb = cols + 4 * C::kGroups;
#pragma unroll
                for (int g = 0; g < C::kGroups; ++g) {
                    copy_scales(ca + 4 * g, scale_desc(sa + g * kScaleTile));
#pragma unroll
                    for (int t = 0; t < C::kNTiles; ++t)      // the columns of one group behind one another, 128 tokens each
                        copy_scales(cb + 4 * (g * C::kNTiles + t), scale_desc(sb + (t * C::kGroups + g) * kScaleTile));
                }
                const uint64_t da = umma_desc(wa), db = umma_desc(xa);
                const uint32_t col = BN < 128 ? (m0 % 128) / 32 : 0;      // tokens 32 to a column
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int g = MX ? k >> 1 : k;
                    umma_fp4<MX>(tmem, da + 2u * k, db + 2u * k, instruction<MX>(BN, MX ? (k & 1) * 2 : 0), ca + 4 * g, cb + 4 * g * C::kNTiles + col,
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
    }
    __syncwarp();

    // epilogue: TMEM lane = output, column = token
    const int quad = warp & 3;
    const int feature = quad * 32 + lane;
    const int n = n0 + feature;
    const bool epi = warp >= 2;
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
        ok = __all_sync(0xFFFFFFFFu, wait_for(done, 0, abort_flag, 3));
        tc_fence_after();
    }
    auto store = [&](float v, int m) {
        if (m < a.M && n < a.N) {
            const float gx = a.x_row != nullptr ? a.x_row[m] : 1.0f;
            v = __fmaf_rn(v, gw * gx, bias);
            if (a.relu && v < 0.0f) v = 0.0f;
            y[static_cast<int64_t>(m) * a.ldy + n] = narrow<OutT>(v);
        }
    };
    if (epi && ok) {
        const uint32_t at = tmem + (static_cast<uint32_t>(quad * 32) << 16);
        constexpr int kPiece = BN < 32 ? 16 : 32;
        for (int c = 0; c < BN && m0 + c < a.M; c += kPiece) {
            int32_t v[32];
            if constexpr (BN < 32) tmem_ld16(at + c, v);
            else tmem_ld32(at + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                if (parts == 1) store(__int_as_float(v[e]), m0 + c + e);
                else sums[(c + e) * kTileM + feature] = __int_as_float(v[e]);
            }
        }
    }
    if (parts > 1) {
        cluster_sync();
        if (epi && ok) {
            // tokens beyond M have no sums; an aborted part leaves its ring's contents, and the status word tells
            const int lo = BN * part / parts, hi = BN * (part + 1) / parts;
            for (int c = lo; c < hi && m0 + c < a.M; ++c) {
                float v = 0.0f;
                for (int p = 0; p < parts; ++p) v += remote_float(smem_u32(sums + c * kTileM + feature), static_cast<uint32_t>(p));
                store(v, m0 + c);
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
    const int tiles_n = (a.N + kTileM - 1) / kTileM, tiles_m = (a.M + BN - 1) / BN;
    const int64_t slots = static_cast<int64_t>(C::kPerSm) * sm_count();
    int parts = 1;
    while (parts < 8 && static_cast<int64_t>(tiles_n) * tiles_m * parts * 2 <= slots && a.blocks >= parts * 4) parts *= 2;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(parts);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(tiles_n * parts), static_cast<unsigned>(tiles_m), 1);
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

template <bool MX, typename OutT>
int launch_width(const Operands& o, const Args& a, cudaStream_t stream) {
    if (a.M <= 16) return launch<16, MX, OutT>(o, a, stream);
    if (a.M <= 32) return launch<32, MX, OutT>(o, a, stream);
    if (a.M <= 64) return launch<64, MX, OutT>(o, a, stream);
    if (a.M <= 128) return launch<128, MX, OutT>(o, a, stream);
    return launch<256, MX, OutT>(o, a, stream);
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
