// Log probabilities of given tokens, and distillation from a teacher's top logits: kernels over rows of logits.
//
// Both need the softmax statistics of every row, so both are one pass over the logits with a running maximum and sum per thread
// (vocab.cuh), joined in a block and then in a cluster. What bounds them is the logits' bytes.
#include <algorithm>

#include "vocab.cuh"

namespace bsi {
namespace {

namespace cg = cooperative_groups;
using vocab::kThreads;
using vocab::kWarps;
using vocab::Piece;
using vocab::RowPlan;
using vocab::Span;
using vocab::Stats;

constexpr int kBatch = 4;               // 16-byte pieces that a thread has under way
constexpr int kMaxTop = 128;            // alternatives of token_logprobs
constexpr int kCandidates = 2048;       // entries at least as large as the block's bound that it keeps
constexpr int kMaxListed = 512;         // teacher entries per row

// ---- log probabilities, ranks, entropy, top alternatives ---------------------------------------------------------------------
//
// For a row z and a token t:  logprob = z_t - lse,  lse = m + log sum exp(z - m),  entropy = lse - sum p z,
// rank = #{z_j > z_t} + #{j < t, z_j = z_t}, top = the k largest, equal values by ascending index.
//
// The top k ride on the same pass. The largest value that each thread met is its running maximum; with B the k-th largest of those
// 512 maxima, at least k entries are >= B, so the k largest all are, and few others. A search over the upper 16 bits of the ordered
// maxima (16 votes of the block) finds a B that is no larger; only threads whose maximum reaches it look at their pieces again
// (out of L2), and the entries found are put in order by counting for each one how many come before it.
// Where more than kCandidates entries reach B (a row that is -inf but for a few, a constant row), the block selects by radix: four
// passes over 8 bits each give the k-th value, one pass the larger entries, one in index order the equal ones.

struct ScoreArgs {
    const void* logits;
    RowPlan rows;
    int64_t V;
    const int64_t* tokens;
    RowPlan tokens_at;
    int top;
    float* logprobs;
    int64_t* ranks;
    float* entropy;
    float* top_logprobs;
    int64_t* top_ids;
};

struct ScoreShared {
    Stats warp[kWarps];
    int warp_ahead[kWarps];
    Stats mine;          // this CTA's part of the row, read by CTA 0
    int ahead;
    int found;           // candidates
    int listed;          // entries in `best`: min(top, elements of this part)
    uint32_t hist[256];
    uint32_t prefix, need;
    unsigned long long best[kMaxTop];      // this CTA's largest, in order
    unsigned long long cand[kCandidates];
};

__device__ __forceinline__ unsigned long long sort_key(float v, int64_t index) {
    return (static_cast<unsigned long long>(vocab::ordered(v)) << 32) | static_cast<uint32_t>(~static_cast<uint32_t>(index));
}

// The exact k largest of [lo, hi) into sh.cand[0 .. k), in no order, for any contents. All threads; k <= hi - lo.
template <typename T>
__device__ void select_by_radix(ScoreShared& sh, const T* row, int64_t lo, int64_t hi, int k) {
    uint32_t prefix = 0;
    int need = k;        // entries still to be found among those that share the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kThreads) sh.hist[i] = 0;
        __syncthreads();
        for (int64_t i0 = lo; i0 < hi; i0 += kThreads) {
            const int64_t i = i0 + threadIdx.x;
            const uint32_t key = i < hi ? vocab::ordered(Piece<T>::one(row[i])) : 0u;
            const bool in = i < hi && (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)));
            const uint32_t bin = in ? (key >> shift) & 255u : 256u;
            const unsigned same = __match_any_sync(0xFFFFFFFFu, bin);      // one addition per warp and bin
            if (in && (__ffs(same) - 1) == static_cast<int>(threadIdx.x & 31)) atomicAdd(&sh.hist[bin], static_cast<uint32_t>(__popc(same)));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int left = need, b = 255;
            while (b > 0 && static_cast<int>(sh.hist[b]) < left) left -= static_cast<int>(sh.hist[b--]);
            sh.prefix = prefix | (static_cast<uint32_t>(b) << shift);
            sh.need = static_cast<uint32_t>(left);
        }
        __syncthreads();
        prefix = sh.prefix;
        need = static_cast<int>(sh.need);
        __syncthreads();
    }
    // k - need entries are larger than the k-th value, and need of those equal to it are wanted, lowest index first
    if (threadIdx.x == 0) sh.found = 0;
    __syncthreads();
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) {
        const float v = Piece<T>::one(row[i]);
        if (vocab::ordered(v) > prefix) sh.cand[atomicAdd(&sh.found, 1)] = sort_key(v, i);
    }
    __syncthreads();
    int taken = 0;
    for (int64_t i0 = lo; i0 < hi && taken < need; i0 += kThreads) {
        const int64_t i = i0 + threadIdx.x;
        const float v = i < hi ? Piece<T>::one(row[i]) : 0.0f;
        const bool eq = i < hi && vocab::ordered(v) == prefix;
        const unsigned votes = __ballot_sync(0xFFFFFFFFu, eq);
        if ((threadIdx.x & 31) == 0) sh.warp_ahead[threadIdx.x >> 5] = __popc(votes);
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < kWarps; ++w) {
            const int n = sh.warp_ahead[w];
            if (w < static_cast<int>(threadIdx.x >> 5)) before += n;
            all += n;
        }
        const int place = taken + before + __popc(votes & ((1u << (threadIdx.x & 31)) - 1u));
        if (eq && place < need) sh.cand[(k - need) + place] = sort_key(v, i);
        taken += all;
        __syncthreads();
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) score_kernel(const ScoreArgs a) {
    constexpr int kVec = Piece<T>::kVec;
    constexpr int N = kBatch * kVec;
    __shared__ ScoreShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = static_cast<int>(cluster.num_blocks());
    const int part = static_cast<int>(cluster.block_rank());
    const int64_t r = blockIdx.x / parts;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    const T* row = static_cast<const T*>(a.logits) + a.rows.at(r);
    const Span<T> span(row, a.V, part, parts);
    const int64_t token = a.tokens == nullptr ? -1 : a.tokens[a.tokens_at.at(r)];
    const bool scored = token >= 0 && token < a.V;
    const float zt = scored ? Piece<T>::one(row[token]) : CUDART_INF_F;

    Stats st{-CUDART_INF_F, 0.0f, 0.0f};
    int ahead = 0;
    for (int64_t v = span.first + tid; v < span.last; v += kBatch * kThreads) {
        float z[N];
        if (v >= span.lo && v + (kBatch - 1) * kThreads < min(span.hi, span.last)) {
            uint4 u[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) u[b] = span.grid[v + b * kThreads];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) Piece<T>::unpack(u[b], z + b * kVec);
        } else {
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int64_t p = v + b * kThreads;
                if (p < span.last) {
                    span.load(p, z + b * kVec);
                } else {
#pragma unroll
                    for (int e = 0; e < kVec; ++e) z[b * kVec + e] = -CUDART_INF_F;
                }
            }
        }
        vocab::take<N, true>(st, z, vocab::kLog2e);
        if (scored) {
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                if (v + b * kThreads >= span.last) break;
                const int64_t e0 = span.element(v + b * kThreads);
                if (e0 > token || e0 + kVec <= token) {
                    // what lies before the token also counts where it is equal; -inf beyond the row's ends is below or, for a
                    // token at -inf, has to be left out
                    const bool before = e0 < token;
#pragma unroll
                    for (int e = 0; e < kVec; ++e) {
                        const float x = z[b * kVec + e];
                        ahead += x > zt || (before && x == zt && e0 + e >= 0);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < kVec; ++e) {
                        const float x = z[b * kVec + e];
                        ahead += x > zt || (x == zt && e0 + e < token && e0 + e >= 0);
                    }
                }
            }
        }
    }

    // the block's statistics
    const float own_max = st.m;
    Stats all = vocab::warp_merge(st, vocab::kLog2e);
    ahead = __reduce_add_sync(0xFFFFFFFFu, ahead);
    if (lane == 0) {
        sh.warp[warp] = all;
        sh.warp_ahead[warp] = ahead;
    }
    if (tid == 0) sh.found = 0;
    __syncthreads();
    if (warp == 0) {
        all = lane < kWarps ? sh.warp[lane] : Stats{-CUDART_INF_F, 0.0f, 0.0f};
        all = vocab::warp_merge(all, vocab::kLog2e);
        const int n = __reduce_add_sync(0xFFFFFFFFu, lane < kWarps ? sh.warp_ahead[lane] : 0);
        if (lane == 0) {
            sh.mine = all;
            sh.ahead = n;
        }
    }

    if (a.top > 0) {
        const int64_t mine = span.end() - span.begin();
        const int k = static_cast<int>(min(static_cast<int64_t>(a.top), mine > 0 ? mine : 0));
        // pieces without a thread of their own never raise a maximum: such threads do not vote
        const bool has = span.first + tid < span.last;
        const uint32_t key = vocab::ordered(own_max);
        uint32_t bound = 0;
        for (int bit = 31; bit >= 16; --bit) {
            const uint32_t tryit = bound | (1u << bit);
            if (__syncthreads_count(has && key >= tryit) >= k) bound = tryit;
        }
        if (has && (key >= bound)) {
            for (int64_t v = span.first + tid; v < span.last; v += kThreads) {
                float z[kVec];
                span.load(v, z);
                const int64_t e0 = span.element(v);
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    if (vocab::ordered(z[e]) >= bound && e0 + e >= 0 && e0 + e < a.V) {
                        const int place = atomicAdd(&sh.found, 1);
                        if (place < kCandidates) sh.cand[place] = sort_key(z[e], e0 + e);
                    }
                }
            }
        }
        __syncthreads();
        int n = sh.found;
        __syncthreads();
        if (n > kCandidates) {
            select_by_radix<T>(sh, row, span.begin(), span.end(), k);
            n = k;
        }
        for (int i = tid; i < n; i += kThreads) {
            const unsigned long long own = sh.cand[i];
            int place = 0;
            for (int j = 0; j < n; ++j) place += sh.cand[j] > own;
            if (place < k) sh.best[place] = own;
        }
        if (tid == 0) sh.listed = k;
    }
    cluster.sync();

    if (part == 0) {
        Stats total = sh.mine;
        int before = sh.ahead;
        for (int p = 1; p < parts; ++p) {
            const ScoreShared* other = cluster.map_shared_rank(&sh, p);
            total = vocab::merge(total, other->mine, vocab::kLog2e);
            before += other->ahead;
        }
        const float log_s = logf(total.s);
        if (tid == 0) {
            if (a.logprobs != nullptr) a.logprobs[r] = scored ? (zt - total.m) - log_s : 0.0f;
            if (a.ranks != nullptr) a.ranks[r] = scored ? before : -1;
            // entropy = lse - sum p z = log s - (sum e d) ln 2 / s with d = log2 e; a row of -inf has none
            if (a.entropy != nullptr) a.entropy[r] = total.m == -CUDART_INF_F ? CUDART_NAN_F : log_s - total.w * vocab::kLn2 / total.s;
        }
        // every CTA's list is in order: an entry's place is its own plus, in each other list, how many come before it
        for (int i = tid; i < parts * a.top; i += kThreads) {
            const int p = i / a.top, q = i % a.top;
            const ScoreShared* list = cluster.map_shared_rank(&sh, p);
            if (q >= list->listed) continue;
            const unsigned long long key = list->best[q];
            int place = q;
            for (int o = 0; o < parts; ++o) {
                if (o == p) continue;
                const ScoreShared* other = cluster.map_shared_rank(&sh, o);
                int lo = 0, hi = other->listed;
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (other->best[mid] > key) lo = mid + 1;
                    else hi = mid;
                }
                place += lo;
            }
            if (place < a.top) {
                const float z = vocab::from_ordered(static_cast<uint32_t>(key >> 32));
                a.top_logprobs[r * a.top + place] = (z - total.m) - log_s;
                a.top_ids[r * a.top + place] = static_cast<int64_t>(~static_cast<uint32_t>(key));
            }
        }
    }
    cluster.sync();      // CTA 0 reads the others' shared memory
}

// CTAs per row: as many as fill the GPU once with two CTAs per SM, each with at least two batches of the threads' pieces.
int parts_for(int64_t rows, int64_t V, int esz) {
    const int64_t pieces = (V * esz + 15) / 16;
    int parts = 1;
    while (parts < vocab::kMaxCluster && rows * parts * 2 <= 2 * static_cast<int64_t>(sm_count()) && pieces >= static_cast<int64_t>(parts) * 2 * kThreads * 2) parts *= 2;
    return parts;
}

template <typename Kernel, typename... Args>
int launch_rows(Kernel kernel, int64_t rows, int parts, int64_t smem, cudaStream_t stream, const char* what, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(parts);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(rows * parts), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e != cudaSuccess) {
        set_error("%s: %s", what, cudaGetErrorString(e));
        return BSI_ERR_CUDA;
    }
    return BSI_OK;
}

constexpr int64_t kMaxRows = 0x7FFFFFFFll / vocab::kMaxCluster;

int check_rows(const char* what, const void* logits, int dtype, int64_t rows, int64_t V, const bsi_row_plan* plan) {
    if (dtype != BSI_DTYPE_F32 && dtype != BSI_DTYPE_F16 && dtype != BSI_DTYPE_BF16) {
        set_error("%s: dtype must be a BSI_DTYPE_* code, got %d", what, dtype);
        return BSI_ERR_INVALID;
    }
    if (rows < 0 || V < 1 || rows > kMaxRows || V > 0x7FFFFFFFll) {
        set_error("%s: %lld rows of %lld logits", what, static_cast<long long>(rows), static_cast<long long>(V));
        return BSI_ERR_INVALID;
    }
    if (rows > 0 && logits == nullptr) {
        set_error("%s: null logits", what);
        return BSI_ERR_INVALID;
    }
    const int esz = dtype == BSI_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % esz != 0 || plan == nullptr || plan->per < 0) {
        set_error("%s: misaligned logits or no row plan", what);
        return BSI_ERR_INVALID;
    }
    return BSI_OK;
}

RowPlan plan_of(const bsi_row_plan* p) { return RowPlan{p->per, p->block_stride, p->row_stride}; }

// ---- distillation from a teacher's top logits ---------------------------------------------------------------------------------
//
// Per row, with q = softmax(z / T) and the teacher's entries (id_k, t_k):
//   tail off:  p = softmax over the listed entries of t / T;        loss = T^2 sum p_k (log p_k - log q_{id_k})
//   tail on:   p_k = exp(t_k), rest = max(0, 1 - sum p_k) stands for all that is not listed:  loss += T^2 rest (log rest - log q_rest)
//   dloss/dz_j = T (q_j - sum of the p_k with id_k = j)             listed, or tail off
//   dloss/dz_j = T q_j (1 - rest / q_rest)                          not listed, tail on
// Entries whose id lies outside the vocabulary are not there. The row's weight and the reduction's factor go on top.
//
// With the tail on, what is not listed is summed by itself (a bit per logit says which pieces hold a listed one; such a logit is
// read as -inf) and the listed ones are added at the end: the rest's mass is no difference of two sums near each other.
// What a backward pass needs of the forward one is four numbers a row: m, 1 / s, rest's factor, and nothing of the vocabulary's size.

struct DistillArgs {
    const void* logits;
    RowPlan rows;
    int64_t V;
    const int64_t* ids;          // [rows, K]
    const void* teacher;         // [rows, K]
    int teacher_dtype;
    int K;
    float temperature;
    int tail;
    const float* weights;        // [rows] or null
    float* row_loss;             // [rows], weight and T^2 included
    float4* saved;               // [rows]: m, 1 / s, factor of q_j outside the list, whether the row is on
    // gradient
    const float* upstream;       // null: 1
    int64_t upstream_stride;     // 0: one value for all rows
    const float* denominator;    // null: 1
    void* grad;
    int64_t grad_stride;
};

struct Entry {
    int id;          // -1: not there
    float p;
    float logp;
    float z;
};

struct DistillShared {
    Stats warp[kWarps];
    float part[kWarps];
    Stats rest, listed;          // of this CTA's part of the row, read by the other CTAs
    float total_p;
    Entry entry[kMaxListed];
};

__device__ __forceinline__ float teacher_value(const void* t, int dtype, int64_t i) {
    if (dtype == BSI_DTYPE_F32) return static_cast<const float*>(t)[i];
    if (dtype == BSI_DTYPE_F16) return __half2float(static_cast<const __half*>(t)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(t)[i]);
}

// The row's entries with their probabilities and logits, by warp 0 alone (a few values per lane); the caller synchronises.
template <typename T>
__device__ void read_entries(DistillShared& sh, const DistillArgs& a, int64_t r, const T* row) {
    const int lane = threadIdx.x & 31;
    const float inv_t = 1.0f / a.temperature;
    float top = -CUDART_INF_F;
    for (int k = lane; k < a.K; k += 32) {
        const int64_t id = a.ids[r * a.K + k];
        const bool there = id >= 0 && id < a.V;
        float t = there ? teacher_value(a.teacher, a.teacher_dtype, r * a.K + k) : -CUDART_INF_F;
        if (!a.tail) t *= inv_t;
        sh.entry[k].id = there ? static_cast<int>(id) : -1;
        sh.entry[k].logp = t;
        sh.entry[k].z = there ? Piece<T>::one(row[id]) : 0.0f;
        top = vocab::max_nan(top, t);
    }
    float norm = 0.0f;
    if (!a.tail) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = vocab::max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        float s = 0.0f;
        if (top != -CUDART_INF_F) {
            for (int k = lane; k < a.K; k += 32) s += expf(sh.entry[k].logp - top);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        norm = top == -CUDART_INF_F ? 0.0f : top + logf(s);
    }
    float sum = 0.0f;
    for (int k = lane; k < a.K; k += 32) {
        const float lp = sh.entry[k].logp - norm;
        const float p = expf(lp);
        sh.entry[k].logp = lp;
        sh.entry[k].p = p;
        sum += p;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) sh.total_p = sum;
}

// One value per thread summed over the block, the same on every call with the same values.
__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += part[w];
    return s;
}

// An entry's p over all entries of its id, and whether it is the first of them.
__device__ __forceinline__ bool first_of_id(const DistillShared& sh, int K, int k, float* p) {
    const int id = sh.entry[k].id;
    if (id < 0) return false;
    float sum = 0.0f;
    bool first = true;
    for (int j = 0; j < K; ++j) {
        if (sh.entry[j].id == id) {
            sum += sh.entry[j].p;
            first = first && j >= k;
        }
    }
    *p = sum;
    return first;
}

// The gradient of the pieces [first, last) of a row: factor * q_j everywhere, then the listed logits by themselves.
// cached: the pieces as they were read by this CTA, or null to read them again.
template <typename T>
__device__ void write_grad(DistillShared& sh, const DistillArgs& a, int64_t r, const Span<T>& span, const uint4* cached, float4 saved,
                           float scale) {
    constexpr int kVec = Piece<T>::kVec;
    T* out = static_cast<T*>(a.grad) + r * a.grad_stride;
    const float c = vocab::kLog2e / a.temperature;
    const float rest = scale * saved.z * saved.y, top = scale * saved.y;
    const bool vector = (reinterpret_cast<uintptr_t>(out) & 15u) / sizeof(T) == static_cast<unsigned>(span.shift);
    uint4* out_grid = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(out) & ~uintptr_t(15));
    const bool on = saved.w != 0.0f && scale != 0.0f;
    for (int64_t v0 = span.first + threadIdx.x; v0 < span.last; v0 += kBatch * kThreads) {
        uint4 u[kBatch];
        if (on) {
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int64_t v = v0 + b * kThreads;
                if (v < span.last && (cached != nullptr || span.whole(v))) u[b] = cached != nullptr ? cached[v - span.first] : span.grid[v];
            }
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int64_t v = v0 + b * kThreads;
            if (v >= span.last) break;
            float z[kVec], g[kVec];
            if (on) {
                if (cached != nullptr || span.whole(v)) Piece<T>::unpack(u[b], z);
                else span.load_edge(v, z);
#pragma unroll
                for (int e = 0; e < kVec; ++e) g[e] = rest * vocab::exp2_fast((z[e] - saved.x) * c);
            } else {
#pragma unroll
                for (int e = 0; e < kVec; ++e) g[e] = 0.0f;
            }
            if (vector && span.whole(v)) {
                out_grid[v] = Piece<T>::pack(g);
            } else {
                const int64_t e0 = span.element(v);
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if (e0 + e >= 0 && e0 + e < a.V) out[e0 + e] = Piece<T>::narrow(g[e]);
            }
        }
    }
    if (!on) return;
    __syncthreads();       // the pieces are written before the listed logits' own values
    const int64_t lo = span.begin(), hi = span.end();
    for (int k = threadIdx.x; k < a.K; k += kThreads) {
        const int id = sh.entry[k].id;
        if (id < lo || id >= hi) continue;
        float p;
        if (!first_of_id(sh, a.K, k, &p)) continue;
        out[id] = Piece<T>::narrow(top * vocab::exp2_fast((sh.entry[k].z - saved.x) * c) - scale * p);
    }
}

__device__ __forceinline__ float grad_scale(const DistillArgs& a, int64_t r) {
    const float w = a.weights != nullptr ? a.weights[r] : 1.0f;
    const float up = a.upstream != nullptr ? a.upstream[r * a.upstream_stride] : 1.0f;
    const float d = a.denominator != nullptr ? *a.denominator : 1.0f;
    if (w == 0.0f || d == 0.0f) return 0.0f;
    return up * a.temperature * (w / d);
}

// The forward pass; GRAD: the gradient too, from the row's pieces that the cluster keeps in shared memory.
// Dynamic shared memory: with the tail on, one bit per logit of the part; with GRAD, the part's pieces.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(kThreads) distill_kernel(const DistillArgs a, int bit_words) {
    constexpr int kVec = Piece<T>::kVec;
    constexpr int N = kBatch * kVec;
    extern __shared__ uint4 dyn[];
    __shared__ DistillShared sh;
    uint32_t* bits = reinterpret_cast<uint32_t*>(dyn);
    uint4* cache = dyn + bit_words / 4;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = static_cast<int>(cluster.num_blocks());
    const int part = static_cast<int>(cluster.block_rank());
    const int64_t r = blockIdx.x / parts;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* row = static_cast<const T*>(a.logits) + a.rows.at(r);
    const Span<T> span(row, a.V, part, parts);

    if (a.weights != nullptr && a.weights[r] == 0.0f) {      // every CTA of the cluster alike: a padded row is not read
        if (part == 0 && tid == 0) {
            a.row_loss[r] = 0.0f;
            if (a.saved != nullptr) a.saved[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        if (GRAD) write_grad<T>(sh, a, r, span, nullptr, make_float4(0.0f, 0.0f, 0.0f, 0.0f), 0.0f);
        return;
    }

    if (warp == 0) read_entries<T>(sh, a, r, row);
    if (a.tail) {
        for (int i = tid; i < bit_words; i += kThreads) bits[i] = 0u;
    }
    __syncthreads();
    const float c = vocab::kLog2e / a.temperature;
    const int64_t bit0 = span.first * kVec - span.shift;         // the part's bit 0; kVec bits for each piece
    if (a.tail) {
        for (int k = tid; k < a.K; k += kThreads) {
            const int64_t id = sh.entry[k].id;
            if (id >= span.begin() && id < span.end()) atomicOr(&bits[(id - bit0) >> 5], 1u << ((id - bit0) & 31));
        }
        __syncthreads();
    }

    Stats st{-CUDART_INF_F, 0.0f, 0.0f};
    for (int64_t v = span.first + tid; v < span.last; v += kBatch * kThreads) {
        float z[N];
        if (v >= span.lo && v + (kBatch - 1) * kThreads < min(span.hi, span.last)) {
            uint4 u[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) u[b] = span.grid[v + b * kThreads];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                Piece<T>::unpack(u[b], z + b * kVec);
                if (GRAD) cache[v + b * kThreads - span.first] = u[b];
            }
        } else {
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int64_t p = v + b * kThreads;
                if (p < span.last) {
                    span.load(p, z + b * kVec);
                    if (GRAD) cache[p - span.first] = Piece<T>::pack(z + b * kVec);
                } else {
#pragma unroll
                    for (int e = 0; e < kVec; ++e) z[b * kVec + e] = -CUDART_INF_F;
                }
            }
        }
        if (a.tail) {
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int64_t p = v + b * kThreads - span.first;
                if (p >= span.last - span.first) break;
                const uint32_t mask = (bits[p * kVec >> 5] >> ((p * kVec) & 31)) & ((1u << kVec) - 1u);
                if (mask != 0u) {
#pragma unroll
                    for (int e = 0; e < kVec; ++e)
                        if ((mask >> e) & 1u) z[b * kVec + e] = -CUDART_INF_F;
                }
            }
        }
        vocab::take<N, false>(st, z, c);
    }

    Stats listed{-CUDART_INF_F, 0.0f, 0.0f};
    if (a.tail) {
        for (int k = tid; k < a.K; k += kThreads) {
            const int64_t id = sh.entry[k].id;
            float p;
            if (id >= span.begin() && id < span.end() && first_of_id(sh, a.K, k, &p)) {
                const float z[1] = {sh.entry[k].z};
                vocab::take<1, false>(listed, z, c);
            }
        }
    }
    st = vocab::warp_merge(st, c);
    if (lane == 0) sh.warp[warp] = st;
    __syncthreads();
    if (warp == 0) {
        st = vocab::warp_merge(lane < kWarps ? sh.warp[lane] : Stats{-CUDART_INF_F, 0.0f, 0.0f}, c);
        if (lane == 0) sh.rest = st;
    }
    if (a.tail) {
        listed = vocab::warp_merge(listed, c);
        __syncthreads();
        if (lane == 0) sh.warp[warp] = listed;
        __syncthreads();
        if (warp == 0) {
            listed = vocab::warp_merge(lane < kWarps ? sh.warp[lane] : Stats{-CUDART_INF_F, 0.0f, 0.0f}, c);
            if (lane == 0) sh.listed = listed;
        }
    } else if (tid == 0) {
        sh.listed = Stats{-CUDART_INF_F, 0.0f, 0.0f};
    }
    cluster.sync();

    // every CTA joins the parts in the same order
    Stats rest = cluster.map_shared_rank(&sh, 0)->rest, all = cluster.map_shared_rank(&sh, 0)->listed;
    for (int p = 1; p < parts; ++p) {
        const DistillShared* other = cluster.map_shared_rank(&sh, p);
        rest = vocab::merge(rest, other->rest, c);
        all = vocab::merge(all, other->listed, c);
    }
    all = vocab::merge(rest, all, c);
    cluster.sync();      // nobody's shared memory is read after this

    // Rows of at most K logits may be listed whole: then there is no rest, whatever rounding leaves of the teacher's sum.
    bool outside = true;
    if (a.tail && a.K >= a.V && part == 0) {
        float distinct = 0.0f, p;
        for (int k = tid; k < a.K; k += kThreads) distinct += first_of_id(sh, a.K, k, &p) ? 1.0f : 0.0f;
        outside = block_sum(distinct, sh.part) < static_cast<float>(a.V);
    }
    const float log_s = logf(all.s);
    const float inv_t = 1.0f / a.temperature;
    const float p_rest = a.tail ? fmaxf(1.0f - sh.total_p, 0.0f) : 0.0f;
    // log of the rest's share, from its own maximum and sum; nothing there: the share is 0
    const float log_rest = rest.s != 0.0f ? (rest.m - all.m) * inv_t + logf(rest.s) - log_s : -CUDART_INF_F;
    float factor = 1.0f;
    if (a.tail && rest.s != 0.0f) factor = 1.0f - p_rest * expf(-log_rest);
    // a row without any entry has no loss and no gradient
    const bool on = a.tail || sh.total_p != 0.0f;
    const float4 saved = make_float4(all.m, 1.0f / all.s, factor, on ? 1.0f : 0.0f);
    if (part == 0) {
        float loss = 0.0f;
        for (int k = tid; k < a.K; k += kThreads) {
            const Entry e = sh.entry[k];
            if (e.id >= 0 && e.p != 0.0f) loss += e.p * (e.logp - ((e.z - all.m) * inv_t - log_s));
        }
        loss = block_sum(loss, sh.part);
        if (tid == 0) {
            if (p_rest != 0.0f && outside) loss += p_rest * (logf(p_rest) - log_rest);
            const float w = a.weights != nullptr ? a.weights[r] : 1.0f;
            a.row_loss[r] = loss * (a.temperature * a.temperature) * w;
            if (a.saved != nullptr) a.saved[r] = saved;
        }
    }
    if (GRAD) write_grad<T>(sh, a, r, span, cache, saved, grad_scale(a, r));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(const DistillArgs a, int parts) {
    __shared__ DistillShared sh;
    const int64_t r = blockIdx.x / parts;
    const T* row = static_cast<const T*>(a.logits) + a.rows.at(r);
    const Span<T> span(row, a.V, static_cast<int>(blockIdx.x % parts), parts);
    const float4 saved = a.saved[r];
    if (saved.w != 0.0f) {
        if (threadIdx.x < 32) read_entries<T>(sh, a, r, row);
        __syncthreads();
    }
    write_grad<T>(sh, a, r, span, nullptr, saved, grad_scale(a, r));
}

// totals[0] = the rows' losses summed (mean: over the weights' sum), totals[1] = the weights' sum. One block: a fixed order.
// row_loss may be null (only the weights are wanted), weights too (each row counts one).
constexpr int kTotalThreads = 1024;
__global__ void __launch_bounds__(kTotalThreads) distill_totals_kernel(const float* row_loss, const float* weights, int64_t rows, int mean,
                                                                       float* loss, float* weight_sum) {
    __shared__ double part[2][kTotalThreads / 32];
    double l = 0.0, w = 0.0;        // sums over any number of rows
    for (int64_t i = threadIdx.x; i < rows; i += kTotalThreads) {
        if (row_loss != nullptr) l += row_loss[i];
        w += weights != nullptr ? weights[i] : 1.0f;
    }
    for (int o = 16; o > 0; o >>= 1) {
        l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
        w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
    }
    if ((threadIdx.x & 31) == 0) {
        part[0][threadIdx.x >> 5] = l;
        part[1][threadIdx.x >> 5] = w;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        l = part[0][threadIdx.x];
        w = part[1][threadIdx.x];
        for (int o = 16; o > 0; o >>= 1) {
            l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
            w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
        }
        if (threadIdx.x == 0) {
            if (loss != nullptr) *loss = static_cast<float>(mean ? (w != 0.0 ? l / w : 0.0) : l);
            if (weight_sum != nullptr) *weight_sum = static_cast<float>(w);
        }
    }
}

// Shared memory of a part in distill_kernel; the bits first, whole 16-byte pieces.
template <typename T>
int part_bytes(int64_t V, int parts, bool tail, bool grad, int* bit_words) {
    const int64_t pieces = (V + 2 * Piece<T>::kVec - 2) / Piece<T>::kVec;      // whatever the row's offset
    const int64_t mine = (pieces + parts - 1) / parts + 1;
    *bit_words = tail ? static_cast<int>((mine * Piece<T>::kVec + 127) / 128 * 4) : 0;
    const int64_t bytes = *bit_words * 4ll + (grad ? mine * 16 : 0);
    return bytes > 0x7FFFFFFF ? 0x7FFFFFFF : static_cast<int>(bytes);
}

constexpr int kPartLimit = 200 * 1024;      // dynamic shared memory of a CTA, beside about 10 KB of static

template <typename T, bool GRAD>
int launch_distill(const DistillArgs& a, int64_t rows, cudaStream_t stream) {
    static bool attr_set[64] = {false};
    int dev = 0;
    BSI_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        BSI_CUDA_TRY(cudaFuncSetAttribute(distill_kernel<T, GRAD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPartLimit));
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    int parts = parts_for(rows, a.V, sizeof(T)), words = 0;
    while (parts < vocab::kMaxCluster && part_bytes<T>(a.V, parts, a.tail != 0, GRAD, &words) > kPartLimit) parts *= 2;
    const int bytes = part_bytes<T>(a.V, parts, a.tail != 0, GRAD, &words);
    if (bytes > kPartLimit) return fail(BSI_ERR_UNSUPPORTED, "distill: a row of this length does not fit the shared memory of a cluster");
    return launch_rows(distill_kernel<T, GRAD>, rows, parts, bytes, stream, "distill", a, words);
}

template <typename T>
int launch_distill_backward(const DistillArgs& a, int64_t rows, cudaStream_t stream) {
    const int parts = parts_for(rows, a.V, sizeof(T));
    distill_backward_kernel<T><<<static_cast<unsigned>(rows * parts), kThreads, 0, stream>>>(a, parts);
    return check_launch("distill_backward launch");
}

int check_distill(const char* what, const void* logits, int dtype, int64_t rows, int64_t V, const bsi_row_plan* plan, const int64_t* ids,
                  const void* teacher, int teacher_dtype, int K, float temperature) {
    const int rc = check_rows(what, logits, dtype, rows, V, plan);
    if (rc != BSI_OK) return rc;
    if (K < 1 || K > kMaxListed) {
        set_error("%s: %d teacher entries a row, 1 to %d are taken", what, K, kMaxListed);
        return BSI_ERR_INVALID;
    }
    if (rows > 0 && (ids == nullptr || teacher == nullptr)) {
        set_error("%s: null ids or teacher", what);
        return BSI_ERR_INVALID;
    }
    if (teacher_dtype != BSI_DTYPE_F32 && teacher_dtype != BSI_DTYPE_F16 && teacher_dtype != BSI_DTYPE_BF16) {
        set_error("%s: teacher dtype must be a BSI_DTYPE_* code, got %d", what, teacher_dtype);
        return BSI_ERR_INVALID;
    }
    if (!(temperature > 0.0f) || !(temperature <= 3.0e38f)) {
        set_error("%s: temperature must be positive and finite", what);
        return BSI_ERR_INVALID;
    }
    return BSI_OK;
}

}  // namespace
}  // namespace bsi

extern "C" int bsi_b200_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t V, const bsi_row_plan* plan,
                                       const int64_t* tokens, const bsi_row_plan* token_plan, int top,
                                       float* logprobs, int64_t* ranks, float* entropy, float* top_logprobs, int64_t* top_ids,
                                       bsi_stream_t stream) {
    using namespace bsi;
    int rc = check_rows("token_logprobs", logits, dtype, rows, V, plan);
    if (rc != BSI_OK) return rc;
    if (top < 0 || top > kMaxTop || top > V) {
        set_error("token_logprobs: top %d, at most %d and the %lld logits of a row", top, kMaxTop, static_cast<long long>(V));
        return BSI_ERR_INVALID;
    }
    if (tokens != nullptr && token_plan == nullptr) return fail(BSI_ERR_INVALID, "token_logprobs: tokens without a plan");
    if (rows == 0) return BSI_OK;
    if (top > 0 && (top_logprobs == nullptr || top_ids == nullptr)) return fail(BSI_ERR_INVALID, "token_logprobs: null output for the top alternatives");
    rc = require_sm100();
    if (rc != BSI_OK) return rc;
    ScoreArgs a{logits, plan_of(plan), V, tokens, tokens != nullptr ? plan_of(token_plan) : RowPlan{0, 0, 0}, top,
                logprobs, ranks, entropy, top_logprobs, top_ids};
    const int parts = parts_for(rows, V, dtype == BSI_DTYPE_F32 ? 4 : 2);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case BSI_DTYPE_F32: return launch_rows(score_kernel<float>, rows, parts, 0, s, "token_logprobs", a);
        case BSI_DTYPE_F16: return launch_rows(score_kernel<__half>, rows, parts, 0, s, "token_logprobs", a);
        default: return launch_rows(score_kernel<__nv_bfloat16>, rows, parts, 0, s, "token_logprobs", a);
    }
}

extern "C" int bsi_b200_distill_forward(const void* logits, int dtype, int64_t rows, int64_t V, const bsi_row_plan* plan,
                                        const int64_t* ids, const void* teacher, int teacher_dtype, int K, float temperature, int tail,
                                        const float* weights, int mean, float* row_loss, float* saved, float* loss, float* weight_sum,
                                        bsi_stream_t stream) {
    using namespace bsi;
    int rc = check_distill("distill_forward", logits, dtype, rows, V, plan, ids, teacher, teacher_dtype, K, temperature);
    if (rc != BSI_OK) return rc;
    if (rows > 0 && row_loss == nullptr) return fail(BSI_ERR_INVALID, "distill_forward: null row_loss");
    if (reinterpret_cast<uintptr_t>(saved) & 15u) return fail(BSI_ERR_INVALID, "distill_forward: saved must be 16-byte aligned");
    rc = require_sm100();
    if (rc != BSI_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    DistillArgs a{logits, plan_of(plan), V, ids, teacher, teacher_dtype, K, temperature, tail != 0, weights, row_loss,
                  reinterpret_cast<float4*>(saved), nullptr, 0, nullptr, nullptr, 0};
    if (rows > 0) {
        rc = dtype == BSI_DTYPE_F32 ? launch_distill<float, false>(a, rows, s)
             : dtype == BSI_DTYPE_F16 ? launch_distill<__half, false>(a, rows, s) : launch_distill<__nv_bfloat16, false>(a, rows, s);
        if (rc != BSI_OK) return rc;
    }
    if (loss == nullptr && weight_sum == nullptr) return BSI_OK;
    distill_totals_kernel<<<1, kTotalThreads, 0, s>>>(row_loss, weights, rows, mean, loss, weight_sum);
    return check_launch("distill totals launch");
}

extern "C" int bsi_b200_distill_backward(const void* logits, int dtype, int64_t rows, int64_t V, const bsi_row_plan* plan,
                                         const int64_t* ids, const void* teacher, int teacher_dtype, int K, float temperature, int tail,
                                         const float* weights, const float* saved, const float* upstream, int64_t upstream_stride,
                                         const float* denominator, void* grad, int64_t grad_stride, bsi_stream_t stream) {
    using namespace bsi;
    int rc = check_distill("distill_backward", logits, dtype, rows, V, plan, ids, teacher, teacher_dtype, K, temperature);
    if (rc != BSI_OK) return rc;
    if (rows == 0) return BSI_OK;
    if (saved == nullptr || grad == nullptr || grad_stride < V || (reinterpret_cast<uintptr_t>(saved) & 15u) ||
        reinterpret_cast<uintptr_t>(grad) % (dtype == BSI_DTYPE_F32 ? 4 : 2) != 0)
        return fail(BSI_ERR_INVALID, "distill_backward: null or misaligned saved or grad, or gradient rows shorter than the vocabulary");
    rc = require_sm100();
    if (rc != BSI_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    DistillArgs a{logits, plan_of(plan), V, ids, teacher, teacher_dtype, K, temperature, tail != 0, weights, nullptr,
                  const_cast<float4*>(reinterpret_cast<const float4*>(saved)), upstream, upstream_stride, denominator, grad, grad_stride};
    return dtype == BSI_DTYPE_F32 ? launch_distill_backward<float>(a, rows, s)
           : dtype == BSI_DTYPE_F16 ? launch_distill_backward<__half>(a, rows, s) : launch_distill_backward<__nv_bfloat16>(a, rows, s);
}

extern "C" int bsi_b200_distill_fused_fits(int dtype, int64_t V, int tail) {
    using namespace bsi;
    int words = 0;
    if (V < 1 || V > 0x7FFFFFFFll) return 0;
    const int bytes = dtype == BSI_DTYPE_F32 ? part_bytes<float>(V, vocab::kMaxCluster, tail != 0, true, &words)
                                             : part_bytes<__half>(V, vocab::kMaxCluster, tail != 0, true, &words);
    return bytes <= kPartLimit ? 1 : 0;
}

extern "C" int bsi_b200_distill_fused(const void* logits, int dtype, int64_t rows, int64_t V, const bsi_row_plan* plan,
                                      const int64_t* ids, const void* teacher, int teacher_dtype, int K, float temperature, int tail,
                                      const float* weights, int mean, float* row_loss, float* loss, float* weight_sum,
                                      void* grad, int64_t grad_stride, bsi_stream_t stream) {
    using namespace bsi;
    int rc = check_distill("distill_fused", logits, dtype, rows, V, plan, ids, teacher, teacher_dtype, K, temperature);
    if (rc != BSI_OK) return rc;
    if (loss == nullptr || weight_sum == nullptr || (rows > 0 && (row_loss == nullptr || grad == nullptr || grad_stride < V)) ||
        reinterpret_cast<uintptr_t>(grad) % (dtype == BSI_DTYPE_F32 ? 4 : 2) != 0)
        return fail(BSI_ERR_INVALID, "distill_fused: null output, or gradient rows shorter than the vocabulary");
    rc = require_sm100();
    if (rc != BSI_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (mean) {       // the gradient's rows need the weights' sum
        distill_totals_kernel<<<1, kTotalThreads, 0, s>>>(nullptr, weights, rows, 0, nullptr, weight_sum);
        rc = check_launch("distill weights launch");
        if (rc != BSI_OK) return rc;
    }
    DistillArgs a{logits, plan_of(plan), V, ids, teacher, teacher_dtype, K, temperature, tail != 0, weights, row_loss,
                  nullptr, nullptr, 0, mean ? weight_sum : nullptr, grad, grad_stride};
    if (rows > 0) {
        rc = dtype == BSI_DTYPE_F32 ? launch_distill<float, true>(a, rows, s)
             : dtype == BSI_DTYPE_F16 ? launch_distill<__half, true>(a, rows, s) : launch_distill<__nv_bfloat16, true>(a, rows, s);
        if (rc != BSI_OK) return rc;
    }
    distill_totals_kernel<<<1, kTotalThreads, 0, s>>>(row_loss, weights, rows, mean, loss, weight_sum);
    return check_launch("distill totals launch");
}
