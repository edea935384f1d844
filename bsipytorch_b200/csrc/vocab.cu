// Log probabilities of given tokens, and distillation from a teacher's top logits: kernels over rows of logits.
//
// Both need the softmax statistics of every row, so both are one pass over the logits with a running maximum and sum per thread
// (vocab.cuh), joined in a block and then in a cluster. What bounds them is the logits' bytes.
#include <algorithm>
#include <cmath>

#include "vocab.cuh"

namespace bsi {

__device__ int g_vocab_status = 0;

int take_vocab_status(int* v) {
    int s = 0;
    BSI_CUDA_TRY(cudaMemcpyFromSymbol(&s, g_vocab_status, sizeof(int)));
    if (s != 0) {
        const int zero = 0;
        BSI_CUDA_TRY(cudaMemcpyToSymbol(g_vocab_status, &zero, sizeof(int)));
    }
    *v = s;
    return BSI_OK;
}

namespace {

namespace cg = cooperative_groups;
__device__ __forceinline__ vocab::Factor natural() { return vocab::Factor{1.44269502162933349609375f, 1.92596299e-8f}; }      // log2(e)
using vocab::kBatch;
using vocab::kChunk;
using vocab::kThreads;
using vocab::kWarps;
using vocab::Piece;
using vocab::Ring;
using vocab::RowPlan;
using vocab::Span;
using vocab::Stats;

constexpr int kMaxTop = 128;            // alternatives of token_logprobs
constexpr int kCandidates = 1024;       // entries at least as large as the last bound that a block keeps
constexpr int kPerSm = 4;               // CTAs of 256 threads with 64 registers: a row's end takes as long as a third of 100 KB, and others fill it
constexpr int kStages = 2;              // chunks under way in each: 128 KB an SM
constexpr int kMaxListed = 512;         // teacher entries per row
static_assert(vocab::kMaxCluster * kMaxTop <= kCandidates, "CTA 0 gathers the others' lists where its candidates were");

// ---- log probabilities, ranks, entropy, top alternatives ---------------------------------------------------------------------
//
// For a row z and a token t:  logprob = z_t - lse,  lse = m + log sum exp(z - m),  entropy = lse - sum p z,
// rank = #{z_j > z_t} + #{j < t, z_j = z_t}, top = the k largest, equal values by ascending index.
//
// The top k ride on the same pass. Every warp knows the j-th largest of its lanes' running maxima, j = ceil(k / 8); with B the t-th
// largest of these over the 8 warps, t = ceil(k / j), at least k entries are >= B, so the k largest all are, and few others. It is
// worked out behind chunks 1, 2, 3, 4, 8, 16, ... without any barrier, as a bound of an earlier time is one too; a thread only notes which of
// its batches reached the bound of their time, a bit each. At the row's end the last bound is a tight one, and the few batches noted
// are read again, out of L2, for the entries that reach it, which are put in order by counting for each one how many come before it.
// (633 x 128011 float32, k = 64: keeping the entries themselves as the row goes by took 138 us, reading again all that a thread whose
// maximum reaches the last bound had read, 163.)
// Where more than kCandidates entries are kept (a row in ascending order, a constant one), the block selects by radix: four passes over
// 8 bits each give the k-th value, one pass the larger entries, one in index order the equal ones. -inf is kept only where a row has
// fewer than k other entries.

struct ScoreArgs {
    const void* logits;
    RowPlan rows;
    uint32_t count;      // rows
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
    int lengths[vocab::kMaxCluster];      // CTA 0: the others' `listed`
    int listed;          // entries in `best`: min(top, elements of this part)
    volatile uint32_t bound[kWarps];      // the warps' own
    uint32_t agreed_bound;                // the highest that has come of them
    uint64_t bars[2 * kStages];
    vocab::Feed feed;
    uint32_t hist[256];
    uint32_t prefix, need;
    unsigned long long best[kMaxTop];      // this CTA's largest, in order
    unsigned long long cand[kCandidates];

    // The t-th largest of the voting warps' bounds, by whole warps. Equal ones by their number, so that each has a rank of its own.
    __device__ __forceinline__ uint32_t agreed(int voters, int t) const {
        const int lane = threadIdx.x & 31;
        const uint32_t own = lane < voters ? bound[lane] * kWarps + static_cast<uint32_t>(lane) : 0u;
        int rank = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) rank += __shfl_sync(0xFFFFFFFFu, own, w) > own;
        const unsigned it = __ballot_sync(0xFFFFFFFFu, lane < voters && rank == t - 1);
        return it == 0u ? 0u : __shfl_sync(0xFFFFFFFFu, own, __ffs(it) - 1) / kWarps;
    }
};

__device__ __forceinline__ unsigned long long sort_key(float v, int64_t index) {
    return (static_cast<unsigned long long>(vocab::ordered(v)) << 32) | static_cast<uint32_t>(~static_cast<uint32_t>(index));
}

// The first `need` entries of [lo, hi), in index order, whose place in the order is `prefix`, into sh.cand[at ..). All threads.
template <typename T>
__device__ void take_equal(ScoreShared& sh, const T* row, int64_t lo, int64_t hi, uint32_t prefix, int at, int need) {
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
        if (eq && place < need) sh.cand[at + place] = sort_key(v, i);
        taken += all;
        __syncthreads();
    }
    __syncthreads();
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
    take_equal<T>(sh, row, lo, hi, prefix, k - need, need);
}

// The j-th largest of a warp's places, by halving: the largest place that at least j lanes reach (0: none is).
__device__ __forceinline__ uint32_t warp_bound(uint32_t place, int j) {
    if (j == 1) return __reduce_max_sync(0xFFFFFFFFu, place);
    uint32_t bound = 0;
#pragma unroll 4
    for (int bit = 15; bit >= 0; --bit) {
        const uint32_t tryit = bound | (1u << bit);
        if (__popc(__ballot_sync(0xFFFFFFFFu, place >= tryit)) >= j) bound = tryit;
    }
    return bound;
}

// The row's ends and the few pieces of a CTA's last round go one by one; the rest in batches.
template <typename T>
struct ScoreThread {
    vocab::Running<T, true> run;
    int ahead;
    uint32_t at, behind;       // thresholds in front of the token's piece and from it on, as words
    int token_piece;
    float bound;               // of the entries that are kept, and as a word
    uint32_t thr;

    __device__ __forceinline__ void set_bound(uint32_t place) {
        const T b = Piece<T>::smallest(max(place, Piece<T>::kFloor));
        bound = Piece<T>::one(b);
        thr = Piece<T>::word(b);
    }

    template <int B>
    __device__ __forceinline__ float take(const uint4 (&u)[B], int v) {
        const float top = run.take(u, natural());
        typename Piece<T>::Count count;
#pragma unroll
        for (int b = 0; b < B; ++b) count.add(u[b], v + b * kThreads < token_piece ? at : behind);
        ahead += count.total();
        return top;
    }
    // Keeps the entries that reach the bound; top: the largest of them all, from: where the pieces lie, kThreads pieces apart.
    template <int B>
    __device__ __forceinline__ void keep(ScoreShared& sh, const Span<T>& span, const uint4 (&u)[B], int v, float top, const T* from) {
        if (top < bound) return;
        uint32_t reached = 0;
#pragma unroll
        for (int b = 0; b < B; ++b) reached |= Piece<T>::reach(u[b], thr) << (b * Piece<T>::kVec);
        while (reached != 0u) {
            const int bit = __ffs(reached) - 1;
            reached &= reached - 1u;
            const int off = bit / Piece<T>::kVec * kThreads * Piece<T>::kVec + bit % Piece<T>::kVec, i = span.element(v) + off;
            if (i < 0 || i >= span.V) continue;
            const int place = atomicAdd(&sh.found, 1);
            if (place < kCandidates) sh.cand[place] = sort_key(Piece<T>::one(from[off]), i);
        }
    }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, kPerSm) score_kernel(const ScoreArgs a) {
    constexpr int kVec = Piece<T>::kVec;
    extern __shared__ uint4 dyn[];       // the ring
    __shared__ ScoreShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = static_cast<int>(cluster.num_blocks());
    const int part = static_cast<int>(cluster.block_rank());
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int V = static_cast<int>(a.V);
    const bool top = a.top > 0;
    const uint32_t step = gridDim.x / static_cast<unsigned>(parts);
    uint32_t r = blockIdx.x / static_cast<unsigned>(parts);
    Ring<T> ring(dyn, sh.bars, kStages, &sh.feed, a.logits, a.rows, V, part, parts, nullptr, r, step, a.count, &g_vocab_status);

    auto token_of = [&](uint32_t row) { return a.tokens == nullptr || row >= a.count ? int64_t(-1) : a.tokens[a.tokens_at.at(row)]; };
    int64_t wanted = token_of(r);
    T zt = Piece<T>::nan();
    if (wanted >= 0 && wanted < V) zt = (static_cast<const T*>(a.logits) + a.rows.at(r))[wanted];
    typename Ring<T>::Place place{0, 0};
    for (; r < a.count; r += step) {
    const T* row = static_cast<const T*>(a.logits) + a.rows.at(r);
    const Span<T> span(row, V, part, parts);
    const bool scored = wanted >= 0 && wanted < V;
    const int token = scored ? static_cast<int>(wanted) : -1;
    const int64_t wanted_next = token_of(r + step);
    // What is ahead of the token: values >= its own in pieces before its own, values >= the type's next larger one from there on,
    // and what equals it in front of it in its own piece, which is counted apart.
    ScoreThread<T> me;
    me.ahead = 0;
    me.token_piece = (token + span.shift) / kVec;
    me.at = me.behind = Piece<T>::word(Piece<T>::nan());
    if (scored) {
        me.at = Piece<T>::word(zt);
        me.behind = Piece<T>::word(Piece<T>::next_up(zt));
        if (tid < kVec && me.token_piece >= span.first && me.token_piece < span.last) {
            const int i = span.element(me.token_piece) + tid;
            if (i >= 0 && i < token) me.ahead += Piece<T>::one(row[i]) == Piece<T>::one(zt);
        }
    }

    const int mine = max(span.end() - span.begin(), 0);
    const int k = min(a.top, mine);
    const int pieces = span.whole_last() - span.whole_first();
    // warps whose lanes all have a piece from the start vote
    const int voters = max(1, min(kWarps, pieces / 32)), j = max(1, (k + voters - 1) / voters), t = (k + j - 1) / j;
    if (tid == 0) {
        sh.found = 0;
        sh.agreed_bound = 0;
    }
    if (tid < kWarps) sh.bound[tid] = 0;       // no warp has one for this row yet
    me.set_bound(0);
    __syncthreads();       // the ring's barriers, the count, and nobody is at the row before
    auto publish = [&]() {
        const uint32_t own = warp_bound(Piece<T>::place(me.run.m), j);
        if (lane == 0) sh.bound[warp] = own;
        __syncwarp();
        return sh.agreed(voters, t);
    };
    // bit: one batch, or as many as 64 bits have to share (rows of more than a megabyte a part)
    const int share = (pieces + 64 * kChunk - 1) / (64 * kChunk);
    unsigned long long noted = 0;
    // the batches with the four highest maxima of those noted: place << 16 | bit, descending; lost: the highest place that did not fit
    uint32_t best_batch[4] = {0u, 0u, 0u, 0u}, lost = 0;
    for (int i = 0, n = 0; i < pieces; i += kChunk, ++n) {
        const uint4* chunk = ring.arrive(place);
        const int v = span.whole_first() + i + tid;
        float largest = -CUDART_INF_F;
        if (i + kChunk <= pieces) {
            uint4 u[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) u[b] = chunk[tid + b * kThreads];
            largest = me.take(u, v);
        } else {
            // the part's last pieces
            for (int b = 0; i + b * kThreads + tid < pieces; ++b) {
                const uint4 u[1] = {chunk[tid + b * kThreads]};
                largest = vocab::max_nan(largest, me.take(u, v + b * kThreads));
            }
            __syncwarp();
        }
        ring.release(place);
        ring.advance(place);
        if (top) {
            if (n == 0 || !(largest < me.bound)) {
                const int bit = n / share;
                noted |= 1ull << bit;
                uint32_t in = Piece<T>::place(largest) << 16 | static_cast<uint32_t>(bit);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t low = min(best_batch[q], in);
                    best_batch[q] = max(best_batch[q], in);
                    in = low;
                }
                lost = max(lost, in >> 16);
            }
            if ((n & (n + 1)) == 0 || n == 2) {
                const uint32_t all = publish();
                if (lane == 0) atomicMax(&sh.agreed_bound, all);
            }
            me.set_bound(*static_cast<volatile uint32_t*>(&sh.agreed_bound));
        }
    }
    if (top) publish();
    T zt_next = Piece<T>::nan();
    if (wanted_next >= 0 && wanted_next < V) zt_next = (static_cast<const T*>(a.logits) + a.rows.at(r + step))[wanted_next];
    // the row's ends; -inf in the places that are not the row's, which a token at -inf would count on the left
    if ((tid == 0 && span.has_left()) || (tid == 32 && span.has_right())) {
        const int v = tid == 0 ? span.first : span.last - 1;
        const uint4 u[1] = {span.load_edge(v)};
        me.take(u, v);
        if (span.element(v) < 0 && v < me.token_piece && Piece<T>::one(zt) == -CUDART_INF_F) me.ahead += span.element(v);
    }

    // the block's statistics
    __syncwarp();
    Stats all = vocab::warp_merge(me.run.stats(natural()), natural());
    const int ahead = __reduce_add_sync(0xFFFFFFFFu, me.ahead);
    if (lane == 0) {
        sh.warp[warp] = all;
        sh.warp_ahead[warp] = ahead;
    }
    __syncthreads();
    if (warp == 0) {
        all = lane < kWarps ? sh.warp[lane] : Stats{-CUDART_INF_F, 0.0f, 0.0f};
        all = vocab::warp_merge(all, natural());
        const int n = __reduce_add_sync(0xFFFFFFFFu, lane < kWarps ? sh.warp_ahead[lane] : 0);
        if (lane == 0) {
            sh.mine = ring.gave_up() ? Stats{CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F} : all;
            sh.ahead = n;
        }
    }

    if (top) {
        const uint32_t last_bound = max(sh.agreed(voters, t), Piece<T>::kFloor);
        me.set_bound(last_bound);
        auto look_again = [&](int n) {
            const int v = span.whole_first() + n * kChunk + tid;
            if (v >= span.whole_last()) return;
            uint4 u[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                u[b] = v + b * kThreads < span.whole_last() ? span.grid[v + b * kThreads] : make_uint4(Piece<T>::kNone, Piece<T>::kNone, Piece<T>::kNone, Piece<T>::kNone);
            me.keep(sh, span, u, v, Piece<T>::top(u), row + span.element(v));
        };
        if (share == 1 && lost < last_bound) {
            // a thread has seldom more than one or two of them: each look takes memory's whole latency
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (best_batch[q] >> 16 >= last_bound) look_again(static_cast<int>(best_batch[q] & 63u));
        } else if (Piece<T>::place(me.run.m) >= last_bound) {
            while (noted != 0ull) {
                const int bit = __ffsll(static_cast<long long>(noted)) - 1;
                noted &= noted - 1ull;
                for (int n = bit * share; n < (bit + 1) * share; ++n) look_again(n);
            }
        }
        if ((tid == 0 && span.has_left()) || (tid == 32 && span.has_right())) {
            const int v = tid == 0 ? span.first : span.last - 1;
            const uint4 u[1] = {span.load_edge(v)};
            me.keep(sh, span, u, v, Piece<T>::top(u), row + span.element(v));
        }
        __syncthreads();
        int n = sh.found;
        if (n > kCandidates) {
            __syncthreads();      // everybody has read how many there were
            select_by_radix<T>(sh, row, span.begin(), span.end(), k);
            n = k;
        } else if (n < k) {
            // fewer entries than that are above -inf, and all of them are kept
            __syncthreads();
            take_equal<T>(sh, row, span.begin(), span.end(), vocab::ordered(-CUDART_INF_F), n, k - n);
            n = k;
        }
        for (int i = tid; i < n; i += kThreads) {
            const unsigned long long key = sh.cand[i];
            int place = 0;
#pragma unroll 8
            for (int q = 0; q < n; ++q) place += sh.cand[q] > key;
            if (place < k) sh.best[place] = key;
        }
        if (tid == 0) sh.listed = k;
    }
    if (parts > 1) cluster.sync();
    else __syncthreads();

    if (part == 0) {
        if (parts > 1) {
            // the others' statistics, a lane each, and lists, all at once
            if (warp == 0) {
                const ScoreShared* other = cluster.map_shared_rank(&sh, min(lane, parts - 1));
                const Stats total = vocab::warp_merge(lane < parts ? other->mine : Stats{-CUDART_INF_F, 0.0f, 0.0f}, natural());
                const int before = __reduce_add_sync(0xFFFFFFFFu, lane < parts ? other->ahead : 0);
                if (lane < parts) sh.lengths[lane] = other->listed;
                __syncwarp();
                if (lane == 0) {
                    sh.mine = total;
                    sh.ahead = before;
                }
            }
            for (int i = tid; i < parts * a.top; i += kThreads) sh.cand[i] = cluster.map_shared_rank(&sh, i / a.top)->best[i % a.top];
            __syncthreads();
        }
        const Stats total = sh.mine;
        const float log_s = logf(total.s);
        if (tid == 0) {
            if (a.logprobs != nullptr) a.logprobs[r] = scored ? (Piece<T>::one(zt) - total.m) - log_s : 0.0f;
            if (a.ranks != nullptr) a.ranks[r] = scored ? sh.ahead : -1;
            // entropy = lse - sum p z = log s - (sum e d) ln 2 / s with d = log2 e; a row of -inf has none
            if (a.entropy != nullptr) a.entropy[r] = total.m == -CUDART_INF_F ? CUDART_NAN_F : log_s - total.w * vocab::kLn2 / total.s;
        }
        // every CTA's list is in order: an entry's place is its own plus, in each other list, how many come before it
        for (int i = tid; i < parts * a.top; i += kThreads) {
            const int p = i / a.top, q = i % a.top;
            if (q >= (parts > 1 ? sh.lengths[p] : sh.listed)) continue;
            const unsigned long long key = parts > 1 ? sh.cand[i] : sh.best[q];
            int place = q;
            for (int o = 0; o < parts; ++o) {
                if (o == p) continue;
                int lo = 0, hi = sh.lengths[o];
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (sh.cand[o * a.top + mid] > key) lo = mid + 1;
                    else hi = mid;
                }
                place += lo;
            }
            if (place < a.top) {
                const float z = vocab::from_ordered(static_cast<uint32_t>(key >> 32));
                const int64_t at = static_cast<int64_t>(r) * a.top + place;
                a.top_logprobs[at] = (z - total.m) - log_s;
                a.top_ids[at] = static_cast<int64_t>(~static_cast<uint32_t>(key));
            }
        }
    }
    if (parts > 1) cluster.sync();      // CTA 0 reads the others' shared memory
    else __syncthreads();
    wanted = wanted_next;
    zt = zt_next;
    }
    ring.finish();
}

// CTAs per row and rows under way: as many CTAs as the GPU holds walk over the rows. A row by itself is read at 20 bytes per ns and CTA,
// so few rows are shared by clusters (one row of 128011 float32: 31.5 us alone, 8.8 by eight CTAs); but a cluster joins its parts at the
// row's end, and where rows follow one another that costs more than it gives (512 rows: 52 us alone, 57 by two, 124 by eight). Shared as
// long as every part has 8 KB and the parts are no more than two to an SM, or four with 96 KB each. Eight lists of many alternatives
// are joined more slowly than they are found (64 of one row: 14.5 us by four, 17.9 by eight; 20: 16.7 and 14.8).
struct Walk {
    int parts;
    int64_t clusters;
};
Walk walk_over(int64_t rows, int64_t V, int esz, int least_parts, int most_parts, int per_sm) {
    const int64_t sms = sm_count(), bytes = V * esz;
    int parts = least_parts;
    while (parts * 2 <= most_parts && bytes >= 8192 * parts * 2 &&
           (rows * parts * 2 <= 2 * sms || (rows * parts * 2 <= 4 * sms && bytes >= 98304 * parts * 2))) parts *= 2;
    return Walk{parts, std::min(rows, std::max<int64_t>(1, sms * per_sm / parts))};
}

template <typename Kernel, typename... Args>
int launch_rows(Kernel kernel, const Walk& walk, int64_t smem, cudaStream_t stream, const char* what, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(walk.parts);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(walk.clusters * walk.parts), 1, 1);
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

constexpr int kRingBytes = kStages * kChunk * 16;

template <typename Kernel>
int allow_shared(Kernel kernel, int bytes, bool (&set)[64]) {
    int dev = 0;
    BSI_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !set[dev]) {
        BSI_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (dev >= 0 && dev < 64) set[dev] = true;
    }
    return BSI_OK;
}

template <typename T>
int launch_score(const ScoreArgs& a, int64_t rows, cudaStream_t stream) {
    static bool set[64] = {false};
    if (int rc = allow_shared(score_kernel<T>, kRingBytes, set)) return rc;
    return launch_rows(score_kernel<T>, walk_over(rows, a.V, sizeof(T), 1, a.top > 32 ? 4 : vocab::kMaxCluster, kPerSm), kRingBytes, stream, "token_logprobs", a);
}

constexpr int64_t kMaxRows = 0x7FFFFFFFll / vocab::kMaxCluster;

// Pointers that a kernel reads or writes whole numbers or float32 values through, of `bytes` each.
template <typename... Pointers>
bool aligned(uintptr_t bytes, const Pointers*... p) {
    return (((reinterpret_cast<uintptr_t>(p) % bytes) | ...) == 0);
}

int check_rows(const char* what, const void* logits, int dtype, int64_t rows, int64_t V, const bsi_row_plan* plan) {
    if (dtype != BSI_DTYPE_F32 && dtype != BSI_DTYPE_F16 && dtype != BSI_DTYPE_BF16) {
        set_error("%s: dtype must be a BSI_DTYPE_* code, got %d", what, dtype);
        return BSI_ERR_INVALID;
    }
    if (rows < 0 || V < 1 || rows > kMaxRows || V > (1ll << 30)) {      // pieces' elements are counted in 32 bits
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

// Rows that are all in the first block need no division; what is left of `per` is below the number of rows, 31 bits (a multiple of 2^32 as
// 32 bits would be a division by 0, and the row it gave no row of the tensor's).
RowPlan plan_of(const bsi_row_plan* p, int64_t rows) {
    return p->per >= rows ? RowPlan{0, 0, p->row_stride} : RowPlan{p->per, p->block_stride, p->row_stride};
}

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
// read as -inf) and the listed ones are added at the end: the rest's mass is no difference of two sums near each other. With m_out and
// s_out its own statistics, q_j (1 - rest / q_rest) = exp((z_j - m_out) / T) (q_rest - rest) / s_out: this holds where q_rest is below
// what a number can be, as where everything outside the list is masked by the type's lowest value.
// What a backward pass needs of the forward one is four numbers a row: m, 1 / s, (q_rest - rest) / s_out, m_out, and nothing of the
// vocabulary's size. (Tail off: the third is 1 / s, the last m.)

struct DistillArgs {
    const void* logits;
    RowPlan rows;
    uint32_t count;              // rows
    int64_t V;
    const int64_t* ids;          // [rows, K]
    const void* teacher;         // [rows, K]
    int teacher_dtype;
    int K;
    vocab::Factor c;             // log2(e) / T
    double temperature, inv_t;
    int tail;
    const float* weights;        // [rows] or null
    float* row_loss;             // [rows], weight and T^2 included
    float4* saved;               // [rows]: see above; 1 / s as -1: the row has no loss
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

// A row's softmax: maximum, 1 / sum; factor and reference of the exponentials outside the list; log of the sum, log of what is not
// listed's share.
struct Joined {
    float m, inv_s, factor, ref, log_s, log_share;
};

struct DistillShared {
    Stats warp[kWarps];
    float part[kWarps];
    double listed_part[kWarps];
    vocab::Feed feed;
    Stats rest;                  // of this CTA's part of the row, read by the other CTAs
    Joined joined;
    float listed_top;                  // the largest of the logits that the entries name
    double rest_p;                     // what the entries' probabilities leave of 1
    float total_p;                     // their sum
    long long raw_id[kMaxListed];      // as they lie in memory
    float raw_t[kMaxListed];
    uint32_t raw_z[kMaxListed];
    Entry entry[kMaxListed];
};

__device__ __forceinline__ float teacher_value(const void* t, int dtype, int64_t i) {
    if (dtype == BSI_DTYPE_F32) return static_cast<const float*>(t)[i];
    if (dtype == BSI_DTYPE_F16) return __half2float(static_cast<const __half*>(t)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(t)[i]);
}

// The row's entries with their probabilities and logits, by one warp in three steps. Each step's values come from memory while something
// else goes on: ids and the teacher's values during the end of the row before, the logits that they name while the row streams.
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool eight) {
    const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
    if (eight) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_done() {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
}

__device__ __forceinline__ void ask_entries(DistillShared& sh, const DistillArgs& a, int64_t r) {
    for (int k = threadIdx.x & 31; k < a.K; k += 32) {
        copy_async(&sh.raw_id[k], a.ids + r * a.K + k, true);
        // 16-bit values are read when they are used: there is no copy of two bytes
        if (a.teacher_dtype == BSI_DTYPE_F32) copy_async(&sh.raw_t[k], static_cast<const float*>(a.teacher) + r * a.K + k, false);
    }
}
template <typename T>
__device__ __forceinline__ void ask_logits(DistillShared& sh, const DistillArgs& a, const T* row) {
    copies_done();
    for (int k = threadIdx.x & 31; k < a.K; k += 32) {
        const int64_t id = sh.raw_id[k];
        const bool there = id >= 0 && id < a.V;
        sh.entry[k].id = there ? static_cast<int>(id) : -1;
        // the 4 bytes that hold it
        if (there) copy_async(&sh.raw_z[k], reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(row + id) & ~uintptr_t(3)), false);
    }
}
// A handful of values a row, of whose differences the gradient is made: in double.
template <typename T>
__device__ void finish_entries(DistillShared& sh, const DistillArgs& a, int64_t r, const T* row) {
    const int lane = threadIdx.x & 31;
    copies_done();
    float top = -CUDART_INF_F, top_z = -CUDART_INF_F;
    for (int k = lane; k < a.K; k += 32) {
        const int id = sh.entry[k].id;
        float t = -CUDART_INF_F, z = -CUDART_INF_F;
        if (id >= 0) {
            t = a.teacher_dtype == BSI_DTYPE_F32 ? sh.raw_t[k] : teacher_value(a.teacher, a.teacher_dtype, r * a.K + k);
            const uint32_t word = sh.raw_z[k];
            if constexpr (sizeof(T) == 4) {
                z = __uint_as_float(word);
            } else {
                const unsigned short half = static_cast<unsigned short>((reinterpret_cast<uintptr_t>(row + id) & 2u) ? word >> 16 : word & 0xFFFFu);
                z = Piece<T>::one(*reinterpret_cast<const T*>(&half));
            }
        }
        sh.entry[k].logp = t;
        sh.entry[k].z = z;
        top = vocab::max_nan(top, t);
        top_z = vocab::max_nan(top_z, z);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        top = vocab::max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        top_z = vocab::max_nan(top_z, __shfl_xor_sync(0xFFFFFFFFu, top_z, o));
    }
    const double scale = a.tail ? 1.0 : a.inv_t;
    // log p = (t - top) / T - log sum exp((t - top) / T), or t as it is
    const double from = a.tail || top == -CUDART_INF_F ? 0.0 : static_cast<double>(top);
    double norm = 0.0;
    if (!a.tail && top != -CUDART_INF_F) {
        double s = 0.0;
        for (int k = lane; k < a.K; k += 32) s += exp((sh.entry[k].logp - from) * scale);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        norm = log(s);
    }
    double sum = 0.0;
    for (int k = lane; k < a.K; k += 32) {
        const double lp = (sh.entry[k].logp - from) * scale - norm, p = exp(lp);
        sh.entry[k].logp = static_cast<float>(lp);
        sh.entry[k].p = static_cast<float>(p);
        sum += p;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) {
        sh.listed_top = top_z;
        sh.total_p = static_cast<float>(sum);
        sh.rest_p = 1.0 - sum;
    }
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

// A warp's share of the listed logits' sum of exponentials against the largest of them, in double and by every CTA for the whole row:
// they hold most of the mass, and a gradient is the difference of a listed q and its p. (With ex2.approx single entries of
// 96 x 128011 float32 were off by 5e-4 of the gradient's rms.)
__device__ __noinline__ double listed_sum(const DistillShared& sh, int K, double inv_t) {
    double sum = 0.0;
    for (int k = threadIdx.x; k < K; k += kThreads) {
        const float z = sh.entry[k].z;
        float p;
        if (z != -CUDART_INF_F && first_of_id(sh, K, k, &p)) sum += exp((static_cast<double>(z) - sh.listed_top) * inv_t);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    return sum;
}

// The gradient of a part of a row: rest * exp((z_j - ref) / T) everywhere, then the listed logits by themselves.
template <typename T>
struct Gradient {
    static constexpr int kVec = Piece<T>::kVec;
    T* out;
    uint4* out_grid;
    vocab::Factor c;
    double inv_t;
    float m, ref, rest, inv_s, scale;
    bool vector, on;

    __device__ __forceinline__ Gradient(const DistillArgs& a, uint32_t r, const Span<T>& span, const float4& saved, float s)
        : out(static_cast<T*>(a.grad) + r * a.grad_stride), c(a.c), inv_t(a.inv_t), m(saved.x), ref(saved.w), rest(s * saved.z), inv_s(saved.y),
          scale(s), vector((reinterpret_cast<uintptr_t>(out) & 15u) / sizeof(T) == static_cast<unsigned>(span.shift)), on(!(saved.y < 0.0f) && s != 0.0f) {
        out_grid = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(out) & ~uintptr_t(15));
    }
    __device__ __forceinline__ void write(const Span<T>& span, const uint4& u, int v) const {
        float z[kVec];
        if (on) {
            Piece<T>::unpack(u, z);
            const vocab::Two less(-ref, -ref), cc(c.hi, c.hi), ll(c.lo, c.lo), rr(rest, rest);
#pragma unroll
            for (int e = 0; e < kVec; e += 2) {
                float d0, d1;
                const vocab::Two x = vocab::add2(vocab::Two(z[e], z[e + 1]), less);
                vocab::fma2(x, ll, vocab::mul2(x, cc)).split(d0, d1);
                vocab::mul2(vocab::Two(vocab::exp2_fast(d0), vocab::exp2_fast(d1)), rr).split(z[e], z[e + 1]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e) z[e] = 0.0f;
        }
        if (vector && span.whole(v)) {
            out_grid[v] = Piece<T>::pack(z);
        } else {
            const int e0 = span.element(v);
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (e0 + e >= 0 && e0 + e < span.V) out[e0 + e] = Piece<T>::narrow(z[e]);
        }
    }
    // From memory.
    __device__ __forceinline__ void write_part(const Span<T>& span) const {
        const int last = span.whole_last();
        int v = span.whole_first() + threadIdx.x;
        const uint4 none = make_uint4(0u, 0u, 0u, 0u);
        for (; v + (kBatch - 1) * kThreads < last; v += kChunk) {
            uint4 u[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) u[b] = on ? span.grid[v + b * kThreads] : none;
#pragma unroll
            for (int b = 0; b < kBatch; ++b) write(span, u[b], v + b * kThreads);
        }
        for (; v < last; v += kThreads) write(span, on ? span.grid[v] : none, v);
    }
    __device__ __forceinline__ void write_ends(const Span<T>& span) const {
        if ((threadIdx.x == 0 && span.has_left()) || (threadIdx.x == 32 && span.has_right())) {
            const int v = threadIdx.x == 0 ? span.first : span.last - 1;
            write(span, span.load_edge(v), v);
        }
    }
    // Behind a barrier of the block: the pieces are written, and the entries have been read.
    __device__ __forceinline__ void write_listed(const DistillShared& sh, const Span<T>& span, int K) const {
        const int lo = span.begin(), hi = span.end();
        for (int k = threadIdx.x; k < K; k += kThreads) {
            const int id = sh.entry[k].id;
            if (id < lo || id >= hi) continue;
            float p;
            if (!first_of_id(sh, K, k, &p)) continue;
            const double q = exp((static_cast<double>(sh.entry[k].z) - m) * inv_t);
            out[id] = Piece<T>::narrow(static_cast<float>(scale * (inv_s * q - p)));
        }
    }
};

__device__ __forceinline__ float grad_scale(const DistillArgs& a, int64_t r) {
    const float w = a.weights != nullptr ? a.weights[r] : 1.0f;
    const float up = a.upstream != nullptr ? a.upstream[r * a.upstream_stride] : 1.0f;
    const float d = a.denominator != nullptr ? *a.denominator : 1.0f;
    if (w == 0.0f || d == 0.0f) return 0.0f;
    return up * static_cast<float>(a.temperature) * (w / d);
}

// The forward pass; GRAD: the gradient too, while L2 still holds the row. Dynamic shared memory: with the tail on, one bit per logit of
// the part; the ring.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(kThreads, kPerSm) distill_kernel(const DistillArgs a, int bit_words, int stages) {
    constexpr int kVec = Piece<T>::kVec;
    extern __shared__ uint4 dyn[];
    __shared__ DistillShared sh;
    uint32_t* bits = reinterpret_cast<uint32_t*>(dyn);
    uint64_t* bars = reinterpret_cast<uint64_t*>(dyn + bit_words / 4);
    uint4* data = dyn + bit_words / 4 + stages;      // two barriers a stage
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = static_cast<int>(cluster.num_blocks());
    const int part = static_cast<int>(cluster.block_rank());
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int V = static_cast<int>(a.V);
    const uint32_t step = gridDim.x / static_cast<unsigned>(parts);
    uint32_t r = blockIdx.x / static_cast<unsigned>(parts);
    Ring<T> ring(data, bars, stages, &sh.feed, a.logits, a.rows, V, part, parts, a.weights, r, step, a.count, &g_vocab_status);
    typename Ring<T>::Place place{0, 0};
    auto next_read = [&](uint32_t q) {       // the first row from q on that is read
        while (q < a.count && a.weights != nullptr && a.weights[q] == 0.0f) q += step;
        return q;
    };
    if (warp == kWarps - 1) {
        const uint32_t q = next_read(r);
        if (q < a.count) ask_entries(sh, a, q);
    }
    for (; r < a.count; r += step) {
    const T* row = static_cast<const T*>(a.logits) + a.rows.at(r);
    const Span<T> span(row, V, part, parts);

    if (a.weights != nullptr && a.weights[r] == 0.0f) {      // every CTA of the cluster alike: a padded row is not read
        if (part == 0 && tid == 0) {
            a.row_loss[r] = 0.0f;
            if (a.saved != nullptr) a.saved[r] = make_float4(0.0f, -1.0f, 0.0f, 0.0f);
        }
        if (GRAD) {
            const Gradient<T> g(a, r, span, make_float4(0.0f, -1.0f, 0.0f, 0.0f), 0.0f);
            g.write_part(span);
            g.write_ends(span);
        }
        continue;
    }
    __syncthreads();      // nobody is at the row before

    // The last warp has the entries
    if (warp == kWarps - 1) ask_logits<T>(sh, a, row);
    const vocab::Factor c = a.c;
    const int bit0 = span.element(span.first);         // the part's bit 0; kVec bits for each piece
    const int lo = span.begin(), hi = span.end();
    if (a.tail) {
        for (int i = tid; i < bit_words; i += kThreads) bits[i] = 0u;
        __syncthreads();
        for (int k = tid; k < a.K; k += kThreads) {
            const int id = sh.entry[k].id;
            if (id >= lo && id < hi) atomicOr(&bits[(id - bit0) >> 5], 1u << ((id - bit0) & 31));
        }
        __syncthreads();
    }

    vocab::Running<T, false> run;
    // a piece as the statistics see it: listed logits out where they are summed apart
    auto seen = [&](uint4& u, int v) {
        if (a.tail) {
            const int p = (v - span.first) * kVec;
            const uint32_t mask = (bits[p >> 5] >> (p & 31)) & ((1u << kVec) - 1u);
            if (mask != 0u) {
                float z[kVec];
                Piece<T>::unpack(u, z);
#pragma unroll
                for (int e = 0; e < kVec; ++e)
                    if ((mask >> e) & 1u) z[e] = -CUDART_INF_F;
                u = Piece<T>::pack(z);
            }
        }
    };
    const int pieces = span.whole_last() - span.whole_first();
    for (int i = 0; i < pieces; i += kChunk) {
        const uint4* chunk = ring.arrive(place);
        const int v = span.whole_first() + i + tid;
        if (i + kChunk <= pieces) {
            uint4 u[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) u[b] = chunk[tid + b * kThreads];
            ring.release(place);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) seen(u[b], v + b * kThreads);
            run.take(u, c);
        } else {
            for (int b = 0; i + b * kThreads + tid < pieces; ++b) {
                uint4 u[1] = {chunk[tid + b * kThreads]};
                seen(u[0], v + b * kThreads);
                run.take(u, c);
            }
            ring.release(place);
        }
        ring.advance(place);
    }
    if ((tid == 0 && span.has_left()) || (tid == 32 && span.has_right())) {
        const int v = tid == 0 ? span.first : span.last - 1;
        uint4 u[1] = {span.load_edge(v)};
        seen(u[0], v);
        run.take(u, c);
    }
    __syncwarp();

    Stats st = vocab::warp_merge(run.stats(c), c);
    if (lane == 0) sh.warp[warp] = st;
    if (warp == kWarps - 1) {
        finish_entries<T>(sh, a, r, row);
        const uint32_t q = next_read(r + step);
        if (q < a.count) ask_entries(sh, a, q);
    }
    __syncthreads();
    if (a.tail) {
        const double in = listed_sum(sh, a.K, a.inv_t);
        if (lane == 0) sh.listed_part[warp] = in;
    }
    if (warp == 0) {
        st = vocab::warp_merge(lane < kWarps ? sh.warp[lane] : Stats{-CUDART_INF_F, 0.0f, 0.0f}, c);
        if (lane == 0) sh.rest = ring.gave_up() ? Stats{CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F} : st;
    }
    if (parts > 1) cluster.sync();
    else __syncthreads();

    // every CTA joins the parts in the same way, a lane for each
    if (parts > 1) {
        if (warp == 0) {
            const Stats none{-CUDART_INF_F, 0.0f, 0.0f};
            const DistillShared* other = cluster.map_shared_rank(&sh, min(lane, parts - 1));
            st = vocab::warp_merge(lane < parts ? other->rest : none, c);
        }
        cluster.sync();      // nobody's shared memory is read by another after this
        if (tid == 0) sh.rest = st;
        __syncthreads();
    }
    if (a.tail) {
        // What is listed and what is not, joined in double by one thread: the gradient of what is not listed goes with q_rest - rest,
        // which is small where the teacher's rest and the student's are alike.
        if (tid == 0) {
            const Stats rest = sh.rest;
            double in = 0.0;
            for (int w = 0; w < kWarps; ++w) in += sh.listed_part[w];
            const float m = vocab::max_nan(rest.m, sh.listed_top);
            const double r_s = rest.s != 0.0f ? rest.s * exp((static_cast<double>(rest.m) - m) * a.inv_t) : 0.0;
            const double l_s = in != 0.0 ? in * exp((static_cast<double>(sh.listed_top) - m) * a.inv_t) : 0.0;
            const double total = r_s + l_s, p = fmax(sh.rest_p, 0.0);
            sh.joined = Joined{m, static_cast<float>(1.0 / total), 0.0f, m, static_cast<float>(log(total)), -CUDART_INF_F};
            if (rest.s != 0.0f) {
                sh.joined.factor = static_cast<float>((r_s / total - p) / rest.s);
                sh.joined.ref = rest.m;
                sh.joined.log_share = static_cast<float>((static_cast<double>(rest.m) - m) * a.inv_t + log(rest.s / total));
            }
        }
        __syncthreads();
    }
    const Joined all = a.tail ? sh.joined : Joined{sh.rest.m, 1.0f / sh.rest.s, 1.0f / sh.rest.s, sh.rest.m, logf(sh.rest.s), 0.0f};

    // Rows of at most K logits may be listed whole: then there is no rest, whatever rounding leaves of the teacher's sum.
    bool outside = true;
    if (a.tail && a.K >= a.V && part == 0) {
        float distinct = 0.0f, p;
        for (int k = tid; k < a.K; k += kThreads) distinct += first_of_id(sh, a.K, k, &p) ? 1.0f : 0.0f;
        outside = block_sum(distinct, sh.part) < static_cast<float>(a.V);
    }
    const float p_rest = a.tail ? static_cast<float>(fmax(sh.rest_p, 0.0)) : 0.0f;
    // a row without any entry has no loss and no gradient
    const bool on = a.tail || sh.total_p != 0.0f;
    const float4 saved = make_float4(all.m, on ? all.inv_s : -1.0f, all.factor, all.ref);
    if (part == 0) {
        float loss = 0.0f;
        for (int k = tid; k < a.K; k += kThreads) {
            const Entry e = sh.entry[k];
            if (e.id >= 0 && e.p != 0.0f) loss += e.p * static_cast<float>(e.logp - ((static_cast<double>(e.z) - all.m) * a.inv_t - all.log_s));
        }
        loss = block_sum(loss, sh.part);
        if (tid == 0) {
            if (p_rest != 0.0f && outside) loss += p_rest * (logf(p_rest) - all.log_share);
            const float w = a.weights != nullptr ? a.weights[r] : 1.0f;
            a.row_loss[r] = static_cast<float>(static_cast<double>(loss) * (a.temperature * a.temperature) * w);      // T^2 alone may pass float32's range
            if (a.saved != nullptr) a.saved[r] = saved;
        }
    }
    if (GRAD) {
        // the row again, out of L2: what the resident CTAs are at is a third of it
        const Gradient<T> g(a, r, span, saved, grad_scale(a, r));
        g.write_part(span);
        g.write_ends(span);
        __syncthreads();
        if (g.on) g.write_listed(sh, span, a.K);
    }
    }
    ring.finish();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) distill_backward_kernel(const DistillArgs a, int parts) {
    __shared__ DistillShared sh;
    const uint32_t r = blockIdx.x / static_cast<unsigned>(parts);
    const T* row = static_cast<const T*>(a.logits) + a.rows.at(r);
    const Span<T> span(row, static_cast<int>(a.V), static_cast<int>(blockIdx.x % parts), parts);
    const float4 saved = a.saved[r];
    if (!(saved.y < 0.0f) && threadIdx.x >= kThreads - 32) {
        ask_entries(sh, a, r);
        ask_logits<T>(sh, a, row);
        finish_entries<T>(sh, a, r, row);
    }
    const Gradient<T> g(a, r, span, saved, grad_scale(a, r));
    g.write_part(span);
    g.write_ends(span);
    __syncthreads();
    if (g.on) g.write_listed(sh, span, a.K);
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

// Dynamic shared memory of a part in distill_kernel: bits (in the row's pieces, whatever its offset), two barriers a stage, the stages.
template <typename T>
int64_t part_bytes(int64_t V, int parts, bool tail, int* bit_words) {
    const int64_t mine = ((V + 2 * Piece<T>::kVec - 2) / Piece<T>::kVec + parts - 1) / parts + 1;
    *bit_words = tail ? static_cast<int>((mine * Piece<T>::kVec + 127) / 128 * 4) : 0;
    return *bit_words * 4ll + kStages * 16ll + kRingBytes;
}

constexpr int64_t kSmShared = 227 * 1024;
constexpr int kPartLimit = 200 * 1024;      // dynamic shared memory of a CTA, beside 17 KB of static

template <typename T, bool GRAD>
int launch_distill(const DistillArgs& a, int64_t rows, cudaStream_t stream) {
    static bool set[64] = {false};
    if (int rc = allow_shared(distill_kernel<T, GRAD>, kPartLimit, set)) return rc;
    // a vocabulary whose bits no part holds alone is shared by more
    int least = 1, words = 0;
    while (least < vocab::kMaxCluster && part_bytes<T>(a.V, least, a.tail != 0, &words) > kPartLimit) least *= 2;
    const int64_t largest = part_bytes<T>(a.V, least, a.tail != 0, &words);
    if (largest > kPartLimit) return fail(BSI_ERR_UNSUPPORTED, "distill: the bits of a vocabulary of this size do not fit a cluster's shared memory");
    const int per_sm = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kPerSm, kSmShared / (largest + static_cast<int64_t>(sizeof(DistillShared)) + 1024))));
    const Walk walk = walk_over(rows, a.V, sizeof(T), least, vocab::kMaxCluster, per_sm);
    const int64_t bytes = part_bytes<T>(a.V, walk.parts, a.tail != 0, &words);
    return launch_rows(distill_kernel<T, GRAD>, walk, bytes, stream, "distill", a, words, kStages);
}

// CTAs per row of the backward pass, which has nothing to join: at least two rounds of the GPU's slots, and chunks enough for each.
int pieces_apart(int64_t rows, int64_t V, int esz) {
    const int64_t chunks = (V * esz + kChunk * 16 - 1) / (kChunk * 16);
    int64_t parts = 1;
    while (parts < 64 && rows * parts < 8ll * sm_count() && chunks >= parts * 2) parts *= 2;
    return static_cast<int>(parts);
}

template <typename T>
int launch_distill_backward(const DistillArgs& a, int64_t rows, cudaStream_t stream) {
    const int parts = pieces_apart(rows, a.V, sizeof(T));
    distill_backward_kernel<T><<<static_cast<unsigned>(rows * parts), kThreads, 0, stream>>>(a, parts);
    return check_launch("distill_backward launch");
}

vocab::Factor factor_of(double temperature) {
    // the upper part rounded down and never the whole: -inf times the lower one is -inf, not NaN
    const double c = 1.4426950408889634074 / temperature;
    float hi = static_cast<float>(c);
    if (static_cast<double>(hi) >= c) hi = std::nextafter(hi, 0.0f);
    return vocab::Factor{hi, static_cast<float>(c - hi)};
}

int check_distill(const char* what, const void* logits, int dtype, int64_t rows, int64_t V, const bsi_row_plan* plan, const int64_t* ids,
                  const void* teacher, int teacher_dtype, int K, double temperature) {
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
    if (reinterpret_cast<uintptr_t>(ids) % 8 != 0 || reinterpret_cast<uintptr_t>(teacher) % (teacher_dtype == BSI_DTYPE_F32 ? 4 : 2) != 0) {
        set_error("%s: misaligned ids or teacher", what);
        return BSI_ERR_INVALID;
    }
    if (!(temperature >= 1.0e-30) || !(temperature <= 1.0e30)) {
        set_error("%s: temperature must lie in [1e-30, 1e30]", what);
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
    if (tokens != nullptr && (token_plan == nullptr || token_plan->per < 0)) return fail(BSI_ERR_INVALID, "token_logprobs: tokens without a plan");
    if (!aligned(8, tokens, ranks, top_ids) || !aligned(4, logprobs, entropy, top_logprobs)) return fail(BSI_ERR_INVALID, "token_logprobs: misaligned tokens or outputs");
    if (rows == 0) return BSI_OK;
    if (top > 0 && (top_logprobs == nullptr || top_ids == nullptr)) return fail(BSI_ERR_INVALID, "token_logprobs: null output for the top alternatives");
    rc = require_sm100();
    if (rc != BSI_OK) return rc;
    ScoreArgs a{logits, plan_of(plan, rows), static_cast<uint32_t>(rows), V, tokens, tokens != nullptr ? plan_of(token_plan, rows) : RowPlan{0, 0, 0}, top,
                logprobs, ranks, entropy, top_logprobs, top_ids};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case BSI_DTYPE_F32: return launch_score<float>(a, rows, s);
        case BSI_DTYPE_F16: return launch_score<__half>(a, rows, s);
        default: return launch_score<__nv_bfloat16>(a, rows, s);
    }
}

extern "C" int bsi_b200_distill_forward(const void* logits, int dtype, int64_t rows, int64_t V, const bsi_row_plan* plan,
                                        const int64_t* ids, const void* teacher, int teacher_dtype, int K, double temperature, int tail,
                                        const float* weights, int mean, float* row_loss, float* saved, float* loss, float* weight_sum,
                                        bsi_stream_t stream) {
    using namespace bsi;
    int rc = check_distill("distill_forward", logits, dtype, rows, V, plan, ids, teacher, teacher_dtype, K, temperature);
    if (rc != BSI_OK) return rc;
    if (rows > 0 && row_loss == nullptr) return fail(BSI_ERR_INVALID, "distill_forward: null row_loss");
    if (reinterpret_cast<uintptr_t>(saved) & 15u) return fail(BSI_ERR_INVALID, "distill_forward: saved must be 16-byte aligned");
    if (!aligned(4, weights, row_loss, loss, weight_sum)) return fail(BSI_ERR_INVALID, "distill_forward: misaligned weights or outputs");
    rc = require_sm100();
    if (rc != BSI_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    DistillArgs a{logits, plan_of(plan, rows), static_cast<uint32_t>(rows), V, ids, teacher, teacher_dtype, K, factor_of(temperature), temperature, 1.0 / temperature, tail != 0, weights, row_loss,
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
                                         const int64_t* ids, const void* teacher, int teacher_dtype, int K, double temperature, int tail,
                                         const float* weights, const float* saved, const float* upstream, int64_t upstream_stride,
                                         const float* denominator, void* grad, int64_t grad_stride, bsi_stream_t stream) {
    using namespace bsi;
    int rc = check_distill("distill_backward", logits, dtype, rows, V, plan, ids, teacher, teacher_dtype, K, temperature);
    if (rc != BSI_OK) return rc;
    if (!aligned(4, weights, upstream, denominator)) return fail(BSI_ERR_INVALID, "distill_backward: misaligned weights, upstream or denominator");
    if (rows == 0) return BSI_OK;
    if (saved == nullptr || grad == nullptr || grad_stride < V || (reinterpret_cast<uintptr_t>(saved) & 15u) ||
        reinterpret_cast<uintptr_t>(grad) % (dtype == BSI_DTYPE_F32 ? 4 : 2) != 0)
        return fail(BSI_ERR_INVALID, "distill_backward: null or misaligned saved or grad, or gradient rows shorter than the vocabulary");
    rc = require_sm100();
    if (rc != BSI_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    DistillArgs a{logits, plan_of(plan, rows), static_cast<uint32_t>(rows), V, ids, teacher, teacher_dtype, K, factor_of(temperature), temperature, 1.0 / temperature, tail != 0, weights, nullptr,
                  const_cast<float4*>(reinterpret_cast<const float4*>(saved)), upstream, upstream_stride, denominator, grad, grad_stride};
    return dtype == BSI_DTYPE_F32 ? launch_distill_backward<float>(a, rows, s)
           : dtype == BSI_DTYPE_F16 ? launch_distill_backward<__half>(a, rows, s) : launch_distill_backward<__nv_bfloat16>(a, rows, s);
}

extern "C" int bsi_b200_distill_fused(const void* logits, int dtype, int64_t rows, int64_t V, const bsi_row_plan* plan,
                                      const int64_t* ids, const void* teacher, int teacher_dtype, int K, double temperature, int tail,
                                      const float* weights, int mean, float* row_loss, float* loss, float* weight_sum,
                                      void* grad, int64_t grad_stride, bsi_stream_t stream) {
    using namespace bsi;
    int rc = check_distill("distill_fused", logits, dtype, rows, V, plan, ids, teacher, teacher_dtype, K, temperature);
    if (rc != BSI_OK) return rc;
    if (loss == nullptr || weight_sum == nullptr || (rows > 0 && (row_loss == nullptr || grad == nullptr || grad_stride < V)) ||
        reinterpret_cast<uintptr_t>(grad) % (dtype == BSI_DTYPE_F32 ? 4 : 2) != 0)
        return fail(BSI_ERR_INVALID, "distill_fused: null output, or gradient rows shorter than the vocabulary");
    if (!aligned(4, weights, row_loss, loss, weight_sum)) return fail(BSI_ERR_INVALID, "distill_fused: misaligned weights or outputs");
    rc = require_sm100();
    if (rc != BSI_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (mean) {       // the gradient's rows need the weights' sum
        distill_totals_kernel<<<1, kTotalThreads, 0, s>>>(nullptr, weights, rows, 0, nullptr, weight_sum);
        rc = check_launch("distill weights launch");
        if (rc != BSI_OK) return rc;
    }
    DistillArgs a{logits, plan_of(plan, rows), static_cast<uint32_t>(rows), V, ids, teacher, teacher_dtype, K, factor_of(temperature), temperature, 1.0 / temperature, tail != 0, weights, row_loss,
                  nullptr, nullptr, 0, mean ? weight_sum : nullptr, grad, grad_stride};
    if (rows > 0) {
        rc = dtype == BSI_DTYPE_F32 ? launch_distill<float, true>(a, rows, s)
             : dtype == BSI_DTYPE_F16 ? launch_distill<__half, true>(a, rows, s) : launch_distill<__nv_bfloat16, true>(a, rows, s);
        if (rc != BSI_OK) return rc;
    }
    distill_totals_kernel<<<1, kTotalThreads, 0, s>>>(row_loss, weights, rows, mean, loss, weight_sum);
    return check_launch("distill totals launch");
}
