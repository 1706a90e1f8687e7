// Eviction from the paged cache by accumulated attention weight.
//
// For every sequence and KV head, of its len tokens the last `recent` stay and, of the others, those of the largest scores, keep in all (a tie goes
// to the lower position, a NaN counts as -inf).  The tokens that stay keep their order: with kept[0] < kept[1] < ... the row of
// token kept[j] moves to position j, in other pages or in the sequence's own.  Attention over the cache does not care that another head
// has another token at that position: a key carries its position with it.
//
//   select   A cluster of blocks for each (sequence, head) finds the score of rank k = keep - recent by its bits, eight at a time from the top:
//            a histogram of the digit among the tokens that agree with the digits found so far, summed over the cluster through distributed shared
//            memory, then the digit at which the count from above reaches k.  A score becomes an unsigned word that sorts as the float does.
//            Then every warp counts what it keeps of its own run of tokens, the counts are summed over the warps and blocks in front, and
//            the warp writes its tokens at consecutive places.  No order of atomics reaches the result.
//   move     A block for each page of the destination: all its slots of K and V, 16 bytes a thread and step, so that the stores cover
//            whole lines; the loads are gathered slots.
//
// What bounds it: the scores are read once (4 bytes a token and head), the kept slots are read and written (160 bytes each way for a
// head of 128).
#include "tq_common.cuh"

namespace tq {

constexpr int kEvictThreads = 512, kEvictWarps = kEvictThreads / 32;
constexpr int kEvictRun = 128;                 // tokens a warp takes at once: four a lane
constexpr int kEvictDigits = 256;
constexpr int kEvictMaxCluster = 16;
// The histogram has a column for every lane, so that 32 scores of one exponent (sums of softmax weights mostly share two or three) are 32 banks and
// not one counter.
constexpr int kEvictHistBytes = kEvictDigits * 32 * 4;
constexpr int kEvictMostKeys = 48 * 1024;      // sort keys a block keeps in shared memory; a longer share is read again from L2 in every pass

struct EvictParams {
    uint8_t* kv_cache;
    const int32_t* table;
    const int32_t* out_table;      // null: the pages of `table`
    const int32_t* seq_lens;
    const float* scores;
    float* score_to;               // where kept scores are written: out_scores, or the staging copy
    float* out_scores;
    int32_t* kept;
    int32_t* new_lens;
    uint8_t* staging;              // rows on their way within the same pages: [page of the output][2][16][kv heads][slot]
    int64_t num_blocks, half_bytes, slab_bytes;
    int64_t score_b, score_h, to_b, to_h, out_b, out_h;
    int batch, kv_heads, slot_bytes, max_pages, out_max_pages, out_pages, max_tokens, keep, recent, cluster, key_room, wide;
    int scores_staged;
};

static __device__ int32_t g_evict_faults = 0;

// Lengths as all kernels here see them: a sequence longer than its pages or its scores, or of a negative length, has nothing that stays.
__device__ __forceinline__ int evict_len(const EvictParams& p, int b, bool& bad) {
    const int len = p.seq_lens[b];
    bad = len < 0 || len > p.max_tokens;
    return bad ? 0 : len;
}

// Sorts as the score does; -0 is +0, a NaN is -inf.
__device__ __forceinline__ uint32_t evict_key(float v) {
    if (v != v) v = -INFINITY;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ int cluster_load(const int* local, uint32_t rank) {
    uint32_t at;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

__global__ void __launch_bounds__(kEvictThreads, 1) evict_select_kernel(const __grid_constant__ EvictParams p) {
    extern __shared__ __align__(16) uint32_t evict_smem[];
    uint32_t* const hist = evict_smem;                            // [digit][lane]
    uint32_t* const keys = evict_smem + kEvictDigits * 32;        // the block's share
    __shared__ int sums[2][kEvictDigits], counts[2], warp_gt[kEvictWarps], warp_eq[kEvictWarps], found[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int C = p.cluster, rank = C > 1 ? (int)cluster_rank() : 0;
    const int unit = blockIdx.x / C, b = unit / p.kv_heads, h = unit - b * p.kv_heads;
    grid_launch_dependents();
    for (int i = tid; i < kEvictDigits * 32; i += kEvictThreads) hist[i] = 0;
    grid_dependency_wait();

    bool bad;
    const int len = evict_len(p, b, bad);
    const int n = min(len, p.keep), recent = min(p.recent, n), M = len - recent, k = n - recent;
    if (h == 0 && rank == 0 && tid == 0) {
        p.new_lens[b] = n;
        if (bad) atomicAdd(&g_evict_faults, 1);
    }
    const float* const row = p.scores + b * p.score_b + h * p.score_h;
    float* const to = p.score_to + b * p.to_b + h * p.to_h;
    int32_t* const kept = p.kept + (int64_t)unit * p.keep;
    const int me = rank * kEvictThreads + tid, all = C * kEvictThreads;
    for (int j = me; j < recent; j += all) {
        kept[k + j] = M + j;
        to[k + j] = row[M + j];
    }
    for (int j = n + me; j < p.keep; j += all) kept[j] = -1;
    if (k == M) {                      // all of them (uniform over the cluster, as the ways out below are)
        for (int j = me; j < k; j += all) {
            kept[j] = j;
            to[j] = row[j];
        }
        return;
    }
    if (k == 0) return;

    // This warp's run of tokens, and the block's.
    const int W = ((M + kEvictWarps * C - 1) / (kEvictWarps * C) + kEvictRun - 1) / kEvictRun * kEvictRun;
    const int64_t first = (int64_t)rank * kEvictWarps * W;
    const int64_t begin64 = first + (int64_t)warp * W;
    const int begin = begin64 < M ? (int)begin64 : M, end = begin64 + W < M ? (int)(begin64 + W) : M;
    const bool resident = kEvictWarps * W <= p.key_room;
    uint32_t* const my_keys = keys + (size_t)warp * W;
    auto load = [&](int at, uint32_t (&key)[4]) {                // tokens at + 4 lane ...; past the run: nothing
        const int i = at + 4 * lane;
        if (p.wide && i + 3 < end) {
            const float4 v = *reinterpret_cast<const float4*>(row + i);
            key[0] = evict_key(v.x); key[1] = evict_key(v.y); key[2] = evict_key(v.z); key[3] = evict_key(v.w);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) key[e] = i + e < end ? evict_key(row[i + e]) : 0u;
        }
    };
    auto again = [&](int at, uint32_t (&key)[4]) {
        if (resident) {
            const uint4 v = *reinterpret_cast<const uint4*>(my_keys + (at - begin) + 4 * lane);
            key[0] = v.x; key[1] = v.y; key[2] = v.z; key[3] = v.w;
        } else {
            load(at, key);
        }
    };

    uint32_t prefix = 0;
    int left = k;                      // the rank looked for among the tokens that agree with the prefix
    __syncthreads();                   // the histogram is zero
    for (int pass = 0; pass < 4; pass++) {
        const int shift = 24 - 8 * pass;
        for (int at = begin; at < end; at += kEvictRun) {
            uint32_t key[4];
            if (pass == 0) {
                load(at, key);
                if (resident) *reinterpret_cast<uint4*>(my_keys + (at - begin) + 4 * lane) = make_uint4(key[0], key[1], key[2], key[3]);
            } else {
                again(at, key);
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (at + 4 * lane + e < end && (pass == 0 || key[e] >> (shift + 8) == prefix)) atomicAdd(&hist[((key[e] >> shift) & 255u) * 32 + lane], 1u);
        }
        __syncthreads();
        {   // two threads a digit, 16 columns each
            const int digit = tid >> 1;
            uint32_t sum = 0;
#pragma unroll
            for (int c = 0; c < 16; c++) {
                const int at = digit * 32 + 16 * (tid & 1) + ((c + digit) & 15);
                sum += hist[at];
                hist[at] = 0;
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            if ((tid & 1) == 0) sums[pass & 1][digit] = (int)sum;
        }
        if (C > 1) cluster_sync();
        else __syncthreads();
        if (warp == 0) {               // lane l: digits 255 - 8 l downwards
            int c[8], mine = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                c[e] = 0;
                for (int r = 0; r < C; r++) c[e] += C > 1 ? cluster_load(&sums[pass & 1][255 - 8 * lane - e], (uint32_t)r) : sums[pass & 1][255 - 8 * lane - e];
                mine += c[e];
            }
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += t;
            }
            int above = upto - mine;
            if (above < left && upto >= left) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (above < left && above + c[e] >= left) {
                        found[0] = 255 - 8 * lane - e;
                        found[1] = left - above;
                        break;
                    }
                    above += c[e];
                }
            }
        }
        __syncthreads();
        prefix = prefix << 8 | (uint32_t)found[0];
        left = found[1];
        __syncthreads();               // found is read before the next pass writes it
    }
    // prefix is now the key of rank k, and `left` of the tokens that have it stay: those of the lowest positions.

    int gt = 0, eq = 0;
    for (int at = begin; at < end; at += kEvictRun) {
        uint32_t key[4];
        again(at, key);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool in = at + 4 * lane + e < end;
            gt += in && key[e] > prefix;
            eq += in && key[e] == prefix;
        }
    }
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) {
        warp_gt[warp] = gt;
        warp_eq[warp] = eq;
    }
    __syncthreads();
    if (warp == 0) {                   // sums of the warps in front, and the block's
        int g = lane < kEvictWarps ? warp_gt[lane] : 0, q = lane < kEvictWarps ? warp_eq[lane] : 0;
        const int g0 = g, q0 = q;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, g, o), c = __shfl_up_sync(0xffffffffu, q, o);
            if (lane >= o) {
                g += a;
                q += c;
            }
        }
        if (lane < kEvictWarps) {
            warp_gt[lane] = g - g0;
            warp_eq[lane] = q - q0;
        }
        if (lane == 31) {
            counts[0] = g;
            counts[1] = q;
        }
    }
    if (C > 1) cluster_sync();
    else __syncthreads();
    int before_gt = warp_gt[warp], before_eq = warp_eq[warp];
    for (int r = 0; r < rank; r++) {
        before_gt += cluster_load(&counts[0], (uint32_t)r);
        before_eq += cluster_load(&counts[1], (uint32_t)r);
    }
    if (C > 1) cluster_sync();         // no block of the cluster leaves while another reads its counts
    int ties = left - before_eq;       // of this warp's tokens with the key of rank k, the first `ties` stay
    int place = before_gt + min(before_eq, left);
    const uint32_t lower = (1u << lane) - 1u;
    for (int at = begin; at < end; at += kEvictRun) {
        uint32_t key[4];
        again(at, key);
        bool is_eq[4], stays[4];
        int eq_before = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool in = at + 4 * lane + e < end;
            stays[e] = in && key[e] > prefix;
            is_eq[e] = in && key[e] == prefix;
        }
        if (__any_sync(0xffffffffu, is_eq[0] | is_eq[1] | is_eq[2] | is_eq[3])) {
            int total = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t m = __ballot_sync(0xffffffffu, is_eq[e]);
                eq_before += __popc(m & lower);
                total += __popc(m);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (is_eq[e]) stays[e] = eq_before < ties;
                eq_before += is_eq[e];
            }
            ties -= total;
        }
        int j = place;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t m = __ballot_sync(0xffffffffu, stays[e]);
            j += __popc(m & lower);
            place += __popc(m);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (stays[e]) {
                kept[j] = at + 4 * lane + e;
                to[j] = row[at + 4 * lane + e];
                j++;
            }
        }
    }
}

// One block for each page of the output.  STAGE 0: from the cache to the cache, 1: from the cache to the staging copy, 2: from there to the cache.
// T: the piece of a slot that a thread moves at once.
constexpr int kMoveThreads = 256, kMoveMaxRows = 1024;      // rows (slots of one half) whose sources a block notes at once
template <int STAGE, typename T>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p) {
    __shared__ int64_t source[kMoveMaxRows];      // byte of the row in the cache's K half, -1: nothing to move
    grid_launch_dependents();
    grid_dependency_wait();
    const int b = blockIdx.x / p.out_pages, page = blockIdx.x - b * p.out_pages;
    bool bad;
    const int n = min(evict_len(p, b, bad), p.keep), tokens = min(16, n - 16 * page);
    if (tokens <= 0) return;
    if (STAGE != 1 && p.scores_staged) {          // the kept scores of this page's positions back to where they came from
        for (int i = threadIdx.x; i < p.kv_heads * 16; i += kMoveThreads) {
            const int h = i >> 4, j = 16 * page + (i & 15);
            if ((i & 15) < tokens) p.out_scores[b * p.out_b + h * p.out_h + j] = p.score_to[b * p.to_b + h * p.to_h + j];
        }
    }
    const int32_t* const in = p.table + (int64_t)b * p.max_pages;
    int64_t to_page = 0;
    if (STAGE != 1) {
        to_page = p.out_table ? p.out_table[(int64_t)b * p.out_max_pages + page] : in[page];
        if ((uint64_t)to_page >= (uint64_t)p.num_blocks) {
            if (threadIdx.x == 0) atomicAdd(&g_evict_faults, 1);
            return;
        }
    }
    uint8_t* const stage = p.staging + (int64_t)blockIdx.x * 2 * p.half_bytes;
    const int pieces = p.slot_bytes / (int)sizeof(T), H = p.kv_heads, rows = tokens * H;
    for (int r0 = 0; r0 < rows; r0 += kMoveMaxRows) {
        const int some = min(kMoveMaxRows, rows - r0);
        __syncthreads();
        for (int i = threadIdx.x; i < some; i += kMoveThreads) {
            const int s = (r0 + i) / H, h = r0 + i - s * H, j = 16 * page + s;
            const int t = p.kept[((int64_t)b * H + h) * p.keep + j];
            int64_t at = -1;
            if (STAGE == 0 || t != j) {           // within the same pages a row that stays in its place is left alone
                if (STAGE == 2) {
                    at = 0;
                } else {
                    const int64_t from = in[t >> 4];
                    if ((uint64_t)from < (uint64_t)p.num_blocks) at = from * p.half_bytes + ((int64_t)(t & 15) * H + h) * p.slot_bytes;
                    else atomicAdd(&g_evict_faults, 1);
                }
            }
            source[i] = at;
        }
        __syncthreads();
        const int work = some * pieces;           // of one half
        for (int i = threadIdx.x; i < 2 * work; i += kMoveThreads) {
            const int half = i >= work, rest = i - half * work, r = rest / pieces, piece = rest - r * pieces;
            if (source[r] < 0) continue;
            const int64_t place = (int64_t)(r0 + r) * p.slot_bytes + piece * (int)sizeof(T);      // within a page half
            const T* from = reinterpret_cast<const T*>(STAGE == 2 ? stage + half * p.half_bytes + place
                                                                  : p.kv_cache + half * p.slab_bytes + source[r] + piece * (int)sizeof(T));
            T* to = reinterpret_cast<T*>(STAGE == 1 ? stage + half * p.half_bytes + place
                                                    : p.kv_cache + half * p.slab_bytes + to_page * p.half_bytes + place);
            *to = *from;
        }
    }
}

int device_sm_count(int* out);

int evict_fault_count(int32_t* out) {
    TQ_CUDA(cudaMemcpyFromSymbol(out, g_evict_faults, sizeof(int32_t)));
    return TQ_OK;
}

static size_t evict_up(size_t x) { return (x + 255) & ~(size_t)255; }

template <int STAGE>
static int launch_move(const EvictParams& p, cudaStream_t s) {
    const dim3 grid((unsigned)(p.batch * p.out_pages));
    const bool wide = p.slot_bytes % 16 == 0 && ((uintptr_t)p.kv_cache & 15) == 0;
    if (wide) TQ_CUDA(launch_serialized(evict_move_kernel<STAGE, uint4>, grid, dim3(kMoveThreads), 0, s, p));
    else TQ_CUDA(launch_serialized(evict_move_kernel<STAGE, uint32_t>, grid, dim3(kMoveThreads), 0, s, p));
    return TQ_OK;
}

}  // namespace tq

extern "C" size_t tq_evict_workspace_bytes(int batch, int num_kv_heads, int slot_bytes, int max_tokens, int keep, int in_place, int scores_in_place) {
    if (batch < 1 || num_kv_heads < 1 || slot_bytes < 1 || max_tokens < 0 || keep < 1) return 0;
    const size_t n = (size_t)(keep < max_tokens ? keep : max_tokens), pages = (n + 15) / 16;
    size_t bytes = 0;
    if (in_place) bytes += tq::evict_up((size_t)batch * pages * 32 * num_kv_heads * slot_bytes);
    if (scores_in_place) bytes += tq::evict_up((size_t)batch * num_kv_heads * keep * sizeof(float));
    return bytes;
}

extern "C" int tq_evict(void* kv_cache, int64_t num_blocks, int block_size, int num_kv_heads, int slot_bytes, const int32_t* page_table, int max_pages,
                        const int32_t* seq_lens, int batch, const float* scores, int64_t score_batch_stride, int64_t score_head_stride, int max_tokens,
                        int keep, int recent, const int32_t* out_page_table, int out_max_pages, float* out_scores, int64_t out_batch_stride,
                        int64_t out_head_stride, int32_t* kept, int32_t* new_lens, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace tq;
    TQ_REQUIRE(batch >= 0 && num_blocks >= 0, TQ_ERR_INVALID, "negative size");
    if (batch == 0) return TQ_OK;
    TQ_REQUIRE(kv_cache && page_table && seq_lens && scores && out_scores && kept && new_lens, TQ_ERR_INVALID, "null pointer");
    TQ_REQUIRE(block_size == 16, TQ_ERR_UNSUPPORTED, "block_size must be 16, got %d", block_size);
    TQ_REQUIRE(num_kv_heads >= 1 && slot_bytes >= 4 && slot_bytes % 4 == 0 && max_pages >= 1 && max_tokens >= 1, TQ_ERR_INVALID, "bad geometry");
    TQ_REQUIRE(((uintptr_t)kv_cache & 3) == 0 && ((uintptr_t)scores & 3) == 0, TQ_ERR_INVALID, "kv_cache and scores must be 4-byte aligned");
    TQ_REQUIRE(keep >= 1, TQ_ERR_INVALID, "keep must be at least 1, got %d", keep);
    TQ_REQUIRE(recent >= 0 && recent <= keep, TQ_ERR_INVALID, "recent must be in 0 ... keep = %d, got %d", keep, recent);
    const int64_t room = (int64_t)max_pages * 16;
    const int most = room < max_tokens ? (int)room : max_tokens;      // the longest sequence that the table and the scores can hold
    const int longest = keep < most ? keep : most, out_pages = (longest + 15) / 16;
    TQ_REQUIRE(out_page_table == nullptr || out_max_pages >= out_pages, TQ_ERR_INVALID, "the output table has %d pages a row, %d tokens need %d", out_max_pages,
               longest, out_pages);
    TQ_REQUIRE(most <= 1 << 30, TQ_ERR_UNSUPPORTED, "sequences of more than 2^30 tokens");
    TQ_REQUIRE(score_batch_stride >= 0 && score_head_stride >= 0 && out_batch_stride >= 0 && out_head_stride >= 0, TQ_ERR_INVALID, "negative stride");
    TQ_REQUIRE((batch == 1 || out_batch_stride >= longest) && (num_kv_heads == 1 || out_head_stride >= longest), TQ_ERR_INVALID,
               "the rows of out_scores overlap");
    // Scores that are written where scores are read wait until all have been read.
    auto last = [&](int64_t sb, int64_t sh, int64_t n) { return (batch - 1) * sb + (num_kv_heads - 1) * sh + n; };
    const bool in_place = out_page_table == nullptr;
    const bool scores_staged = out_scores < scores + last(score_batch_stride, score_head_stride, most) &&
                               scores < out_scores + last(out_batch_stride, out_head_stride, longest);
    const size_t need = tq_evict_workspace_bytes(batch, num_kv_heads, slot_bytes, most, keep, in_place, scores_staged);
    TQ_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), TQ_ERR_WORKSPACE, "workspace too small: %zu < %zu", workspace_bytes, need);
    TQ_REQUIRE((int64_t)batch * num_kv_heads < 1 << 26 && (int64_t)batch * out_pages < 1ll << 31, TQ_ERR_UNSUPPORTED, "too many rows for one launch");

    EvictParams p{};
    p.kv_cache = static_cast<uint8_t*>(kv_cache);
    p.table = page_table;
    p.out_table = out_page_table;
    p.seq_lens = seq_lens;
    p.scores = scores;
    p.out_scores = out_scores;
    p.kept = kept;
    p.new_lens = new_lens;
    p.num_blocks = num_blocks;
    p.half_bytes = (int64_t)16 * num_kv_heads * slot_bytes;
    p.slab_bytes = num_blocks * p.half_bytes;
    p.score_b = score_batch_stride;
    p.score_h = score_head_stride;
    p.out_b = out_batch_stride;
    p.out_h = out_head_stride;
    p.batch = batch;
    p.kv_heads = num_kv_heads;
    p.slot_bytes = slot_bytes;
    p.max_pages = max_pages;
    p.out_max_pages = out_max_pages;
    p.out_pages = out_pages;
    p.max_tokens = most;
    p.keep = keep;
    p.recent = recent;
    p.wide = ((uintptr_t)scores & 15) == 0 && score_batch_stride % 4 == 0 && score_head_stride % 4 == 0;
    p.scores_staged = scores_staged;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.staging = in_place ? ws : nullptr;
    if (scores_staged) {
        p.score_to = reinterpret_cast<float*>(ws + (in_place ? evict_up((size_t)batch * out_pages * 2 * p.half_bytes) : 0));
        p.to_h = keep;
        p.to_b = (int64_t)num_kv_heads * keep;
    } else {
        p.score_to = out_scores;
        p.to_h = out_head_stride;
        p.to_b = out_batch_stride;
    }

    // Blocks of a cluster: as many as leave each 4096 tokens, while all clusters together are at most two blocks an SM.
    int sms = 0;
    const int rc = device_sm_count(&sms);
    if (rc != TQ_OK) return rc;
    const int units = batch * num_kv_heads;
    int C = 1;
    while (C < kEvictMaxCluster && most / (2 * C) >= 4096 && (int64_t)units * 2 * C <= 2 * sms) C *= 2;
    p.cluster = C;
    const int share = ((most + kEvictWarps * C - 1) / (kEvictWarps * C) + kEvictRun - 1) / kEvictRun * kEvictRun * kEvictWarps;
    p.key_room = share <= kEvictMostKeys ? share : 0;
    const size_t smem = kEvictHistBytes + (size_t)p.key_room * 4;
    static bool configured[64] = {};
    int dev = 0;
    TQ_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        TQ_CUDA(cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvictHistBytes + kEvictMostKeys * 4));
        TQ_CUDA(cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(units * C));
    cfg.blockDim = dim3(kEvictThreads);
    cfg.dynamicSmemBytes = smem;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)C;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    TQ_CUDA(cudaLaunchKernelEx(&cfg, evict_select_kernel, p));
    if (!in_place) return launch_move<0>(p, s);
    const int moved = launch_move<1>(p, s);
    return moved != TQ_OK ? moved : launch_move<2>(p, s);
}
