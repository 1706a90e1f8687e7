// Eviction from the paged cache by accumulated attention weight.
//
// For every sequence and KV head, of its len tokens the last `recent` stay and, of the others, those of the largest scores, keep in all (a tie goes
// to the lower position, a NaN counts as -inf).  The tokens that stay keep their order: with kept[0] < kept[1] < ... the row of
// token kept[j] moves to position j, in other pages or in the sequence's own.  Attention over the cache does not care that another head
// has another token at that position: a key carries its position with it.
//
//   select   A cluster of blocks for each (sequence, head) finds the score of rank k = keep - recent by its bits from the top.  A score becomes an
//            unsigned word that sorts as the float does.  The leading eleven bits (sign, exponent, two of the fraction) come from a histogram of all
//            tokens, summed over the cluster through distributed shared memory; a second walk over the tokens counts those above that bin,
//            lists those in it, a few in a hundred, and the places of both; the other bits, 8, 8 and 5 at a time, come from the lists.  Then the counts of what stays
//            are summed over the warps and blocks in front, each of which has a run of tokens of its own, and from the places (or a
//            third walk, where there are too many) every warp writes its tokens one behind the other (a million tokens, 1 in 16 stays: 124 us with
//            the third walk, 112 so; 1 in 4 of 32768, keys in shared memory: 66.5 and 67.2).  No order of atomics reaches the result.
//   move     A block for each page of the destination: all its slots of K and V, 16 bytes a thread and step, so that the stores cover
//            whole lines; the loads are gathered slots.
//
// What bounds it: the scores are read once (4 bytes a token and head), the kept slots are read and written (160 bytes each way for a
// head of 128).  Memory is read in 64-byte pieces, of which a slot of 80 bytes anywhere touches 2.2: the move of 8 sequences' 8192 tokens of 32768,
// 8 heads, takes 45 us for 166 MB read and 84 MB written, 5.5 TB/s; the selection before it 21 us, the walks of 16384 scores by 16 warps an SM
// and the cluster's waits between them.  One sequence of a million tokens, 8 heads: 112 us, the selection 63 of them, as a cluster has no more than 16 SMs for a head and
// issues 60 percent of their slots.
#include "tq_common.cuh"

namespace tq {

// Threads of a block of the selection: two blocks an SM; or one, where its share has no room in shared memory and each walk over it waits for L2 (a million
// tokens, 8 heads, three walks: 138 us with 512 threads a block, 124 with 1024; shares of 16384 tokens in shared memory: 66.5 and 66.9).
constexpr int kEvictThreads = 512, kEvictManyThreads = 1024;
constexpr int kEvictRun = 128;                 // tokens of a warp's load: four a lane
constexpr int kEvictAhead = 4;                 // loads in flight together
constexpr int kEvictMaxCluster = 16;
// First histogram: 2048 bins of eight columns (lane % 8), as sums of softmax weights share few exponents.  Then, in its place, that of eight bits with a
// column for every lane, and the lists, one for each warp; a warp whose list does not hold its tokens walks over all of them instead.
constexpr int kEvictBins = 2048, kEvictColumns = 8, kEvictDigits = 256;
constexpr int kEvictHistBytes = kEvictBins * kEvictColumns * 4, kEvictDigitBytes = kEvictDigits * 32 * 4;
constexpr int kEvictListBytes = kEvictHistBytes - kEvictDigitBytes;
constexpr int kEvictMost = 221184, kEvictHalf = 104448;      // shared memory of one block an SM, of two, without the fixed arrays
constexpr int kEvictMostKeys = 36 * 1024;      // sort keys a block keeps in shared memory beside them; longer shares are read from L2 in every walk

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
    int batch, kv_heads, slot_bytes, max_pages, out_max_pages, out_pages, max_tokens, keep, recent, cluster, wide;
    int scores_staged;
    int listed;                    // places that a warp has for its tokens that may stay
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
// The sum over the cluster's C blocks of N neighbouring counts each: all loads are on their way before the first is used.
template <int N>
__device__ __forceinline__ void cluster_sums(const int* local, int C, int (&sum)[N]) {
    int part[kEvictMaxCluster][N];
#pragma unroll
    for (int r = 0; r < kEvictMaxCluster; r++) {
#pragma unroll
        for (int i = 0; i < N; i++) part[r][i] = 0;
        if (r < C) {
            uint32_t at;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local)), "r"(r));
            if constexpr (N == 4) asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(part[r][0]), "=r"(part[r][1]), "=r"(part[r][2]), "=r"(part[r][3]) : "r"(at) : "memory");
            else if constexpr (N == 2) asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(part[r][0]), "=r"(part[r][1]) : "r"(at) : "memory");
            else asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(part[r][0]) : "r"(at) : "memory");
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        sum[i] = 0;
#pragma unroll
        for (int r = 0; r < kEvictMaxCluster; r++) sum[i] += part[r][i];
    }
}
__device__ __forceinline__ int cluster_load(const int* local, uint32_t rank) {
    uint32_t at;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

template <bool KEPT>
__global__ void __launch_bounds__(KEPT ? kEvictThreads : kEvictManyThreads, KEPT ? 2 : 1) evict_select_kernel(const __grid_constant__ EvictParams p) {
    constexpr int THREADS = KEPT ? kEvictThreads : kEvictManyThreads, kWarps = THREADS / 32, kList = kEvictListBytes / 4 / kWarps;
    extern __shared__ __align__(16) uint32_t evict_smem[];
    uint32_t* const hist = evict_smem;                            // [bin][column], then [digit][lane]
    uint32_t* const lists = evict_smem + kEvictDigitBytes / 4;
    uint32_t* const keys = evict_smem + kEvictHistBytes / 4;      // the block's share, KEPT; behind it the places of tokens that may stay
    __shared__ __align__(16) int sums[kEvictBins], sums8[2][kEvictDigits];
    __shared__ int counts[2], warp_gt[32], warp_eq[32], found[2][2], above_s[2][32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int C = p.cluster, rank = C > 1 ? (int)cluster_rank() : 0;
    const int unit = blockIdx.x / C, b = unit / p.kv_heads, h = unit - b * p.kv_heads;
    for (int i = tid; i < kEvictHistBytes / 16; i += THREADS) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0u, 0u, 0u, 0u);
    grid_dependency_wait();

    bool bad;
    const int len = evict_len(p, b, bad);
    const int n = min(len, p.keep), recent = min(p.recent, n), M = len - recent, k = n - recent;
    if (bad && h == 0 && rank == 0 && tid == 0) atomicAdd(&g_evict_faults, 1);
    const float* const row = p.scores + b * p.score_b + h * p.score_h;
    float* const to = p.score_to + b * p.to_b + h * p.to_h;
    int32_t* const kept = p.kept + (int64_t)unit * p.keep;
    const int me = rank * THREADS + tid, all = C * THREADS;
    // The blocks of the move are let in late: waiting ones would keep other selecting blocks out (or ask for another split of the SM's memory).
    auto leave = [&] { grid_launch_dependents(); };
    for (int j = me; j < recent; j += all) {
        kept[k + j] = M + j;
        to[k + j] = row[M + j];
    }
    for (int64_t j = n + me; j < p.keep; j += all) kept[j] = -1;      // (keep may be the largest int)
    if (k == M) {                      // all of them (uniform over the cluster, as the way out below is)
        for (int j = me; j < k; j += all) {
            kept[j] = j;
            to[j] = row[j];
        }
        leave();
        return;
    }
    if (k == 0) {
        leave();
        return;
    }

    // This warp's run of tokens.
    const int W = ((M + kWarps * C - 1) / (kWarps * C) + kEvictRun - 1) / kEvictRun * kEvictRun;
    const int64_t begin64 = ((int64_t)rank * kWarps + warp) * W;
    const int begin = begin64 < M ? (int)begin64 : M, end = begin64 + W < M ? (int)(begin64 + W) : M;
    uint32_t* const my_keys = keys + (size_t)warp * W;
    uint16_t* const mays = reinterpret_cast<uint16_t*>(keys + (KEPT ? (size_t)kWarps * W : 0)) + (size_t)warp * p.listed;
    const bool wide = p.wide;
    // Goes over the warp's tokens, four a lane in each of kEvictAhead runs: body(first token of the lane in a run, keys, a run).  Past the end the key is zero, which
    // no score has.
    auto walk = [&](bool from_keys, auto&& body) {
        for (int at = begin; at < end; at += kEvictRun * kEvictAhead) {
            uint32_t key[kEvictAhead][4];
            if (KEPT && from_keys) {
#pragma unroll
                for (int u = 0; u < kEvictAhead; u++) {
                    const bool in = at + kEvictRun * u < end;
                    const uint4 k4 = in ? *reinterpret_cast<const uint4*>(my_keys + (at - begin) + kEvictRun * u + 4 * lane) : make_uint4(0u, 0u, 0u, 0u);
                    key[u][0] = k4.x; key[u][1] = k4.y; key[u][2] = k4.z; key[u][3] = k4.w;
                }
            } else if (wide && at + kEvictRun * kEvictAhead <= end) {
                float4 v[kEvictAhead];
#pragma unroll
                for (int u = 0; u < kEvictAhead; u++) v[u] = *reinterpret_cast<const float4*>(row + at + kEvictRun * u + 4 * lane);
#pragma unroll
                for (int u = 0; u < kEvictAhead; u++) {
                    key[u][0] = evict_key(v[u].x); key[u][1] = evict_key(v[u].y); key[u][2] = evict_key(v[u].z); key[u][3] = evict_key(v[u].w);
                }
            } else {
#pragma unroll
                for (int u = 0; u < kEvictAhead; u++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int i = at + kEvictRun * u + 4 * lane + e;
                        key[u][e] = i < end ? evict_key(row[i]) : 0u;
                    }
            }
#pragma unroll
            for (int u = 0; u < kEvictAhead; u++) body(at + kEvictRun * u + 4 * lane, key[u]);
        }
    };
    auto all_sync = [&] {
        if (C > 1) cluster_sync();
        else __syncthreads();
    };
    // Of counts by thread, the first thread's bins uppermost: how many lie above this thread's.  Two calls use different `turn`s.
    auto above_all = [&](int mine, int turn) {
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        if (lane == 31) above_s[turn][warp] = upto;
        __syncthreads();
        const int t = lane < warp ? above_s[turn][lane] : 0;
        return upto - mine + __reduce_add_sync(0xffffffffu, t);
    };

    // ---- the leading eleven bits ------------------------------------------------------------------------
    __syncthreads();                   // the histogram is zero
    walk(false, [&](int at, const uint32_t (&key)[4]) {
        if (KEPT && at - 4 * lane < end) *reinterpret_cast<uint4*>(my_keys + (at - begin)) = make_uint4(key[0], key[1], key[2], key[3]);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (key[e] != 0u) atomicAdd(&hist[(key[e] >> 21) * kEvictColumns + (lane & (kEvictColumns - 1))], 1u);
    });
    __syncthreads();
    constexpr int kMine = kEvictBins / THREADS;
    int left = k;                      // the rank looked for among the tokens that agree with what is known of the key
    {
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            const uint4* const at = reinterpret_cast<const uint4*>(hist + (tid + THREADS * i) * kEvictColumns);
            const uint4 x = at[0], y = at[1];
            sums[tid + THREADS * i] = (int)(x.x + x.y + x.z + x.w + y.x + y.y + y.z + y.w);
        }
        all_sync();
        int up[kMine], c[kMine], mine = 0;      // bins 2047 - kMine tid - i, the uppermost first
        const int* const at = &sums[kEvictBins - kMine * (tid + 1)];
        if (C > 1) {
            cluster_sums<kMine>(at, C, up);
        } else {
#pragma unroll
            for (int i = 0; i < kMine; i++) up[i] = at[i];
        }
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            c[i] = up[kMine - 1 - i];
            mine += c[i];
        }
        // (the histogram becomes the digits', zero)
        for (int i = tid; i < kEvictDigitBytes / 16; i += THREADS) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0u, 0u, 0u, 0u);
        int above = above_all(mine, 0);
        if (above < left && above + mine >= left) {
#pragma unroll
            for (int i = 0; i < kMine; i++) {
                if (above < left && above + c[i] >= left) {
                    found[0][0] = kEvictBins - 1 - kMine * tid - i;
                    found[0][1] = left - above;
                }
                above += c[i];
            }
        }
        __syncthreads();
    }
    uint32_t prefix = (uint32_t)found[0][0];
    left = found[0][1];

    // ---- what lies above, and the list of what lies in the bin ---------------------------------------------
    const uint32_t lower = (1u << lane) - 1u;
    uint32_t* const list = lists + warp * kList;
    int gt = 0, listed = 0, may = 0;
    walk(true, [&](int at, const uint32_t (&key)[4]) {
        // those in the bin or above it, by position: what the last walk has to look at
        uint32_t mine = 0, below = 0, all = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            gt += key[e] >> 21 > prefix;
            const bool stays = key[e] >> 21 >= prefix && key[e] != 0u;
            const uint32_t m = __ballot_sync(0xffffffffu, stays);
            mine |= (uint32_t)stays << e;
            below += __popc(m & lower);
            all += __popc(m);
        }
        int place = may + (int)below;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (mine >> e & 1u) {
                if (place < p.listed) mays[place] = (uint16_t)(at + e - begin);
                place++;
            }
        may += (int)all;
        const bool in[4] = {key[0] >> 21 == prefix && key[0] != 0u, key[1] >> 21 == prefix && key[1] != 0u, key[2] >> 21 == prefix && key[2] != 0u,
                            key[3] >> 21 == prefix && key[3] != 0u};
        if (__any_sync(0xffffffffu, in[0] | in[1] | in[2] | in[3])) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t m = __ballot_sync(0xffffffffu, in[e]);
                const int at = listed + __popc(m & lower);
                if (in[e] && at < kList) list[at] = key[e];
                listed += __popc(m);
            }
        }
    });
    const bool fits = listed <= kList;
    __syncwarp();
    auto candidates = [&](auto&& body) {       // body(key) of every token in the bin, and of some zeros
        if (fits) {
            for (int i = 0; i < listed; i += 32) body(i + lane < listed ? list[i + lane] : 0u);
        } else {
            const uint32_t bin = (uint32_t)found[0][0];
            walk(true, [&](int, const uint32_t (&key)[4]) {
#pragma unroll
                for (int e = 0; e < 4; e++) body(key[e] >> 21 == bin ? key[e] : 0u);
            });
        }
    };

    // ---- the other bits -----------------------------------------------------------------------------------
    // A single block with no more tokens in the bin than threads compares each with all: one step in place of three.
    bool done = false;
    if (C == 1) {
        if (lane == 0) warp_gt[warp] = listed;
        __syncthreads();
        const int others = lane < kWarps ? warp_gt[lane] : 0, total = __reduce_add_sync(0xffffffffu, others);
        const int first = __reduce_add_sync(0xffffffffu, lane < warp ? others : 0);
        done = total <= THREADS && !__any_sync(0xffffffffu, others > kList);
        if (done) {                    // (the digits' histogram is not needed)
            for (int i = lane; i < listed; i += 32) hist[first + i] = list[i];
            if (tid < 4) hist[total + tid] = 0u;
            __syncthreads();
            const uint32_t key = tid < total ? hist[tid] : 0u;
            int above = 0, same = 0;
            for (int i = 0; i < total; i += 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(hist + i);
                above += (v.x > key) + (v.y > key) + (v.z > key) + (v.w > key);
                same += (v.x == key) + (v.y == key) + (v.z == key) + (v.w == key);
            }
            if (tid < total && above < left && above + same >= left) {       // (all threads of that key write the same)
                found[1][0] = (int)key;
                found[1][1] = left - above;
            }
            __syncthreads();
            prefix = (uint32_t)found[1][0];
            left = found[1][1];
        }
    }
    for (int pass = 0; pass < 3 && !done; pass++) {
        const int shift = pass == 0 ? 13 : pass == 1 ? 5 : 0, bits = pass == 2 ? 5 : 8;
        const uint32_t mask = (1u << bits) - 1u;
        candidates([&](uint32_t key) {
            if (key != 0u && key >> (shift + bits) == prefix) atomicAdd(&hist[((key >> shift) & mask) * 32 + lane], 1u);
        });
        __syncthreads();
        {   // THREADS / 256 threads a digit, the columns shared out
            constexpr int kShare = THREADS / kEvictDigits, kEach = 32 / kShare;
            const int digit = tid / kShare, first_column = kEach * (tid % kShare);
            uint32_t sum = 0;
#pragma unroll
            for (int c = 0; c < kEach; c++) {
                const int at = digit * 32 + first_column + ((c + digit) & (kEach - 1));
                sum += hist[at];
                hist[at] = 0;
            }
#pragma unroll
            for (int o = 1; o < kShare; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (tid % kShare == 0) sums8[pass & 1][digit] = (int)sum;
        }
        all_sync();
        int mine = 0;                  // thread t < 256: digit 255 - t
        if (tid < kEvictDigits) {
            int sum[1] = {sums8[pass & 1][255 - tid]};
            if (C > 1) cluster_sums<1>(&sums8[pass & 1][255 - tid], C, sum);
            mine = sum[0];
        }
        const int above = above_all(mine, ~pass & 1);
        if (above < left && above + mine >= left) {
            found[1][0] = 255 - tid;
            found[1][1] = left - above;
        }
        __syncthreads();
        prefix = prefix << bits | (uint32_t)found[1][0];
        left = found[1][1];
        __syncthreads();               // found is read before it is written again
    }
    // prefix is now the key of rank k, and `left` of the tokens that have it stay: those of the lowest positions.

    int eq = 0;
    candidates([&](uint32_t key) {
        gt += key > prefix;
        eq += key == prefix;
    });
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) {
        warp_gt[warp] = gt;
        warp_eq[warp] = eq;
    }
    __syncthreads();
    if (warp == 0) {                   // sums of the warps in front, and the block's
        int g = lane < kWarps ? warp_gt[lane] : 0, q = lane < kWarps ? warp_eq[lane] : 0;
        const int g0 = g, q0 = q;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, g, o), c = __shfl_up_sync(0xffffffffu, q, o);
            if (lane >= o) {
                g += a;
                q += c;
            }
        }
        warp_gt[lane] = g - g0;
        warp_eq[lane] = q - q0;
        if (lane == 31) {
            counts[0] = g;
            counts[1] = q;
        }
    }
    all_sync();
    int before_gt = warp_gt[warp], before_eq = warp_eq[warp];
    if (C > 1) {
        before_gt += __reduce_add_sync(0xffffffffu, lane < rank ? cluster_load(&counts[0], (uint32_t)min(lane, C - 1)) : 0);
        before_eq += __reduce_add_sync(0xffffffffu, lane < rank ? cluster_load(&counts[1], (uint32_t)min(lane, C - 1)) : 0);
        cluster_sync();                // no block of the cluster leaves while another reads its counts
    }
    leave();
    int ties = left - before_eq;       // of this warp's tokens with the key of rank k, the first `ties` stay
    int place = before_gt + min(before_eq, left);
    if (may <= p.listed) {
        __syncwarp();
        for (int i = 0; i < may; i += 32) {
            const bool in = i + lane < may;
            const int at = begin + (in ? (int)mays[i + lane] : 0);
            uint32_t key = 0;
            float score = 0.0f;
            if constexpr (KEPT) {
                key = in ? my_keys[at - begin] : 0u;
                score = __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
                if (key == 0x80000000u || key == 0x007fffffu) score = row[at];      // a key that stands for two (zeros, a NaN and -inf)
            } else if (in) {
                score = row[at];
                key = evict_key(score);
            }
            const bool is_eq = key == prefix;
            const uint32_t same = __ballot_sync(0xffffffffu, is_eq);
            const bool stays = key > prefix || (is_eq && __popc(same & lower) < ties);
            const uint32_t m = __ballot_sync(0xffffffffu, stays);
            if (stays) {
                const int j = place + __popc(m & lower);
                kept[j] = at;
                to[j] = score;
            }
            ties -= __popc(same);
            place += __popc(m);
        }
        return;
    }
    walk(true, [&](int at, const uint32_t (&key)[4]) {
        bool is_eq[4], stays[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            stays[e] = key[e] > prefix;
            is_eq[e] = key[e] == prefix;
        }
        if (__any_sync(0xffffffffu, is_eq[0] | is_eq[1] | is_eq[2] | is_eq[3])) {
            int total = 0, eq_before = 0;
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
        float score[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {   // the score from its key; a key that stands for two (zeros, a NaN and -inf) is looked up
            score[e] = __uint_as_float(key[e] ^ (key[e] >> 31 ? 0x80000000u : 0xffffffffu));
            if (stays[e] && (key[e] == 0x80000000u || key[e] == 0x007fffffu)) score[e] = row[at + e];
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (stays[e]) {
                kept[j] = at + e;
                to[j] = score[e];
                j++;
            }
        }
    });
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
    // The new lengths may replace the old ones: they are written behind the selection, whose blocks all have to see the same length, and a block of this
    // launch that reads one already replaced comes to the same n.
    if (STAGE != 1 && page == 0 && threadIdx.x == 0) p.new_lens[b] = n;
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
                const int64_t from = in[t >> 4];
                if ((uint64_t)from < (uint64_t)p.num_blocks) at = STAGE == 2 ? 0 : from * p.half_bytes + ((int64_t)(t & 15) * H + h) * p.slot_bytes;
                else if (STAGE != 2) atomicAdd(&g_evict_faults, 1);      // (nothing was staged for it: it is left out on the way back too)
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

// Launches the selection with the largest cluster of up to C blocks of which all run at the same time.  too_long: a block's keys have no room in shared memory.
template <bool KEPT>
static int launch_select(EvictParams& p, int units, int C, int too_long, cudaStream_t s) {
    // (A cluster stays inside one of the device's groups of SMs, which have not all the same number: eight of sixteen blocks would run seven and one.)
    static int active[64][2][kEvictMaxCluster + 1] = {};      // by device, and one block an SM or two: clusters of c blocks that run at the same time, plus one
    int dev = 0;
    TQ_CUDA(cudaGetDevice(&dev));
    TQ_REQUIRE(dev >= 0 && dev < 64, TQ_ERR_UNSUPPORTED, "device %d", dev);
    const auto kernel = evict_select_kernel<KEPT>;
    constexpr int THREADS = KEPT ? kEvictThreads : kEvictManyThreads, kWarps = THREADS / 32;
    if (active[dev][0][1] == 0) {
        TQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvictMost));
        TQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        active[dev][0][1] = 1;
    }
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(THREADS);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    auto run = [&](int c) { return ((p.max_tokens + kWarps * c - 1) / (kWarps * c) + kEvictRun - 1) / kEvictRun * kEvictRun; };      // tokens of a warp
    auto need = [&](int c) { return kEvictHistBytes + (KEPT ? (int64_t)run(c) * kWarps * 4 : 0); };
    auto two = [&](int c) { return KEPT && need(c) <= kEvictHalf; };
    for (; C > 1; C--) {
        int& known = active[dev][two(C)][C];
        if (known == 0) {
            cfg.gridDim = dim3((unsigned)(64 * C));
            cfg.dynamicSmemBytes = two(C) ? kEvictHalf : kEvictMost;
            attr[0].val.clusterDim.x = (unsigned)C;
            cfg.numAttrs = 1;
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
                cudaGetLastError();
                n = 0;
            }
            known = n + 1;
        }
        if (known - 1 >= units) break;
    }
    if (need(C) > kEvictHistBytes + kEvictMostKeys * 4) return too_long;
    p.cluster = C;
    // What is left of the memory has the places of tokens that may stay; a warp with more of them walks over all its tokens.
    const int room = (int)((two(C) ? kEvictHalf : kEvictMost) - need(C)) / 2 / kWarps;
    p.listed = run(C) <= 65536 ? (run(C) < room ? run(C) : room) : 0;
    cfg.gridDim = dim3((unsigned)(units * C));
    cfg.dynamicSmemBytes = (size_t)need(C) + (size_t)p.listed * 2 * kWarps;
    attr[0].val.clusterDim.x = (unsigned)C;
    cfg.numAttrs = 2;
    TQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return TQ_OK;
}

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
    TQ_REQUIRE(!rows_overlap(batch, num_kv_heads, out_batch_stride, out_head_stride, longest), TQ_ERR_INVALID, "the rows of out_scores overlap");
    // Scores that are written where scores are read wait until all have been read.
    auto last = [&](int64_t sb, int64_t sh, int64_t n) { return (batch - 1) * sb + (num_kv_heads - 1) * sh + n; };
    const bool in_place = out_page_table == nullptr;
    const bool scores_staged = out_scores < scores + last(score_batch_stride, score_head_stride, most) &&
                               scores < out_scores + last(out_batch_stride, out_head_stride, longest);
    const size_t need = tq_evict_workspace_bytes(batch, num_kv_heads, slot_bytes, most, keep, in_place, scores_staged);
    TQ_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), TQ_ERR_WORKSPACE, "workspace too small: %zu < %zu", workspace_bytes, need);
    // Blocks read lengths, tables and scores while others write: what is written may be `scores` and, word for word, `seq_lens`, nothing else that is read.
    struct Span { const void* at; int64_t words; };
    auto meet = [](Span a, Span b) {
        return a.at && b.at && (uintptr_t)a.at < (uintptr_t)b.at + 4 * (uint64_t)b.words && (uintptr_t)b.at < (uintptr_t)a.at + 4 * (uint64_t)a.words;
    };
    const Span s_lens{seq_lens, batch}, s_table{page_table, (int64_t)batch * max_pages}, s_out_table{out_page_table, (int64_t)batch * out_max_pages},
        s_scores{scores, last(score_batch_stride, score_head_stride, most)}, s_out{out_scores, last(out_batch_stride, out_head_stride, longest)},
        s_kept{kept, (int64_t)batch * num_kv_heads * keep}, s_new{new_lens, batch};
    for (const Span& w : {s_out, s_kept, s_new})
        TQ_REQUIRE(!meet(w, s_table) && !meet(w, s_out_table) && (!meet(w, s_lens) || w.at == new_lens && new_lens == seq_lens), TQ_ERR_INVALID,
                   "an output overlaps the lengths or a table");
    TQ_REQUIRE(!meet(s_kept, s_scores) && !meet(s_kept, s_out) && !meet(s_kept, s_new) && !meet(s_new, s_scores) && !meet(s_new, s_out), TQ_ERR_INVALID,
               "kept or new_lens overlaps scores, or one the other");
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

    // Blocks of a cluster: as many as leave each 4096 tokens, up to an SM each.
    int sms = 0;
    int rc = device_sm_count(&sms);
    if (rc != TQ_OK) return rc;
    const int units = batch * num_kv_heads;
    int C = 1;
    while (C < kEvictMaxCluster && most / (C + 1) >= 4096 && (int64_t)units * (C + 1) <= sms) C++;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    constexpr int kTooLong = -1;
    rc = launch_select<true>(p, units, C, kTooLong, s);
    if (rc == kTooLong) rc = launch_select<false>(p, units, C, kTooLong, s);
    if (rc != TQ_OK) return rc;
    if (!in_place) return launch_move<0>(p, s);
    const int moved = launch_move<1>(p, s);
    return moved != TQ_OK ? moved : launch_move<2>(p, s);
}
