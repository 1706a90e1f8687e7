// One-token decode that also gives the attention weights: out = softmax(q K^T) V over the quantized cache, and to the score of every
// cached token is added its weight, summed over the query heads that share its KV head.
//
// A weight exp(x - lse) needs the whole row's lse, which is known only at the end.  So the decode kernel, beside its online softmax, keeps the
// logits x (fp32, 4 bytes a query head and token: 16 for four heads against the 160 bytes of codes and norms just read), and the
// kernel that joins the partials goes over them once more.  Reading K a second time instead would cost 80 bytes and all its lookups.
//
// The scores are sums of many steps and their order decides what an eviction keeps, so the logits are worked out to about 2^-20: the codebook
// has two tables, the fp16 levels and what fp16 leaves of them, and a query row is two MMA columns, its fp16 part and the rest
//     x = K_hi (q_hi + q_lo) + K_lo (q_hi + q_lo).
// An MMA tile has eight columns; four query heads fill it so.  The levels are scaled by 1.42803, at which the eight of them lie within
// 4e-5 (rms) of fp16 values instead of 2.6e-4: V is read from the first table alone.  Up to four query heads the columns that the second
// part of a head has in P V take what fp16 leaves of its probabilities, at no cost.
//
// The plan, the page rings and the fragment scheme are those of tq_decode_split.cu (one tile of eight columns there): a group of four warps takes
// one head of a page range, every warp whole pages of its own.
//
// What bounds it: the look-ups.  A code byte of K is looked up twice and one of V once, and with the page loads that fills shared memory's pipe to 74 percent while
// 63 percent of the issue slots are taken: 8 sequences of 32768 tokens, 32 heads on 8, 113 us, of which the decode 95 (342 MB, 3.6 TB/s) and the
// join 18; a second walk over K in the join's place would be as long as the decode.  Short sequences: the launches, 1024 tokens 10.4 us.
#include <cmath>
#include <cstring>

#include "tq_split.cuh"

namespace tq {

constexpr int kScoredGroups = 4, kScoredGroupWarps = 4, kScoredWarps = 16, kScoredThreads = 512;
constexpr int kScoredRow = 80, kScoredHalf = 16 * kScoredRow, kScoredStage = 2 * kScoredHalf, kScoredStages = 3, kScoredRing = kScoredStages * kScoredStage;
constexpr int kScoredBelow = 7;              // rings below the tables at 64 KB; the others above them, then queries and plans
constexpr int kScoredItemCost = 20;          // pages that starting an item is worth, as in the split decode
constexpr uint32_t kScoredQ = kLutAddr + kLutSpan + (kScoredWarps - kScoredBelow) * kScoredRing;
constexpr uint32_t kScoredPlan = kScoredQ + kScoredGroups * 16 * 256;
constexpr size_t kScoredSmem = kScoredPlan + kScoredWarps * 512 - 1024;
constexpr double kLevelScale = 1.42803;
static_assert(kScoredRing >= 8 * kHeadDim * 4, "a warp's partial output goes through its ring");

struct ScoredParams {
    SplitParams d;
    float* logits;             // [batch x KV heads][room][query heads of a KV head], base 2
    int2* plan;                // [batch], up to kSplitSelf sequences: pages of the sequence, its place in the work list
    float* row_lse;            // [batch x KV heads][query heads of a KV head], base 2: rows that one group finished
    float* scores;
    int64_t score_b, score_h;
    int64_t room;              // tokens of a row of logits
    int score_room, new_tokens, chunks;
    int lose;                  // tests: no copy comes
    uint16_t rest_h[16];       // second table
};

static __device__ int32_t g_scored_faults = 0;
static int g_scored_lose = 0;
// The running maximum that a warp leaves behind a copy that never came, with a sum of +inf: the rows' lse is +inf then, which no logits add up to
// (one of +inf gives NaN), and tells the join.
constexpr float kScoredVoid = 3.0e38f;

// The slots of a page in one tensor copy, as in the split decode, but first to leave L2: read once, while the logits written meanwhile are read again.
__device__ __forceinline__ void scored_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar, uint64_t policy) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %6;"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(0), "r"(bar), "l"(policy) : "memory");
}
// Four code bytes through both tables: the rest is 128 bytes behind the level.
__device__ __forceinline__ void scored_lookup(uint32_t w, uint32_t lut_lane, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t at = prmt(w, lut_lane, 0x7604u | (j << 4));
        hi[j] = lds32(at);
        asm volatile("ld.shared.u32 %0, [%1+128];" : "=r"(lo[j]) : "r"(at));
    }
}

// NT: MMA tiles of four query heads.
template <int NT, bool MANY>
__global__ void __launch_bounds__(kScoredThreads, 1) decode_scored_kernel(const __grid_constant__ ScoredParams sp) {
    constexpr int PD = kHeadDim, E = PD / 32, NG = kScoredGroups, GW = kScoredGroupWarps;
    const SplitParams& p = sp.d;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float m_s[NG][GW][8], l_s[NG][GW][8], v_s[NG][GW], q_scale_s[NG][8];
    __shared__ float sign_s[PD];
    __shared__ uint64_t full_s[kScoredWarps][kScoredStages];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int gg = warp / GW, wg = warp % GW;
    const int g = lane >> 2, tg = lane & 3;
    const uint32_t smem_base = smem_u32(smem);
    const int G = p.group;
    if (smem_base + kScoredBelow * kScoredRing > kLutAddr) {   // the map does not fit: nothing is computed, the join finds a list without work
        grid_dependency_wait();
        if (tid == 0 && blockIdx.x == 0) {
            p.header[1] = 0;
            atomicAdd(&g_scored_faults, 1);
        }
        return;
    }
    auto at_smem = [&](uint32_t at) -> uint8_t* { return smem + (at - smem_base); };
    auto ring_of = [&](int w) -> uint32_t { return w < kScoredBelow ? smem_base + (uint32_t)w * kScoredRing : kLutAddr + kLutSpan + (uint32_t)(w - kScoredBelow) * kScoredRing; };
    const uint32_t ring_at = ring_of(warp);
    auto group_sync = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + gg), "r"(GW * 32) : "memory"); };

    {   // the tables: entry v, column c = {level(v & 15), level(v >> 4)}, and the rests behind them
        const uint32_t mine = p.centroid_h[lane & 15], rest = sp.rest_h[lane & 15];
        uint8_t* const lut = at_smem(kLutAddr);
        for (int v = 4 * warp + (lane >> 3); v < 256; v += 4 * kScoredWarps) {
            const uint32_t e = __shfl_sync(0xffffffffu, mine, v & 15) | (__shfl_sync(0xffffffffu, mine, v >> 4) << 16);
            const uint32_t f = __shfl_sync(0xffffffffu, rest, v & 15) | (__shfl_sync(0xffffffffu, rest, v >> 4) << 16);
            *reinterpret_cast<uint4*>(lut + v * 256 + 16 * (lane & 7)) = make_uint4(e, e, e, e);
            *reinterpret_cast<uint4*>(lut + v * 256 + 128 + 16 * (lane & 7)) = make_uint4(f, f, f, f);
        }
    }
    for (int i = tid; i < PD; i += kScoredThreads) sign_s[i] = p.signs[i];
    if (tid == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&p.cache_map) : "memory");
    if (lane < kScoredStages) mbar_init(&full_s[warp][lane], 1);
    fence_barrier_init();
    __syncthreads();
    grid_dependency_wait();
    grid_launch_dependents();

    SplitPlan s;
    if constexpr (MANY) split_plan_many<GW, NG>(p, s, lane);
    else split_plan<GW, NG>(p, s, lane);
    const int hs = s.head_set;
    const int sub = hs == 1 ? gg : hs == 2 ? gg >> 1 : gg >> 2, hsub = gg - sub * hs;
    const int worker = sub * p.grid + (int)blockIdx.x;
    int pos = 0, hi = 0;
    if (s.piece) {
        pos = worker;
        hi = worker < s.total ? worker + 1 : worker;
    } else if (worker < s.workers) {
        pos = split_cut(worker, s.total, s.workers);
        hi = split_cut(worker + 1, s.total, s.workers);
    }
    if constexpr (MANY) {
        if (blockIdx.x == 0 && warp == 0) split_keep_plan(p, s);
        split_jump(p, s, pos < hi ? __ffs(__ballot_sync(0xffffffffu, s.ends > pos)) - 1 : 0);
    } else if (blockIdx.x == gridDim.x - 1 && warp == 0) {      // for the join, whose blocks start when this kernel's end: there is no room beside them
        if (lane == 0) {
            p.header[1] = s.total;
            p.header[2] = s.workers;
            p.header[3] = s.piece;
        }
        SplitPlan all = s;
        for (int first = 0;;) {
            if (first + lane < p.batch) sp.plan[first + lane] = make_int2(all.np, all.vstart);
            const int run = __shfl_sync(0xffffffffu, all.vend, 31);
            first += 32;
            if (first >= p.batch) break;
            split_load(p, all, first, run, false);
        }
    }
    int4* const plan = reinterpret_cast<int4*>(at_smem(kScoredPlan + (uint32_t)warp * 512u + (uint32_t)lane * 16u));
    *plan = make_int4(s.np, s.len, s.vstart, s.vend);
    const int piece = s.piece;
    int base = MANY ? s.base : 0;
    const uint32_t lut_lane = split_keep(kLutAddr + 4u * lane);
    const int ta = g, tb = g + 8;
    const uint32_t k_at = split_keep(ring_at + g * kScoredRow + tg * 16), kn_at = split_keep(ring_at + g * kScoredRow + PD / 2);
    const uint32_t v_at = split_keep(ring_at + kScoredHalf + 2 * tg * kScoredRow + g * 8), vn_at = kn_at + kScoredHalf;
    const uint32_t full_at = split_keep(smem_u32(&full_s[warp][0]));
    uint32_t stage = 0, parity = 0;
    bool lost = sp.lose != 0, bad_page = false;

    while (pos < hi) {
        // ---- the next segment: a page range of one head -------------------------------------------------
        int4 e = *plan;
        int run_end = __shfl_sync(0xffffffffu, e.w, 31);
        while (pos >= run_end && base + 32 < p.batch) {
            base += 32;
            s.piece = piece;
            s.head_set = hs;
            split_load(p, s, base, run_end, false);
            e = make_int4(s.np, s.len, s.vstart, s.vend);
            *plan = e;
            run_end = __shfl_sync(0xffffffffu, e.w, 31);
        }
        const uint32_t ahead = __ballot_sync(0xffffffffu, e.w > pos);
        if (ahead == 0) break;
        const int bl = __ffs(ahead) - 1, b = base + bl;
        const int np = __shfl_sync(0xffffffffu, e.x, bl), rel = pos - __shfl_sync(0xffffffffu, e.z, bl);
        const int len = __shfl_sync(0xffffffffu, e.y, bl);
        int hset, p0, p1;
        if (piece) {
            const int pieces = split_div_up(np, piece);
            hset = split_div(rel, pieces);
            const int j = rel - hset * pieces, size = split_div(np, pieces), more = np - size * pieces;
            p0 = j * size + (j < more ? j : more);
            p1 = p0 + size + (j < more ? 1 : 0);
            pos = hi;
        } else {
            const int item = np + p.item_cost;
            hset = split_div(rel, item);
            const int off = rel - hset * item;
            const int left = hi - pos, rest = item - off;
            const int take = left < rest ? left : rest;
            p0 = off > p.item_cost ? off - p.item_cost : 0;
            p1 = off + take - p.item_cost;
            pos += take;
            if (p1 <= p0) continue;
        }
        const int head = hset * hs + hsub;

        // ---- page ids, the first stages' copies, the queries ------------------------------------------------
        const int n = p1 - p0 > wg ? (p1 - p0 - wg + GW - 1) / GW : 0;      // this warp's pages: p0 + wg + GW i
        const int32_t* ids = p.page_indices + (int64_t)b * p.max_pages + p0 + wg;
        auto fetch_ids = [&](int i) -> int {
            int id = 0;
            if (i + lane < n) {
                id = ids[(i + lane) * GW];
                if ((uint64_t)(int64_t)id >= (uint64_t)p.num_blocks) {       // no address is formed from it: page 0 in its place
                    id = 0;
                    bad_page = true;
                }
            }
            return id;
        };
        int id_now = fetch_ids(0), id_next = n > 32 ? fetch_ids(32) : 0;
        float qv[NT][E];                                                     // this warp's heads wg, wg + 4
#pragma unroll
        for (int i = 0; i < NT; i++)
            if (wg + 4 * i < G) {
                split_load_row<E>(p.q, p.q_dtype, (int64_t)b * p.real_heads + head * G + wg + 4 * i, p.head_dim, lane * E, qv[i]);
            } else {
#pragma unroll
                for (int j = 0; j < E; j++) qv[i][j] = 0.0f;
            }
        const int x = head * p.slot_bytes;
        auto issue = [&](int i, uint32_t to) {       // page i of this warp into stage `to`
            const int id = __shfl_sync(0xffffffffu, id_now, i & 31);
            if (lane == 0 && i < n && !lost) {
                const uint32_t bar = full_at + 8 * to;
                split_expect(bar, kScoredStage);
                scored_box(ring_at + to * kScoredStage, &p.cache_map, x, id * kPageTokens, bar, l2_policy_evict_first());
            }
        };
#pragma unroll
        for (int i = 0; i < kScoredStages - 1; i++) issue(i, stage + i < kScoredStages ? stage + i : stage + i - kScoredStages);
        // Rotated, brought by a power of two to [512, 1024), in two fp16 parts: columns 2 (head % 4), + 1 of tile head / 4, in the order of B fragments.
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float (&v)[E] = qv[t];
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < E; i++) v[i] *= sign_s[lane * E + i];
            split_fwht<E>(v, lane);
#pragma unroll
            for (int i = 0; i < E; i++) {
                v[i] *= p.scale;
                top = fmaxf(top, fabsf(v[i]));
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            // exponents of 2^-110 ... 2^110: the factor and its inverse are normal numbers (anything else is left as it is)
            const int ex = (int)(__float_as_uint(top) >> 23) - 127;
            const int by = ex > -110 && ex < 110 ? 9 - ex : 0;
            const float f = __uint_as_float((uint32_t)(127 + by) << 23);
            if (lane == 0) q_scale_s[gg][4 * t + wg] = __uint_as_float((uint32_t)(127 - by) << 23);
#pragma unroll
            for (int i = 0; i < E / 2; i++) {        // a code byte dequantizes to {low half: odd dim, high half: even dim}
                const float a = v[2 * i + 1] * f, c = v[2 * i] * f;
                const uint32_t hi2 = pack_half2(a, c);
                const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi2));
                const uint32_t lo2 = pack_half2(a - back.x, c - back.y);
                const uint32_t off = (uint32_t)(lane * E + 2 * i) * 2u, q = off / 64, piece16 = off % 64 / 16;
                const uint32_t at = kScoredQ + (uint32_t)gg * 4096u + (4 * t + piece16) * 512u + (2 * wg * 4 + q) * 16u + off % 16;
                *reinterpret_cast<uint32_t*>(at_smem(at)) = hi2;
                *reinterpret_cast<uint32_t*>(at_smem(at + 64)) = lo2;
            }
        }
        group_sync();
        uint32_t qf[NT][16];
        float k_scale[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            k_scale[t] = p.k_scale * q_scale_s[gg][4 * t + tg];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint4 v = lds128(kScoredQ + (uint32_t)gg * 4096u + (4 * t + i) * 512u + 16u * lane);
                qf[t][4 * i] = v.x; qf[t][4 * i + 1] = v.y; qf[t][4 * i + 2] = v.z; qf[t][4 * i + 3] = v.w;
            }
        }

        // ---- pages -----------------------------------------------------------------------------------------
        float o_acc[8][4], m[NT], l[NT], v_scale = kVScaleStart;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) o_acc[i][j] = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            m[t] = kNoMax;
            l[t] = 0.0f;
        }
        float* const logits = sp.logits + ((int64_t)b * p.kv_heads + head) * sp.room * G + tg;
        int left = len - (p0 + wg) * kPageTokens;                       // tokens from this warp's page on
        for (int it = 0; it < n; it++, left -= GW * kPageTokens) {
            const int ahead_i = it + kScoredStages - 1;
            if ((ahead_i & 31) == 0) {          // the ids of the next 32 pages, and the load of those after them
                id_now = id_next;
                id_next = ahead_i + 32 < n ? fetch_ids(ahead_i + 32) : 0;
            }
            issue(ahead_i, stage == 0 ? kScoredStages - 1 : stage - 1);
            if (!lost) {
                bool there = false;
                for (uint32_t i = 0; i < kSpinLimit && !there; i++) there = split_try_wait(full_at + 8 * stage, parity);
                if (!__all_sync(0xffffffffu, there)) {
                    lost = true;      // the heads from here on are void; what is still in flight gets its time to land
                    if (lane == 0) atomicAdd(&g_scored_faults, 1);
                    for (uint32_t k = 1; k < kScoredStages; k++) {
                        const bool wraps = stage + k >= kScoredStages;
                        for (uint32_t i = 0; i < kSpinLimit / 64; i++)
                            if (split_try_wait(full_at + 8 * (wraps ? stage + k - kScoredStages : stage + k), wraps ? parity ^ 1 : parity)) break;
                    }
                }
            }
            __syncwarp();
            const uint32_t st = stage * kScoredStage;
            uint32_t v0[2], v1[2], v2[2], v3[2], ka[4], kb[4];
            split_lds<8>(v_at + st, v0);
            split_lds<8>(v_at + st + kScoredRow, v1);
            split_lds<8>(v_at + st + 8 * kScoredRow, v2);
            split_lds<8>(v_at + st + 9 * kScoredRow, v3);
            split_lds<16>(k_at + st, ka);
            split_lds<16>(k_at + st + 8 * kScoredRow, kb);
            // Sums of both tables: apart with one tile, whose chain of products would be twice as long, together with two, for the registers.
            float acc[2][4];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[t][i] = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                uint32_t ra[4], rb[4], la[4], lb[4];
                scored_lookup(ka[w], lut_lane, ra, la);
                scored_lookup(kb[w], lut_lane, rb, lb);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    float (&hi_acc)[4] = acc[t], (&lo_acc)[4] = acc[NT == 1 ? 1 : t];
                    mma16816(hi_acc, ra[0], rb[0], ra[1], rb[1], qf[t][4 * w], qf[t][4 * w + 1]);
                    mma16816(lo_acc, la[0], lb[0], la[1], lb[1], qf[t][4 * w], qf[t][4 * w + 1]);
                    mma16816(hi_acc, ra[2], rb[2], ra[3], rb[3], qf[t][4 * w + 2], qf[t][4 * w + 3]);
                    mma16816(lo_acc, la[2], lb[2], la[3], lb[3], qf[t][4 * w + 2], qf[t][4 * w + 3]);
                }
            }
            float na = lds_half(kn_at + st), nb = lds_half(kn_at + st + 8 * kScoredRow);
            float vfa = lds_half(vn_at + st) * v_scale, vfb = lds_half(vn_at + st + 8 * kScoredRow) * v_scale;
            float bias_a = 0.0f, bias_b = 0.0f;
            if (left < kPageTokens) {            // past the sequence's end: whatever the slots contain
                if (ta >= left) { na = 0.0f; vfa = 0.0f; bias_a = -INFINITY; }
                if (tb >= left) { nb = 0.0f; vfb = 0.0f; bias_b = -INFINITY; }
            }
            float xa[NT], xb[NT];                // logits of tokens ta, tb under head 4 t + tg
            bool over = fmaxf(fabsf(vfa), fabsf(vfb)) > kVNormMost;
            float* const to = logits + (int64_t)(len - left) * G;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                float a = acc[t][0] + acc[t][1], b = acc[t][2] + acc[t][3];
                if constexpr (NT == 1) {
                    a += acc[1][0] + acc[1][1];
                    b += acc[1][2] + acc[1][3];
                }
                xa[t] = fmaf(a, na * k_scale[t], bias_a);
                xb[t] = fmaf(b, nb * k_scale[t], bias_b);
                over |= fmaxf(xa[t], xb[t]) > m[t] + kRaiseThreshold;
                if (4 * t + tg < G) {
                    if (ta < left) to[ta * G + 4 * t] = xa[t];
                    if (tb < left) to[tb * G + 4 * t] = xb[t];
                }
            }
            // ---- online softmax (base 2), the maximum raised only when a logit exceeds it by kRaiseThreshold, and the V norms' scale
            // lowered when P times a norm could leave fp16
            if (__any_sync(0xffffffffu, over)) {
                float f = 1.0f, top = fmaxf(fabsf(vfa), fabsf(vfb));
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                // to [256, 512); a warp's first page sets the scale
                if (top > kVNormMost || (it == 0 && top > 0.0f)) f = __uint_as_float((127 + 8 + 127 - (__float_as_uint(top) >> 23)) << 23);
                vfa *= f;
                vfb *= f;
                v_scale *= f;
                float c[NT];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    float mx = fmaxf(xa[t], xb[t]);
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    const bool raise = mx > m[t] + kRaiseThreshold;
                    c[t] = raise ? fast_exp2(m[t] - mx) : 1.0f;
                    if (raise) m[t] = mx;
                    l[t] *= c[t];
                }
                const float f0 = f * c[0], f1 = f * c[NT - 1];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    o_acc[i][0] *= f0; o_acc[i][1] *= f1; o_acc[i][2] *= f0; o_acc[i][3] *= f1;
                }
            }
            uint32_t pa, pb;
            if constexpr (NT == 1) {             // columns 2 tg, + 1: the two parts of head tg
                const float ea = fast_exp2(xa[0] - m[0]), eb = fast_exp2(xb[0] - m[0]);
                l[0] += ea + eb;
                const float wa = ea * vfa, wb = eb * vfb;
                const float ha = __half2float(__float2half_rn(wa)), hb = __half2float(__float2half_rn(wb));
                pa = pack_half2(wa, wa - ha);
                pb = pack_half2(wb, wb - hb);
            } else {                             // columns 2 tg, + 1: heads tg, 4 + tg
                const float e0 = fast_exp2(xa[0] - m[0]), e1 = fast_exp2(xa[1] - m[1]), e2 = fast_exp2(xb[0] - m[0]), e3 = fast_exp2(xb[1] - m[1]);
                l[0] += e0 + e2;
                l[1] += e1 + e3;
                pa = pack_half2(e0 * vfa, e1 * vfa);
                pb = pack_half2(e2 * vfb, e3 * vfb);
            }
            pa = movmatrix_trans(pa);
            pb = movmatrix_trans(pb);
            // ---- O^T += V^^T P: V^ rows g <- odd dim, g + 8 <- even dim of code byte 4 w + j of four tokens
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const uint32_t lo01 = (v0[w] & 0x0F0F0F0Fu) | ((v1[w] << 4) & 0xF0F0F0F0u), hi01 = ((v0[w] >> 4) & 0x0F0F0F0Fu) | (v1[w] & 0xF0F0F0F0u);
                const uint32_t lo23 = (v2[w] & 0x0F0F0F0Fu) | ((v3[w] << 4) & 0xF0F0F0F0u), hi23 = ((v2[w] >> 4) & 0x0F0F0F0Fu) | (v3[w] & 0xF0F0F0F0u);
                uint32_t a0[4], a1[4], a2[4], a3[4];
                dequant8(lo01, lut_lane, a0);
                dequant8(hi01, lut_lane, a1);
                dequant8(lo23, lut_lane, a2);
                dequant8(hi23, lut_lane, a3);
#pragma unroll
                for (int j = 0; j < 4; j++) mma16816(o_acc[4 * w + j], a0[j], a1[j], a2[j], a3[j], pa, pb);
            }
            __syncwarp();      // every lane has read the stage before a later iteration copies into it
            if (++stage == kScoredStages) {
                stage = 0;
                parity ^= 1;
            }
        }

        // ---- combine the group's warps ------------------------------------------------------------------------
        if (lost) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
                m[t] = kScoredVoid;
                l[t] = INFINITY;
            }
            v_scale = NAN;
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[t] += __shfl_xor_sync(0xffffffffu, l[t], o);
            if (g == 0) {
                m_s[gg][wg][4 * t + tg] = m[t];
                l_s[gg][wg][4 * t + tg] = l[t];
            }
        }
        if (lane == 0) v_s[gg][wg] = p.v_scale / v_scale;
        __syncwarp();
        // rows of PD floats in the warp's own ring; the 16-byte pieces of a row are swapped by the head (banks)
        float* const mine = reinterpret_cast<float*>(at_smem(ring_at));
        if (n > 0) {
#pragma unroll
            for (int w = 0; w < 4; w++) {      // dims d ... d + 3
                const int at = 4 * ((4 * g + w) ^ tg);
                const float(&a)[4] = o_acc[2 * w], (&c)[4] = o_acc[2 * w + 1];
                if constexpr (NT == 1) {
                    *reinterpret_cast<float4*>(mine + tg * PD + at) = make_float4(a[2] + a[3], a[0] + a[1], c[2] + c[3], c[0] + c[1]);
                } else {
                    *reinterpret_cast<float4*>(mine + tg * PD + at) = make_float4(a[2], a[0], c[2], c[0]);
                    *reinterpret_cast<float4*>(mine + (4 + tg) * PD + at) = make_float4(a[3], a[1], c[3], c[1]);
                }
            }
        }
        group_sync();
        const bool whole = p0 == 0 && p1 == np;
        const int slot = (worker * 2 + (p0 == 0 ? 1 : 0)) * hs + hsub;
        for (int r = wg; r < G; r += GW) {
            float mm = kNoMax, ll = 0.0f, o[E];
            const int warps = min(GW, p1 - p0);            // the others had no page
#pragma unroll
            for (int i = 0; i < E; i++) o[i] = 0.0f;
            for (int w = 0; w < warps; w++) mm = fmaxf(mm, m_s[gg][w][r]);
            for (int w = 0; w < warps; w++) {
                const float cl = fast_exp2(m_s[gg][w][r] - mm), c = cl * v_s[gg][w];
                ll += cl * l_s[gg][w][r];
                const float4 t = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(at_smem(ring_of(gg * GW + w))) + r * PD + 4 * (lane ^ (r & 3)));
                o[0] += c * t.x; o[1] += c * t.y; o[2] += c * t.z; o[3] += c * t.w;
            }
            const float inv = ll == 0.0f ? 0.0f : 1.0f / ll, lse2 = ll == 0.0f ? -INFINITY : mm + log2f(ll);
#pragma unroll
            for (int i = 0; i < E; i++) o[i] *= inv;
            if (whole) {
                if (lane == 0) sp.row_lse[((int64_t)b * p.kv_heads + head) * G + r] = lse2;
                split_finish<PD>(p, sign_s, b, head, r, o, lse2, lane);
            } else {
                const int64_t at = (int64_t)slot * G + r;
                *reinterpret_cast<float4*>(p.partial_o + at * PD + lane * E) = make_float4(o[0], o[1], o[2], o[3]);
                if (lane == 0) p.partial_lse[at] = lse2;
            }
        }
        if (pos < hi) {
            fence_proxy_async();       // the ring was written and read as rows
            group_sync();              // rings and query rows are free again
        }
    }
    if (bad_page) atomicAdd(&g_scored_faults, 1);
}

// Joins the partials of the heads that were cut and adds the weights to the scores.  A block takes every chunks-th run of 256 tokens of one (sequence, KV
// head): it works out the lse of the head's rows from the partials (they are few), writes the output rows r = chunk, chunk + chunks, ... , and
// goes over its tokens' logits.
constexpr int kJoinThreads = 256, kJoinAhead = 4;
__global__ void __launch_bounds__(kJoinThreads) scored_join_kernel(const __grid_constant__ ScoredParams sp) {
    constexpr int PD = kHeadDim, E = PD / 32, kWarps = kJoinThreads / 32;
    const SplitParams& p = sp.d;
    __shared__ float acc_s[kWarps][PD], sign_s[PD], lse_s[8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = p.group;
    grid_launch_dependents();
    const int bh = blockIdx.x / sp.chunks, chunk = blockIdx.x - bh * sp.chunks, b = bh / p.kv_heads, head = bh - b * p.kv_heads;
    for (int i = tid; i < PD; i += kJoinThreads) sign_s[i] = p.signs[i];
    grid_dependency_wait();
    const int given = p.seq_lens[b];
    SplitPlan s;
    int np, vstart;
    if (p.batch > kSplitSelf) {
        split_kept_plan(p, s, lane);
        split_jump(p, s, b / (32 * split_bin(p)));
        while (s.base + 32 <= b) split_load(p, s, s.base + 32, __shfl_sync(0xffffffffu, s.vend, 31), false);
        np = __shfl_sync(0xffffffffu, s.np, (b - s.base) & 31);
        vstart = __shfl_sync(0xffffffffu, s.vstart, (b - s.base) & 31);
    } else {
        const int2 place = sp.plan[b];
        np = place.x;
        vstart = place.y;
        s.total = p.header[1];
        s.workers = p.header[2];
        s.piece = p.header[3];
        s.head_set = s.piece ? 1 : p.head_set;
    }
    const int hs = s.head_set, hset = head / hs, hsub = head - hset * hs;
    int first = 0, count = 0;           // workers of this head's parts
    if (np > 0 && s.total > 0) {
        if (s.piece) {
            count = split_div_up(np, s.piece);
            first = vstart + hset * count;
        } else {
            const int64_t at = vstart + (int64_t)hset * (np + p.item_cost) + p.item_cost, end = at + np;
            first = (int)(((at + 1) * s.workers + s.total - 1) / s.total) - 1;
            count = (int)((end * s.workers + s.total - 1) / s.total) - first;
        }
    }
    // (a list without work although there are tokens: nothing was computed)
    const bool fits = given <= sp.score_room && (given <= 0 || s.total > 0) && np == (given > 0 ? (given + kPageTokens - 1) / kPageTokens : 0) && given >= 0;
    if (!fits && head == 0 && chunk == 0 && tid == 0) atomicAdd(&g_scored_faults, 1);
    // The first tokens' logits and scores are on their way while the lse is worked out.
    const int64_t step = (int64_t)sp.chunks * kJoinThreads, t_first = (int64_t)chunk * kJoinThreads + tid;
    float* const score = sp.scores + b * sp.score_b + head * sp.score_h;
    const float* const logits = sp.logits + (int64_t)bh * sp.room * G;
    const int64_t old_end = (int64_t)given - sp.new_tokens;
    float4 v[kJoinAhead];
    float old[kJoinAhead];
    auto fetch = [&](int64_t t0) {
#pragma unroll
        for (int u = 0; u < kJoinAhead; u++) {
            const int64_t t = t0 + step * u;
            if (G == 4) v[u] = t < given ? *reinterpret_cast<const float4*>(logits + t * 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            old[u] = t < old_end ? score[t] : 0.0f;
        }
    };
    if (fits) fetch(t_first);
    auto slot_row = [&](int i, int r) -> int64_t { return ((int64_t)((first + i) * 2 + (i == 0 ? 1 : 0)) * hs + hsub) * G + r; };
    bool gone = false;
    for (int r = warp; r < G; r += kWarps) {
        float lse = -INFINITY;
        if (count == 1) {
            lse = sp.row_lse[(int64_t)bh * G + r];
        } else if (count > 1) {
            float top = -INFINITY, sum = 0.0f;
            for (int i = lane; i < count; i += 32) top = fmaxf(top, p.partial_lse[slot_row(i, r)]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (top == -INFINITY) top = 0.0f;
            for (int i = lane; i < count; i += 32) sum += fast_exp2(p.partial_lse[slot_row(i, r)] - top);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            lse = sum == 0.0f ? -INFINITY : top == INFINITY ? top : top + log2f(sum);
        }
        gone |= lse == INFINITY;
        if (lane == 0) lse_s[r] = lse;
    }
    gone = __syncthreads_or(gone);
    if (count != 1) {
        for (int r = chunk; r < G; r += sp.chunks) {
            const float lse = lse_s[r];
            float acc[E] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (lse != -INFINITY) {
                for (int i = warp; i < count; i += kWarps) {
                    const int64_t at = slot_row(i, r);
                    const float w = fast_exp2(p.partial_lse[at] - lse);
                    const float4 t = *reinterpret_cast<const float4*>(p.partial_o + at * PD + lane * E);
                    acc[0] = fmaf(w, t.x, acc[0]); acc[1] = fmaf(w, t.y, acc[1]); acc[2] = fmaf(w, t.z, acc[2]); acc[3] = fmaf(w, t.w, acc[3]);
                }
            }
            *reinterpret_cast<float4*>(&acc_s[warp][lane * E]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            __syncthreads();
            if (warp == 0) {
#pragma unroll
                for (int w = 1; w < kWarps; w++) {
                    const float4 t = *reinterpret_cast<const float4*>(&acc_s[w][lane * E]);
                    acc[0] += t.x; acc[1] += t.y; acc[2] += t.z; acc[3] += t.w;
                }
                split_finish<PD>(p, sign_s, b, head, r, acc, lse, lane);
            }
            __syncthreads();
        }
    }
    if (!fits || gone) return;          // (void rows have no weights: the scores, which outlast the call, stay as they are)
    float lse[8];
#pragma unroll
    for (int r = 0; r < 8; r++) lse[r] = r < G && lse_s[r] != -INFINITY ? lse_s[r] : INFINITY;      // a row without a weight: exp2(x - inf) = 0
    for (int64_t t0 = t_first; t0 < given; t0 += step * kJoinAhead) {
        float w[kJoinAhead];
        if (t0 != t_first) fetch(t0);
        if (G == 4) {
#pragma unroll
            for (int u = 0; u < kJoinAhead; u++)
                w[u] = (fast_exp2(v[u].x - lse[0]) + fast_exp2(v[u].y - lse[1])) + (fast_exp2(v[u].z - lse[2]) + fast_exp2(v[u].w - lse[3]));
        } else {
            float x[kJoinAhead][8];
#pragma unroll
            for (int u = 0; u < kJoinAhead; u++)
#pragma unroll
                for (int r = 0; r < 8; r++) x[u][r] = r < G && t0 + step * u < given ? logits[(t0 + step * u) * G + r] : 0.0f;
#pragma unroll
            for (int u = 0; u < kJoinAhead; u++) {
                w[u] = 0.0f;
#pragma unroll
                for (int r = 0; r < 8; r++)
                    if (r < G) w[u] += fast_exp2(x[u][r] - lse[r]);
            }
        }
#pragma unroll
        for (int u = 0; u < kJoinAhead; u++)
            if (t0 + step * u < given) score[t0 + step * u] = old[u] + w[u];
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
int device_sm_count(int* out);
int encode_cache_map(CUtensorMap* map, const void* kv_cache, int64_t num_blocks, int64_t row_bytes, int box_bytes, int slabs);

static size_t scored_up(size_t x) { return (x + 255) & ~(size_t)255; }

int scored_fault_count(int32_t* out) {
    TQ_CUDA(cudaMemcpyFromSymbol(out, g_scored_faults, sizeof(int32_t)));
    return TQ_OK;
}

struct ScoredLayout {
    size_t plan, partial_lse, partial_o, row_lse, logits, end;
};
static ScoredLayout scored_layout(int batch, int heads, int kv_heads, int64_t max_pages, int ctas) {
    const size_t G = (size_t)(heads / kv_heads), rows = (size_t)2 * ctas * kScoredGroups * G;
    ScoredLayout l;
    l.plan = 256;
    l.partial_lse = l.plan + scored_up((size_t)kSplitSelf * sizeof(int2));
    l.partial_o = l.partial_lse + scored_up(rows * 4);
    l.row_lse = l.partial_o + scored_up(rows * kHeadDim * 4);
    l.logits = l.row_lse + scored_up((size_t)batch * heads * 4);
    l.end = l.logits + scored_up((size_t)batch * heads * (size_t)max_pages * kPageTokens * 4);
    return l;
}

template <int NT, bool MANY>
static int launch_scored_kernel(const ScoredParams& p, cudaStream_t s) {
    static bool configured[64] = {};
    int dev = 0;
    TQ_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        TQ_CUDA(cudaFuncSetAttribute(decode_scored_kernel<NT, MANY>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kScoredSmem));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    TQ_CUDA(launch_serialized(decode_scored_kernel<NT, MANY>, dim3((unsigned)p.d.grid), dim3(kScoredThreads), kScoredSmem, s, p));
    return TQ_OK;
}

}  // namespace tq

extern "C" int tq_scored_lose_copies(int on) {
    tq::g_scored_lose = on != 0;
    return TQ_OK;
}

extern "C" size_t tq_decode_scored_workspace_bytes(int batch, int num_q_heads, int num_kv_heads, int max_pages) {
    int sms = 0;
    if (batch < 1 || num_kv_heads < 1 || num_q_heads < num_kv_heads || max_pages < 1 || tq::device_sm_count(&sms) != TQ_OK) return 0;
    return tq::scored_layout(batch, num_q_heads, num_kv_heads, max_pages, sms).end;
}

extern "C" int tq_decode_scored(const void* q, int q_dtype, int batch, int num_q_heads, int num_kv_heads, int head_dim, const void* kv_cache,
                                int64_t num_blocks, int block_size, int slot_bytes, const int32_t* page_table, int max_pages, const int32_t* seq_lens,
                                const float* signs, float sm_scale, float* scores, int64_t score_batch_stride, int64_t score_head_stride, int score_tokens,
                                int new_tokens, void* workspace, size_t workspace_bytes, void* out, int out_dtype, float* out_lse, void* stream) {
    using namespace tq;
    TQ_REQUIRE(batch >= 0 && num_blocks >= 0, TQ_ERR_INVALID, "negative size");
    if (batch == 0) return TQ_OK;
    TQ_REQUIRE(q && kv_cache && page_table && seq_lens && signs && scores && workspace && out, TQ_ERR_INVALID, "null pointer");
    TQ_REQUIRE(q_dtype >= TQ_F32 && q_dtype <= TQ_BF16 && out_dtype >= TQ_F32 && out_dtype <= TQ_BF16, TQ_ERR_INVALID, "unknown dtype");
    TQ_REQUIRE(head_dim > 64 && head_dim <= 128, TQ_ERR_UNSUPPORTED, "head_dim must be in 65 ... 128, got %d", head_dim);
    TQ_REQUIRE(block_size == 16 && slot_bytes == kSlotBytes, TQ_ERR_UNSUPPORTED, "16-token pages of 80-byte slots only, got %d and %d", block_size, slot_bytes);
    TQ_REQUIRE(num_kv_heads >= 1 && num_q_heads >= 1 && num_q_heads % num_kv_heads == 0, TQ_ERR_INVALID, "%d query heads on %d KV heads", num_q_heads, num_kv_heads);
    const int G = num_q_heads / num_kv_heads;
    TQ_REQUIRE(G <= 8, TQ_ERR_UNSUPPORTED, "at most 8 query heads per KV head, got %d", G);
    TQ_REQUIRE(max_pages >= 1 && max_pages <= 1 << 26 && score_tokens >= 0 && new_tokens >= 0, TQ_ERR_INVALID, "bad size");
    TQ_REQUIRE(score_batch_stride >= 0 && score_head_stride >= 0, TQ_ERR_INVALID, "negative stride");
    const int64_t most = (int64_t)max_pages * kPageTokens < score_tokens ? (int64_t)max_pages * kPageTokens : score_tokens;
    TQ_REQUIRE(!rows_overlap(batch, num_kv_heads, score_batch_stride, score_head_stride, most), TQ_ERR_INVALID, "the rows of scores overlap");
    TQ_REQUIRE(((uintptr_t)kv_cache & 15) == 0 && ((uintptr_t)workspace & 255) == 0, TQ_ERR_INVALID, "kv_cache must be 16-byte aligned, the workspace 256-byte");
    TQ_REQUIRE((int64_t)batch * num_q_heads < 1 << 24, TQ_ERR_UNSUPPORTED, "too many rows for one launch");
    int sms = 0;
    int rc = device_sm_count(&sms);
    if (rc != TQ_OK) return rc;
    const ScoredLayout lay = scored_layout(batch, num_q_heads, num_kv_heads, max_pages, sms);
    TQ_REQUIRE(workspace_bytes >= lay.end, TQ_ERR_WORKSPACE, "workspace too small: %zu < %zu", workspace_bytes, lay.end);

    ScoredParams sp{};
    SplitParams& p = sp.d;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.q = q;
    p.kv_cache = static_cast<const uint8_t*>(kv_cache);
    p.page_indices = page_table;
    p.seq_lens = seq_lens;
    p.signs = signs;
    p.header = reinterpret_cast<int32_t*>(ws);
    p.partial_lse = reinterpret_cast<float*>(ws + lay.partial_lse);
    p.partial_o = reinterpret_cast<float*>(ws + lay.partial_o);
    p.out = out;
    p.out_lse = out_lse;
    p.num_blocks = num_blocks;
    p.kv_end = -1;
    p.batch = batch;
    p.kv_heads = num_kv_heads;
    p.group = p.real_group = G;
    p.nq = 1;
    p.real_heads = num_q_heads;
    p.max_pages = max_pages;
    p.q_dtype = q_dtype;
    p.out_dtype = out_dtype;
    p.head_dim = head_dim;
    p.slot_bytes = slot_bytes;
    p.grid = sms;
    p.head_set = num_kv_heads % 4 == 0 ? 4 : num_kv_heads % 2 == 0 ? 2 : 1;
    p.head_sets = num_kv_heads / p.head_set;
    p.item_cost = kScoredItemCost;
    p.inv_warps = 1.0f / (float)(sms * kScoredWarps);
    const double inv = 1.0 / std::sqrt((double)kHeadDim);
    p.scale = (float)inv;
    for (int k = 0; k < 16; k++) {
        const double c = kLevelScale * kCentroidsN01_4bit[k];
        const __half h = __float2half_rn((float)c), r = __float2half_rn((float)(c - (double)__half2float(h)));
        memcpy(&p.centroid_h[k], &h, 2);
        memcpy(&sp.rest_h[k], &r, 2);
    }
    p.v_scale = (float)(inv / kLevelScale);
    p.k_scale = (float)(inv / kLevelScale * (double)sm_scale * 1.4426950408889634);
    sp.logits = reinterpret_cast<float*>(ws + lay.logits);
    sp.plan = reinterpret_cast<int2*>(ws + lay.plan);
    sp.row_lse = reinterpret_cast<float*>(ws + lay.row_lse);
    sp.scores = scores;
    sp.score_b = score_batch_stride;
    sp.score_h = score_head_stride;
    sp.room = (int64_t)max_pages * kPageTokens;
    sp.score_room = score_tokens;
    sp.new_tokens = new_tokens;
    sp.lose = g_scored_lose;
    // A block of the join for every 256 tokens, up to eight an SM in all (and one a row at least).
    const int64_t runs = (most + kJoinThreads - 1) / kJoinThreads, fit = (int64_t)8 * sms / ((int64_t)batch * num_kv_heads);
    sp.chunks = (int)(runs < 1 ? 1 : runs < (fit > 1 ? fit : 1) ? runs : (fit > 1 ? fit : 1));
    rc = encode_cache_map(&p.cache_map, kv_cache, num_blocks, (int64_t)num_kv_heads * slot_bytes, kScoredRow, 2);
    if (rc != TQ_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool many = batch > kSplitSelf;
    if (G <= 4) rc = many ? launch_scored_kernel<1, true>(sp, s) : launch_scored_kernel<1, false>(sp, s);
    else rc = many ? launch_scored_kernel<2, true>(sp, s) : launch_scored_kernel<2, false>(sp, s);
    if (rc != TQ_OK) return rc;
    TQ_CUDA(launch_serialized(scored_join_kernel, dim3((unsigned)(batch * num_kv_heads * sp.chunks)), dim3(kJoinThreads), 0, s, sp));
    return TQ_OK;
}
