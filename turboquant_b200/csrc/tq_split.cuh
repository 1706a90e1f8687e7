// Pieces shared by the kernels that split a decode over (sequence, KV head, page range): the launch parameters, the plan that both a decode
// kernel and the kernel that joins its partials make on the device, and the helpers of a warp that works on pages of one head.
#pragma once

#include <cuda.h>  // CUtensorMap only

#include "tq_decode_common.cuh"

namespace tq {

struct SplitParams {
    alignas(64) CUtensorMap cache_map;   // uint8 [2][num_blocks * 16][H * slot], boxes of [kSlabs][16][kRow]
    const void* q;
    const uint8_t* kv_cache;
    const int32_t* page_indices;
    const int32_t* page_indptr;
    const int32_t* seq_lens;
    const float* signs;
    int32_t* header;        // workspace word 0: sticky status
    float* partial_lse;     // [2 x groups of the grid][group columns], base 2
    float* partial_o;       // [2 x groups of the grid][group columns][PD], normalized, rotated domain
    void* out;
    float* out_lse;
    int64_t num_blocks, kv_begin, kv_end;
    int batch, kv_heads, group, max_pages, q_dtype, out_dtype, emit_rotated;
    int nq, real_heads, real_group, head_dim, slot_bytes;
    int causal;             // query i of nq sees the first len - (nq - 1 - i) tokens
    int grid, head_set, head_sets;   // blocks of the decode launch; heads side by side in a block when the work is cut evenly, and kv_heads / head_set
    int item_cost;          // virtual pages that starting an item is worth (SplitShape::kItemCost)
    float inv_warps;        // 1 / warps of the grid
    int all_or_nothing;     // a sequence longer than its table empties the whole batch (128-wide heads), or only itself
    float k_scale, v_scale, scale;
    uint16_t centroid_h[16];
};

// ---------------------------------------------------------------------------------------------
// The plan: which (sequence, head, page range) a worker takes, and which workers a head's partials come from.  Both kernels
// compute it from seq_lens, every warp for itself: a lane holds one sequence of a batch of 32.
//   pieces: every head is cut into equal pieces of at most kGroupWarps x `tiles` pages, with the smallest number of tiles (pages per
//           warp) for which all pieces fit the groups of the grid; a worker is a group and takes one piece.  One start and one combine per
//           group, and a head that fits a piece is not cut at all; but the pieces of a ragged batch are of many sizes.
//   even:   the list of all pages (sequence, head set, page) is cut into equal ranges, one per worker and none of them empty, with
//           item_cost virtual pages in front of every item for what starting it costs (queries to rotate, a combine).  The head_set groups of a worker
//           take neighbouring heads of the same pages, so that the slots they read share their DRAM lines.
// Pieces are taken when their tiles exceed the even share by at most kSplitSlackTiles (about what a second start costs a group).
// ---------------------------------------------------------------------------------------------
constexpr int kSplitSlackTiles = 3;
// The running maximum before any score: finite, so that a column whose tokens are all masked so far has exp2(-inf - m) = 0.
constexpr float kNoMax = -3.402823466e38f;
// P times the V norm is rounded to fp16 as the MMA's operand; 1 / sqrt(128) is taken out in fp32 at the combine (ahead of the rounding it cost V rows of
// norm 1e-3 under 16 ... 32 causal columns 7 ... 8.7e-4 of error against 64 bits, now 4.9e-4 at any norm).  Norms are any fp16 value; a
// page whose largest exceeds kVNormMost (2^kRaiseThreshold times that is still finite in fp16) would overflow.
//   One column tile of padded size 64 / 128: that page's norms are brought to [256, 512) and the accumulators scaled down and up again around
//   it, so that other pages pay a maximum and a comparison (head size 64, 22 x 14327: 67 us as with a fixed scale, 75 with the one below).
//   Else: the warp keeps a power of two for the norms, 16 at first, and lowers it with the accumulators; a word in shared memory, for a register
//   more spills, and so does the code of the other form (8 x 32768 causal, 8 queries 162.6 us with a fixed scale, 163.2 so, 166 the other
//   way; one sequence of 1048576 567 / 577 / 587; head size 256, 1 x 1917 13.0 / 13.3 / 13.4).
constexpr float kVNormMost = 1000.0f, kVScaleStart = 16.0f;

// n / d for 0 <= n < 2^24, d > 0: a reciprocal, then the quotient put right.  (The plan is repeated by every warp, and the compiler's
// division is three times as long.)
__device__ __forceinline__ int split_div(int n, int d) {
    int q = (int)((float)n * __frcp_rn((float)d));
    const int r = n - q * d;
    q += r >= d ? 1 : r < 0 ? -1 : 0;
    return q;
}
// ceil(n / d), as above
__device__ __forceinline__ int split_div_up(int n, int d) { return split_div(n + d - 1, d); }

// the list position where worker c's range begins: c total / workers
__device__ __forceinline__ int split_cut(int c, int total, int workers) {
    if (total < (1 << 20) && workers < (1 << 12)) return (int)((uint32_t)c * (uint32_t)total / (uint32_t)workers);
    return (int)((int64_t)c * total / workers);
}

struct SplitPlan {
    int lane, base;          // this batch of 32 starts at sequence `base`
    int np, len;             // the lane's sequence: pages inside the window, tokens up to the window's end
    int vstart, vend;        // its span in the list, in units of pieces or of virtual pages (even)
    int run;                 // end of the span of the last sequence before this batch
    int ends;                // of many sequences: the list position where the lane's bin of them ends
    int total, workers, head_set;
    int piece;               // pages of a piece at most, 0: the even cut
    bool too_long;           // some sequence is longer than its page table
    bool void_batch;         // ... and that empties the batch
};

__device__ __forceinline__ int split_pages(const SplitParams& p, int b, int& len_out, bool& too_long) {
    int64_t len = p.seq_lens[b];
    if (p.kv_end >= 0 && p.kv_end < len) len = p.kv_end;
    const int first = (int)(p.kv_begin / kPageTokens);
    const int64_t last = (len + kPageTokens - 1) / kPageTokens;
    len_out = (int)len;
    int np = last > first ? (int)(last - first) : 0;
    const int have = p.page_indptr ? p.page_indptr[b + 1] - p.page_indptr[b] : p.max_pages;
    if (np > 0 && first + np > have) {
        too_long = true;
        np = 0;
    }
    return np;
}

__device__ __forceinline__ void split_load(const SplitParams& p, SplitPlan& s, int base, int run, bool keep) {
    bool dummy = false;
    if (!keep) {
        s.np = 0;
        if (base + s.lane < p.batch && !s.void_batch) s.np = split_pages(p, base + s.lane, s.len, dummy);
    }
    s.base = base;
    s.run = run;
    int v = 0;
    if (s.np > 0) v = s.piece ? p.kv_heads * split_div_up(s.np, s.piece) : p.head_sets * (s.np + p.item_cost);
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, o);
        if (s.lane >= o) incl += t;
    }
    s.vstart = run + incl - v;
    s.vend = run + incl;
}

// The cut of a work list of `pages` pages in `nonempty` sequences (and, in pieces, the piece and their number).
template <int NG>
__device__ __forceinline__ void split_cut_list(const SplitParams& p, SplitPlan& s, int pages, int nonempty, int pieces) {
    s.head_set = s.piece ? 1 : p.head_set;
    s.workers = p.grid * (s.head_set == 1 ? NG : s.head_set == 2 ? NG / 2 : NG / 4);
    s.total = s.piece ? pieces * p.kv_heads : p.head_sets * (pages + nonempty * p.item_cost);
    // Every worker of the even cut has a position of the list: one with an empty range would write no partial, and the merge counts
    // all workers between a head's first and last as its parts.  (A short list is cut too: many sequences of which few hold tokens.)
    if (!s.piece && s.workers > s.total) s.workers = s.total;
}
// Up to kSplitSelf sequences: every warp of both kernels plans for itself, and walks the list a batch of 32 at a time.
constexpr int kSplitSelf = 64;
template <int GW, int NG>
__device__ __forceinline__ void split_plan(const SplitParams& p, SplitPlan& s, int lane) {
    s.lane = lane;
    s.too_long = s.void_batch = false;
    s.len = 0;
    int pages = 0, nonempty = 0, np_first = 0, len_first = 0;
    for (int base = 0; base < p.batch; base += 32) {
        int np = 0, len = 0;
        if (base + lane < p.batch) np = split_pages(p, base + lane, len, s.too_long);
        if (base == 0) { np_first = np; len_first = len; }
        nonempty += __popc(__ballot_sync(0xffffffffu, np > 0));
        pages += __reduce_add_sync(0xffffffffu, np);
    }
    s.too_long = __any_sync(0xffffffffu, s.too_long);
    s.void_batch = s.too_long && p.all_or_nothing;
    if (s.void_batch) pages = nonempty = np_first = 0;
    s.np = np_first;
    s.len = len_first;
    // the smallest number of tiles whose pieces fit, from the even share on
    const int groups = p.grid * NG;
    const float even = (float)pages * (float)p.kv_heads * p.inv_warps;     // pages per warp (rounding it either way is fine)
    const int share = (int)even + (even > (float)(int)even ? 1 : 0);
    s.piece = 0;
    int pieces = 0;
    for (int t = share < 1 ? 1 : share; t <= share + kSplitSlackTiles; t++) {
        const int size = t * GW;
        pieces = __reduce_add_sync(0xffffffffu, split_div_up(np_first, size));
        for (int base = 32; base < p.batch && !s.void_batch; base += 32) {
            int len;
            bool dummy;
            const int np = base + lane < p.batch ? split_pages(p, base + lane, len, dummy) : 0;
            pieces += __reduce_add_sync(0xffffffffu, split_div_up(np, size));
        }
        if (pieces * p.kv_heads <= groups) {
            s.piece = size;
            break;
        }
    }
    split_cut_list<NG>(p, s, pages, nonempty, pieces);
    split_load(p, s, 0, 0, true);
}

// More sequences: the decode kernel's warps load the lengths of 256 at a time and remember where each of up to 32 bins of sequences ends in the list (a
// bin is one batch of 32, or as many as make 32 bins do), to find their place in one step.  Up to 256 may be cut in pieces (beyond that it measured slower: 512 of 2048
// tokens, ragged, 8 heads on one 29 -> 41 us).  The merge,
// whose blocks are more than fit the chip at once, reads this plan from the workspace (words 1 ... 4 and 8 ... 39) after its wait.
// The plan above costs a warp two trips over the lengths and half of a third one, in every block of the merge too: 8 heads on one, head size 64, 1000
// sequences of 500 tokens 75 -> 42 us with this one, 2000 of 64 157 -> 52; 64 / 8 heads, 256 ragged ones x 1024 98 -> 56.  At 64
// sequences and fewer the one above is faster by up to 8 %.
__device__ __forceinline__ int split_bin(const SplitParams& p) { return (p.batch + 1023) >> 10; }     // batches of 32 in a bin

template <int GW, int NG>
__device__ __forceinline__ void split_plan_many(const SplitParams& p, SplitPlan& s, int lane) {
    constexpr int kAhead = 8;
    s.lane = lane;
    s.too_long = s.void_batch = false;
    s.np = s.len = 0;
    const int span = split_bin(p);
    int np[kAhead], pages = 0, nonempty = 0, bin_pages = 0, bin_live = 0, bin = 0, in_bin = 0;
    for (int g0 = 0; 32 * g0 < p.batch; g0 += kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const int b = 32 * (g0 + u) + lane;
            int len = 0;
            np[u] = b < p.batch ? split_pages(p, b, len, s.too_long) : 0;
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (32 * (g0 + u) >= p.batch) break;
            const int sum = __reduce_add_sync(0xffffffffu, np[u]), live = __popc(__ballot_sync(0xffffffffu, np[u] > 0));
            if (lane == bin) { bin_pages += sum; bin_live += live; }
            if (++in_bin == span) { in_bin = 0; bin++; }
            pages += sum;
            nonempty += live;
        }
    }
    s.too_long = __any_sync(0xffffffffu, s.too_long);
    s.void_batch = s.too_long && p.all_or_nothing;
    if (s.void_batch) {
        pages = nonempty = bin_pages = bin_live = 0;
#pragma unroll
        for (int u = 0; u < kAhead; u++) np[u] = 0;
    }
    const int groups = p.grid * NG;
    const float even = (float)pages * (float)p.kv_heads * p.inv_warps;
    const int share = (int)even + (even > (float)(int)even ? 1 : 0);
    s.piece = 0;
    int pieces = 0, bin_pieces = 0;
    for (int t = share < 1 ? 1 : share; t <= share + kSplitSlackTiles && p.batch <= 32 * kAhead; t++) {      // np has them all
        const int size = t * GW;
        pieces = 0;
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (32 * u >= p.batch) break;
            const int sum = __reduce_add_sync(0xffffffffu, split_div_up(np[u], size));
            if (lane == u) bin_pieces = sum;
            pieces += sum;
        }
        if (pieces * p.kv_heads <= groups) {
            s.piece = size;
            break;
        }
    }
    split_cut_list<NG>(p, s, pages, nonempty, pieces);
    s.ends = s.piece ? p.kv_heads * bin_pieces : p.head_sets * (bin_pages + bin_live * p.item_cost);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, s.ends, o);
        if (lane >= o) s.ends += t;
    }
}
// to the first sequences of bin i
__device__ __forceinline__ void split_jump(const SplitParams& p, SplitPlan& s, int i) {
    const int before = __shfl_sync(0xffffffffu, s.ends, (i - 1) & 31);
    split_load(p, s, 32 * split_bin(p) * i, i > 0 ? before : 0, false);
}
__device__ __forceinline__ void split_keep_plan(const SplitParams& p, const SplitPlan& s) {
    if (s.lane == 0) {
        p.header[1] = s.total;
        p.header[2] = s.workers;
        p.header[3] = s.piece;
        p.header[4] = s.void_batch;
    }
    p.header[8 + s.lane] = s.ends;
}
__device__ __forceinline__ void split_kept_plan(const SplitParams& p, SplitPlan& s, int lane) {
    s.lane = lane;
    s.total = p.header[1];
    s.workers = p.header[2];
    s.piece = p.header[3];
    s.void_batch = p.header[4] != 0;
    s.ends = p.header[8 + lane];
    s.head_set = s.piece ? 1 : p.head_set;
    s.len = 0;
}

// One box of the cache into shared memory: bytes x ... of 16 token rows from row y of slab z (0: K, 1: V), or of both.  No multicast; x is a
// multiple of the slot, hence of 16.
__device__ __forceinline__ void split_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void split_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool split_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// A value the compiler cannot work out again: a lane's constants stay in registers through the page loop instead of being recomputed
// from the thread index in every iteration.
__device__ __forceinline__ uint32_t split_keep(uint32_t v) {
    asm volatile("" : "+r"(v));
    return v;
}
// BYTES (4, 8, 16 or 32) of a staged code row into words
template <int BYTES>
__device__ __forceinline__ void split_lds(uint32_t addr, uint32_t (&w)[BYTES / 4]) {
    if constexpr (BYTES == 4) {
        w[0] = lds32(addr);
    } else if constexpr (BYTES == 8) {
        const uint2 v = lds64(addr);
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 16; i++) {
            const uint4 v = lds128(addr + 16 * i);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    }
}

// Hadamard butterflies of a row over a warp: lane l holds elements E l ... E l + E - 1.
template <int E>
__device__ __forceinline__ void split_fwht(float (&v)[E], int lane) {
#pragma unroll
    for (int h = 1; h < E; h <<= 1) {
#pragma unroll
        for (int i = 0; i < E; i++) {
            if ((i & h) == 0) {
                const float a = v[i], b = v[i + h];
                v[i] = a + b;
                v[i + h] = a - b;
            }
        }
    }
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
#pragma unroll
        for (int i = 0; i < E; i++) {
            const float o = __shfl_xor_sync(0xffffffffu, v[i], m);
            v[i] = (lane & m) ? o - v[i] : v[i] + o;
        }
    }
}

// E consecutive elements of a 16- or 32-bit row as fp32; `at` is the element index of the first one, rows hold `dim` elements
template <int E>
__device__ __forceinline__ void split_load_row(const void* base, int dtype, int64_t row, int dim, int d0, float (&v)[E]) {
    const int64_t at = row * dim + d0;
    if (dtype != TQ_F32 && dim % E == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0) {   // E 16-bit elements: 4, 8 or 16 bytes
        if (d0 >= dim) {
#pragma unroll
            for (int i = 0; i < E; i++) v[i] = 0.0f;
            return;
        }
        uint32_t w[E / 2];
        const uint16_t* src = reinterpret_cast<const uint16_t*>(base) + at;
        if constexpr (E == 2) w[0] = *reinterpret_cast<const uint32_t*>(src);
        else if constexpr (E == 4) { const uint2 t = *reinterpret_cast<const uint2*>(src); w[0] = t.x; w[1] = t.y; }
        else { const uint4 t = *reinterpret_cast<const uint4*>(src); w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w; }
#pragma unroll
        for (int i = 0; i < E / 2; i++) {
            if (dtype == TQ_BF16) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < E; i++) v[i] = d0 + i < dim ? load_q(base, dtype, at + i) : 0.0f;
}

// A finished row (normalized, rotated domain): back through the rotation and out, or out as it is.
template <int PD>
__device__ __forceinline__ void split_finish(const SplitParams& p, const float* signs, int b, int head, int col, float (&o)[PD / 32], float lse2, int lane) {
    constexpr int E = PD / 32;
    const int qi = col / p.real_group, hh = col - qi * p.real_group;
    const int64_t orow = ((int64_t)b * p.nq + qi) * p.real_heads + head * p.real_group + hh;
    const int d0 = lane * E;
    if (p.emit_rotated) {
        float* dst = reinterpret_cast<float*>(p.out) + orow * PD + d0;
#pragma unroll
        for (int i = 0; i < E; i++) dst[i] = o[i];
        if (p.out_lse && lane == 0) p.out_lse[orow] = lse2;
        return;
    }
    split_fwht<E>(o, lane);
    const int dim = p.head_dim;
#pragma unroll
    for (int i = 0; i < E; i++) o[i] *= p.scale * signs[d0 + i];
    const int64_t at = orow * dim + d0;
    if (p.out_dtype != TQ_F32 && dim % E == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0) {
        if (d0 < dim) {
            uint32_t w[E / 2];
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                if (p.out_dtype == TQ_BF16) {
                    const __nv_bfloat162 t = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
                    w[i] = *reinterpret_cast<const uint32_t*>(&t);
                } else {
                    w[i] = pack_half2(o[2 * i], o[2 * i + 1]);
                }
            }
            uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + at;
            if constexpr (E == 2) *reinterpret_cast<uint32_t*>(dst) = w[0];
            else if constexpr (E == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; i++) {
            if (d0 + i >= dim) continue;
            if (p.out_dtype == TQ_BF16) reinterpret_cast<__nv_bfloat16*>(p.out)[at + i] = __float2bfloat16_rn(o[i]);
            else if (p.out_dtype == TQ_F16) reinterpret_cast<__half*>(p.out)[at + i] = __float2half_rn(o[i]);
            else reinterpret_cast<float*>(p.out)[at + i] = o[i];
        }
    }
    if (p.out_lse && lane == 0) p.out_lse[orow] = lse2 * 0.6931471805599453f;
}

}  // namespace tq
