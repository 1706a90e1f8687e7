// Many queries a sequence over its cached states, every query over all of them: attention of a decoder's prompt to an encoder's states in the
// quantized cache, on the 5th-generation tensor cores.
//
//   out[t, h] = sum_j softmax_j(q[t, h] . k[j] * scale) v[j],      j over the tokens of the cache, t over the query rows of the sequence
//
// Queries and cached rows stay in the rotated domain (K^ = H S K, V^ = H S V): a query is rotated once, an output row is rotated back
// once, and what is between is two matrix products.  A block takes one or two tiles of 128 query rows of one KV head (the query heads that share
// it are rows too: row r is query r / G, head r % G) and a range of the tokens, 128 at a time:
//
//   two warps     bring the slots of K and V into shared memory, 64 tokens at a time (a tiled tensor copy of 16 rows a page), another fetches the norms,
//   four warps    look the K codes up into the 32 KB image that the tensor core reads (rows of 128 bytes, 16-byte pieces swizzled by the row), four
//                 others the V codes into its transpose, nibbles of two tokens zipped into bytes,
//   a warp        issues S = Q K^^T and O += P V^,
//   two warpgroups, a thread a row, take S from tensor memory, keep a running maximum and sum, and put P (fp16) into the same columns.
//
// Where many query rows share a sequence's tokens (prompts), a first kernel writes the images of K and V to memory once and a block only copies them in,
// 32 KB each: the look-ups take longer than the products they feed (405 us looked up, 305 laid out ahead, at four sequences of 1024 queries on 4096
// tokens, 32 heads on 8).  With few rows that would write and read 512 bytes for every 80-byte slot, and the slots are looked up as they
// come (36 us looked up, 56 laid out ahead, with 32 queries).
//
// S, then P, and O of two tiles are all of tensor memory: 2 x (128 + 128) columns.  With two tiles of query rows each warpgroup has one, and while it works out
// exponentials the tensor core works for the other.  With one the warpgroups take the tiles of tokens in turn; at the end each brings its O to the
// larger of their maxima, and the product that rotates back adds them.  The running maximum, of the logit and the logarithm of V's scale in its tile together, is raised
// only when one exceeds it by 2^8, which makes rescaling O rare; a row needs no other thread but its own.  Where few rows have long sequences the tokens are cut over
// several blocks as well: every group leaves a partial, and a second kernel joins them.
//
// The rotations are matrix products too, with a matrix of ones and minus ones, exact in any type: the queries go through the tensor core as they come before the
// first tile, and O, as two fp16 parts, behind the last, which also brings its columns into order.  As butterflies over registers they took as long as ten tiles: code that a
// block runs once is fetched anew by every block, and that is what it costs.  (4 x 2048 queries on 4096 tokens: 645 us with butterflies in front, 573 so.)
//
// What bounds it.  Many rows: products and exponentials follow each other through S and P of a tile, and two tiles in flight, all that tensor memory holds, keep
// the tensor core busy for two thirds of a tile's 3000 cycles: 4 x 2048 queries on 4096 tokens, 32 heads on 8, 560 us, 980 TFLOP/s.  Few rows, long
// sequences: the same chain for one tile, half of its exponentials' time the norms' loads and products (fp16 results), and V's look-ups: 2 x 16
// queries on 65536 tokens, 64 heads on 8, 173 us, 805 GB/s of codes.  Short ones: what a block does before its first tile and behind its last, some 20
// thousand cycles: 24 queries on 1500 tokens, 16 heads on 8, 20.1 us, two tiles a block.
//
// Numbers are fp16 in the tensor core with fp32 sums, brought into fp16's range by powers of two: a query row by its largest element, the norms of
// K and V by the largest of the tile, P by the largest share that a tile can have in the row.  (By the largest weight alone, tiles whose values are small beside those of
// earlier tiles kept few bits, even where they had all the weight: values 2^-24 of the others' none.)
//   16-bit results of 8 bits (bf16): norms are multiplied into K^ and V^, one rounding (2^-12) each.
//   results of 11 bits and more (fp16, fp32): K^ and V^ are bare levels, scaled so that the eight of them lie within 4e-5 of fp16 values;
//             norms multiply S and P in fp32, and a query is two fp16 parts (half again as many operations in the tensor core, and one
//             tile of query rows a block): what is rounded is P.
#include <cmath>
#include <cstring>

#include "tq_split.cuh"
#include "tq_tcgen05.cuh"

namespace tq {

constexpr int kCrossTile = 128;                      // tokens, query rows, padded head size
constexpr int kCrossImage = kCrossTile * kCrossTile * 2;
constexpr int kCrossTeam = 4;                        // warps that look up K, and as many for V
constexpr int kCrossRowThreads = 384, kCrossThreads = kCrossRowThreads + 2 * kCrossTeam * 32;      // two warpgroups of rows, one of copies, norms and products; the teams
// Tiles of query rows a sequence, on the average, above which the images are laid out ahead.  us laid out and looked up, 32 heads on 8, bf16 / fp16 results:
//   320 rows    16 x 1500 tokens 110 and 95 / 128 and 121, 32 x 700 123 and 114 / 161 and 163
//   512 rows    8 x 1500 tokens 59 and 51 / 82 and 82, 4 x 4096 85 and 72 / 89 and 91
//   768 rows    4 x 4096 103 and 106 / 136 and 167;   1200 rows    4 x 32768 1124 and 1418 / 1308 and 1700
// and of one sequence 800 rows on 1500 tokens 35 and 31 / 39 and 35, 1600 rows on 65536 587 and 706 / 815 and 1148.
constexpr int kCrossLaid = 4;
constexpr float kCrossRaise = 8.0f;                  // P up to 2^8
constexpr double kCrossLevelScale = 1.42803;         // see tq_scored.cu
constexpr float kCrossNoNorm = -40.0f;               // the logarithm of V's scale in a tile whose V is all zero: below that of any other
constexpr uint32_t kCrossWaitLimit = 1u << 18, kCrossSuspendNs = 1000;

struct CrossParams {
    SplitParams f;              // what split_load_row / split_finish take: types, head size, signs, out, the cache; its tensor map (boxes of 16 slots)
    const int32_t* cu_q;        // [batch + 1]
    // where the images are laid out ahead:
    uint8_t* kv_images;         // [tile][head][K, V][32 KB]; behind the last, the matrix of the way back
    uint8_t* turn_image;        // and the matrix of the way in behind it
    float2* tile_scales;        // [tile][head]: K's power of two, the logarithm of V's
    uint16_t* tile_norms;       // exact: [tile][head][K, V][128]
    int64_t kv_room;            // tiles that there is room for
    float* partial_o;           // [cut][group][query row][query head][128], rotated domain
    float* partial_lse;
    int total_q, splits;        // of the tokens: most blocks that a sequence is cut over
    uint16_t level_h[16];
};

static __device__ int32_t g_cross_faults = 0;

struct CrossSeq {
    int b, local;               // the sequence, and which of its items the index is
    int len, qlen;              // tokens, query rows (tokens of the prompt)
    int kv0;                    // its first tile of tokens
    int cuts;                   // blocks that its tokens are cut over
};

__device__ __forceinline__ int cross_len(const CrossParams& p, int b, bool& bad) {
    const int len = p.f.seq_lens[b];
    bad = len < 0 || len > (int64_t)p.f.max_pages * kPageTokens;
    return bad ? 0 : len;
}
// Query rows of N times 32 sequences, a lane each, from their bounds.  A range that is none has no rows, and none has one that begins before the end of an earlier one,
// which takes bounds that fall somewhere: only from there on the ends are looked at.  A whole warp, one batch of sequences behind the other.
struct CrossRanges {
    int end = 0;                // of the ranges so far: the lane's, and once bounds have fallen all lanes'
    bool fell = false;
    template <int N>
    __device__ __forceinline__ void rows(const CrossParams& p, const int (&c0)[N], const int (&c1)[N], int lane, int (&rows)[N], int& faults) {
        bool falls = false;
#pragma unroll
        for (int e = 0; e < N; e++) {
            const bool bad = c0[e] < 0 || c1[e] < c0[e] || c1[e] > p.total_q;
            rows[e] = bad ? 0 : c1[e] - c0[e];
            faults += bad;
            falls |= c1[e] < c0[e];
        }
        if (!fell && __any_sync(0xffffffffu, falls)) {
            fell = true;
            end = __reduce_max_sync(0xffffffffu, end);
        }
        if (!fell) {
#pragma unroll
            for (int e = 0; e < N; e++) end = max(end, rows[e] > 0 ? c1[e] : 0);
            return;
        }
#pragma unroll
        for (int e = 0; e < N; e++) {
            const int upto = rows[e] > 0 ? c1[e] : 0;
            int before = __shfl_up_sync(0xffffffffu, upto, 1);
            before = lane == 0 ? end : max(before, end);
#pragma unroll 1
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before = max(before, t);
            }
            if (rows[e] > 0 && c0[e] < before) {
                rows[e] = 0;
                faults++;
            }
            end = max(end, __reduce_max_sync(0xffffffffu, upto));
        }
    }
};
// Blocks that a sequence's tokens are cut over: two tiles each (one a warpgroup) at least.  By its own length: results depend neither on the table's width nor on
// the tokens that the caller makes room for, and no block beside these has work (or a partial).
__device__ __forceinline__ int cross_cuts(const CrossParams& p, int len) { return max(1, min(p.splits, (len + 2 * kCrossTile - 1) / (2 * kCrossTile))); }
__device__ __forceinline__ int cross_upto(int v, int lane) {      // the sum of the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}
// The sequence that item `index` of a kind belongs to (0: tiles of tokens; 1, 2: that many tiles of query rows); false: there are not so many.  A sequence
// without queries has no tiles of tokens; one that ends behind the tiles which the caller's number of tokens makes has no tokens.  A whole warp.
template <int KIND>
__device__ __forceinline__ bool cross_find(const CrossParams& p, int64_t index, int lane, CrossSeq& s) {
    constexpr int kAhead = 4;                         // 32 sequences each, whose numbers are on their way together
    int64_t kv = 0, items = 0;
    CrossRanges ranges;
    for (int base = 0; base < p.f.batch; base += 32 * kAhead) {
        int len[kAhead], qlen[kAhead], c0[kAhead], c1[kAhead], faults = 0;
#pragma unroll
        for (int e = 0; e < kAhead; e++) {
            const int b = base + 32 * e + lane;
            bool bad;
            len[e] = b < p.f.batch ? cross_len(p, b, bad) : 0;
            c0[e] = b < p.f.batch ? p.cu_q[b] : 0;
            c1[e] = b < p.f.batch ? p.cu_q[b + 1] : 0;
        }
        ranges.rows(p, c0, c1, lane, qlen, faults);
        bool hit = false;
        int kt = 0, mine = 0;
#pragma unroll
        for (int e = 0; e < kAhead; e++) {
            if (hit || base + 32 * e >= p.f.batch) continue;
            s.b = base + 32 * e;
            s.len = len[e];
            s.qlen = qlen[e];
            kt = s.qlen > 0 ? (s.len + kCrossTile - 1) / kCrossTile : 0;
            mine = KIND == 0 ? kt : (s.qlen * p.f.real_group + KIND * kCrossTile - 1) / (KIND == 0 ? 1 : KIND * kCrossTile);
            const int all = __reduce_add_sync(0xffffffffu, mine);
            hit = index < items + all;
            if (!hit) {
                items += all;
                kv += __reduce_add_sync(0xffffffffu, kt);
            }
        }
        if (hit) {
            const int to = cross_upto(mine, lane), l = __ffs(__ballot_sync(0xffffffffu, index < items + to)) - 1;
            const int64_t kv_to = kv + cross_upto(kt, lane);
            s.b += l;
            s.local = (int)(index - items) - __shfl_sync(0xffffffffu, to - mine, l);
            if constexpr (KIND != 0) s.cuts = __shfl_sync(0xffffffffu, cross_cuts(p, s.len), l);
            s.len = __shfl_sync(0xffffffffu, kv_to <= p.kv_room ? s.len : 0, l);
            s.qlen = __shfl_sync(0xffffffffu, s.qlen, l);
            s.kv0 = (int)__shfl_sync(0xffffffffu, kv_to - kt, l);
            return true;
        }
    }
    return false;
}
// Counts what is left out.  A whole warp, of one block.
__device__ __forceinline__ void cross_count_faults(const CrossParams& p, int lane) {
    int64_t kv = 0;
    int faults = 0;
    CrossRanges ranges;
    for (int base = 0; base < p.f.batch; base += 32) {
        bool bad_len = false;
        const int b = base + lane, len = b < p.f.batch ? cross_len(p, b, bad_len) : 0;
        const int c0[1] = {b < p.f.batch ? p.cu_q[b] : 0}, c1[1] = {b < p.f.batch ? p.cu_q[b + 1] : 0};
        int qlen[1];
        ranges.rows(p, c0, c1, lane, qlen, faults);
        const int kt = qlen[0] > 0 ? (len + kCrossTile - 1) / kCrossTile : 0, to = cross_upto(kt, lane);
        faults += bad_len + (kt > 0 && kv + to > p.kv_room);
        kv += __shfl_sync(0xffffffffu, to, 31);
    }
    if (faults) atomicAdd(&g_cross_faults, faults);
}

// Byte of 16-byte piece c (0 ... 15) of row r in an image: two halves of 128 rows x 128 bytes, the pieces of a row swizzled within its half.
__device__ __forceinline__ uint32_t cross_piece(int r, int c) { return (uint32_t)((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

__device__ __forceinline__ uint32_t cross_mul2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// The power of two that brings v to [2^to, 2^(to + 1)), as its exponent; 0 for what is not a normal positive number.
__device__ __forceinline__ int cross_exponent(float v, int to) {
    const int ex = (int)(__float_as_uint(v) >> 23) - 127;
    return ex > -110 && ex < 110 ? to - ex : 0;
}
__device__ __forceinline__ float cross_power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// Where the largest norm of a tile goes, as an exponent of two.  In the images: products with levels up to 4 stay inside fp16.  Under P (exact): below one, so that P
// times a norm is no larger than P.
constexpr int kCrossInImage = 6, kCrossUnderP = -1;

// Piece c (eight columns) of row dim of the matrix of the way back: column 16 d + w is dim 8 w + d of O.
__device__ __forceinline__ uint4 cross_turn(int dim, int c, bool negative) {
    const uint32_t same = (uint32_t)__popc(dim & (64 * (c & 1) + (c >> 1))) ^ (uint32_t)negative;      // d = c / 2, w = 8 (c % 2) + ...
    uint32_t v[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t a = (same ^ (uint32_t)__popc((dim >> 3) & (2 * e))) & 1u, b = (same ^ (uint32_t)__popc((dim >> 3) & (2 * e + 1))) & 1u;
        v[e] = 0x3C003C00u | a << 15 | b << 31;
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ uint32_t cross_negative(const float* signs, int c) {      // of eight dims, a bit each
    uint32_t negative = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) negative |= (uint32_t)(signs[8 * c + e] < 0.0f) << e;
    return negative;
}
// Piece c (eight dims, negative: a bit each) of row col of the matrix of the way in, which rotates the queries: column col of a query image is dim col ^ 1, as the codes have
// them.  one: a pair of ones of the queries' type.
__device__ __forceinline__ uint4 cross_way_in(int col, int c, uint32_t negative, uint32_t one) {
    const int j = col ^ 1;
    const uint32_t same = (uint32_t)__popc(j & (8 * c));
    uint32_t v[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t a = (same ^ (uint32_t)__popc(j & (2 * e)) ^ (negative >> (2 * e))) & 1u, b = (same ^ (uint32_t)__popc(j & (2 * e + 1)) ^ (negative >> (2 * e + 1))) & 1u;
        v[e] = one | a << 15 | b << 31;
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// ---------------------------------------------------------------------------------------------
// images laid out ahead
// ---------------------------------------------------------------------------------------------
constexpr int kLayThreads = 256, kLayPitch = 17;      // words of a staged V row (16 and one, for the banks)
// (Registers for three blocks an SM: left to itself the compiler takes 48, and 8 x 512 fp16 queries on 1500 tokens 238 us in place of 230.)
template <bool EXACT>
__global__ void __launch_bounds__(kLayThreads, 3) cross_lay_out_kernel(const __grid_constant__ CrossParams p) {
    __shared__ uint32_t lut[256 * 32];                // entry v, column lane: {level(v & 15), level(v >> 4)}
    __shared__ uint32_t codes_s[kCrossTile * kLayPitch];
    __shared__ int64_t slot_s[kCrossTile];            // byte of each token's K slot
    __shared__ uint16_t norm_s[2][kCrossTile];
    __shared__ float most_s[2][4];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, H = p.f.kv_heads;
    grid_launch_dependents();
    for (int i = tid; i < 256 * 32; i += kLayThreads) lut[i] = (uint32_t)p.level_h[(i >> 5) & 15] | ((uint32_t)p.level_h[i >> 9] << 16);
    grid_dependency_wait();
    if (blockIdx.x == 0 && warp == 0) cross_count_faults(p, lane);
    if (blockIdx.x == gridDim.x - 1) {                // the matrices of the way back and in
        const uint32_t one = p.f.q_dtype == TQ_BF16 ? 0x3F803F80u : 0x3C003C00u, negative = cross_negative(p.f.signs, tid & 15);
        for (int i = tid; i < kCrossTile * 16; i += kLayThreads) {
            *reinterpret_cast<uint4*>(p.turn_image + cross_piece(i >> 4, i & 15)) = cross_turn(i >> 4, i & 15, p.f.signs[i >> 4] < 0.0f);
            *reinterpret_cast<uint4*>(p.turn_image + kCrossImage + cross_piece(i >> 4, i & 15)) = cross_way_in(i >> 4, i & 15, negative, one);
        }
    }
    __syncthreads();

    const uint8_t* lut_lane = reinterpret_cast<const uint8_t*>(lut) + 4 * lane;
    auto level2 = [&](uint32_t byte) { return *reinterpret_cast<const uint32_t*>(lut_lane + (byte << 7)); };
    int64_t unit = blockIdx.x;
    for (;; unit += gridDim.x) {
        CrossSeq s;
        const int64_t tile = unit / H;
        const int h = (int)(unit - tile * H);
        if (!cross_find<0>(p, tile, lane, s)) break;
        if (s.len == 0) continue;                     // does not fit
        const int t0 = s.local * kCrossTile, n = min(kCrossTile, s.len - t0);
        if (tid < kCrossTile) {
            int64_t page = tid < n ? p.f.page_indices[(int64_t)s.b * p.f.max_pages + (t0 + tid) / kPageTokens] : 0;
            if ((uint64_t)page >= (uint64_t)p.f.num_blocks) {
                page = 0;
                if (h == 0 && (tid & 15) == 0) atomicAdd(&g_cross_faults, 1);
            }
            slot_s[tid] = (page * kPageTokens + (tid & 15)) * p.f.kv_heads * kSlotBytes + h * kSlotBytes;
        }
        __syncthreads();
        const int64_t slab = p.f.num_blocks * kPageTokens * p.f.kv_heads * kSlotBytes;
        // K codes: a lane takes 4 bytes (8 dims, one piece) of a row, eight lanes 32 bytes of it
        uint32_t k_code[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = (i & 3) * 32 + warp * 4 + (lane >> 3), c = (i >> 2) * 8 + (lane & 7);
            k_code[i] = r < n ? *reinterpret_cast<const uint32_t*>(p.f.kv_cache + slot_s[r] + 4 * c) : 0u;
        }
        // V codes to shared memory, to be read by columns
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = (tid >> 2) + 64 * i, c = tid & 3;
            const uint4 v = r < n ? *reinterpret_cast<const uint4*>(p.f.kv_cache + slab + slot_s[r] + 16 * c) : make_uint4(0u, 0u, 0u, 0u);
            uint32_t* to = codes_s + r * kLayPitch + 4 * c;
            to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
        }
        const int which = tid >> 7, t = tid & 127;
        const float norm = t < n ? __half2float(__ushort_as_half(*reinterpret_cast<const uint16_t*>(p.f.kv_cache + which * slab + slot_s[t] + kHeadDim / 2))) : 0.0f;
        float most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(norm) < INFINITY ? fabsf(norm) : 0.0f)));
        if (lane == 0) most_s[which][warp & 3] = most;
        __syncthreads();
        most = fmaxf(fmaxf(most_s[which][0], most_s[which][1]), fmaxf(most_s[which][2], most_s[which][3]));
        const int by = cross_exponent(most, EXACT ? kCrossUnderP : kCrossInImage);
        if constexpr (EXACT) p.tile_norms[((tile * H + h) * 2 + which) * kCrossTile + t] = __half_as_ushort(__float2half_rn(norm));      // as they are
        else norm_s[which][t] = __half_as_ushort(__float2half_rn(norm * cross_power(by)));
        if (t == 0) reinterpret_cast<float*>(p.tile_scales + tile * H + h)[which] = which ? most > 0.0f ? (float)-by : kCrossNoNorm : EXACT ? 1.0f : cross_power(-by);
        __syncthreads();
        uint8_t* const image = p.kv_images + (tile * H + h) * 2 * kCrossImage;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = (i & 3) * 32 + warp * 4 + (lane >> 3), c = (i >> 2) * 8 + (lane & 7);
            const uint32_t w = k_code[i], nn = EXACT ? 0u : (uint32_t)norm_s[0][r] * 0x10001u;
            uint32_t v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {             // dims in pairs {odd, even}, as the queries have them
                v[j] = level2((w >> (8 * j)) & 255u);
                if constexpr (!EXACT) v[j] = cross_mul2(v[j], nn);
            }
            *reinterpret_cast<uint4*>(image + cross_piece(r, c)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
        // V^ transposed, dim 8 w + d as row 16 d + w: a lane takes eight tokens (one piece) of eight dims (one code word); nibbles of two tokens are zipped into bytes
        {
            const int c = (lane & 7) + 8 * (warp & 1), word = (lane >> 3) + 4 * (warp >> 1);     // pieces 0 ... 15, words 0 ... 15
            uint32_t out[8][4];
#pragma unroll
            for (int pr = 0; pr < 4; pr++) {
                const uint32_t a = codes_s[(8 * c + 2 * pr) * kLayPitch + word], b = codes_s[(8 * c + 2 * pr + 1) * kLayPitch + word];
                const uint32_t odd = (a & 0x0F0F0F0Fu) | ((b << 4) & 0xF0F0F0F0u), even = ((a >> 4) & 0x0F0F0F0Fu) | (b & 0xF0F0F0F0u);
                const uint32_t nn = EXACT ? 0u : *reinterpret_cast<const uint32_t*>(&norm_s[1][8 * c + 2 * pr]);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    out[2 * j][pr] = level2((even >> (8 * j)) & 255u);
                    out[2 * j + 1][pr] = level2((odd >> (8 * j)) & 255u);
                    if constexpr (!EXACT) {
                        out[2 * j][pr] = cross_mul2(out[2 * j][pr], nn);
                        out[2 * j + 1][pr] = cross_mul2(out[2 * j + 1][pr], nn);
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < 8; d++) *reinterpret_cast<uint4*>(image + kCrossImage + cross_piece(16 * d + word, c)) = make_uint4(out[d][0], out[d][1], out[d][2], out[d][3]);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------------
// SW128, K-major: rows of 128 bytes, eight rows 1024 bytes on
__host__ __device__ constexpr uint64_t cross_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)64 << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// A wait of a whole warp that ends early when another role has given up.
__device__ __forceinline__ bool cross_wait(uint32_t bar, uint32_t parity, volatile int* gone) {
    bool done = false;
    for (uint32_t i = 0; i < kCrossWaitLimit && !done; i++) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar), "r"(parity), "r"(kCrossSuspendNs) : "memory");
        done = ok != 0;
        if ((i & 15) == 15 && *gone) break;
    }
    return __all_sync(0xffffffffu, done);
}
__device__ __forceinline__ void cross_bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void cross_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void cross_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cross_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// Stores that keep their order among themselves and to the barriers, and loads of what does not change (the table), which have none: the compiler is
// free to look codes up ahead of the stores of those before.
__device__ __forceinline__ void cross_sts(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d));
}
__device__ __forceinline__ uint32_t cross_table(uint32_t at) {
    uint32_t v;
    asm("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ float2 cross_lds_f2(uint32_t at) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at));
    return v;
}
// 32 columns of the thread's tensor-memory lane; the values are there after cross_ld_wait of the same registers.
__device__ __forceinline__ void cross_ld(uint32_t taddr, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
          "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
          "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void cross_ld16(uint32_t taddr, float* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
                   "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]) : "r"(taddr));
}
__device__ __forceinline__ void cross_ld_wait16(float* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]),
                   "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]) :: "memory");
}
__device__ __forceinline__ void cross_ld_wait(float* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]),
                   "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]), "+f"(r[16]),
                   "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]),
                   "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
                 :: "memory");
}
__device__ __forceinline__ void cross_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void cross_st(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
          "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
          "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}

// Shared memory as absolute addresses of the block's window, whose first 1024 bytes are the system's.  Where the block looks codes up itself: two rings of slots,
// K's and V's, of three halves of a tile (64 tokens); barriers and small words; the table at a multiple of its size (a shift and one logic
// instruction make an entry's address); the images on their 1024-byte boundaries; the norms.  Where the images come laid out: barriers, images, norms.
constexpr int kCrossHalf = kCrossTile / 2, kCrossUnit = kCrossHalf * kSlotBytes, kCrossStages = 3, kCrossMetas = 4;
constexpr uint32_t kCrossRaw = 1024;                                     // K's ring, then V's
constexpr uint32_t kCrossLut = 32768;                                    // entry v, column lane: {level(v & 15), level(v >> 4)}
template <bool EXACT, bool LAID>
struct CrossMap {
    static constexpr uint32_t kBars = LAID ? 1024 : kCrossRaw + 2 * kCrossStages * kCrossUnit;
    static constexpr uint32_t kScales = kBars + 512;                     // of tile t at t % kCrossMetas: K's power of two, the logarithm of V's
    static constexpr uint32_t kSigns = kScales + kCrossMetas * 8;        // a bit a dim: negative
    static constexpr uint32_t kQ = LAID ? 2048 : 65536;                  // two images: tiles of query rows, or the two parts of one
    // Images in turn, of K and V.  Two tiles of query rows: K0 V0 K1 V1 ... ; one: K0 K1 V0 K2 V1 ... , the order in which they are needed.  Behind the last comes
    // the matrix of the way back, where the next K would be.  Looked up here each is written as two halves (64 tokens); it is free when its product has been formed.
    static constexpr int kImages = LAID ? 5 : 3;
    static constexpr uint32_t kImg = kQ + 2 * kCrossImage;
    static constexpr uint32_t kWay = kImg + (kImages - 1) * kCrossImage; // before its first image: the matrix of the way in
    // The norms of tile t at t % 4: for the rows (exact), fp16, K's and V's; or for the look-ups, fp16, K's twice each.  When S (t - 2) has been formed P (t - 4)
    // has been handed over, so nobody reads the norms of tile t - 4 any more.
    static constexpr uint32_t kNorms = kImg + kImages * kCrossImage;
    static constexpr int kNormBytes = EXACT ? 2 * kCrossTile * 2 : LAID ? 0 : 2 * kCrossTile * 4;
    static constexpr size_t kSmem = kNorms + kCrossMetas * kNormBytes - 1024;
    static_assert(kSigns + 16 <= (LAID ? kQ : kCrossLut) && kSmem <= 232448 && kCrossUnit % 128 == 0, "shared memory of a block");
};

// The exponent that brings the largest of a tile's norms (four a lane) to [2^to, 2^(to + 1)).
__device__ __forceinline__ int cross_norm_exponent(const float (&norm)[4], int to, bool& has) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (fabsf(norm[i]) < INFINITY) most = fmaxf(most, fabsf(norm[i]));
    most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));      // bits of numbers that are not negative sort as they do
    has = most > 0.0f;
    return cross_exponent(most, to);
}

// LAID: the images are there, laid out by the kernel before this one; else the codes are looked up and the queries rotated here.
template <bool EXACT, bool LAID>
__global__ void __launch_bounds__(LAID ? kCrossRowThreads : kCrossThreads, 1) cross_attend_kernel(const __grid_constant__ CrossParams p) {
    constexpr int kTiles = EXACT ? 1 : 2;             // of query rows
    using M = CrossMap<EXACT, LAID>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, H = p.f.kv_heads, G = p.f.real_group;
    uint8_t* const window = smem - smem_u32(smem);    // address 0 of the block's window
    grid_launch_dependents();
    if (smem_u32(smem) != 1024) {                     // the map counts on it
        grid_dependency_wait();
        if (tid == 0 && blockIdx.x == 0) atomicAdd(&g_cross_faults, 1);
        return;
    }
    const uint32_t bars = M::kBars;
    const uint32_t raw_full = bars, raw_empty = raw_full + 16 * kCrossStages, meta_full = raw_empty + 16 * kCrossStages, s_formed = meta_full + 8 * kCrossMetas,
                   img_full = s_formed + 8 * kCrossMetas, img_empty = img_full + 16 * M::kImages, s_full = img_empty + 8 * M::kImages, p_full = s_full + 16,
                   o_full = p_full + 16, a_full = o_full + 16, d_full = a_full + 16, drained = d_full + 16, turned = drained + 8;      // raw: K's stages, then V's; images: two halves
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(window + M::kBars + 400);
    volatile int* const gone = reinterpret_cast<volatile int*>(window + M::kBars + 404);
    if (tid == 9 * 32) {
        for (int i = 0; i < 2 * kCrossStages; i++) {
            cross_bar_init(raw_full + 8 * i, 1);
            cross_bar_init(raw_empty + 8 * i, kCrossTeam);
        }
        for (int i = 0; i < kCrossMetas; i++) {
            cross_bar_init(meta_full + 8 * i, 1);
            cross_bar_init(s_formed + 8 * i, 1);
        }
        for (int i = 0; i < M::kImages; i++) {
            cross_bar_init(img_full + 16 * i, kCrossTeam);
            cross_bar_init(img_full + 16 * i + 8, LAID ? 1 : kCrossTeam);
            cross_bar_init(img_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            cross_bar_init(s_full + 8 * i, 1);
            cross_bar_init(p_full + 8 * i, 4);        // the warps of a group
            cross_bar_init(o_full + 8 * i, 1);
            cross_bar_init(a_full + 8 * i, 4);
            cross_bar_init(d_full + 8 * i, 1);
        }
        cross_bar_init(drained, 1);
        cross_bar_init(turned, 1);
        *gone = 0;
        fence_barrier_init();
    }
    if (!LAID && warp >= 12) {                        // the table, the matrix of the way in and the signs' bits, while the others look for the sequence
        const uint32_t mine = p.level_h[lane & 15];
        for (int v = 4 * (warp - 12) + (lane >> 3); v < 256; v += 8 * kCrossTeam) {
            const uint32_t e = __shfl_sync(0xffffffffu, mine, v & 15) | (__shfl_sync(0xffffffffu, mine, v >> 4) << 16);
            *reinterpret_cast<uint4*>(window + kCrossLut + v * 128 + 16 * (lane & 7)) = make_uint4(e, e, e, e);
        }
        const int c = lane & 15;
        const uint32_t one = p.f.q_dtype == TQ_BF16 ? 0x3F803F80u : 0x3C003C00u, negative = cross_negative(p.f.signs, c);
#pragma unroll 1
        for (int col = 2 * (warp - 12) + (lane >> 4); col < kCrossTile; col += 4 * kCrossTeam) {
            const uint4 v = cross_way_in(col, c, negative, one);
            cross_sts(M::kWay + cross_piece(col, c), v.x, v.y, v.z, v.w);
        }
        if (warp == 12 && lane < 16) (window + M::kSigns)[lane] = (uint8_t)negative;      // a byte every eight dims
        fence_proxy_async();
    }
    grid_dependency_wait();
    if (!LAID && blockIdx.x == 0 && warp == 10) cross_count_faults(p, lane);
    CrossSeq s;
    const int64_t item = blockIdx.x / p.splits;
    const int split = (int)(blockIdx.x - item * p.splits), h = (int)(item % H);
    volatile int* const told = reinterpret_cast<volatile int*>(window + M::kBars + 416);
    auto cut_over = [&] { return (int)lds32(M::kBars + 416 + 20); };      // read again where it is needed: a register less
    if constexpr (LAID) {
        if (!cross_find<kTiles>(p, item / H, lane, s)) return;            // uniform over the block
        if (tid == 0) told[5] = s.cuts;
    } else {
        bool found = true;
        if (warp < 12) found = cross_find<kTiles>(p, item / H, lane, s);
        if (tid == 0) {
            told[0] = found; told[1] = s.b; told[2] = s.local; told[3] = s.len; told[4] = s.qlen; told[5] = s.cuts;
        }
        __syncthreads();
        found = told[0] != 0;
        s.b = told[1]; s.local = told[2]; s.len = told[3]; s.qlen = told[4]; s.cuts = told[5];
        if (!found) return;                           // uniform over the block
    }
    if (split >= s.cuts) return;                      // so is this (as one condition with the search's it costs the laid-out form 200 bytes of spills)
    const int rows = s.qlen * G, row0 = s.local * kTiles * kCrossTile;
    const bool solo = kTiles == 1 || rows - row0 <= kCrossTile;           // one tile of query rows
    const int all = (s.len + kCrossTile - 1) / kCrossTile;
    // The block's tiles of tokens (2^23 at most in all, and no more cuts than SMs: 32 bits).
    const int j0 = (int)((uint32_t)all * (uint32_t)split / (uint32_t)s.cuts), n = (int)((uint32_t)all * (uint32_t)(split + 1) / (uint32_t)s.cuts) - j0;
    if (LAID && tid == 9 * 32 && n > 0) {             // the matrix of the way in, see below
        split_expect(raw_full, kCrossImage);
        cross_copy(M::kWay, p.turn_image + kCrossImage, kCrossImage, raw_full);
    }

    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(M::kBars + 400), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    const int pages = (s.len + kPageTokens - 1) / kPageTokens, page0 = j0 * (kCrossTile / kPageTokens);
    bool bad_page = false;
    auto page_id = [&](int i) -> int {                // page i of the block's range; none and bad ones: page 0
        if (page0 + i >= pages) return 0;
        const int id = p.f.page_indices[(int64_t)s.b * p.f.max_pages + page0 + i];
        const bool good = (uint64_t)(int64_t)id < (uint64_t)p.f.num_blocks;
        bad_page |= !good;
        return good ? id : 0;
    };
    const int units = 2 * n;                          // halves of tiles
    // Item numbers of the images, see M::kImages.
    auto k_item = [&](int t) { return solo ? (t < 2 ? t : 2 * t - 1) : 2 * t; };
    auto v_item = [&](int t) { return solo ? 2 * t + 2 : 2 * t + 1; };

    const int D = p.f.head_dim;
    // K's and V's first slots: there is room.  ids: pages of eight units, and of the next eight.
    const int which = warp == 11, ring8 = which * kCrossStages;
    int id_now = 0, id_next = 0;
    auto copy_unit = [&](int u) {                     // lanes 0 ... 3 a page each
        const int stage = u % kCrossStages, id = __shfl_sync(0xffffffffu, id_now, (4 * (u & 7) + lane) & 31), some = max(0, min(4, pages - page0 - 4 * u));
        const uint32_t bar = raw_full + 8 * (ring8 + stage);
        if (lane == 0) split_expect(bar, (uint32_t)(some * kPageTokens * kSlotBytes));
        __syncwarp();
        if (lane < some)
            split_box(kCrossRaw + (ring8 + stage) * kCrossUnit + lane * kPageTokens * kSlotBytes, &p.f.cache_map, h * kSlotBytes, id * kPageTokens, which, bar);
    };
    const int q_tiles = solo ? 1 : 2, q_rows = min(rows - row0, q_tiles * kCrossTile), q_first = p.cu_q[s.b];
    const bool halves = p.f.q_dtype != TQ_F32;
    auto row_of = [&](int r) -> int64_t {             // of the query tensor
        const int row = row0 + r, qi = row / G;
        return (int64_t)(q_first + qi) * p.f.real_heads + h * G + (row - qi * G);
    };
    // As they come into the images' place, all in flight together, by the block's first `threads` threads.
    auto load_queries = [&](int threads) {
        if (!halves || n == 0) return;
        const uint16_t* const q16 = reinterpret_cast<const uint16_t*>(p.f.q);
        const bool whole = D % 8 == 0 && (reinterpret_cast<uintptr_t>(q16) & 15) == 0;
        const int step = threads / 16, c = tid & 15, on_q = step / G, on_g = step - on_q * G;      // rows on: a query row's place moves by on_q queries and on_g heads
        int r = tid >> 4, qi = (row0 + r) / G, g = row0 + r - qi * G;
#pragma unroll 1
        for (; r < q_tiles * kCrossTile; r += step) {
            const int some = r < q_rows ? min(8, D - 8 * c) : 0;
            const uint32_t to = M::kQ + (r >> 7) * kCrossImage + cross_piece(r & 127, c);
            const uint16_t* const from = some > 0 ? q16 + ((int64_t)(q_first + qi) * p.f.real_heads + h * G + g) * D + 8 * c : q16;
            qi += on_q;
            g += on_g;
            if (g >= G) {
                g -= G;
                qi++;
            }
            if (whole) {                              // (no bytes: zeros)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(some > 0 ? 16 : 0) : "memory");
            } else {
                uint32_t v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = (2 * e < some ? (uint32_t)from[2 * e] : 0u) | (2 * e + 1 < some ? (uint32_t)from[2 * e + 1] << 16 : 0u);
                cross_sts(to, v[0], v[1], v[2], v[3]);
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async();
    };
    if constexpr (LAID) {
        load_queries(kCrossRowThreads);
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
    }

    if (!LAID && warp >= 12) {
        const uint32_t lut_lane = kCrossLut + 4 * lane;
        // byte j of a word through the table: 128 bytes an entry
        auto level2 = [&](uint32_t w, int j) { return cross_table(((j == 0 ? w << 7 : w >> (8 * j - 7)) & 0x7f80u) | lut_lane); };
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const bool on_k = warp < 12 + kCrossTeam;
        const int mate = on_k ? warp - 12 : warp - 12 - kCrossTeam;
        bool ok = true;
        int stage = 0, turn = 0;
        const uint32_t ring = on_k ? 0 : kCrossStages;      // of the barriers and stages: K's first
        for (int u = 0; u < units && ok; u++) {
            const int t = u >> 1, half = u & 1;
            const uint32_t raw = kCrossRaw + (ring + stage) * kCrossUnit, norms = M::kNorms + (uint32_t)(t % kCrossMetas) * M::kNormBytes;
            ok = cross_wait(raw_full + 8 * (ring + stage), turn, gone);
            if (!EXACT && half == 0) ok = ok && cross_wait(meta_full + 8 * (t % kCrossMetas), (t / kCrossMetas) & 1, gone);
            const int item = on_k ? k_item(t) : v_item(t), slot = item % M::kImages;
            if (half == 0) ok = ok && cross_wait(img_empty + 8 * slot, ((item / M::kImages) & 1) ^ 1, gone) && (item != M::kImages - 1 || cross_wait(turned, 0, gone));
            if (!ok) break;
            const uint32_t image = M::kImg + slot * kCrossImage;
            if (on_k) {
                // =========================== K ================================================================
                // A lane takes 16 code bytes of a row, eight lanes the same of eight rows: no bank is met twice, at 80 bytes a row or in the image.
                // Both rows are looked up before either is stored: the assembler keeps loads and stores of shared memory in order.
                const int q = lane >> 3, r0 = 8 * mate + (lane & 7);
                constexpr int kStep = 8 * kCrossTeam, kRows = kCrossHalf / kStep;
                uint32_t v[kRows][16], nn[kRows];
                uint4 code[kRows];
#pragma unroll
                for (int i = 0; i < kRows; i++) {
                    code[i] = lds128(raw + (kStep * i + r0) * kSlotBytes + 16 * q);
                    if constexpr (!EXACT) nn[i] = lds32(norms + 4 * (kCrossHalf * half + kStep * i + r0));
                }
#pragma unroll
                for (int i = 0; i < kRows; i++) {
                    const uint32_t w4[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
#pragma unroll
                    for (int e = 0; e < 16; e++) v[i][e] = level2(w4[e >> 2], e & 3);
                }
#pragma unroll
                for (int i = 0; i < kRows; i++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        if constexpr (!EXACT) {
#pragma unroll
                            for (int j = 0; j < 4; j++) v[i][4 * c + j] = cross_mul2(v[i][4 * c + j], nn[i]);
                        }
                        cross_sts(image + cross_piece(kCrossHalf * half + kStep * i + r0, 4 * q + c), v[i][4 * c], v[i][4 * c + 1], v[i][4 * c + 2], v[i][4 * c + 3]);
                    }
            } else {
                // =========================== V ================================================================
                // A lane takes eight tokens (a piece of the image's rows) of a code word (eight dims); dim 8 w + d is row 16 d + w of the image, so that
                // neighbouring lanes store to rows of different swizzle.
                const int w = lane & 15, c = 2 * mate + (lane >> 4);      // piece of the half
                const uint32_t at = raw + 8 * c * kSlotBytes + 4 * w;
                uint32_t code[8], nn[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 8; e++) code[e] = lds32(at + e * kSlotBytes);
                if constexpr (!EXACT) {
                    const uint4 v = lds128(norms + 4 * kCrossTile + 2 * (kCrossHalf * half + 8 * c));
                    nn[0] = v.x; nn[1] = v.y; nn[2] = v.z; nn[3] = v.w;
                }
                // odd and even dims of token pairs, in place of the codes
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const uint32_t a = code[e], b = code[e + 1];
                    code[e] = ((a >> 4) & 0x0F0F0F0Fu) | (b & 0xF0F0F0F0u);
                    code[e + 1] = (a & 0x0F0F0F0Fu) | ((b << 4) & 0xF0F0F0F0u);
                }
#pragma unroll
                for (int j2 = 0; j2 < 4; j2 += 2) {
                    uint32_t out[2][2][4];
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            out[j][0][e] = level2(code[2 * e], j2 + j);
                            out[j][1][e] = level2(code[2 * e + 1], j2 + j);
                        }
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int d = 0; d < 2; d++) {
                            uint32_t (&o)[4] = out[j][d];
                            if constexpr (!EXACT) {
#pragma unroll
                                for (int e = 0; e < 4; e++) o[e] = cross_mul2(o[e], nn[e]);
                            }
                            cross_sts(image + cross_piece(16 * (2 * (j2 + j) + d) + w, 8 * half + c), o[0], o[1], o[2], o[3]);
                        }
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                cross_arrive(raw_empty + 8 * (ring + stage));
                cross_arrive(img_full + 16 * slot + 8 * half);
            }
            if (++stage == kCrossStages) {
                stage = 0;
                turn ^= 1;
            }
        }
        if (on_k && ok && n > 0 && cut_over() == 1) {
            // =============================== the matrix of the way back ======================================
            const int item = k_item(n), slot = item % M::kImages;
            ok = cross_wait(img_empty + 8 * slot, ((item / M::kImages) & 1) ^ 1, gone) && (item != M::kImages - 1 || cross_wait(turned, 0, gone));
            if (ok) {
#pragma unroll 1
                for (int i = tid - 12 * 32; i < kCrossTile * 16; i += kCrossTeam * 32) {
                    const uint4 v = cross_turn(i >> 4, i & 15, (lds32(M::kSigns + 4 * (i >> 9)) >> ((i >> 4) & 31)) & 1u);
                    cross_sts(M::kImg + slot * kCrossImage + cross_piece(i >> 4, i & 15), v.x, v.y, v.z, v.w);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) cross_arrive(img_full + 16 * slot + 8);
            }
        }
        if (!ok) *gone = 1;
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (LAID && warp == 8) {
            // =============================== copies: images ===============================================
            const int items = n == 0 ? 0 : solo || cut_over() == 1 ? 2 * n + 1 : 2 * n;
            int k = 0;
            for (; k < items; k++) {
                const int slot = k % M::kImages, v = solo ? k > 0 && !(k & 1) : k & 1, t = solo ? v ? (k >> 1) - 1 : (k + 1) >> 1 : k >> 1;      // item k is V (t) or K (t)
                if (t == n && cut_over() > 1) continue;
                if (!cross_wait(img_empty + 8 * slot, ((k / M::kImages) & 1) ^ 1, gone) || (k == M::kImages - 1 && !cross_wait(turned, 0, gone))) break;
                if (lane == 0) {
                    const uint8_t* const from = t == n ? p.turn_image : p.kv_images + (((int64_t)(s.kv0 + j0 + t) * H + h) * 2 + v) * kCrossImage;
                    split_expect(img_full + 16 * slot + 8, kCrossImage);
                    cross_copy(M::kImg + slot * kCrossImage, from, kCrossImage, img_full + 16 * slot + 8);
                }
                __syncwarp();
            }
            if (k < items) {                          // gave up: what is in flight gets its time to land
                if (lane == 0) atomicAdd(&g_cross_faults, 1);
                *gone = 1;
                for (int c = k > M::kImages ? k - M::kImages : 0; c < k; c++)
                    for (uint32_t w = 0; w < kCrossWaitLimit / 64; w++)
                        if (split_try_wait(img_full + 16 * (c % M::kImages) + 8, (c / M::kImages) & 1)) break;
            }
        } else if (LAID && warp == 10) {
            // =============================== norms and scales ============================================
            const int64_t unit0 = (int64_t)(s.kv0 + j0) * H + h;
            float2 scales = make_float2(0.0f, 0.0f);
            uint4 norms = make_uint4(0u, 0u, 0u, 0u);
            auto fetch = [&](int t) {
                if (t >= n) return;
                scales = p.tile_scales[unit0 + (int64_t)t * H];
                if constexpr (EXACT) norms = reinterpret_cast<const uint4*>(p.tile_norms + (unit0 + (int64_t)t * H) * 2 * kCrossTile)[lane];
            };
            fetch(0);
            bool ok = true;
            for (int t = 0; t < n && ok; t++) {
                const int slot = t % kCrossMetas;
                if (t >= kCrossMetas) ok = cross_wait(s_formed + 8 * ((t - 2) % kCrossMetas), ((t - 2) / kCrossMetas) & 1, gone);
                if (!ok) break;
                if constexpr (EXACT) *reinterpret_cast<uint4*>(window + M::kNorms + slot * M::kNormBytes + 16 * lane) = norms;
                if (lane == 0) reinterpret_cast<float2*>(window + M::kScales)[slot] = scales;
                fetch(t + 1);
                __syncwarp();
                if (lane == 0) cross_arrive(meta_full + 8 * slot);
            }
            if (!ok) *gone = 1;
        } else if (!LAID && (warp == 8 || warp == 11)) {
            // =============================== copies: K, V ================================================
            id_now = page_id(lane);
            id_next = page_id(32 + lane);
            int u = 0;
            for (; u < units; u++) {
                if ((u & 7) == 0 && u > 0) {
                    id_now = id_next;
                    id_next = page_id(4 * u + 32 + lane);
                }
                if (!cross_wait(raw_empty + 8 * (ring8 + u % kCrossStages), ((u / kCrossStages) & 1) ^ 1, gone)) break;
                copy_unit(u);
            }
            if (bad_page && which == 0) atomicAdd(&g_cross_faults, 1);
            if (u < units) {                          // gave up: what is in flight gets its time to land
                if (lane == 0) atomicAdd(&g_cross_faults, 1);
                *gone = 1;
                for (int k = u > kCrossStages ? u - kCrossStages : 0; k < u; k++)
                    for (uint32_t w = 0; w < kCrossWaitLimit / 64; w++)
                        if (split_try_wait(raw_full + 8 * (ring8 + k % kCrossStages), (k / kCrossStages) & 1)) break;
            }
        } else if (!LAID && warp == 10) {
            // =============================== norms =======================================================
            // Lane l has tokens l, l + 32, l + 64, l + 96; those of the next tile and the pages of the one after are on their way.
            const int64_t slab = p.f.num_blocks * kPageTokens * H * kSlotBytes;
            int ids[4];
            uint16_t nk[4], nv[4];
            auto fetch_ids = [&](int t) {
#pragma unroll
                for (int e = 0; e < 4; e++) ids[e] = t < n ? page_id(8 * t + 2 * e + (lane >> 4)) : 0;
            };
            auto fetch = [&](int t) {
                const int valid = t < n ? s.len - (j0 + t) * kCrossTile : 0;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint8_t* const at = p.f.kv_cache + (((int64_t)ids[e] * kPageTokens + (lane & 15)) * H + h) * kSlotBytes + kHeadDim / 2;
                    const bool in = lane + 32 * e < valid;
                    nk[e] = in ? *reinterpret_cast<const uint16_t*>(at) : (uint16_t)0;
                    nv[e] = in ? *reinterpret_cast<const uint16_t*>(at + slab) : (uint16_t)0;
                }
            };
            fetch_ids(0);
            fetch(0);
            fetch_ids(1);
            bool ok = true;
            for (int t = 0; t < n && ok; t++) {
                const int slot = t % kCrossMetas;
                float fk[4], fv[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    fk[e] = __half2float(__ushort_as_half(nk[e]));
                    fv[e] = __half2float(__ushort_as_half(nv[e]));
                }
                fetch(t + 1);
                fetch_ids(t + 2);
                if (t >= kCrossMetas) ok = cross_wait(s_formed + 8 * ((t - 2) % kCrossMetas), ((t - 2) / kCrossMetas) & 1, gone);
                if (!ok) break;
                bool has_k, has_v;
                const int by_k = cross_norm_exponent(fk, kCrossInImage, has_k), by_v = cross_norm_exponent(fv, EXACT ? kCrossUnderP : kCrossInImage, has_v);
                const float sk = cross_power(by_k), sv = cross_power(by_v);
                uint8_t* const to = window + M::kNorms + slot * M::kNormBytes;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int tok = lane + 32 * e;
                    if constexpr (EXACT) {
                        reinterpret_cast<__half*>(to)[tok] = __float2half_rn(fk[e]);      // as they are: the powers of two are part of the exponents
                        reinterpret_cast<__half*>(to)[kCrossTile + tok] = __float2half_rn(fv[e]);
                    } else {
                        reinterpret_cast<uint32_t*>(to)[tok] = pack_half2(fk[e] * sk, fk[e] * sk);
                        reinterpret_cast<__half*>(to + 4 * kCrossTile)[tok] = __float2half_rn(fv[e] * sv);
                    }
                }
                if (lane == 0) reinterpret_cast<float2*>(window + M::kScales)[slot] = make_float2(EXACT ? 1.0f : cross_power(-by_k), has_v ? (float)-by_v : kCrossNoNorm);
                __syncwarp();
                if (lane == 0) cross_arrive(meta_full + 8 * slot);
            }
            if (!ok) *gone = 1;
        } else if (warp == 9 && n > 0) {
            // =============================== matrix products ==============================================
            constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(kCrossTile >> 3) << 17) | ((uint32_t)(kCrossTile >> 4) << 24);      // fp16 x fp16 -> fp32, 128 x 128
            const uint64_t q_desc = cross_desc(M::kQ), img_desc = cross_desc(M::kImg);
            constexpr uint64_t kImage16 = kCrossImage / 16;
            auto scores = [&](int i, int slot) {      // S of group i from the K in a slot
                const uint64_t k_desc = img_desc + (uint64_t)slot * kImage16, a_desc = q_desc + (EXACT || solo ? 0 : i) * kImage16;
#pragma unroll
                for (int a = 0; a < (EXACT ? 2 : 1); a++)
#pragma unroll
                    for (int kk = 0; kk < 8; kk++) {
                        const uint64_t off = (uint64_t)((kk >> 2) * 1024 + (kk & 3) * 2);      // 16 dims on, in units of 16 bytes
                        mq_mma(128 * i, a_desc + a * kImage16 + off, k_desc + off, idesc, a || kk ? 1u : 0u);
                    }
                cross_commit(s_full + 8 * i);
            };
            auto formed = [&](int t) {                // S (t) of all groups
                cross_commit(img_empty + 8 * (k_item(t) % M::kImages));
                cross_commit(s_formed + 8 * (t % kCrossMetas));
            };
            auto values = [&](int i, int slot, int half, bool more) {      // O of group i += P V of 64 tokens
                const uint64_t v_desc = img_desc + (uint64_t)slot * kImage16 + (uint64_t)(half * 1024);
#pragma unroll
                for (int kk = 0; kk < 4; kk++) mq_mma_ts(256 + 128 * i, 128 * i + 32 * half + 8 * kk, v_desc + (uint64_t)(kk * 2), idesc, more || half || kk ? 1u : 0u);
            };
            auto image_there = [&](int item, int half) { return cross_wait(img_full + 16 * (item % M::kImages) + (LAID ? 8 : 8 * half), (item / M::kImages) & 1, gone); };
            if constexpr (!LAID) {
                tc_fence_before();
                asm volatile("bar.sync 3, 288;" ::: "memory");     // the rows' warps have the queries in their place
            }
            bool ok = !LAID || cross_wait(raw_full, 0, gone);
            if (ok && halves && elect_one()) {              // the queries' rotation: their own type against ones, into S's place
                const uint32_t q_idesc = idesc | (p.f.q_dtype == TQ_BF16 ? 1u << 7 | 1u << 10 : 0u);
                const uint64_t way = cross_desc(M::kWay);
#pragma unroll 1
                for (int kk = 0; kk < 8 * q_tiles; kk++) {
                    const uint64_t off = (uint64_t)(((kk >> 2) & 1) * 1024 + (kk & 3) * 2);
                    mq_mma(128 * (kk >> 3), q_desc + (uint64_t)(kk >> 3) * kImage16 + off, way + off, q_idesc, kk & 7 ? 1u : 0u);
                }
                cross_commit(turned);
            }
            __syncwarp();
            asm volatile("bar.sync 2, 288;" ::: "memory");         // the rows' warps have written the images
            tc_fence_after();
            if (!halves && elect_one()) cross_commit(turned);
            __syncwarp();
            // Two tiles of query rows: step u is group u % 2 and tile u / 2 of the tokens; one: group u % 2, tile u.  After P V of a step comes the next S
            // of its group.
            const int first = solo ? min(2, n) : 1, steps = solo ? n : 2 * n;
            for (int t = 0; t < first && ok; t++) {
                ok = image_there(k_item(t), 0) && image_there(k_item(t), 1);
                tc_fence_after();
                if (ok && elect_one()) {
                    scores(solo ? t : 0, k_item(t) % M::kImages);
                    if (!solo) scores(1, k_item(0) % M::kImages);
                    formed(t);
                }
                __syncwarp();
            }
            for (int u = 0; u < steps && ok; u++) {
                const int i = u & 1, t = solo ? u : u >> 1, next = t + (solo ? 2 : 1), k = u >> 1;
                const bool last = solo || i == 1;     // group of this tile
                const bool fresh = solo || i == 0;    // images that this step is the first to read
                if constexpr (LAID) {                 // they are there before P is: one wait between P and the products
                    ok = !fresh || (image_there(v_item(t), 1) && (next >= n || image_there(k_item(next), 1)));
                    ok = ok && cross_wait(p_full + 8 * i, k & 1, gone);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        values(i, v_item(t) % M::kImages, 0, k > 0);
                        values(i, v_item(t) % M::kImages, 1, true);
                        if (last) cross_commit(img_empty + 8 * (v_item(t) % M::kImages));
                        if (next >= n) cross_commit(o_full + 8 * i);
                        else scores(i, k_item(next) % M::kImages);
                        if (next < n && last) formed(next);
                    }
                    __syncwarp();
                    continue;
                }
                ok = cross_wait(p_full + 8 * i, k & 1, gone);
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    if (fresh) ok = ok && image_there(v_item(t), half);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        values(i, v_item(t) % M::kImages, half, k > 0);
                        if (half == 1 && last) cross_commit(img_empty + 8 * (v_item(t) % M::kImages));
                        if (half == 1 && next >= n) cross_commit(o_full + 8 * i);
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (next < n) {
                    if (fresh) ok = image_there(k_item(next), 0) && image_there(k_item(next), 1);
                    tc_fence_after();
                    if (ok && elect_one()) {
                        scores(i, k_item(next) % M::kImages);
                        if (last) formed(next);
                    }
                    __syncwarp();
                }
            }
            if (ok && cut_over() == 1) {              // the way back: two parts of O's rows, in S's place, against the matrix in V's; of one tile, both groups' O
                ok = image_there(k_item(n), 1);
                for (int i = 0; i < (solo && n == 1 ? 1 : 2) && ok; i++) {
                    ok = cross_wait(a_full + 8 * i, 0, gone);
                    tc_fence_after();
                    if (ok && elect_one()) {
                        const uint64_t turn = img_desc + (uint64_t)(k_item(n) % M::kImages) * kImage16;
                        const int to = solo ? 0 : i;
#pragma unroll 1
                        for (int kk = 0; kk < 16; kk++)
                            mq_mma_ts(256 + 128 * to, 128 * i + 8 * kk, turn + (uint64_t)(((kk >> 2) & 1) * 1024 + (kk & 3) * 2), idesc, kk || to != i ? 1u : 0u);
                        if (!solo || i == 1 || n == 1) cross_commit(d_full + 8 * to);
                    }
                    __syncwarp();
                }
            }
            if (!ok) {
                if (lane == 0 && !*gone) atomicAdd(&g_cross_faults, 1);
                *gone = 1;
                if (elect_one()) cross_commit(drained);      // products in flight end before tensor memory is given back
                __syncwarp();
                for (uint32_t w = 0; w < kCrossWaitLimit / 64; w++)
                    if (split_try_wait(drained, 0)) break;
            }
        }
    } else {
        // =============================== a row a thread ===================================================
        // A row of S is read 32 columns at a time: kept in registers it would take more than the 128 a thread that leave the look-ups theirs, and there is no
        // first-level cache to speak of behind this much shared memory for what spills.
        if constexpr (LAID) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
        const int i = warp >> 2, r = tid & 127, row = row0 + (solo ? 0 : i * kCrossTile) + r;
        const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tm_s = 128 * i + lane_at, tm_o = 256 + 128 * i + lane_at;      // tensor memory is allocated whole: it begins at zero
        bool ok = true;
        // ---- the queries: rotated, by a power of two to [512, 1024), into the images.  One tile: half of a row's columns each group --------------
        float q_scale = 0.0f;
        if (n > 0) {
            if constexpr (!LAID) {
                load_queries(256);
                asm volatile("bar.sync 3, 288;" ::: "memory");      // and tensor memory is there
                tc_fence_after();
            }
            const uint32_t image = M::kQ + (solo ? 0 : i) * kCrossImage;
            auto take = [&](float top) {              // the largest of the row: what its numbers are multiplied by
                const int by = cross_exponent(top * p.f.scale, 9);
                q_scale = fabsf(p.f.k_scale) * cross_power(-by);
                return (p.f.k_scale < 0.0f ? -cross_power(by) : cross_power(by)) * p.f.scale;
            };
            if (halves) {
                ok = cross_wait(turned, 0, gone);
                tc_fence_after();
                if (ok) {
                    float top = 0.0f, v[32];
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        cross_ld(tm_s - (solo ? 128 * i : 0) + 32 * c, v);
                        cross_ld_wait(v);
#pragma unroll
                        for (int e = 0; e < 32; e++) top = fmaxf(top, fabsf(v[e]));
                    }
                    const float f = take(top);
#pragma unroll 1
                    for (int c = solo ? 2 * i : 0; c < (solo ? 2 * i + 2 : 4); c++) {
                        cross_ld(tm_s - (solo ? 128 * i : 0) + 32 * c, v);
                        cross_ld_wait(v);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            uint32_t a[4], b[4];
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const float x = v[8 * e + 2 * k] * f, y = v[8 * e + 2 * k + 1] * f;
                                a[k] = pack_half2(x, y);
                                const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&a[k]));
                                b[k] = pack_half2(x - back.x, y - back.y);
                            }
                            cross_sts(image + cross_piece(r, 4 * c + e), a[0], a[1], a[2], a[3]);
                            if constexpr (EXACT) cross_sts(image + kCrossImage + cross_piece(r, 4 * c + e), b[0], b[1], b[2], b[3]);
                        }
                    }
                }
            } else {                                  // 32-bit queries: a warp a row, each warp the rows of its threads
                const float4 sign = reinterpret_cast<const float4*>(p.f.signs)[lane];
#pragma unroll 1
                for (int j = 0; j < 32; j++) {
                    const int rr = (warp & 3) * 32 + j, rq = rr + (solo ? 0 : i * kCrossTile);
                    float v[4], top = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = rq < q_rows && 4 * lane + e < D ? load_q(p.f.q, TQ_F32, row_of(rq) * D + 4 * lane + e) : 0.0f;
                    v[0] *= sign.x; v[1] *= sign.y; v[2] *= sign.z; v[3] *= sign.w;
                    split_fwht<4>(v, lane);
#pragma unroll
                    for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(v[e]));
                    const float keep = q_scale, f = take(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top))));
                    if (lane != j) q_scale = keep;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] *= f;
                    if (solo && i == 1) continue;     // (the first group writes them)
                    const uint32_t a = pack_half2(v[1], v[0]), b = pack_half2(v[3], v[2]), to = image + cross_piece(rr, lane >> 1) + 8 * (lane & 1);
                    *reinterpret_cast<uint2*>(window + to) = make_uint2(a, b);
                    if constexpr (EXACT) {
                        const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a)), fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
                        *reinterpret_cast<uint2*>(window + to + kCrossImage) = make_uint2(pack_half2(v[1] - fa.x, v[0] - fa.y), pack_half2(v[3] - fb.x, v[2] - fb.y));
                    }
                }
            }
            fence_proxy_async();
            tc_fence_before();
            asm volatile("bar.sync 2, 288;" ::: "memory");
            if (!ok) *gone = 1;
        }
        // P is taken relative to 2^m, m the running maximum of (logit + ev), 2^ev the scale of the tile's V: a token's share of the row, not its weight alone, decides
        // how many bits of it are left.  l is the sum of the weights, s that of P, both in units of 2^m; |O| is below s times the largest entry of V's image.
        float m = kNoMax, l = 0.0f, s_p = 0.0f;
        const int turns = solo ? (n + 1 - i) >> 1 : n;
        for (int k = 0; k < turns && ok; k++) {
            const int t = solo ? 2 * k + i : k;
            ok = cross_wait(meta_full + 8 * (t % kCrossMetas), (t / kCrossMetas) & 1, gone) && cross_wait(s_full + 8 * i, k & 1, gone);
            if (!ok) break;
            tc_fence_after();
            const uint32_t norms = M::kNorms + (uint32_t)(t % kCrossMetas) * M::kNormBytes;
            const float2 scales = cross_lds_f2(M::kScales + 8 * (t % kCrossMetas));
            // A masked logit is -inf times kf: kf is no zero (a scale of zero).
            const float kf = fmaxf(scales.x * q_scale, 1e-36f), ev = scales.y;
            const int valid = s.len - (j0 + t) * kCrossTile;
            const P2 kf2 = pk(kf, kf);
            // Where the norms multiply P as they are (exact) it is the weight that comes from the exponential, else P.
            const float weight = EXACT ? 1.0f : cross_power(-(int)ev), share = EXACT ? cross_power((int)ev) : 1.0f;      // of one of its sum
            // Norms of eight tokens, fp16 as in the cache (a broadcast load costs a wavefront for every four bytes: half of what fp32 ones would).
            auto times_norms = [&](int which, int col, float* v) {
                const uint4 a = lds128(norms + 2 * (kCrossTile * which + col));
                const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                    up(mul2(pk(v[2 * e], v[2 * e + 1]), pk(f.x, f.y)), v[2 * e], v[2 * e + 1]);
                }
            };
            // exp2 of 16 columns into fp16 pairs, and their sum
            auto exponentials = [&](int col, float* v, P2 sub, P2& sum, uint32_t* ph) {
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    up(fma2(pk(v[e], v[e + 1]), kf2, sub), v[e], v[e + 1]);
                    v[e] = fast_exp2(v[e]);
                    v[e + 1] = fast_exp2(v[e + 1]);
                    sum = add2(sum, pk(v[e], v[e + 1]));
                }
                if constexpr (EXACT) {
#pragma unroll
                    for (int e = 0; e < 16; e += 8) times_norms(1, col + e, v + e);
                }
#pragma unroll
                for (int e = 0; e < 16; e += 2) ph[e >> 1] = pack_half2(v[e], v[e + 1]);
            };
            P2 sum = pk(0.0f, 0.0f);
            bool done = false;
            // In the common case the running maximum needs no look at the row: P is worked out from the maximum that there is, and its sum tells whether any of it
            // is too large (2^9; NaN and infinity too).  P waits in registers until the warp knows, as it takes the place of S.
            if (k > 0 && valid >= kCrossTile) {
                const float from = EXACT ? -m : ev - m;
                const P2 sub = pk(from, from);
                uint32_t ph[64];
                float v[2][16];                       // the next columns are on their way
                cross_ld16(tm_s, v[0]);
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    cross_ld_wait16(v[c & 1]);
                    if (c < 7) cross_ld16(tm_s + 16 * (c + 1), v[(c + 1) & 1]);
                    if constexpr (EXACT) {
#pragma unroll
                        for (int e = 0; e < 16; e += 8) times_norms(0, 16 * c + e, v[c & 1] + e);
                    }
                    exponentials(16 * c, v[c & 1], sub, sum, ph + 8 * c);
                }
                float sa, sb;
                up(sum, sa, sb);
                done = __all_sync(0xffffffffu, (sa + sb) * share <= 512.0f);
                if (done) {
                    cross_st(tm_s, ph);
                    cross_st(tm_s + 32, ph + 32);
                }
            }
            if (!done) {
                // The maximum first, then P, 32 columns at a time: the columns of P (c) are those of S (c / 2), read already.
                auto columns = [&](int c, float (&v)[32]) {      // S of 32 columns, as it counts
                    cross_ld(tm_s + 32 * c, v);
                    cross_ld_wait(v);
                    if constexpr (EXACT) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) times_norms(0, 32 * c + e, v + e);
                    }
                    if (valid < 32 * c + 32) {        // the last tile of the sequence
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            if (32 * c + e >= valid) v[e] = -INFINITY;
                    }
                };
                float v[32], top = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < 4; c++) {
                    columns(c, v);
#pragma unroll
                    for (int e = 0; e < 32; e++) top = fmaxf(top, v[e]);
                }
                top = top * kf + ev;                  // kf > 0
                const bool raise = top > m + kCrossRaise;
                if (__any_sync(0xffffffffu, raise)) {
                    const float c = raise ? fast_exp2(m - top) : 1.0f;
                    if (raise) m = top;
                    l *= c;
                    s_p *= c;
                    if (k > 0) {                      // S is there, so the products before it are done with O
#pragma unroll 1
                        for (int a = 0; a < 4; a++) {
                            cross_ld(tm_o + 32 * a, v);
                            cross_ld_wait(v);
#pragma unroll
                            for (int e = 0; e < 32; e++) v[e] *= c;
                            cross_st(tm_o + 32 * a, reinterpret_cast<const uint32_t*>(v));
                        }
                    }
                }
                const float from = EXACT ? -m : ev - m;
                const P2 sub = pk(from, from);
                sum = pk(0.0f, 0.0f);
#pragma unroll 1
                for (int c = 0; c < 4; c++) {
                    uint32_t ph[16];
                    columns(c, v);
                    exponentials(32 * c, v, sub, sum, ph);
                    exponentials(32 * c + 16, v + 16, sub, sum, ph + 8);
                    cross_st16(tm_s + 16 * c, ph);
                }
            }
            float sa, sb;
            up(sum, sa, sb);
            l += (sa + sb) * weight;
            s_p += (sa + sb) * share;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) cross_arrive(p_full + 8 * i);
        }
        // ---- the row: normalized, brought back, out or to the partials ---------------------------------
        if (ok && n > 0) ok = cross_wait(o_full + 8 * (turns > 0 ? i : 0), 0, gone);
        if (!ok) *gone = 1;
        tc_fence_after();
        // One tile's two groups bring their sums to the larger of their maxima.  (What is written to the queries' place: by now all S are formed.)
        float scale = 1.0f;
        const bool cut = cut_over() > 1;
        if (solo && n > 0 && !cut) {
            float4* const sums = reinterpret_cast<float4*>(window + M::kQ);
            sums[tid] = make_float4(m, l, s_p, 0.0f);
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float4 other = sums[tid ^ 128];
            const float mm = fmaxf(m, other.x), c1 = fast_exp2(other.x - mm);
            scale = fast_exp2(m - mm);
            // (Each product rounded by itself: the two groups have to come to the same bits, as the power of two that their parts are brought to follows from them.)
            l = __fadd_rn(__fmul_rn(l, scale), __fmul_rn(other.y, c1));
            s_p = __fadd_rn(__fmul_rn(s_p, scale), __fmul_rn(other.z, c1));
            m = mm;
            if (*gone) ok = false;
        }
        if (__all_sync(0xffffffffu, ok)) {
            const bool none = l == 0.0f, live = row < rows;
            const int by = cross_exponent(s_p, EXACT ? 12 : 5);
            const float to_parts = cross_power(by);
            const int qi = row / G, g = row - qi * G;
            const int64_t to = live ? (int64_t)(q_first + qi) * p.f.real_heads + h * G + g : -1;
            const float lse2 = none ? -INFINITY : m + log2f(l);
            if (cut) {
                // A partial of the group's own, as O has its columns.  There are two for each cut; rows that one group has to itself leave the other empty.
                const int64_t part = (int64_t)p.total_q * p.f.real_heads, at = (2 * split + (solo ? i : 0)) * part + to;
                if (live) {
                    p.partial_lse[at] = lse2;
                    if (!solo) p.partial_lse[at + part] = -INFINITY;
                }
                scale = p.f.v_scale / l;
#pragma unroll 1
                for (int c = 0; c < 4 && turns > 0; c++) {
                    float v[32];
                    __syncwarp();
                    cross_ld(tm_o + 32 * c, v);
                    cross_ld_wait(v);
                    float4* const dst = reinterpret_cast<float4*>(p.partial_o + at * kCrossTile + 32 * c);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (live && !none) dst[e] = make_float4(v[4 * e] * scale, v[4 * e + 1] * scale, v[4 * e + 2] * scale, v[4 * e + 3] * scale);
                }
            }
            if (turns > 0 && !cut) {
                // O as two fp16 parts in S's place, by a power of two to below 2^15: the images have levels below 4, in the one form times norms below 2^7.
                scale *= to_parts;
#pragma unroll 1
                for (int c = 0; c < 4; c++) {
                    float v[32];
                    cross_ld(tm_o + 32 * c, v);
                    cross_ld_wait(v);
                    uint32_t a[16], b[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const float x = none ? 0.0f : v[2 * e] * scale, y = none ? 0.0f : v[2 * e + 1] * scale;
                        a[e] = pack_half2(x, y);
                        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&a[e]));
                        b[e] = pack_half2(x - back.x, y - back.y);
                    }
                    cross_st16(tm_s + 16 * c, a);
                    cross_st16(tm_s + 64 + 16 * c, b);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) cross_arrive(a_full + 8 * i);
            }
            if (p.f.out_lse && live && !cut && !(solo && i == 1)) p.f.out_lse[to] = lse2 * 0.6931471805599453f;
            const int mine = solo ? 0 : i;            // whose O's place the result is in
            if (n > 0 && !cut) ok = cross_wait(d_full + 8 * mine, 0, gone);
            tc_fence_after();
            // 64 bytes each of the warp's rows go to memory by way of shared memory, neighbouring lanes to neighbouring pieces of a row.
            const uint32_t stage = M::kQ + 4096 + warp * 2048;
            auto place = [&](int row, int piece) { return stage + row * 64 + 16 * (piece ^ ((row >> 1) & 3)); };
            auto rows_out = [&](const uint32_t* v, int at_byte) {
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 4; e++) cross_sts(place(lane, e), v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int r = 8 * j + (lane >> 2), piece = lane & 3;
                    const uint4 x = lds128(place(r, piece));
                    const int64_t row_to = __shfl_sync(0xffffffffu, to, r);
                    if (row_to >= 0 && at_byte + 16 * piece < 2 * D) *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.f.out) + row_to * 2 * D + at_byte + 16 * piece) = x;
                }
            };
            const bool whole = p.f.out_dtype != TQ_F32 && D % 8 == 0 && (reinterpret_cast<uintptr_t>(p.f.out) & 15) == 0;
            const float f = p.f.v_scale * p.f.scale * cross_power(-by) * (1.0f / l);
#pragma unroll 1
            for (int c = solo ? 2 * i : 0; c < (solo ? 2 * i + 2 : 4) && ok && !cut; c++) {
                float v[32];
                __syncwarp();
                if (n > 0) {
                    cross_ld(256 + 128 * mine + lane_at + 32 * c, v);
                    cross_ld_wait(v);
                }
#pragma unroll
                for (int e = 0; e < 32; e++) v[e] = none ? 0.0f : v[e] * f;
                if (whole) {
                    uint32_t u[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        if (p.f.out_dtype == TQ_BF16) {
                            const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
                            u[e] = *reinterpret_cast<const uint32_t*>(&t);
                        } else {
                            u[e] = pack_half2(v[2 * e], v[2 * e + 1]);
                        }
                    }
                    rows_out(u, 64 * c);
                } else if (live) {
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        if (32 * c + e >= D) continue;
                        const int64_t o = to * D + 32 * c + e;
                        if (p.f.out_dtype == TQ_BF16) reinterpret_cast<__nv_bfloat16*>(p.f.out)[o] = __float2bfloat16_rn(v[e]);
                        else if (p.f.out_dtype == TQ_F16) reinterpret_cast<__half*>(p.f.out)[o] = __float2half_rn(v[e]);
                        else reinterpret_cast<float*>(p.f.out)[o] = v[e];
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(512));
    }
}

// A warp a row (query row, query head): the parts of the splits.
__global__ void __launch_bounds__(128) cross_join_kernel(const __grid_constant__ CrossParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), rows = (int64_t)p.total_q * p.f.real_heads;
    grid_launch_dependents();
    grid_dependency_wait();
    if (at >= rows) return;
    float lse = lane < 2 * p.splits ? p.partial_lse[lane * rows + at] : -INFINITY;      // of the first 32 parts, a lane each; fewer count, see below
    // a row that belongs to no sequence, to one that was left out or to one that a single block takes is left as it is
    const int t = (int)(at / p.f.real_heads);
    int cuts = 1;
    CrossRanges ranges;
    for (int base = 0; base < p.f.batch; base += 32) {
        const int b = base + lane, c0[1] = {b < p.f.batch ? p.cu_q[b] : 0}, c1[1] = {b < p.f.batch ? p.cu_q[b + 1] : 0};
        int qlen[1], faults = 0;
        ranges.rows(p, c0, c1, lane, qlen, faults);
        const uint32_t where = __ballot_sync(0xffffffffu, qlen[0] > 0 && c0[0] <= t && t < c1[0]);
        if (where) {
            bool bad;
            cuts = cross_cuts(p, cross_len(p, base + __ffs(where) - 1, bad));
            break;
        }
    }
    if (cuts == 1) return;
    const int parts = 2 * cuts;
    if (lane >= parts) lse = -INFINITY;
    float m = lse, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 32 + lane; s < parts; s += 32) m = fmaxf(m, p.partial_lse[s * rows + at]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    for (int base = 0; base < parts; base += 32) {
        if (base > 0) lse = base + lane < parts ? p.partial_lse[(base + lane) * rows + at] : -INFINITY;
        const float mine = lse == -INFINITY ? 0.0f : fast_exp2(lse - m);
#pragma unroll 4
        for (int s = 0; s < min(32, parts - base); s++) {
            const float w = __shfl_sync(0xffffffffu, mine, s);
            const float* const v = p.partial_o + ((base + s) * rows + at) * kCrossTile + 64 * (lane & 1) + (lane >> 1);      // dim 8 w + d is column 16 d + w
            l += w;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float x = v[16 * e];
                if (w != 0.0f) o[e] = fmaf(w, x, o[e]);      // (else nothing has been written there)
            }
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] *= inv;
    SplitParams f = p.f;
    f.real_group = 1;
    split_finish<kCrossTile>(f, p.f.signs, t, (int)(at - (int64_t)t * p.f.real_heads), 0, o, l == 0.0f ? -INFINITY : m + log2f(l), lane);
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
int device_sm_count(int* out);
int encode_cache_map(CUtensorMap* map, const void* kv_cache, int64_t num_blocks, int64_t row_bytes, int box_bytes, int slabs);

int cross_fault_count(int32_t* out) {
    TQ_CUDA(cudaMemcpyFromSymbol(out, g_cross_faults, sizeof(int32_t)));
    return TQ_OK;
}

static size_t cross_up(size_t x) { return (x + 255) & ~(size_t)255; }

struct CrossLayout {
    bool laid;
    int64_t items, kv_room;     // tiles or pairs of tiles of query rows, tiles of tokens, at most
    int splits;
    size_t turn, scales, norms, partial_lse, partial_o, end;      // the images of K and V are in front
};
static bool cross_exact(int out_dtype) { return out_dtype != TQ_BF16; }
static CrossLayout cross_layout(int batch, int total_q, int64_t total_tokens, int heads, int kv_heads, int max_pages, int out_dtype, int sms) {
    CrossLayout l;
    const bool exact = cross_exact(out_dtype);
    const int64_t per = (exact ? 1 : 2) * kCrossTile, rows = (int64_t)total_q * (heads / kv_heads);
    l.items = rows / per + batch;                           // every sequence may end inside one
    l.kv_room = total_tokens / kCrossTile + batch;
    l.laid = rows > (int64_t)kCrossLaid * kCrossTile * batch;
    // As many cuts of the longest sequence's tokens as fill the SMs, of two tiles (one a warpgroup) at least; see cross_cuts.
    const int64_t some = (rows + per - 1) / per, blocks = (some > batch ? some : batch) * kv_heads;
    const int64_t longest = (int64_t)max_pages * kPageTokens < total_tokens ? (int64_t)max_pages * kPageTokens : total_tokens;
    const int64_t most = (longest + 2 * kCrossTile - 1) / (2 * kCrossTile), fit = sms / blocks;
    l.splits = (int)(fit < most ? fit : most);
    if (l.splits < 1) l.splits = 1;
    const size_t units = l.laid ? (size_t)l.kv_room * kv_heads : 0;
    l.turn = units * 2 * kCrossImage;
    l.scales = l.turn + (l.laid ? 2 * kCrossImage : 0);
    l.norms = l.scales + cross_up(units * sizeof(float2));
    l.partial_lse = l.norms + (exact ? cross_up(units * 2 * kCrossTile * 2) : 0);
    const size_t cut = l.splits > 1 ? (size_t)2 * l.splits * total_q * heads : 0;
    l.partial_o = l.partial_lse + cross_up(cut * 4);
    l.end = l.partial_o + cross_up(cut * kCrossTile * 4);
    return l;
}

template <bool EXACT, bool LAID>
static int launch_cross(const CrossParams& p, int sms, int64_t blocks, cudaStream_t s) {
    constexpr size_t kSmem = CrossMap<EXACT, LAID>::kSmem;
    static bool configured[64] = {};
    int dev = 0;
    TQ_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        TQ_CUDA(cudaFuncSetAttribute(cross_attend_kernel<EXACT, LAID>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    if constexpr (LAID) {
        const int64_t units = p.kv_room * p.f.kv_heads, lay = units < 4 * sms ? units : 4 * sms;
        TQ_CUDA(launch_serialized(cross_lay_out_kernel<EXACT>, dim3((unsigned)lay), dim3(kLayThreads), 0, s, p));
    }
    TQ_CUDA(launch_serialized(cross_attend_kernel<EXACT, LAID>, dim3((unsigned)blocks), dim3(LAID ? kCrossRowThreads : kCrossThreads), kSmem, s, p));
    if (p.splits > 1) {
        const int64_t rows = (int64_t)p.total_q * p.f.real_heads;
        TQ_CUDA(launch_serialized(cross_join_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, s, p));
    }
    return TQ_OK;
}

}  // namespace tq

extern "C" size_t tq_cross_workspace_bytes(int batch, int total_q, int64_t total_tokens, int num_q_heads, int num_kv_heads, int max_pages, int out_dtype) {
    int sms = 0;
    if (batch < 1 || total_q < 1 || total_tokens < 0 || num_kv_heads < 1 || num_q_heads < num_kv_heads || max_pages < 1 || tq::device_sm_count(&sms) != TQ_OK) return 0;
    return tq::cross_layout(batch, total_q, total_tokens, num_q_heads, num_kv_heads, max_pages, out_dtype, sms).end;
}

extern "C" int tq_cross(const void* q, int q_dtype, int total_q, const int32_t* cu_seqlens_q, int batch, int num_q_heads, int num_kv_heads, int head_dim,
                        const void* kv_cache, int64_t num_blocks, int block_size, int slot_bytes, const int32_t* page_table, int max_pages,
                        const int32_t* seq_lens, int64_t total_tokens, const float* signs, float sm_scale, void* workspace, size_t workspace_bytes, void* out,
                        int out_dtype, float* out_lse, void* stream) {
    using namespace tq;
    TQ_REQUIRE(batch >= 0 && total_q >= 0 && num_blocks >= 0 && total_tokens >= 0, TQ_ERR_INVALID, "negative size");
    if (batch == 0 || total_q == 0) return TQ_OK;
    TQ_REQUIRE(q && cu_seqlens_q && kv_cache && page_table && seq_lens && signs && workspace && out, TQ_ERR_INVALID, "null pointer");
    TQ_REQUIRE(q_dtype >= TQ_F32 && q_dtype <= TQ_BF16 && out_dtype >= TQ_F32 && out_dtype <= TQ_BF16, TQ_ERR_INVALID, "unknown dtype");
    TQ_REQUIRE(head_dim > 64 && head_dim <= 128, TQ_ERR_UNSUPPORTED, "head_dim must be in 65 ... 128, got %d", head_dim);
    TQ_REQUIRE(block_size == 16 && slot_bytes == kSlotBytes, TQ_ERR_UNSUPPORTED, "16-token pages of 80-byte slots only, got %d and %d", block_size, slot_bytes);
    TQ_REQUIRE(num_kv_heads >= 1 && num_q_heads >= 1 && num_q_heads % num_kv_heads == 0, TQ_ERR_INVALID, "%d query heads on %d KV heads", num_q_heads, num_kv_heads);
    TQ_REQUIRE(max_pages >= 1 && max_pages <= 1 << 26, TQ_ERR_INVALID, "bad size");
    TQ_REQUIRE(((uintptr_t)kv_cache & 15) == 0 && ((uintptr_t)signs & 15) == 0 && ((uintptr_t)workspace & 255) == 0, TQ_ERR_INVALID,
               "kv_cache and signs must be 16-byte aligned, the workspace 256-byte");
    TQ_REQUIRE(num_blocks > 0, TQ_ERR_INVALID, "the cache has no pages");
    int sms = 0;
    int rc = device_sm_count(&sms);
    if (rc != TQ_OK) return rc;
    const bool exact = cross_exact(out_dtype);
    const int G = num_q_heads / num_kv_heads;
    const CrossLayout l = cross_layout(batch, total_q, total_tokens, num_q_heads, num_kv_heads, max_pages, out_dtype, sms);
    const int64_t blocks = l.items * num_kv_heads * l.splits;
    TQ_REQUIRE((int64_t)total_q * num_q_heads < 1ll << 31 && l.kv_room < 1 << 30 && blocks < 1ll << 31, TQ_ERR_UNSUPPORTED,
               "too many rows or tokens for one launch");
    TQ_REQUIRE(workspace_bytes >= l.end, TQ_ERR_WORKSPACE, "workspace too small: %zu < %zu", workspace_bytes, l.end);

    CrossParams p{};
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.f.q = q;
    p.f.kv_cache = static_cast<const uint8_t*>(kv_cache);
    p.f.page_indices = page_table;
    p.f.seq_lens = seq_lens;
    p.f.signs = signs;
    p.f.out = out;
    p.f.out_lse = out_lse;
    p.f.num_blocks = num_blocks;
    p.f.batch = batch;
    p.f.kv_heads = num_kv_heads;
    p.f.max_pages = max_pages;
    p.f.q_dtype = q_dtype;
    p.f.out_dtype = out_dtype;
    p.f.nq = 1;
    p.f.real_heads = num_q_heads;
    p.f.real_group = G;
    p.f.head_dim = head_dim;
    p.cu_q = cu_seqlens_q;
    p.kv_images = ws;
    p.turn_image = ws + l.turn;
    p.tile_scales = reinterpret_cast<float2*>(ws + l.scales);
    p.tile_norms = reinterpret_cast<uint16_t*>(ws + l.norms);
    p.partial_lse = reinterpret_cast<float*>(ws + l.partial_lse);
    p.kv_room = l.kv_room;
    p.partial_o = reinterpret_cast<float*>(ws + l.partial_o);
    p.total_q = total_q;
    p.splits = l.splits;
    const double inv = 1.0 / std::sqrt((double)kHeadDim);
    p.f.scale = (float)inv;
    for (int k = 0; k < 16; k++) {
        const __half v = __float2half_rn((float)(kCrossLevelScale * kCentroidsN01_4bit[k]));
        memcpy(&p.level_h[k], &v, 2);
    }
    p.f.v_scale = (float)(inv / kCrossLevelScale);
    p.f.k_scale = (float)(inv / kCrossLevelScale * (double)sm_scale * 1.4426950408889634);
    rc = encode_cache_map(&p.f.cache_map, kv_cache, num_blocks, (int64_t)num_kv_heads * slot_bytes, slot_bytes, 1);
    if (rc != TQ_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (l.laid) return exact ? launch_cross<true, true>(p, sms, blocks, s) : launch_cross<false, true>(p, sms, blocks, s);
    return exact ? launch_cross<true, false>(p, sms, blocks, s) : launch_cross<false, false>(p, sms, blocks, s);
}
