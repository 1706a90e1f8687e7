// Many queries a sequence over its cached states, every query over all of them: attention of a decoder's prompt to an encoder's states in the
// quantized cache, on the 5th-generation tensor cores.
//
//   out[t, h] = sum_j softmax_j(q[t, h] . k[j] * scale) v[j],      j over the tokens of the cache, t over the query rows of the sequence
//
// Queries and cached rows stay in the rotated domain (K^ = H S K, V^ = H S V): a query is rotated once, an output row is rotated back
// once, and what is between is two matrix products.  With hundreds of query rows those bound it, 4 x 128 operations for each row and
// token, and a cached row would be dequantized again for every 256 query rows; so a first kernel does that once.
//
//   lay out   K^ and V^ of 128 tokens and one head, and 128 rotated query rows of one head, become the two 32 KB shared-memory images that the
//             tensor core reads (rows of 128 bytes, 16-byte pieces swizzled by the row, V^ transposed), so that the second kernel
//             brings a tile with one contiguous bulk copy and needs no tensor map.  The query heads that share a KV head are rows of
//             one tile: row r is query r / G, head r % G.
//   attend    A block takes 256 query rows (two tiles) of one head and a range of the tokens.  Two warpgroups own a tile each, a thread a
//             row; one warp copies tiles into a ring, one issues S = Q K^^T and O += P V^.  S and then P (fp16, in the same columns) of a
//             tile and its O are all of tensor memory: 2 x (128 + 128) columns.  While one tile's row maxima and exponentials are worked
//             out, the tensor core works for the other tile.  The running maximum is raised only when a logit exceeds it by 2^8, which
//             makes rescaling O rare; a row needs no other thread but its own.
//   join      Where few rows have long sequences, the tokens are cut over several blocks, whose rows a third kernel joins.
//
// Numbers are fp16 in the tensor core with fp32 sums, brought into fp16's range by powers of two: a query row by its largest element, the norms of
// K and V by the largest of the tile.
//   16-bit results of 8 bits (bf16): norms are multiplied into K^ and V^, one rounding (2^-12) each.
//   results of 11 bits and more (fp16, fp32): K^ and V^ are bare levels, scaled so that the eight of them lie within 4e-5 of fp16 values;
//             norms multiply S and P in fp32, and a query is two fp16 parts (half again as many operations in the tensor core): what is rounded is P.
#include <cmath>
#include <cstring>

#include "tq_split.cuh"
#include "tq_tcgen05.cuh"

namespace tq {

constexpr int kCrossTile = 128;                      // tokens, query rows, padded head size
constexpr int kCrossImage = kCrossTile * kCrossTile * 2;
constexpr int kCrossThreads = 384;                   // two softmax warpgroups, and one of a copying, an issuing and two idle warps
constexpr float kCrossRaise = 8.0f;                  // P up to 2^8
constexpr double kCrossLevelScale = 1.42803;         // see tq_scored.cu
constexpr float kCrossNoNorm = -1000.0f;             // the logarithm of V's scale in a tile whose V is all zero
constexpr uint32_t kCrossWaitLimit = 1u << 18, kCrossSuspendNs = 1000;

struct CrossParams {
    SplitParams f;              // what split_load_row / split_finish take: types, head size, signs, out, the cache
    const int32_t* cu_q;        // [batch + 1]
    uint8_t* kv_images;         // [tile][head][K, V][32 KB]
    float2* tile_scales;        // [tile][head]: powers of two that the norms were divided by, K and V (their logarithm)
    float* tile_norms;          // exact: [tile][head][K, V][128]
    uint8_t* q_images;          // [query tile][head][part][32 KB]
    float* q_scales;            // [query tile][head][128], times the scale of the logits (base 2)
    float* partial_o;           // [split][query row][query head][128], rotated domain
    float* partial_lse;
    int64_t kv_room, q_room;    // tiles that the workspace holds
    int total_q, splits, heads;
    uint16_t level_h[16];
};

static __device__ int32_t g_cross_faults = 0;

struct CrossSeq {
    int b, local;               // the sequence, and which of its tiles (pairs of query tiles) the index is
    int len, qlen;              // tokens, query rows (tokens of the prompt)
    int kv0, q0;                // its first tiles
};

__device__ __forceinline__ int cross_len(const CrossParams& p, int b, bool& bad) {
    const int len = p.f.seq_lens[b];
    bad = len < 0 || len > (int64_t)p.f.max_pages * kPageTokens;
    return bad ? 0 : len;
}
__device__ __forceinline__ int cross_qlen(const CrossParams& p, int b, bool& bad) {
    const int c0 = p.cu_q[b], c1 = p.cu_q[b + 1];
    bad = c0 < 0 || c1 < c0 || c1 > p.total_q;
    return bad ? 0 : c1 - c0;
}
// The sequence that item `index` of a kind belongs to (0: tiles of tokens, 1: tiles of query rows, 2: pairs of these); false: there are not so many.  A
// sequence without queries has no tiles of tokens; one whose tiles the workspace does not hold has no tokens (or queries).  A whole warp.
template <int KIND>
__device__ __forceinline__ bool cross_find(const CrossParams& p, int64_t index, int lane, CrossSeq& s, int* faults = nullptr) {
    int64_t kv = 0, q = 0, pairs = 0;
    for (int base = 0; base < p.f.batch; base += 32) {
        int len = 0, qlen = 0, kt = 0, qt = 0;
        if (base + lane < p.f.batch) {
            bool bad_len, bad_q;
            len = cross_len(p, base + lane, bad_len);
            qlen = cross_qlen(p, base + lane, bad_q);
            qt = (qlen * p.f.real_group + kCrossTile - 1) / kCrossTile;
            kt = qlen > 0 ? (len + kCrossTile - 1) / kCrossTile : 0;
            if (faults) *faults += bad_len + bad_q;
        }
        int kt_to = kt, qt_to = qt, pair_to = (qt + 1) / 2;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, kt_to, o), c = __shfl_up_sync(0xffffffffu, qt_to, o), d = __shfl_up_sync(0xffffffffu, pair_to, o);
            if (lane >= o) { kt_to += a; qt_to += c; pair_to += d; }
        }
        const bool kv_fits = kv + kt_to <= p.kv_room, q_fits = q + qt_to <= p.q_room;
        if (faults) *faults += (kt > 0 && !kv_fits) + (qt > 0 && !q_fits);
        const int mine = KIND == 0 ? kt : KIND == 1 ? qt : (qt + 1) / 2;
        const int64_t end = KIND == 0 ? kv + kt_to : KIND == 1 ? q + qt_to : pairs + pair_to;
        const uint32_t hit = __ballot_sync(0xffffffffu, index < end);
        if (hit) {
            const int l = __ffs(hit) - 1;
            s.b = base + l;
            s.local = (int)(index - (__shfl_sync(0xffffffffu, end, l) - __shfl_sync(0xffffffffu, mine, l)));
            s.len = __shfl_sync(0xffffffffu, kv_fits ? len : 0, l);
            s.qlen = __shfl_sync(0xffffffffu, q_fits ? qlen : 0, l);
            s.kv0 = (int)(kv + __shfl_sync(0xffffffffu, kt_to - kt, l));
            s.q0 = (int)(q + __shfl_sync(0xffffffffu, qt_to - qt, l));
            return true;
        }
        kv += __shfl_sync(0xffffffffu, kt_to, 31);
        q += __shfl_sync(0xffffffffu, qt_to, 31);
        pairs += __shfl_sync(0xffffffffu, pair_to, 31);
    }
    return false;
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

constexpr int kLayThreads = 256, kLayPitch = 17;      // words of a staged V row (16 and one, for the banks)
template <bool EXACT>
__global__ void __launch_bounds__(kLayThreads) cross_lay_out_kernel(const __grid_constant__ CrossParams p) {
    __shared__ uint32_t lut[256 * 32];                // entry v, column lane: {level(v & 15), level(v >> 4)}
    __shared__ uint32_t codes_s[kCrossTile * kLayPitch];
    __shared__ int64_t slot_s[kCrossTile];            // byte of each token's K slot
    __shared__ uint16_t norm_s[2][kCrossTile];
    __shared__ float most_s[2][4];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, H = p.f.kv_heads, G = p.f.real_group;
    grid_launch_dependents();
    for (int i = tid; i < 256 * 32; i += kLayThreads) lut[i] = (uint32_t)p.level_h[(i >> 5) & 15] | ((uint32_t)p.level_h[i >> 9] << 16);
    grid_dependency_wait();
    if (blockIdx.x == 0 && warp == 0) {               // what is left out is counted once
        CrossSeq s;
        int faults = 0;
        cross_find<0>(p, (int64_t)1 << 60, lane, s, &faults);
        if (faults) atomicAdd(&g_cross_faults, faults);
    }
    __syncthreads();

    // ---- tiles of tokens -------------------------------------------------------------------------------
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
        float most = fabsf(norm) < INFINITY ? fabsf(norm) : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        if (lane == 0) most_s[which][warp & 3] = most;
        __syncthreads();
        // norms to [64, 128): with levels up to 4 the products stay inside fp16, and so do their sums' terms
        most = fmaxf(fmaxf(most_s[which][0], most_s[which][1]), fmaxf(most_s[which][2], most_s[which][3]));
        const bool has = most > 0.0f;
        const int by = cross_exponent(most, 6);
        norm_s[which][t] = __half_as_ushort(__float2half_rn(norm * cross_power(by)));
        if constexpr (EXACT) p.tile_norms[((tile * H + h) * 2 + which) * kCrossTile + t] = norm * cross_power(by);
        if (t == 0) {
            float* const to = reinterpret_cast<float*>(p.tile_scales + tile * H + h) + which;
            *to = !which ? cross_power(-by) : has ? (float)-by : kCrossNoNorm;
        }
        __syncthreads();
        uint8_t* const image = p.kv_images + (tile * H + h) * 2 * kCrossImage;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = (i & 3) * 32 + warp * 4 + (lane >> 3), c = (i >> 2) * 8 + (lane & 7);
            const uint32_t w = k_code[i], nn = (uint32_t)norm_s[0][r] * 0x10001u;
            uint32_t v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {             // dims in pairs {odd, even}, as the queries have them
                v[j] = level2((w >> (8 * j)) & 255u);
                if constexpr (!EXACT) v[j] = cross_mul2(v[j], nn);
            }
            *reinterpret_cast<uint4*>(image + cross_piece(r, c)) = make_uint4(v[0], v[1], v[2], v[3]);
        }
        // V^ transposed: a lane takes eight tokens (one piece) of eight dims (one code word); nibbles of two tokens are zipped into bytes
        {
            const int c = (lane & 7) + 8 * (warp & 1), word = (lane >> 3) + 4 * (warp >> 1);     // pieces 0 ... 15, words 0 ... 15
            uint32_t out[8][4];
#pragma unroll
            for (int pr = 0; pr < 4; pr++) {
                const uint32_t a = codes_s[(8 * c + 2 * pr) * kLayPitch + word], b = codes_s[(8 * c + 2 * pr + 1) * kLayPitch + word];
                const uint32_t odd = (a & 0x0F0F0F0Fu) | ((b << 4) & 0xF0F0F0F0u), even = ((a >> 4) & 0x0F0F0F0Fu) | (b & 0xF0F0F0F0u);
                const uint32_t nn = *reinterpret_cast<const uint32_t*>(&norm_s[1][8 * c + 2 * pr]);
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
            for (int d = 0; d < 8; d++) *reinterpret_cast<uint4*>(image + kCrossImage + cross_piece(8 * word + d, c)) = make_uint4(out[d][0], out[d][1], out[d][2], out[d][3]);
        }
        __syncthreads();
    }

    // ---- tiles of query rows: a warp a row ------------------------------------------------------------
    const float4 sign = reinterpret_cast<const float4*>(p.f.signs)[lane];
    int64_t tiles = 0;                                // units are dealt on from where the tiles of tokens ended
    {
        int64_t kv = 0;
        for (int base = 0; base < p.f.batch; base += 32) {
            int kt = 0;
            if (base + lane < p.f.batch) {
                bool bad;
                const int len = cross_len(p, base + lane, bad);
                if (cross_qlen(p, base + lane, bad) > 0) kt = (len + kCrossTile - 1) / kCrossTile;
            }
            kv += __reduce_add_sync(0xffffffffu, kt);
        }
        tiles = kv * H;
    }
    for (unit -= tiles;; unit += gridDim.x) {
        CrossSeq s;
        const int64_t tile = unit / H;
        const int h = (int)(unit - tile * H);
        if (!cross_find<1>(p, tile, lane, s)) break;
        if (s.qlen == 0) continue;
        constexpr int kParts = EXACT ? 2 : 1;
        uint8_t* const image = p.q_images + (tile * H + h) * kParts * kCrossImage;
        const int row0 = s.local * kCrossTile, rows = s.qlen * G, first = p.cu_q[s.b];
        for (int r = warp; r < kCrossTile; r += kLayThreads / 32) {
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const int row = row0 + r;
            if (row < rows) {
                const int qi = row / G, g = row - qi * G;
                split_load_row<4>(p.f.q, p.f.q_dtype, (int64_t)(first + qi) * p.f.real_heads + h * G + g, p.f.head_dim, 4 * lane, v);
            }
            v[0] *= sign.x; v[1] *= sign.y; v[2] *= sign.z; v[3] *= sign.w;
            split_fwht<4>(v, lane);
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[i] *= p.f.scale;
                top = fmaxf(top, fabsf(v[i]));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int by = cross_exponent(top, 9);    // to [512, 1024)
            const float f = p.f.k_scale < 0.0f ? -cross_power(by) : cross_power(by);
            if (lane == 0) p.q_scales[(tile * H + h) * kCrossTile + r] = fabsf(p.f.k_scale) * cross_power(-by);
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] *= f;
            const uint32_t at = cross_piece(r, lane >> 1) + 8 * (lane & 1);
            const uint32_t a = pack_half2(v[1], v[0]), b = pack_half2(v[3], v[2]);
            *reinterpret_cast<uint2*>(image + at) = make_uint2(a, b);
            if constexpr (EXACT) {
                const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a)), fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
                *reinterpret_cast<uint2*>(image + kCrossImage + at) = make_uint2(pack_half2(v[1] - fa.x, v[0] - fa.y), pack_half2(v[3] - fb.x, v[2] - fb.y));
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------------
template <bool EXACT>
struct CrossShape {
    static constexpr int kParts = EXACT ? 2 : 1;
    static constexpr int kSlots = EXACT ? 3 : 5;                           // of the ring: K, V, K, V, ... of the tiles in turn
    static constexpr uint32_t kQ = 0, kRing = 2 * kParts * kCrossImage;
    // Norms of a tile travel with its K into one of two buffers.  The copy of K (j + 2) waits for the slot of V (j) at the latest, which is free
    // when both warpgroups have handed over P (j), and so have read the norms of tile j.
    static constexpr uint32_t kNorms = kRing + kSlots * kCrossImage, kNormBytes = EXACT ? 2 * kCrossTile * 4 : 0;
    static constexpr uint32_t kBars = kNorms + 2 * kNormBytes;
    static constexpr size_t kSmem = kBars + 256;
    static_assert(!EXACT || kSlots <= 3, "the norms' buffers");
    static_assert(kSmem <= 232448, "shared memory of a block");
};

// SW128, K-major: rows of 128 bytes, eight rows 1024 bytes on
__device__ __forceinline__ uint64_t cross_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)64 << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// A wait of a whole warp that ends early when another role has given up.
__device__ __forceinline__ bool cross_wait(uint32_t bar, uint32_t parity, volatile int* gone) {
    bool done = false;
    for (uint32_t i = 0; i < kCrossWaitLimit && !done && !*gone; i++) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar), "r"(parity), "r"(kCrossSuspendNs) : "memory");
        done = ok != 0;
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
__device__ __forceinline__ void cross_ld_wait(float* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]),
                   "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]), "+f"(r[16]),
                   "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]),
                   "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
                 :: "memory");
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

template <bool EXACT>
__global__ void __launch_bounds__(kCrossThreads, 1) cross_attend_kernel(const __grid_constant__ CrossParams p) {
    using F = CrossShape<EXACT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, H = p.f.kv_heads, G = p.f.real_group;
    const uint32_t base = smem_u32(smem);
    grid_launch_dependents();
    if (base & 1023) {                                // the swizzle counts on it
        grid_dependency_wait();
        if (tid == 0 && blockIdx.x == 0) atomicAdd(&g_cross_faults, 1);
        return;
    }
    // barriers of 8 bytes: Q, the ring's full and empty, S and P and O of the two tiles; then the tensor-memory address and the flag of a role that gave up
    const uint32_t bars = base + F::kBars;
    const uint32_t q_full = bars, ring_full = bars + 8, ring_empty = ring_full + 8 * F::kSlots, s_full = ring_empty + 8 * F::kSlots, p_full = s_full + 16,
                   o_full = p_full + 16, drained = o_full + 16;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + F::kBars + 192);
    volatile int* const gone = reinterpret_cast<volatile int*>(smem + F::kBars + 196);
    if (tid == 0) {
        cross_bar_init(q_full, 1);
        for (int i = 0; i < F::kSlots; i++) {
            cross_bar_init(ring_full + 8 * i, 1);
            cross_bar_init(ring_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; i++) {
            cross_bar_init(s_full + 8 * i, 1);
            cross_bar_init(p_full + 8 * i, 4);        // the warps of the tile
            cross_bar_init(o_full + 8 * i, 1);
        }
        cross_bar_init(drained, 1);
        *gone = 0;
        fence_barrier_init();
    }
    grid_dependency_wait();
    CrossSeq s;
    const int64_t item = blockIdx.x / p.splits;
    const int split = (int)(blockIdx.x - item * p.splits), h = (int)(item % H);
    if (!cross_find<2>(p, item / H, lane, s) || s.qlen == 0) return;      // uniform over the block
    const int rows = s.qlen * G, qt = (rows + kCrossTile - 1) / kCrossTile, q_tile = 2 * s.local, both = q_tile + 1 < qt ? 2 : 1;
    const int all = (s.len + kCrossTile - 1) / kCrossTile;
    const int j0 = (int)((int64_t)all * split / p.splits), n = (int)((int64_t)all * (split + 1) / p.splits) - j0;      // the block's tiles of tokens
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + F::kBars + 192), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;                 // S / P of tile i at 128 i, O at 256 + 128 i
    const int64_t kv_at = (int64_t)(s.kv0 + j0) * H + h;      // image of the block's tile j: kv_at + j H

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 8) {
            // =============================== copies ======================================================
            if (n > 0 && lane == 0) {
                split_expect(q_full, both * F::kParts * kCrossImage);
                for (int i = 0; i < both; i++)
                    for (int a = 0; a < F::kParts; a++)
                        cross_copy(base + F::kQ + (i * F::kParts + a) * kCrossImage,
                                   p.q_images + (((int64_t)(s.q0 + q_tile + i) * H + h) * F::kParts + a) * kCrossImage, kCrossImage, q_full);
            }
            int k = 0, slot = 0, parity = 1;          // of the wait for an empty slot: free at first
            for (; k < 2 * n; k++) {
                if (!cross_wait(ring_empty + 8 * slot, parity, gone)) break;
                if (lane == 0) {
                    const int64_t image = kv_at + (int64_t)(k >> 1) * H;
                    const uint32_t bar = ring_full + 8 * slot, more = (k & 1) == 0 ? F::kNormBytes : 0;
                    split_expect(bar, kCrossImage + more);
                    cross_copy(base + F::kRing + slot * kCrossImage, p.kv_images + (image * 2 + (k & 1)) * kCrossImage, kCrossImage, bar);
                    if (more) cross_copy(base + F::kNorms + ((k >> 1) & 1) * F::kNormBytes, p.tile_norms + image * 2 * kCrossTile, F::kNormBytes, bar);
                }
                __syncwarp();
                if (++slot == F::kSlots) {
                    slot = 0;
                    parity ^= 1;
                }
            }
            if (k < 2 * n) {                          // gave up: what is in flight gets its time to land
                if (lane == 0) atomicAdd(&g_cross_faults, 1);
                *gone = 1;
                for (int i = k > F::kSlots ? k - F::kSlots : 0; i < k; i++)
                    for (uint32_t w = 0; w < kCrossWaitLimit / 64; w++)
                        if (split_try_wait(ring_full + 8 * (i % F::kSlots), (i / F::kSlots) & 1)) break;
                for (uint32_t w = 0; w < kCrossWaitLimit / 64; w++)
                    if (split_try_wait(q_full, 0)) break;
            }
        } else if (warp == 9 && n > 0) {
            // =============================== matrix products ==============================================
            constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(kCrossTile >> 3) << 17) | ((uint32_t)(kCrossTile >> 4) << 24);      // fp16 x fp16 -> fp32, 128 x 128
            bool ok = cross_wait(q_full, 0, gone);
            int slot = 0, parity = 0;
            auto next_slot = [&] {
                if (++slot == F::kSlots) {
                    slot = 0;
                    parity ^= 1;
                }
            };
            auto scores = [&](int i) {                // S of tile i from the K image in the slot
                const uint64_t b0 = cross_desc(base + F::kRing + slot * kCrossImage);
#pragma unroll
                for (int a = 0; a < F::kParts; a++) {
                    const uint64_t a0 = cross_desc(base + F::kQ + (i * F::kParts + a) * kCrossImage);
#pragma unroll
                    for (int kk = 0; kk < 8; kk++) {
                        const uint64_t off = (uint64_t)((kk >> 2) * 1024 + (kk & 3) * 2);      // 16 dims on, in units of 16 bytes
                        mq_mma(tmem + 128 * i, a0 + off, b0 + off, idesc, a || kk ? 1u : 0u);
                    }
                }
                cross_commit(s_full + 8 * i);
            };
            if (ok) ok = cross_wait(ring_full, 0, gone);
            tc_fence_after();
            if (ok && elect_one()) {
                for (int i = 0; i < both; i++) scores(i);
                cross_commit(ring_empty);
            }
            __syncwarp();
            next_slot();
            for (int j = 0; j < n && ok; j++) {
                const int v_slot = slot, v_parity = parity;
                next_slot();
                ok = cross_wait(ring_full + 8 * v_slot, v_parity, gone);
                const bool more = j + 1 < n;
                if (ok && more) ok = cross_wait(ring_full + 8 * slot, parity, gone);
                for (int i = 0; i < both && ok; i++) {
                    ok = cross_wait(p_full + 8 * i, j & 1, gone);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t b0 = cross_desc(base + F::kRing + v_slot * kCrossImage);
#pragma unroll
                        for (int kk = 0; kk < 8; kk++)
                            mq_mma_ts(tmem + 256 + 128 * i, tmem + 128 * i + 8 * kk, b0 + (uint64_t)((kk >> 2) * 1024 + (kk & 3) * 2), idesc, j || kk ? 1u : 0u);
                        if (i == both - 1) cross_commit(ring_empty + 8 * v_slot);
                        if (more) scores(i);
                        else cross_commit(o_full + 8 * i);
                        if (more && i == both - 1) cross_commit(ring_empty + 8 * slot);
                    }
                    __syncwarp();
                }
                next_slot();
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
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int i = warp >> 2, r = tid & 127, row = (q_tile + i) * kCrossTile + r;
        const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tm_s = tmem + 128 * i + lane_at, tm_o = tmem + 256 + 128 * i + lane_at;
        bool ok = true;
        float m = kNoMax, l = 0.0f, x[128];
        float ev_most = -1000.0f;
        const bool mine = i < both;
        const float q_scale = mine ? p.q_scales[((int64_t)(s.q0 + q_tile + i) * H + h) * kCrossTile + r] : 0.0f;
        // The scale of V that the sums are kept in: the largest of the block's tiles.
        for (int j = lane; j < n; j += 32) ev_most = fmaxf(ev_most, p.tile_scales[kv_at + (int64_t)j * H].y);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ev_most = fmaxf(ev_most, __shfl_xor_sync(0xffffffffu, ev_most, o));
        float2 scales = n > 0 ? p.tile_scales[kv_at] : make_float2(0.0f, 0.0f);
        for (int j = 0; j < n && mine && ok; j++) {
            // A masked logit is -inf times kf: kf is no zero (a scale of zero).  A tile whose V is zero, or as good as that beside the largest, has P
            // scaled by 2^-60: out of fp16, not out of the row's sum.
            const float kf = fmaxf(scales.x * q_scale, 1e-36f), dv = fmaxf(scales.y - ev_most, -60.0f);
            if (j + 1 < n) scales = p.tile_scales[kv_at + (int64_t)(j + 1) * H];
            ok = cross_wait(s_full + 8 * i, j & 1, gone);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < 4; c++) cross_ld(tm_s + 32 * c, x + 32 * c);
#pragma unroll
            for (int c = 0; c < 4; c++) cross_ld_wait(x + 32 * c);
            const float* const norms = reinterpret_cast<const float*>(smem + F::kNorms + (j & 1) * F::kNormBytes);
            if constexpr (EXACT) {
#pragma unroll
                for (int c = 0; c < 128; c += 4) {
                    const float4 t = *reinterpret_cast<const float4*>(norms + c);
                    x[c] *= t.x; x[c + 1] *= t.y; x[c + 2] *= t.z; x[c + 3] *= t.w;
                }
            }
            const int valid = s.len - (j0 + j) * kCrossTile;
            if (valid < kCrossTile) {                 // the last tile of the sequence
#pragma unroll
                for (int c = 0; c < 128; c++)
                    if (c >= valid) x[c] = -INFINITY;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 128; c += 4) {
                mx[0] = fmaxf(mx[0], x[c]); mx[1] = fmaxf(mx[1], x[c + 1]); mx[2] = fmaxf(mx[2], x[c + 2]); mx[3] = fmaxf(mx[3], x[c + 3]);
            }
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * kf;      // kf >= 0
            const bool raise = top > m + kCrossRaise;
            if (__any_sync(0xffffffffu, raise)) {
                const float c = raise ? fast_exp2(m - top) : 1.0f;
                if (raise) m = top;
                l *= c;
                if (j > 0) {                          // S (j) is there, so the products before it are done with O
#pragma unroll
                    for (int a = 0; a < 4; a++) {
                        float o[32];
                        cross_ld(tm_o + 32 * a, o);
                        cross_ld_wait(o);
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] *= c;
                        cross_st(tm_o + 32 * a, reinterpret_cast<const uint32_t*>(o));
                    }
                }
            }
            const P2 kf2 = pk(kf, kf), sub = pk(dv - m, dv - m);
            P2 sum = pk(0.0f, 0.0f);
            uint32_t ph[64];
#pragma unroll
            for (int c = 0; c < 128; c += 2) {
                float a, b;
                up(fma2(pk(x[c], x[c + 1]), kf2, sub), a, b);
                a = fast_exp2(a);
                b = fast_exp2(b);
                sum = add2(sum, pk(a, b));
                if constexpr (EXACT) {
                    const float2 t = *reinterpret_cast<const float2*>(norms + kCrossTile + c);
                    a *= t.x;
                    b *= t.y;
                }
                ph[c >> 1] = pack_half2(a, b);
            }
            cross_st(tm_s, ph);
            cross_st(tm_s + 32, ph + 32);
            float sa, sb;
            up(sum, sa, sb);
            l += (sa + sb) * fast_exp2(-dv);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) cross_arrive(p_full + 8 * i);
        }
        // ---- the row: normalized, rotated back, out; or a partial ------------------------------------------
        if (mine && ok && n > 0) ok = cross_wait(o_full + 8 * i, 0, gone);
        if (mine && !ok) *gone = 1;
        if (mine && ok) {
            tc_fence_after();
            if (n > 0) {
#pragma unroll
                for (int c = 0; c < 4; c++) cross_ld(tm_o + 32 * c, x + 32 * c);
#pragma unroll
                for (int c = 0; c < 4; c++) cross_ld_wait(x + 32 * c);
            }
            const float f = l == 0.0f ? 0.0f : p.f.v_scale * fast_exp2(ev_most) / l;
            const float lse2 = l == 0.0f ? -INFINITY : m + log2f(l);
#pragma unroll
            for (int c = 0; c < 128; c++) x[c] = l == 0.0f ? 0.0f : x[c] * f;
            if (row < rows) {
                const int qi = row / G, g = row - qi * G;
                const int64_t to = (int64_t)(p.cu_q[s.b] + qi) * p.f.real_heads + h * G + g;
                if (p.splits > 1) {
                    const int64_t at = (int64_t)split * p.total_q * p.f.real_heads + to;
                    float4* dst = reinterpret_cast<float4*>(p.partial_o + at * kCrossTile);
#pragma unroll
                    for (int c = 0; c < 32; c++) dst[c] = make_float4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
                    p.partial_lse[at] = lse2;
                } else {
#pragma unroll
                    for (int w = 1; w < 128; w <<= 1) {
#pragma unroll
                        for (int c = 0; c < 128; c++) {
                            if ((c & w) == 0) {
                                const float a = x[c], b = x[c + w];
                                x[c] = a + b;
                                x[c + w] = a - b;
                            }
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 128; c += 4) {
                        const float4 sg = reinterpret_cast<const float4*>(p.f.signs)[c >> 2];
                        x[c] *= p.f.scale * sg.x; x[c + 1] *= p.f.scale * sg.y; x[c + 2] *= p.f.scale * sg.z; x[c + 3] *= p.f.scale * sg.w;
                    }
                    const int D = p.f.head_dim;
                    if (p.f.out_dtype != TQ_F32 && D % 8 == 0 && (reinterpret_cast<uintptr_t>(p.f.out) & 15) == 0) {
                        uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.f.out) + to * D);
#pragma unroll
                        for (int c = 0; c < 16; c++) {
                            uint32_t w[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                if (p.f.out_dtype == TQ_BF16) {
                                    const __nv_bfloat162 t = __floats2bfloat162_rn(x[8 * c + 2 * e], x[8 * c + 2 * e + 1]);
                                    w[e] = *reinterpret_cast<const uint32_t*>(&t);
                                } else {
                                    w[e] = pack_half2(x[8 * c + 2 * e], x[8 * c + 2 * e + 1]);
                                }
                            }
                            if (8 * c < D) dst[c] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 128; c++) {
                            if (c >= D) continue;
                            if (p.f.out_dtype == TQ_BF16) reinterpret_cast<__nv_bfloat16*>(p.f.out)[to * D + c] = __float2bfloat16_rn(x[c]);
                            else if (p.f.out_dtype == TQ_F16) reinterpret_cast<__half*>(p.f.out)[to * D + c] = __float2half_rn(x[c]);
                            else reinterpret_cast<float*>(p.f.out)[to * D + c] = x[c];
                        }
                    }
                    if (p.f.out_lse) p.f.out_lse[to] = lse2 * 0.6931471805599453f;
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// A warp a row (query row, query head): the parts of the splits.
__global__ void __launch_bounds__(128) cross_join_kernel(const __grid_constant__ CrossParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), rows = (int64_t)p.total_q * p.f.real_heads;
    grid_launch_dependents();
    grid_dependency_wait();
    if (at >= rows) return;
    // a row that belongs to no sequence, or to one that was left out, is left as it is
    const int t = (int)(at / p.f.real_heads);
    bool live = false;
    for (int base = 0; base < p.f.batch && !live; base += 32) {
        bool bad;
        const bool in = base + lane < p.f.batch && cross_qlen(p, base + lane, bad) > 0 && p.cu_q[base + lane] <= t && t < p.cu_q[base + lane + 1];
        live = __any_sync(0xffffffffu, in);
    }
    if (!live) return;
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < p.splits; s++) m = fmaxf(m, p.partial_lse[s * rows + at]);
    if (m == -INFINITY) m = 0.0f;
    for (int s = 0; s < p.splits; s++) {
        const float w = fast_exp2(p.partial_lse[s * rows + at] - m);
        l += w;
        const float4 v = *reinterpret_cast<const float4*>(p.partial_o + (s * rows + at) * kCrossTile + 4 * lane);
        o[0] = fmaf(w, v.x, o[0]); o[1] = fmaf(w, v.y, o[1]); o[2] = fmaf(w, v.z, o[2]); o[3] = fmaf(w, v.w, o[3]);
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

int cross_fault_count(int32_t* out) {
    TQ_CUDA(cudaMemcpyFromSymbol(out, g_cross_faults, sizeof(int32_t)));
    return TQ_OK;
}

static size_t cross_up(size_t x) { return (x + 255) & ~(size_t)255; }

struct CrossLayout {
    int64_t kv_room, q_room;
    int splits;
    size_t scales, norms, q_images, q_scales, partial_lse, partial_o, end;      // the images of K and V are in front
};
static CrossLayout cross_layout(int batch, int total_q, int64_t total_tokens, int heads, int kv_heads, int max_pages, bool exact, int sms) {
    CrossLayout l;
    const int64_t G = heads / kv_heads, rows = total_q * G;
    l.kv_room = total_tokens / kCrossTile + batch;          // every sequence may end inside a tile
    l.q_room = rows / kCrossTile + batch;
    // As many cuts of the tokens as fill the SMs, of four tiles at least.
    const int64_t pairs = (rows + 2 * kCrossTile - 1) / (2 * kCrossTile), blocks = (pairs > batch ? pairs : batch) * kv_heads;
    const int64_t longest = (int64_t)max_pages * kPageTokens < total_tokens ? (int64_t)max_pages * kPageTokens : total_tokens;
    const int64_t most = longest / (4 * kCrossTile), fit = blocks > 0 ? sms / blocks : 1;
    l.splits = (int)(fit < most ? fit : most);
    if (l.splits < 1) l.splits = 1;
    const size_t units = (size_t)l.kv_room * kv_heads, q_units = (size_t)l.q_room * kv_heads, parts = exact ? 2 : 1;
    l.scales = units * 2 * kCrossImage;
    l.norms = l.scales + cross_up(units * sizeof(float2));
    l.q_images = l.norms + (exact ? cross_up(units * 2 * kCrossTile * 4) : 0);
    l.q_scales = l.q_images + q_units * parts * kCrossImage;
    l.partial_lse = l.q_scales + cross_up(q_units * kCrossTile * 4);
    const size_t cut = l.splits > 1 ? (size_t)l.splits * total_q * heads : 0;
    l.partial_o = l.partial_lse + cross_up(cut * 4);
    l.end = l.partial_o + cross_up(cut * kCrossTile * 4);
    return l;
}
static bool cross_exact(int out_dtype) { return out_dtype != TQ_BF16; }

template <bool EXACT>
static int launch_cross(const CrossParams& p, int sms, int64_t pairs, cudaStream_t s) {
    using F = CrossShape<EXACT>;
    static bool configured[64] = {};
    int dev = 0;
    TQ_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        TQ_CUDA(cudaFuncSetAttribute(cross_attend_kernel<EXACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F::kSmem));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    const int64_t units = (p.kv_room + p.q_room) * p.f.kv_heads, lay = units < 4 * sms ? units : 4 * sms;
    TQ_CUDA(launch_serialized(cross_lay_out_kernel<EXACT>, dim3((unsigned)lay), dim3(kLayThreads), 0, s, p));
    TQ_CUDA(launch_serialized(cross_attend_kernel<EXACT>, dim3((unsigned)(pairs * p.f.kv_heads * p.splits)), dim3(kCrossThreads), F::kSmem, s, p));
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
    return tq::cross_layout(batch, total_q, total_tokens, num_q_heads, num_kv_heads, max_pages, tq::cross_exact(out_dtype), sms).end;
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
    const CrossLayout l = cross_layout(batch, total_q, total_tokens, num_q_heads, num_kv_heads, max_pages, exact, sms);
    const int64_t pairs = ((int64_t)total_q * G) / (2 * kCrossTile) + batch;
    TQ_REQUIRE((int64_t)total_q * num_q_heads < 1ll << 31 && l.kv_room < 1 << 30 && pairs * num_kv_heads * l.splits < 1ll << 31, TQ_ERR_UNSUPPORTED,
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
    p.tile_scales = reinterpret_cast<float2*>(ws + l.scales);
    p.tile_norms = reinterpret_cast<float*>(ws + l.norms);
    p.q_images = ws + l.q_images;
    p.q_scales = reinterpret_cast<float*>(ws + l.q_scales);
    p.partial_lse = reinterpret_cast<float*>(ws + l.partial_lse);
    p.partial_o = reinterpret_cast<float*>(ws + l.partial_o);
    p.kv_room = l.kv_room;
    p.q_room = l.q_room;
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
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return exact ? launch_cross<true>(p, sms, pairs, s) : launch_cross<false>(p, sms, pairs, s);
}
