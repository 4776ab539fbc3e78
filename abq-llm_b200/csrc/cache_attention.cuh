// Attention of a token step over the quantised cache (abq_cache_attention): one token of a decode step, or a tree of drafted tokens.
//
// Keys are k_j = kmin_j + ks_j c_j with codes c_j (16 bits hold min and scale, the tensor cores multiply the codes, centred: c' = c - 2^(bits-1), exact
// in fp16), so  q . k_j = ks_j (q . c'_j) + (kmin_j + 2^(bits-1) ks_j) sum(q), and likewise  sum_j p_j v_j = sum_j (p_j vs_j) c'_j + sum_j p_j (vmin_j + ..).
// Products are transposed (tokens are the 16 rows of an m16n8k16 MMA, query rows its 8 columns): a granule of 16 tokens costs D / 16 instructions for
// S^T = K Q^T and D / 16 for O^T += V^T P^T per 8 query rows, and one conversion of its codes however many rows there are.
//
// What bounds it is HBM (2 * bits / 8 bytes per feature and token, read once) as long as a granule costs few instructions and enough warps are under way.  So
// every warp works for itself: the granules of all sequences, heads and row blocks are one line that the warps of the grid cut into equal runs, whatever the
// lengths, each with a ring of bulk copies of its own (a granule is one contiguous copy), queries straight from global memory to registers, no barrier of the
// block anywhere.  An item (sequence, head, row block) counts for kCaExtra granules more than it has: its queries and its result cost about that much
// (without it, runs over many short sequences took twice as long as those over long ones).  Pieces of an item that several warps hold meet in the
// workspace, added by a second kernel in order (no atomics): joined by whichever warp comes last they took twice the time of both kernels, since one warp has
// too few loads under way.
//
// Measured (us, one call in a chain; the bytes' floor at the copy rate): 2 sequences of 128 K tokens, 32 heads on 8, 8 bits 95 to 99 (76.7, so 78 to 81 % of the rate); 32 of
// up to 4096 tokens, 4 bits 20.6 (4.8): a granule is a chain of dependent steps of 1750 clocks for its warp, three warps a scheduler; one of 1024 tokens, 32 heads 8.0
// to 8.5 (1.3): 3 us until a warp has found its run and its first copy is there, and 3 us for the second kernel, are what short calls cost.
//
//  * Running maximum: raised only when a score passes it by more than 2^8 (checked with one vote), so that shuffles and the scaling of O are rare.
//  * p vs_j is rounded to fp16 after scaling by a power of two that keeps the largest vs seen so far near 2^6: with p <= 2^8 the product is below 2^15 and
//    keeps 11 bits down to 2^-29 of it, so that many small weights are not lost beside one large.  With fp16 results and up to 8 rows the rounding's remainder
//    is multiplied too (a second MMA per tile): rounded alone it would be an error as large as the result's own rounding.  With more rows, where the products
//    count, it is left out; bf16 results do not show it.
//  * Keys are multiplied as 1024 + c (8 bits) or 1 + c / 64 (4 bits), which are single logic operations away from the codes; the constant times sum(q) goes
//    with the row's offset.  The running sum of one score's D / 16 products is rounded at each of them, at a size of up to (1024 + 255) sum|q| (64 + 15 with 4 bits):
//    at most D / 16 times 2^-23 of that, 2^-20 for D = 128.  In practice it is far less: over 1024 tokens of 8 bits the result's error against 64 bits (2.1e-4,
//    fp16) is that of its own rounding.  Values are summed over thousands of tokens and are multiplied centred.
//  * Queries: fp16 as they are; bf16 rows are scaled by a power of two to [1, 2) and held in fp16 (exact down to 2^-14 of the row's largest).
#pragma once
#include "abq_kernels.h"
#include "kv_cache.cuh"

namespace abq {

constexpr int kCaWarps = 4;
constexpr int kCaThreads = 32 * kCaWarps;
constexpr int kCaSms = 148;
// Granules a warp takes at least: fewer take less time, but more pieces have to be joined.  Measured with 1, 2, 3, 4, 6 (us, 32 heads): one sequence of 1024 tokens, one row 9.1 8.0
// 8.6 8.8 10.1; of 300 6.9 7.1 7.8 8.6 10.0; 12 rows on 8 key heads, 1024 tokens 12.7 12.7 11.3 11.6 12.9.
__host__ __device__ constexpr int ca_min_quota(int tiles) { return tiles == 1 ? 2 : 3; }
// What an item costs beside its granules, in granules.  Measured with 1, 2, 3, 4, 5, 6 (us): 29 sequences of up to 4096 tokens, one row 21.5 20.7 20.0 20.2 19.9 19.9; 4 of up to
// 2049, 26 rows 35.4 35.6 34.4 33.7 33.7 35.0; one of 1024, one row 9.9 8.9 9.1 9.0 8.9 9.0.
constexpr int kCaExtra = 4;

// 128, 168 or 255 registers a thread: as many CTAs as fit without spills (heads of 64 with one more than heads of 128: two sequences of 64 K tokens, 40 heads, one
// row 137 us instead of 149, 26 rows over 4 of up to 2049 27 instead of 29; heads of 128 with spills for one more 45 instead of 35)
__host__ __device__ constexpr int ca_ctas_per_sm(int head_dim, int tiles) { return (tiles == 1 ? 3 : 2) + (head_dim == 64); }

struct CacheAttnArgs {
    const uint8_t *data;
    const uint8_t *q;
    uint8_t *out;
    long long q_stride, q_head_stride, out_stride, out_head_stride; // bytes
    const int *table, *seq_lens;
    const uint64_t *tree;
    float *part; // [2 * runs][slot_rows][D] sums, then [2 * runs][slot_rows] pairs (maximum, sum of p)
    int *status;
    int num_pages, page_granules, kv_heads, batch, n, group, row_blocks, slot_rows, table_stride, runs;
    int unit_log2, extra, min_quota; // the line's unit: 16 tokens (a warp's granule) or 128 (a CTA's tile)
    float scale_log2;
    unsigned long long page_magic;
};

__device__ __forceinline__ int ca_tokens(const CacheAttnArgs &a, int b)
{
    const long long cap = (long long)a.table_stride * a.page_granules * kGranuleTokens;
    const int len = a.seq_lens[b];
    return len < 0 ? 0 : (int)min((long long)min(len, 0x7fffff00), cap);
}
__device__ __forceinline__ int ca_granules(const CacheAttnArgs &a, int b) // (or tiles: units)
{
    return (int)(((long long)ca_tokens(a, b) + (1 << a.unit_log2) - 1) >> a.unit_log2);
}
__device__ __forceinline__ int ca_units(const CacheAttnArgs &a, int granules) { return granules ? granules + a.extra : 0; } // an item's length on the line

// Units of all sequences, and of those before sequence `before`, one item each; by a warp.
__device__ __forceinline__ void ca_sums(const CacheAttnArgs &a, int before, long long &all, long long &prefix)
{
    long long s = 0, p = 0;
    for (int b = threadIdx.x & 31; b < a.batch; b += 32) {
        const int u = ca_units(a, ca_granules(a, b));
        s += u;
        p += b < before ? u : 0;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        p += __shfl_xor_sync(0xffffffffu, p, o);
    }
    all = s;
    prefix = p;
}
// Quotient of numbers that hardly ever need 64 bits (their division is some ten times slower)
__device__ __forceinline__ long long ca_div(long long x, long long y)
{
    return ((unsigned long long)(x | y) >> 32) == 0 ? (long long)((uint32_t)x / (uint32_t)y) : x / y;
}
__device__ __forceinline__ long long ca_quota(const CacheAttnArgs &a, long long total) { return max(ca_div(total + a.runs - 1, a.runs), (long long)a.min_quota); }
// Entry of a block table that holds granule g (page_magic = ceil(2^34 / page_granules): exact for granule numbers below 2^28)
__device__ __forceinline__ int ca_entry(const CacheAttnArgs &a, int g) { return (int)(((unsigned long long)(uint32_t)g * a.page_magic) >> 34); }

// A part of an item that one run holds, and the walk over a run's parts (by a warp, all lanes alike).
struct CaPiece {
    int b, item, G, g0, g1; // units g0 .. g1 - 1 of G
    bool first;             // the run starts in this item
};
struct CaRun {
    int b, G, item, pos;
    long long left;
    bool first;

    __device__ __forceinline__ bool begin(const CacheAttnArgs &a, int run, int lane)
    {
        const int items = a.kv_heads * a.row_blocks;
        long long units = 0, quota = 0, rem = 0, unused;
        first = true;
        if (a.batch > 32) {
            ca_sums(a, 0, units, unused);
            quota = ca_quota(a, units * items);
        }
        for (int b0 = 0;; b0 += 32) { // 32 sequences at a time
            const int own = b0 + lane < a.batch ? ca_granules(a, b0 + lane) : 0;
            uint32_t upto = ca_units(a, own);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
                upto += lane >= o ? x : 0;
            }
            if (b0 == 0) {
                if (a.batch <= 32) {
                    units = __shfl_sync(0xffffffffu, upto, 31);
                    quota = ca_quota(a, units * items);
                }
                rem = run * quota; // from the start of sequence b0
                left = min(units * items, rem + quota) - rem;
                if (left <= 0)
                    return false;
            }
            const uint32_t behind = __ballot_sync(0xffffffffu, rem < (long long)upto * items);
            if (behind) {
                const int at = __ffs(behind) - 1;
                b = b0 + at;
                G = __shfl_sync(0xffffffffu, own, at);
                rem -= (long long)(__shfl_sync(0xffffffffu, upto, at) - ca_units(a, G)) * items;
                break;
            }
            rem -= (long long)__shfl_sync(0xffffffffu, upto, 31) * items;
        }
        item = (int)ca_div(rem, ca_units(a, G));
        pos = (int)(rem - (long long)item * ca_units(a, G));
        return true;
    }
    __device__ __forceinline__ bool next(const CacheAttnArgs &a, CaPiece &p) // the next part that has units
    {
        while (left > 0) {
            if (pos == ca_units(a, G)) {
                pos = 0;
                first = false;
                if (++item == a.kv_heads * a.row_blocks) {
                    item = 0;
                    do {
                        G = ca_granules(a, ++b);
                    } while (G == 0);
                }
            }
            const int span = (int)min((long long)(ca_units(a, G) - pos), left);
            p.b = b, p.item = item, p.G = G, p.first = first;
            p.g0 = max(0, pos - a.extra), p.g1 = max(0, pos + span - a.extra);
            pos += span;
            left -= span;
            if (p.g1 > p.g0)
                return true;
        }
        return false;
    }
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_sub(uint32_t a, uint32_t b)
{
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// 0x6400 | c is the fp16 number 1024 + c, and 0x3c00 | c << 4 is 1 + c / 64.  Pairs of codes as they are multiplied with the queries, from bytes 0 and 1, bytes 2 and
// 3, or bits 4-7 of both halves ...
__device__ __forceinline__ uint32_t key_bytes_lo(uint32_t w) { return __byte_perm(w, 0x64646464u, 0x4140); }
__device__ __forceinline__ uint32_t key_bytes_hi(uint32_t w) { return __byte_perm(w, 0x64646464u, 0x4342); }
__device__ __forceinline__ uint32_t key_nibbles(uint32_t w) { return (w & 0x00f000f0u) | 0x3c003c00u; }
// ... and centred, from ...
__device__ __forceinline__ uint32_t bytes_lo(uint32_t w) { return half2_sub(__byte_perm(w, 0x64646464u, 0x4140), 0x64806480u); } // ... bytes 0, 1
__device__ __forceinline__ uint32_t bytes_hi(uint32_t w) { return half2_sub(__byte_perm(w, 0x64646464u, 0x4342), 0x64806480u); } // ... bytes 2, 3
__device__ __forceinline__ uint32_t nibbles_lo(uint32_t w) { return half2_sub((w & 0x000f000fu) | 0x64006400u, 0x64086408u); }  // ... bits 0-3 of both halves
__device__ __forceinline__ uint32_t nibbles_hi(uint32_t w) // ... bits 4-7: (1024 + 16 c) / 16 - 72
{
    const uint32_t x = (w & 0x00f000f0u) | 0x64006400u, sixteenth = 0x2c002c00u, off = 0xd480d480u;
    const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&x), *reinterpret_cast<const __half2 *>(&sixteenth), *reinterpret_cast<const __half2 *>(&off));
    return *reinterpret_cast<const uint32_t *>(&r);
}

template <int BYTES>
__device__ __forceinline__ void lds(uint32_t *dst, const uint8_t *src)
{
    if (BYTES == 16) {
        const uint4 v = *reinterpret_cast<const uint4 *>(src);
        dst[0] = v.x, dst[1] = v.y, dst[2] = v.z, dst[3] = v.w;
    } else if (BYTES == 8) {
        const uint2 v = *reinterpret_cast<const uint2 *>(src);
        dst[0] = v.x, dst[1] = v.y;
    } else {
        dst[0] = *reinterpret_cast<const uint32_t *>(src);
    }
}

template <int D, int BITS, int NT>
struct CaShape {
    static constexpr int RB = kv_row_bytes(D, BITS), kGranule = kv_granule_bytes(RB), kRows = 8 * NT, kSteps = D / 16;
    static constexpr int kFixed = kCaWarps * kRows * 8;
    static constexpr int kRoom = 226 * 1024 / ca_ctas_per_sm(D, NT) - 1024 - kFixed;
    static constexpr int kFit = kRoom / (kCaWarps * (kGranule + 8));
    static constexpr int kStages = kFit < 10 ? kFit : 10;
    static constexpr int kSmem = kFixed + kCaWarps * kStages * (kGranule + 8);
    static_assert(kStages >= 3 && kStages <= 32, "ring");
};

template <int D, int BITS, int NT, bool BF16>
__global__ void __launch_bounds__(kCaThreads, ca_ctas_per_sm(D, NT)) cache_attention_kernel(const __grid_constant__ CacheAttnArgs a)
{
    using Sh = CaShape<D, BITS, NT>;
    constexpr int RB = Sh::RB, kGranule = Sh::kGranule, kRows = Sh::kRows, kSteps = Sh::kSteps, kStages = Sh::kStages, kTiles = D / 16;
    constexpr int kKW = RB / 16, kVW = RB / 32; // 32-bit words of codes per lane and token
    constexpr float kCentre = (float)(1 << (BITS - 1));
    constexpr float kKeyScale = BITS == 8 ? 1.f : 64.f, kKeyOffset = BITS == 8 ? -1024.f : -64.f; // code = factor * kKeyScale + kKeyOffset
    constexpr bool kRemainder = NT == 1 && !BF16;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;
    uint8_t *ring = smem + warp * kStages * kGranule;
    uint64_t *masks = reinterpret_cast<uint64_t *>(smem + kCaWarps * kStages * kGranule) + warp * kRows;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + kCaWarps * kStages * kGranule + Sh::kFixed) + warp * kStages;
    if (lane < kStages)
        mbar_init(&full[lane], 1);
    fence_mbar_init();
    __syncwarp();
    pdl_wait_prior_grid();
    pdl_launch_dependents();

    const int run = blockIdx.x * kCaWarps + warp;
    CaRun line;
    if (!line.begin(a, run, lane))
        return; // (before any copy)

    // ---- ring of granules: lane i % 32 owns the address of granule i of the piece
    using Piece = CaPiece;
    struct Batch {
        uint32_t at;   // index of the granule in the cache, or ~0
        uint32_t good; // ballot: which of the 32 lie in the cache
    };
    auto batch_of = [&](const Piece &p, int base) {
        Batch t;
        const int g = p.g0 + base + lane;
        t.at = ~0u;
        if (g < p.g1) {
            const int entry = ca_entry(a, g), page = a.table[(size_t)p.b * a.table_stride + entry];
            if (page >= 0 && page < a.num_pages)
                t.at = ((uint32_t)page * a.kv_heads + p.item / a.row_blocks) * a.page_granules + (g - entry * a.page_granules);
            else if (a.status)
                atomicOr(a.status, ABQ_STATUS_BAD_PAGE);
        }
        t.good = __ballot_sync(0xffffffffu, t.at != ~0u);
        return t;
    };
    uint32_t put_stage = 0, get_stage = 0, get_phase = 0; // over all pieces
    int pending = 0;                                      // copies not yet waited for
    auto issue = [&](uint32_t at, int owner) {
        ++pending;
        if (lane == owner) {
            uint64_t *bar = &full[put_stage];
            if (at != ~0u) {
                mbar_arrive_expect_tx(bar, kGranule);
                bulk_load(ring + put_stage * kGranule, a.data + (size_t)at * kGranule, kGranule, bar);
            } else {
                mbar_arrive(bar); // nothing to wait for
            }
        }
        put_stage = put_stage + 1 == kStages ? 0 : put_stage + 1;
    };
    const int rows = a.n * a.group;
    // the 16 bytes x of this lane's queries in tile t of an item
    auto query = [&](const Piece &p, int t, int x) -> const uint8_t * {
        const int head = p.item / a.row_blocks, at = (p.item - head * a.row_blocks) * kRows + 8 * t + r, i = at / a.group;
        // 8 bits: features 16 q .. of each 64; 4 bits: a quarter of the row
        const int byte = BITS == 8 ? (x >> 1) * 128 + q * 32 + (x & 1) * 16 : q * (D / 2) + x * 16;
        return at < rows ? a.q + ((long long)p.b * a.n + i) * a.q_stride + (long long)(head * a.group + at - i * a.group) * a.q_head_stride + byte : nullptr;
    };
    auto prefetch_queries = [&](const Piece &p) { // (they are used behind the first copies, which need the block table first)
#pragma unroll
        for (int t = 0; t < NT; ++t)
            if (const uint8_t *at = query(p, t, 0))
                asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
    };

    Piece cur;
    if (!line.next(a, cur))
        return;
    prefetch_queries(cur);
    Batch now = batch_of(cur, 0), ahead = now;
    if (cur.g1 - cur.g0 > 32)
        ahead = batch_of(cur, 32);
    for (int i = 0; i < min(cur.g1 - cur.g0, kStages); ++i)
        issue(now.at, i);
    const int tok = (r & 1) * 4 + (r >> 1); // MMA row r holds token tok, row r + 8 token tok + 8: then P's columns are tokens q, 4 + q, 8 + q, 12 + q
    const int koff = kv_place<RB>(tok, q * (RB == 32 ? 8 : 16)), voff = kv_place<RB>(q, r * (RB / 8));
    const float inf = INFINITY;

    for (;;) {
        const int head = cur.item / a.row_blocks, row0 = (cur.item - head * a.row_blocks) * kRows;
        const int len = ca_tokens(a, cur.b), ctx = len - a.n;
        // ---- queries: this lane's fragments of the MMA's B operand lie together in global memory, 16 bytes at a time
        uint2 qr[NT][kSteps];
        float m[NT][2], l[NT][2], bias[NT][2], O[NT][kTiles][4], rf[NT][2], rs[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int at = row0 + 8 * t + r, i = at / a.group;
            uint4 v[D / 32];
#pragma unroll
            for (int x = 0; x < D / 32; ++x) {
                const uint8_t *src = query(cur, t, x);
                v[x] = src ? *reinterpret_cast<const uint4 *>(src) : make_uint4(0, 0, 0, 0);
            }
            float back = 1.f, sum = 0.f;
            if (BF16) {
                uint32_t top = 0;
#pragma unroll
                for (int x = 0; x < D / 32; ++x)
                    top = __vmaxu2(__vmaxu2(top, v[x].x & 0x7fff7fffu), __vmaxu2(__vmaxu2(v[x].y & 0x7fff7fffu, v[x].z & 0x7fff7fffu), v[x].w & 0x7fff7fffu));
                top = max(top & 0xffffu, top >> 16);
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                int e = (int)(top >> 7) - 127; // exponent of the largest magnitude
                e = e > 127 || top == 0 ? 0 : max(e, -126);
                const float down = __int_as_float(e == 127 ? 0x00400000 : (127 - e) << 23); // 2^-e (e = 127: a subnormal)
                back = __int_as_float((127 + e) << 23);
#pragma unroll
                for (int x = 0; x < D / 32; ++x) {
                    uint32_t *w = &v[x].x;
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const float2 f = half_pair_to_float(w[y], true);
                        w[y] = float_pair_to_half(f.x * down, f.y * down, false);
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < D / 32; ++x) {
                const uint32_t w[4] = { v[x].x, v[x].y, v[x].z, v[x].w };
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const float2 f = half_pair_to_float(w[y], false);
                    sum += f.x + f.y;
                }
                // 8 bits: 4 features a step; 4 bits: a word of 8 codes is two steps, its pairs (1, 5), (0, 4) and (2, 6), (3, 7) apart
                const uint2 f0 = BITS == 8 ? make_uint2(w[0], w[1]) : make_uint2(__byte_perm(w[0], w[2], 0x5410), __byte_perm(w[0], w[2], 0x7632));
                const uint2 f1 = BITS == 8 ? make_uint2(w[2], w[3]) : make_uint2(__byte_perm(w[1], w[3], 0x5410), __byte_perm(w[1], w[3], 0x7632));
                qr[t][2 * x] = f0;
                qr[t][2 * x + 1] = f1;
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const float f = a.scale_log2 * back;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                rf[t][c] = __shfl_sync(0xffffffffu, f, 8 * q + 4 * c);
                rs[t][c] = __shfl_sync(0xffffffffu, sum * f, 8 * q + 4 * c);
                m[t][c] = -inf;
                l[t][c] = bias[t][c] = 0.f;
            }
            if (q == 0)
                masks[8 * t + r] = at >= rows ? 0 : a.tree ? a.tree[(size_t)cur.b * a.n + i] : i >= 63 ? ~0ull : (2ull << i) - 1;
#pragma unroll
            for (int x = 0; x < kTiles; ++x)
                O[t][x][0] = O[t][x][1] = O[t][x][2] = O[t][x][3] = 0.f;
        }
        __syncwarp();
        float vmax = 0.f, vnorm = 1.f; // value scales below vmax = 2^(L + 1) are brought to 2^6 by vnorm = 2^(6 - L)
        int L = -121;

        // ---- granules
        const int mine = cur.g1 - cur.g0;
        uint32_t good = now.good;
        bool dead = false;
        for (int i = 0; i < mine; ++i) {
            if ((i & 31) == 0 && i) {
                good = ahead.good;
                now = ahead;
                ahead = batch_of(cur, i + 32);
            }
            const int g = cur.g0 + i;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[get_stage], get_phase, a.status, STATUS_TIMEOUT_TMA))) {
                dead = true;
                break;
            }
            const uint8_t *st = ring + get_stage * kGranule;
            if (good >> (i & 31) & 1) {
                uint32_t kw[2][kKW], vw[4][kVW];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    lds<(RB == 32 ? 8 : 16)>(kw[h], st + koff + h * 8 * RB);
                    if (RB == 128)
                        lds<16>(&kw[h][kKW / 2], st + (koff ^ 64) + h * 8 * RB);
                }
                const uint8_t *par = st + kv_param_offset(RB, 0) + 4 * tok;
                float2 kp[2], vp[2];
                kp[0] = half_pair_to_float(*reinterpret_cast<const uint32_t *>(par), BF16);
                kp[1] = half_pair_to_float(*reinterpret_cast<const uint32_t *>(par + 32), BF16);
                vp[0] = half_pair_to_float(*reinterpret_cast<const uint32_t *>(par + 64), BF16);
                vp[1] = half_pair_to_float(*reinterpret_cast<const uint32_t *>(par + 96), BF16);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    lds<RB / 8>(vw[e], st + 16 * RB + ((voff + e * 4 * RB) ^ ((e & 1) * 64)));
                float s[NT][4];
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    uint32_t f0, f1, f2, f3;
                    if (BITS == 8) {
                        f0 = key_bytes_lo(kw[0][k]), f1 = key_bytes_lo(kw[1][k]), f2 = key_bytes_hi(kw[0][k]), f3 = key_bytes_hi(kw[1][k]);
                    } else { // the pairs of nibbles 0 and 1, or 2 and 3, of both halves of the word
                        const uint32_t x = kw[0][k >> 1], y = kw[1][k >> 1];
                        f0 = key_nibbles(k & 1 ? x >> 4 : x << 4), f1 = key_nibbles(k & 1 ? y >> 4 : y << 4);
                        f2 = key_nibbles(k & 1 ? x >> 8 : x), f3 = key_nibbles(k & 1 ? y >> 8 : y);
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        mma_f16(s[t], f0, f1, f2, f3, qr[t][k].x, qr[t][k].y);
                    }
                }
                const float ks0 = kp[0].x * kKeyScale, ks1 = kp[1].x * kKeyScale;
                const float ko0 = fmaf(kKeyOffset, kp[0].x, kp[0].y), ko1 = fmaf(kKeyOffset, kp[1].x, kp[1].y);
                float vo0 = fmaf(kCentre, vp[0].x, vp[0].y), vo1 = fmaf(kCentre, vp[1].x, vp[1].y);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        s[t][c] = fmaf(s[t][c], ks0 * rf[t][c], ko0 * rs[t][c]);
                        s[t][2 + c] = fmaf(s[t][2 + c], ks1 * rf[t][c], ko1 * rs[t][c]);
                    }
                const bool edge = 16 * g + 16 > ctx; // some of these tokens are drafts, or lie behind the end
                uint32_t seen = ~0u;
                if (edge) {
                    const int t0 = 16 * g + tok;
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int at = t0 + (c >> 1) * 8;
                            const bool see = at < ctx || (at < len && (masks[8 * t + 2 * q + (c & 1)] >> (at - ctx) & 1));
                            if (!see) {
                                s[t][c] = -inf;
                                seen &= ~(1u << (4 * t + c));
                            }
                        }
                    if (t0 >= len) // (what lies there belongs to no token)
                        vp[0].x = vo0 = 0.f;
                    if (t0 + 8 >= len)
                        vp[1].x = vo1 = 0.f;
                }
                // ---- running maximum, and the largest value scale
                bool raise = (vp[0].x >= vmax && vp[0].x < inf) || (vp[1].x >= vmax && vp[1].x < inf);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        raise |= fmaxf(s[t][c], s[t][2 + c]) > m[t][c] + 8.f;
                if (__any_sync(0xffffffffu, raise)) {
                    const uint32_t v0 = vp[0].x < inf ? __float_as_uint(vp[0].x) : 0u, v1 = vp[1].x < inf ? __float_as_uint(vp[1].x) : 0u;
                    const uint32_t top = __reduce_max_sync(0xffffffffu, max(v0, v1)); // scales are not negative: ordered like their bits
                    const int Ln = max(L, max((int)(top >> 23) - 127, -120));
                    const float down = ex2((float)(L - Ln));
                    L = Ln;
                    vmax = __int_as_float(min(128 + L, 255) << 23);
                    vnorm = __int_as_float((133 - L) << 23);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        float f[2];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float x = fmaxf(s[t][c], s[t][2 + c]);
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                            const float mn = fmaxf(m[t][c], x);
                            f[c] = mn == -inf ? 1.f : ex2(m[t][c] - mn);
                            m[t][c] = mn;
                            l[t][c] *= f[c];
                            bias[t][c] *= f[c];
                            f[c] *= down;
                        }
#pragma unroll
                        for (int x = 0; x < kTiles; ++x) {
                            O[t][x][0] *= f[0];
                            O[t][x][1] *= f[1];
                            O[t][x][2] *= f[0];
                            O[t][x][3] *= f[1];
                        }
                    }
                }
                // ---- weights
                const float vf0 = vp[0].x * vnorm, vf1 = vp[1].x * vnorm;
                uint32_t pb[NT][2], pl[2];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float pv[4], pw[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float mm = m[t][c & 1] == -inf ? 0.f : m[t][c & 1];
                        const float p = ex2(s[t][c] - mm);
                        l[t][c & 1] += p;
                        pv[c] = p * (c < 2 ? vf0 : vf1);
                        pw[c] = p * (c < 2 ? vo0 : vo1);
                    }
                    if (edge) { // an unseen value may be Inf or NaN: 0 times that is no 0
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (!(seen >> (4 * t + c) & 1))
                                pv[c] = pw[c] = 0.f;
                    }
                    bias[t][0] += pw[0] + pw[2];
                    bias[t][1] += pw[1] + pw[3];
                    const uint32_t h0 = float_pair_to_half(pv[0], pv[1], false), h1 = float_pair_to_half(pv[2], pv[3], false);
                    pb[t][0] = movmatrix(h0);
                    pb[t][1] = movmatrix(h1);
                    if (kRemainder) {
                        const float2 x0 = half_pair_to_float(h0, false), x1 = half_pair_to_float(h1, false);
                        pl[0] = movmatrix(float_pair_to_half(pv[0] - x0.x, pv[1] - x0.y, false));
                        pl[1] = movmatrix(float_pair_to_half(pv[2] - x1.x, pv[3] - x1.y, false));
                    }
                }
                // ---- O^T += V^T P^T: this lane's features are D / 8 neighbours, two an MMA
                auto add = [&](int tile, uint32_t f0, uint32_t f1, uint32_t f2, uint32_t f3) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        mma_f16(O[t][tile], f0, f1, f2, f3, pb[t][0], pb[t][1]);
                    if (kRemainder)
                        mma_f16(O[0][tile], f0, f1, f2, f3, pl[0], pl[1]);
                };
#pragma unroll
                for (int w = 0; w < kVW; ++w) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (BITS == 8) {
                            const uint32_t x = __byte_perm(vw[0][w], vw[1][w], h ? 0x7362 : 0x5140), y = __byte_perm(vw[2][w], vw[3][w], h ? 0x7362 : 0x5140);
                            add(2 * w + h, bytes_lo(x), bytes_hi(x), bytes_lo(y), bytes_hi(y));
                        } else {
                            const uint32_t x = __byte_perm(vw[0][w], vw[1][w], h ? 0x7632 : 0x5410), y = __byte_perm(vw[2][w], vw[3][w], h ? 0x7632 : 0x5410);
                            add((4 * w + 2 * h) % kTiles, nibbles_lo(x), nibbles_hi(x), nibbles_lo(y), nibbles_hi(y));
                            add((4 * w + 2 * h + 1) % kTiles, nibbles_lo(x >> 8), nibbles_hi(x >> 8), nibbles_lo(y >> 8), nibbles_hi(y >> 8));
                        }
                    }
                }
            }
            __syncwarp(); // every lane has read the slot
            --pending;
            if (i + kStages < mine) {
                const int j = i + kStages;
                issue((j >> 5) == (i >> 5) ? now.at : ahead.at, j & 31);
            }
            get_stage = get_stage + 1 == kStages ? 0 : get_stage + 1;
            get_phase ^= get_stage == 0;
        }
        if (dead)
            break;

        // ---- the next piece's first copies go out before this one's result is written
        Piece next;
        const bool more = line.next(a, next);
        if (more) {
            prefetch_queries(next);
            now = batch_of(next, 0);
            if (next.g1 - next.g0 > 32)
                ahead = batch_of(next, 32);
            for (int i = 0; i < min(next.g1 - next.g0, kStages); ++i)
                issue(now.at, i);
        }
        const float undo = __int_as_float((121 + L) << 23); // 2^(L - 6); L >= -121
        const bool whole = cur.g0 == 0 && cur.g1 == cur.G;
        const size_t slot = 2 * (size_t)run + (cur.first ? 0 : 1);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    l[t][c] += __shfl_xor_sync(0xffffffffu, l[t][c], o);
                    bias[t][c] += __shfl_xor_sync(0xffffffffu, bias[t][c], o);
                }
                const int row = 8 * t + 2 * q + c, at = row0 + row;
                if (at >= rows)
                    continue;
                float v[D / 8];
#pragma unroll
                for (int x = 0; x < kTiles; ++x) {
                    v[2 * x] = fmaf(O[t][x][c], undo, bias[t][c]);
                    v[2 * x + 1] = fmaf(O[t][x][2 + c], undo, bias[t][c]);
                }
                if (whole) {
                    const float inv = l[t][c] == 0.f ? 0.f : 1.f / l[t][c];
                    const int i = at / a.group;
                    uint8_t *dst = a.out + ((long long)cur.b * a.n + i) * a.out_stride + (long long)(head * a.group + at - i * a.group) * a.out_head_stride + r * (D / 4);
#pragma unroll
                    for (int x = 0; x < D / 8; x += 8)
                        *reinterpret_cast<uint4 *>(dst + 2 * x) =
                            make_uint4(float_pair_to_half(v[x] * inv, v[x + 1] * inv, BF16), float_pair_to_half(v[x + 2] * inv, v[x + 3] * inv, BF16),
                                       float_pair_to_half(v[x + 4] * inv, v[x + 5] * inv, BF16), float_pair_to_half(v[x + 6] * inv, v[x + 7] * inv, BF16));
                } else {
                    float *dst = a.part + (slot * a.slot_rows + row) * D + r * (D / 8);
#pragma unroll
                    for (int x = 0; x < D / 8; x += 4)
                        *reinterpret_cast<float4 *>(dst + x) = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
                    if (r == 0)
                        reinterpret_cast<float2 *>(a.part + 2 * (size_t)a.runs * a.slot_rows * D)[slot * a.slot_rows + row] = make_float2(m[t][c], l[t][c]);
                }
            }
        if (!more)
            break;
        cur = next;
    }
    for (; pending > 0; --pending) { // a wait ran out: no copy may be under way when the warp ends
        mbar_wait_bounded(&full[get_stage], get_phase, a.status, STATUS_TIMEOUT_TMA);
        get_stage = get_stage + 1 == kStages ? 0 : get_stage + 1;
        get_phase ^= get_stage == 0;
    }
}

// Items that several warps hold: their pieces in order.  Sequences without a token: rows of 0.  D / 8 threads a row; what is left of the block's groups of
// them takes pieces in turn (`row_groups` rows at a time, a power of two).
template <int D, bool BF16>
__global__ void __launch_bounds__(kCaThreads) cache_attention_combine_kernel(const __grid_constant__ CacheAttnArgs a, int tile_rows, int row_groups)
{
    constexpr int kLanes = D / 8, kGroups = kCaThreads / kLanes;
    __shared__ float sums[kCaThreads][9];
    const int items = a.kv_heads * a.row_blocks, b = blockIdx.x / items, item = blockIdx.x - b * items;
    long long units, prefix;
    ca_sums(a, b, units, prefix);
    const long long quota = ca_quota(a, units * items);
    const int G = ca_granules(a, b);
    const long long start = prefix * items + (long long)item * ca_units(a, G);
    int c0 = 0, c1 = 0;
    if (G) {
        c0 = (int)ca_div(start + a.extra, quota);
        c1 = (int)ca_div(start + a.extra + G - 1, quota);
    }
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    if (G && c0 == c1)
        return;
    const int head = item / a.row_blocks, row0 = (item - head * a.row_blocks) * tile_rows, rows = min(a.n * a.group - row0, tile_rows);
    const int sub = threadIdx.x % kLanes, grp = threadIdx.x / kLanes, row = blockIdx.y * row_groups + grp % row_groups, turn = grp / row_groups, turns = kGroups / row_groups;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + 2 * (size_t)a.runs * a.slot_rows * D);
    float v[8] = {}, lsum = 0.f;
    if (row < rows && G) {
        auto slot_of = [&](int c) { return 2 * (size_t)c + (c == c0 && c0 * quota < start ? 1 : 0); };
        float2 p[4];
        float4 lo[4], hi[4];
        auto fetch = [&](int c) { // four pieces under way
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int at = c + u * turns;
                p[u] = make_float2(-INFINITY, 0.f);
                lo[u] = hi[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (at <= c1) {
                    const size_t slot = slot_of(at) * a.slot_rows + row;
                    const float *src = a.part + slot * D + sub * 8;
                    p[u] = ml[slot];
                    lo[u] = *reinterpret_cast<const float4 *>(src);
                    hi[u] = *reinterpret_cast<const float4 *>(src + 4);
                }
            }
        };
        fetch(c0 + turn); // (used behind the maximum)
        float top = -INFINITY;
        for (int c = c0 + sub; c <= c1; c += 4 * kLanes) {
            float x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                x[u] = c + u * kLanes <= c1 ? ml[slot_of(c + u * kLanes) * a.slot_rows + row].x : -INFINITY;
            top = fmaxf(top, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
        }
        const unsigned lanes = kLanes == 16 ? 0xffffu << (threadIdx.x & 16) : 0xffu << (threadIdx.x & 24);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1)
            top = fmaxf(top, __shfl_xor_sync(lanes, top, o));
        for (int c = c0 + turn; c <= c1;) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float f = p[u].x == -INFINITY ? 1.f : ex2(p[u].x - top);
                lsum = fmaf(f, p[u].y, lsum);
                v[0] = fmaf(f, lo[u].x, v[0]), v[1] = fmaf(f, lo[u].y, v[1]), v[2] = fmaf(f, lo[u].z, v[2]), v[3] = fmaf(f, lo[u].w, v[3]);
                v[4] = fmaf(f, hi[u].x, v[4]), v[5] = fmaf(f, hi[u].y, v[5]), v[6] = fmaf(f, hi[u].z, v[6]), v[7] = fmaf(f, hi[u].w, v[7]);
            }
            c += 4 * turns;
            if (c <= c1)
                fetch(c);
        }
    }
    if (turns > 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            sums[threadIdx.x][e] = v[e];
        sums[threadIdx.x][8] = lsum;
        __syncthreads();
        if (turn)
            return;
        for (int x = 1; x < turns; ++x) {
            const float *s = sums[threadIdx.x + x * row_groups * kLanes];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] += s[e];
            lsum += s[8];
        }
    }
    if (row >= rows)
        return;
    const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
    const int at = row0 + row, i = at / a.group, hh = at - i * a.group;
    *reinterpret_cast<uint4 *>(a.out + ((long long)b * a.n + i) * a.out_stride + (long long)(head * a.group + hh) * a.out_head_stride + sub * 16) =
        make_uint4(float_pair_to_half(v[0] * inv, v[1] * inv, BF16), float_pair_to_half(v[2] * inv, v[3] * inv, BF16),
                   float_pair_to_half(v[4] * inv, v[5] * inv, BF16), float_pair_to_half(v[6] * inv, v[7] * inv, BF16));
}

} // namespace abq
