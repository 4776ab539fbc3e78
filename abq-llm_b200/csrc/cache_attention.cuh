// Attention of a token step over the quantised cache (abq_cache_attention): one token of a decode step, or a tree of drafted tokens.
//
// Keys are k_j = kmin_j + ks_j c_j with codes c_j (16 bits hold min and scale, the tensor cores multiply the codes, centred: c' = c - 2^(bits-1), exact
// in fp16), so  q . k_j = ks_j (q . c'_j) + (kmin_j + 2^(bits-1) ks_j) sum(q), and likewise  sum_j p_j v_j = sum_j (p_j vs_j) c'_j + sum_j p_j (vmin_j + ..).
// Products are transposed (tokens are the 16 rows of an m16n8k16 MMA, query rows its 8 columns): a granule of 16 tokens costs D / 16 instructions for
// S^T = K Q^T and D / 16 for O^T += V^T P^T per 8 query rows, and one conversion of its codes however many rows there are.
//
// What bounds it is HBM (2 * bits / 8 bytes per feature and token, read once) as long as a granule costs few instructions. So the work is split evenly:
// the granules of all sequences and heads are one line that the CTAs cut into equal runs, whatever the lengths; a CTA's warps take granules in turn, each
// through a ring of its own of bulk copies (a granule is one contiguous copy), and keep their own running maxima and sums.  Pieces of a
// (sequence, head) that several CTAs hold meet in the workspace, added by a second kernel in order (no atomics).
//
//  * Running maximum: raised only when a score passes it by more than 2^8 (checked with one vote), so that shuffles and the scaling of O are rare.
//  * p vs_j is rounded to fp16 after scaling by a power of two that keeps the largest vs seen so far near 2^6: with p <= 2^8 the product is below 2^15 and
//    keeps 11 bits down to 2^-29 of it, so that many small weights are not lost beside one large.
//  * Queries: fp16 as they are; bf16 rows are scaled by a power of two to [1, 2) and held in fp16 (exact down to 2^-14 of the row's largest).
#pragma once
#include "abq_kernels.h"
#include "kv_cache.cuh"

namespace abq {

constexpr int kCaWarps = 4;
constexpr int kCaThreads = 32 * kCaWarps;
constexpr int kCaMaxCtas = 296; // two per SM
constexpr int kCaMinQuota = 8;  // granules a CTA takes at least: two per warp

struct CacheAttnArgs {
    const uint8_t *data;
    const uint8_t *q;
    uint8_t *out;
    long long q_stride, q_head_stride, out_stride, out_head_stride; // bytes
    const int *table, *seq_lens;
    const uint64_t *tree;
    float *part; // [2 * ctas][8 NT][D] sums, then [2 * ctas][8 NT] pairs (maximum, sum of p)
    int *status;
    int num_pages, page_granules, kv_heads, batch, n, group, row_blocks, table_stride, ctas;
    float scale_log2;
    bool bf16;
};

// How the granules of all (sequence, head, row block) items are dealt: item k of sequence b starts at heads * prefix(b) + k * granules(b).
struct CaSplit {
    long long total;
    long long quota;
};

__device__ __forceinline__ int ca_tokens(const CacheAttnArgs &a, int b)
{
    const long long cap = (long long)a.table_stride * a.page_granules * kGranuleTokens;
    const int len = a.seq_lens[b];
    return len < 0 ? 0 : (int)min((long long)min(len, 0x7fffff00), cap);
}
__device__ __forceinline__ int ca_granules(const CacheAttnArgs &a, int b) { return (int)(((long long)ca_tokens(a, b) + 15) >> 4); }

// Block-wide: granules of all sequences, and of those before sequence `before` (one head each).
__device__ __forceinline__ void ca_sums(const CacheAttnArgs &a, int before, long long *scratch, long long &all, long long &prefix)
{
    long long s = 0, p = 0;
    for (int b = threadIdx.x; b < a.batch; b += kCaThreads) {
        const int g = ca_granules(a, b);
        s += g;
        p += b < before ? g : 0;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        p += __shfl_xor_sync(0xffffffffu, p, o);
    }
    if ((threadIdx.x & 31) == 0) {
        scratch[threadIdx.x >> 5] = s;
        scratch[kCaWarps + (threadIdx.x >> 5)] = p;
    }
    __syncthreads();
    all = prefix = 0;
#pragma unroll
    for (int w = 0; w < kCaWarps; ++w) {
        all += scratch[w];
        prefix += scratch[kCaWarps + w];
    }
}
__device__ __forceinline__ CaSplit ca_split(const CacheAttnArgs &a, long long granules)
{
    CaSplit s;
    s.total = granules * a.kv_heads * a.row_blocks;
    s.quota = max((s.total + a.ctas - 1) / a.ctas, (long long)kCaMinQuota);
    return s;
}

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
// 0x6400 | c is the fp16 number 1024 + c.  Pairs of centred codes from ...
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
    static constexpr int kMerge = kCaWarps * 8 * D * 4, kQ = NT * kSteps * 32 * 8;
    static constexpr int kFixed = kMerge + kQ + kRows * (4 + 4 + 8) + kCaWarps * kRows * 12 + 128;
    static constexpr int kRoom = 112 * 1024 - kFixed; // two CTAs per SM
    static constexpr int kStages = kRoom / (kCaWarps * (kGranule + 8)) < 12 ? kRoom / (kCaWarps * (kGranule + 8)) : 12;
    static constexpr int kSmem = kFixed + kCaWarps * kStages * (kGranule + 8);
    static_assert(kStages >= 2 && kStages <= 32, "ring");
};

template <int D, int BITS, int NT>
__global__ void __launch_bounds__(kCaThreads, 2) cache_attention_kernel(const __grid_constant__ CacheAttnArgs a)
{
    using Sh = CaShape<D, BITS, NT>;
    constexpr int RB = Sh::RB, kGranule = Sh::kGranule, kRows = Sh::kRows, kSteps = Sh::kSteps, kStages = Sh::kStages, kTiles = D / 16;
    constexpr int kKW = RB / 16, kVW = RB / 32; // 32-bit words of codes per lane and token
    constexpr float kCentre = (float)(1 << (BITS - 1));
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem;
    float *merge = reinterpret_cast<float *>(ring + kCaWarps * kStages * kGranule);
    uint2 *qfrag = reinterpret_cast<uint2 *>(merge + kCaWarps * 8 * D);
    uint64_t *masks = reinterpret_cast<uint64_t *>(qfrag + NT * kSteps * 32);
    uint64_t *bars = masks + kRows;
    long long *scratch = reinterpret_cast<long long *>(bars + kCaWarps * kStages);
    float *row_f = reinterpret_cast<float *>(scratch + 2 * kCaWarps), *row_sum = row_f + kRows;
    float *w_m = row_sum + kRows, *w_l = w_m + kCaWarps * kRows, *w_b = w_l + kCaWarps * kRows;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;
    uint64_t *full = bars + warp * kStages;
    uint8_t *wring = ring + warp * kStages * kGranule;
    if (lane < kStages)
        mbar_init(&full[lane], 1);
    fence_mbar_init();
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait_prior_grid();

    // ---- this CTA's run of the line
    long long granules, unused;
    ca_sums(a, 0, scratch, granules, unused);
    const CaSplit split = ca_split(a, granules);
    const long long run0 = (long long)blockIdx.x * split.quota, run1 = min(split.total, run0 + split.quota);
    if (run0 >= run1)
        return; // (before any copy)
    const int items = a.kv_heads * a.row_blocks;
    int b = 0, G = 0;
    long long rem = run0; // granules from the start of sequence b
    for (int b0 = 0;; b0 += 32) { // 32 sequences at a time
        const int own = b0 + lane < a.batch ? ca_granules(a, b0 + lane) : 0;
        long long end = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, end, o);
            end += lane >= o ? x : 0;
        }
        end *= items;
        const uint32_t behind = __ballot_sync(0xffffffffu, rem < end);
        if (behind) {
            const int at = __ffs(behind) - 1;
            b = b0 + at;
            G = __shfl_sync(0xffffffffu, own, at);
            rem -= __shfl_sync(0xffffffffu, end, at) - (long long)G * items;
            break;
        }
        rem -= __shfl_sync(0xffffffffu, end, 31);
    }
    int item = (int)(rem / G), g0 = (int)(rem - (long long)item * G);
    long long left = run1 - run0;

    // ---- ring of granules: lane i % 32 owns the address of this warp's granule i of the piece
    struct Batch {
        uint32_t at;   // index of the granule in the cache, or ~0
        uint32_t good; // ballot: which of the 32 lie in the cache
    };
    auto batch_of = [&](int base, int pb, int pitem, int pg0, int pg1) {
        Batch t;
        const int g = pg0 + warp + kCaWarps * (base + lane);
        t.at = ~0u;
        if (g < pg1) {
            const int entry = g / a.page_granules, page = a.table[(size_t)pb * a.table_stride + entry];
            if (page >= 0 && page < a.num_pages)
                t.at = ((uint32_t)page * a.kv_heads + pitem / a.row_blocks) * a.page_granules + (g - entry * a.page_granules);
            else if (a.status)
                atomicOr(a.status, ABQ_STATUS_BAD_PAGE);
        }
        t.good = __ballot_sync(0xffffffffu, t.at != ~0u);
        return t;
    };
    uint32_t put_stage = 0, get_stage = 0, get_phase = 0; // of the warp's ring, over all pieces
    int pending = 0; // copies not yet waited for
    bool dead = false;
    auto issue = [&](uint32_t at, int owner) {
        ++pending;
        if (lane == owner) {
            uint64_t *bar = &full[put_stage];
            if (at != ~0u) {
                mbar_arrive_expect_tx(bar, kGranule);
                bulk_load(wring + put_stage * kGranule, a.data + (size_t)at * kGranule, kGranule, bar);
            } else {
                mbar_arrive(bar); // nothing to wait for
            }
        }
        put_stage = put_stage + 1 == kStages ? 0 : put_stage + 1;
    };
    auto piece_end = [&](int pg0, int pG, long long pleft) { return (int)min((long long)pG, pg0 + pleft); };
    auto count_of = [&](int pg0, int pg1) { return (pg1 - pg0 - warp + kCaWarps - 1) / kCaWarps; }; // granules of this warp

    int g1 = piece_end(g0, G, left);
    Batch cur = batch_of(0, b, item, g0, g1), nxt = batch_of(32, b, item, g0, g1);
    int mine = count_of(g0, g1);
    for (int i = 0; i < min(mine, kStages); ++i)
        issue(cur.at, i);
    bool first_piece = true;

    for (;;) {
        const int head = item / a.row_blocks, row0 = (item - head * a.row_blocks) * kRows, rows = a.n * a.group;
        const int len = ca_tokens(a, b), ctx = len - a.n;
        // ---- queries: fragments of the MMA's B operand in shared memory; row factors; masks
        for (int x = threadIdx.x; x < kRows * (D / 8); x += kCaThreads) {
            const int row = x / (D / 8), sub = x % (D / 8), at = row0 + row;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (at < rows) {
                const int i = at / a.group, hh = at - i * a.group;
                v = *reinterpret_cast<const uint4 *>(a.q + ((long long)b * a.n + i) * a.q_stride + (long long)(head * a.group + hh) * a.q_head_stride + sub * 16);
            }
            uint32_t w[4] = { v.x, v.y, v.z, v.w };
            float back = 1.f, sum = 0.f;
            if (a.bf16) {
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    top = max(top, max(w[e] & 0x7fffu, w[e] >> 16 & 0x7fffu));
#pragma unroll
                for (int o = 1; o < D / 8; o <<= 1)
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                int e = (int)(top >> 7) - 127; // exponent of the largest magnitude
                e = e > 127 || top == 0 ? 0 : max(e, -126);
                const float down = __int_as_float((127 - e) << 23 ? (127 - e) << 23 : 0x00400000); // 2^-e (e = 127: a subnormal)
                back = __int_as_float((127 + e) << 23);
#pragma unroll
                for (int e2 = 0; e2 < 4; ++e2) {
                    const float2 f = half_pair_to_float(w[e2], true);
                    w[e2] = float_pair_to_half(f.x * down, f.y * down, false);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = half_pair_to_float(w[e], false);
                sum += f.x + f.y;
            }
#pragma unroll
            for (int o = 1; o < D / 8; o <<= 1)
                sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (sub == 0) {
                row_f[row] = a.scale_log2 * back;
                row_sum[row] = sum * (a.scale_log2 * back);
                const int i = at / a.group;
                masks[row] = at >= rows ? 0 : a.tree ? a.tree[(size_t)b * a.n + i] : i >= 63 ? ~0ull : (2ull << i) - 1;
            }
            uint2 *dst = qfrag + (size_t)(row >> 3) * kSteps * 32 + (row & 7) * 4;
            if (BITS == 8) { // lane q: 16 features of each half (64 wide) of the row, 4 a step
                const int d = sub * 8, s = (d >> 6) * 4 + ((d & 15) >> 2), qq = (d & 63) >> 4;
                dst[s * 32 + qq] = make_uint2(w[0], w[1]);
                dst[(s + 1) * 32 + qq] = make_uint2(w[2], w[3]);
            } else { // a word of 8 codes is two steps; its pairs are (0, 4), (1, 5) and (2, 6), (3, 7)
                constexpr int kWords = D / 32; // words per lane and token
                const int s = (sub % kWords) * 2, qq = sub / kWords;
                dst[s * 32 + qq] = make_uint2(__byte_perm(w[0], w[2], 0x5410), __byte_perm(w[0], w[2], 0x7632));
                dst[(s + 1) * 32 + qq] = make_uint2(__byte_perm(w[1], w[3], 0x5410), __byte_perm(w[1], w[3], 0x7632));
            }
        }
        __syncthreads();
        constexpr bool kQRegs = NT <= 2;
        uint2 qr[kQRegs ? NT : 1][kSteps];
        if (kQRegs) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
                    qr[t][s] = qfrag[(t * kSteps + s) * 32 + lane];
        }
        float m[NT][2], l[NT][2], bias[NT][2], O[NT][kTiles][4], rf[NT][2], rs[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m[t][c] = -INFINITY;
                l[t][c] = bias[t][c] = 0.f;
                rf[t][c] = row_f[8 * t + 2 * q + c];
                rs[t][c] = row_sum[8 * t + 2 * q + c];
            }
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
                O[t][i][0] = O[t][i][1] = O[t][i][2] = O[t][i][3] = 0.f;
        }
        float vmax = 0.f, vnorm = 1.f; // value scales below vmax = 2^(L + 1) are brought to 2^6 by vnorm = 2^(6 - L)
        int L = -121;

        // ---- this warp's granules
        const int tok = (r & 1) * 4 + (r >> 1); // MMA row r holds token tok, row r + 8 token tok + 8: then P's columns are tokens q, 4 + q, 8 + q, 12 + q
        const int koff = kv_place<RB>(tok, q * (RB == 32 ? 8 : 16)), voff = kv_place<RB>(q, r * (RB / 8));
        uint32_t good = cur.good;
        for (int i = 0; i < mine; ++i) {
            if ((i & 31) == 0 && i) { // (the batch that is being issued from is at most one ahead)
                good = nxt.good;
                cur = nxt;
                nxt = batch_of(i + 32, b, item, g0, g1);
            }
            const int g = g0 + warp + kCaWarps * i;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[get_stage], get_phase, a.status, STATUS_TIMEOUT_TMA))) {
                dead = true;
                break;
            }
            const uint8_t *st = wring + get_stage * kGranule;
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
                kp[0] = half_pair_to_float(*reinterpret_cast<const uint32_t *>(par), a.bf16);
                kp[1] = half_pair_to_float(*reinterpret_cast<const uint32_t *>(par + 32), a.bf16);
                vp[0] = half_pair_to_float(*reinterpret_cast<const uint32_t *>(par + 64), a.bf16);
                vp[1] = half_pair_to_float(*reinterpret_cast<const uint32_t *>(par + 96), a.bf16);
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
                        f0 = bytes_lo(kw[0][k]), f1 = bytes_lo(kw[1][k]), f2 = bytes_hi(kw[0][k]), f3 = bytes_hi(kw[1][k]);
                    } else {
                        const uint32_t x = kw[0][k >> 1] >> (8 * (k & 1)), y = kw[1][k >> 1] >> (8 * (k & 1));
                        f0 = nibbles_lo(x), f1 = nibbles_lo(y), f2 = nibbles_hi(x), f3 = nibbles_hi(y);
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const uint2 qq = kQRegs ? qr[kQRegs ? t : 0][k] : qfrag[(t * kSteps + k) * 32 + lane];
                        mma_f16(s[t], f0, f1, f2, f3, qq.x, qq.y);
                    }
                }
                const float ko0 = fmaf(kCentre, kp[0].x, kp[0].y), ko1 = fmaf(kCentre, kp[1].x, kp[1].y);
                float vo0 = fmaf(kCentre, vp[0].x, vp[0].y), vo1 = fmaf(kCentre, vp[1].x, vp[1].y);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        s[t][c] = fmaf(s[t][c], kp[0].x * rf[t][c], ko0 * rs[t][c]);
                        s[t][2 + c] = fmaf(s[t][2 + c], kp[1].x * rf[t][c], ko1 * rs[t][c]);
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
                                s[t][c] = -INFINITY;
                                seen &= ~(1u << (4 * t + c));
                            }
                        }
                    if (t0 >= len) // (what lies there belongs to no token)
                        vp[0].x = vo0 = 0.f;
                    if (t0 + 8 >= len)
                        vp[1].x = vo1 = 0.f;
                }
                // ---- running maximum, and the largest value scale
                const float inf = INFINITY;
                bool raise = (vp[0].x >= vmax && vp[0].x < inf) || (vp[1].x >= vmax && vp[1].x < inf);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        raise |= s[t][c] > m[t][c & 1] + 8.f;
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
                uint32_t pb[NT][2];
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
                    pb[t][0] = movmatrix(float_pair_to_half(pv[0], pv[1], false));
                    pb[t][1] = movmatrix(float_pair_to_half(pv[2], pv[3], false));
                }
                // ---- O^T += V^T P^T: this lane's features are D / 8 neighbours, two an MMA
#pragma unroll
                for (int w = 0; w < kVW; ++w) {
                    if (BITS == 8) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t x = __byte_perm(vw[0][w], vw[1][w], h ? 0x7362 : 0x5140), y = __byte_perm(vw[2][w], vw[3][w], h ? 0x7362 : 0x5140);
                            const uint32_t f0 = bytes_lo(x), f1 = bytes_hi(x), f2 = bytes_lo(y), f3 = bytes_hi(y);
#pragma unroll
                            for (int t = 0; t < NT; ++t)
                                mma_f16(O[t][2 * w + h], f0, f1, f2, f3, pb[t][0], pb[t][1]);
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t x = __byte_perm(vw[0][w], vw[1][w], h ? 0x7632 : 0x5410), y = __byte_perm(vw[2][w], vw[3][w], h ? 0x7632 : 0x5410);
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                const uint32_t f0 = nibbles_lo(x >> (8 * u)), f1 = nibbles_hi(x >> (8 * u)), f2 = nibbles_lo(y >> (8 * u)), f3 = nibbles_hi(y >> (8 * u));
#pragma unroll
                                for (int t = 0; t < NT; ++t)
                                    mma_f16(O[t][(4 * w + 2 * h + u) % kTiles], f0, f1, f2, f3, pb[t][0], pb[t][1]);
                            }
                        }
                    }
                }
            }
            __syncwarp(); // every lane has read the slot
            --pending;
            if (i + kStages < mine) {
                const int j = i + kStages;
                issue((j >> 5) == (i >> 5) ? cur.at : nxt.at, j & 31);
            }
            get_stage = get_stage + 1 == kStages ? 0 : get_stage + 1;
            get_phase ^= get_stage == 0;
        }

        // ---- the next piece's first copies go out before this one is finished
        const int pb_ = b, phead = head, prow0 = row0, pg0 = g0, pg1 = g1, pG = G;
        left -= g1 - g0;
        const bool more = left > 0;
        if (more) {
            g0 = 0;
            if (++item == items) {
                item = 0;
                do {
                    G = ca_granules(a, ++b);
                } while (G == 0);
            }
            g1 = piece_end(0, G, left);
            mine = dead ? 0 : count_of(0, g1);
            cur = batch_of(0, b, item, 0, g1);
            nxt = batch_of(32, b, item, 0, g1);
            for (int i = 0; i < min(mine, kStages); ++i)
                issue(cur.at, i);
        }

        // ---- the warps' sums meet
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    l[t][c] += __shfl_xor_sync(0xffffffffu, l[t][c], o);
                    bias[t][c] += __shfl_xor_sync(0xffffffffu, bias[t][c], o);
                }
        if (r == 0) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int row = 8 * t + 2 * q + c;
                    w_m[warp * kRows + row] = m[t][c];
                    w_l[warp * kRows + row] = l[t][c];
                    w_b[warp * kRows + row] = bias[t][c];
                }
        }
        __syncthreads();
        const float undo = __int_as_float((121 + L) << 23); // 2^(L - 6); L >= -121
        const bool whole = pg0 == 0 && pg1 == pG;
        const int slot = 2 * blockIdx.x + (first_piece ? 0 : 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int row = 8 * t + 2 * q + c;
                float top = w_m[row];
#pragma unroll
                for (int w = 1; w < kCaWarps; ++w)
                    top = fmaxf(top, w_m[w * kRows + row]);
                const float f = m[t][c] == -INFINITY ? (l[t][c] == 0.f ? 0.f : 1.f) * undo : ex2(m[t][c] - top) * undo;
                float *dst = merge + ((size_t)warp * 8 + 2 * q + c) * D + r * (D / 8);
#pragma unroll
                for (int x = 0; x < kTiles; x += 2)
                    *reinterpret_cast<float4 *>(dst + 2 * x) = make_float4(O[t][x][c] * f, O[t][x][2 + c] * f, O[t][x + 1][c] * f, O[t][x + 1][2 + c] * f);
            }
            __syncthreads();
            for (int x = threadIdx.x; x < 8 * (D / 8); x += kCaThreads) {
                const int row = x / (D / 8), sub = x % (D / 8), at = prow0 + 8 * t + row;
                float top = -INFINITY, lsum = 0.f, bsum = 0.f, v[8] = {};
#pragma unroll
                for (int w = 0; w < kCaWarps; ++w)
                    top = fmaxf(top, w_m[w * kRows + 8 * t + row]);
#pragma unroll
                for (int w = 0; w < kCaWarps; ++w) {
                    const float mw = w_m[w * kRows + 8 * t + row], f = mw == -INFINITY ? 1.f : ex2(mw - top);
                    lsum = fmaf(f, w_l[w * kRows + 8 * t + row], lsum);
                    bsum = fmaf(f, w_b[w * kRows + 8 * t + row], bsum);
                    const float *src = merge + ((size_t)w * 8 + row) * D + sub * 8;
                    const float4 lo = *reinterpret_cast<const float4 *>(src), hi = *reinterpret_cast<const float4 *>(src + 4);
                    v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w, v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
                }
                if (at < rows) {
                    if (whole) {
                        const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            v[e] = (v[e] + bsum) * inv;
                        const int i = at / a.group, hh = at - i * a.group;
                        *reinterpret_cast<uint4 *>(a.out + ((long long)pb_ * a.n + i) * a.out_stride + (long long)(phead * a.group + hh) * a.out_head_stride + sub * 16) =
                            make_uint4(float_pair_to_half(v[0], v[1], a.bf16), float_pair_to_half(v[2], v[3], a.bf16), float_pair_to_half(v[4], v[5], a.bf16),
                                       float_pair_to_half(v[6], v[7], a.bf16));
                    } else {
                        float *dst = a.part + ((size_t)slot * kRows + 8 * t + row) * D + sub * 8;
                        *reinterpret_cast<float4 *>(dst) = make_float4(v[0] + bsum, v[1] + bsum, v[2] + bsum, v[3] + bsum);
                        *reinterpret_cast<float4 *>(dst + 4) = make_float4(v[4] + bsum, v[5] + bsum, v[6] + bsum, v[7] + bsum);
                        if (sub == 0)
                            reinterpret_cast<float2 *>(a.part + (size_t)2 * a.ctas * kRows * D)[(size_t)slot * kRows + 8 * t + row] = make_float2(top, lsum);
                    }
                }
            }
            __syncthreads();
        }
        if (!more)
            break;
        first_piece = false;
    }
    for (; pending > 0; --pending) { // a wait ran out: no copy may be under way when the block ends
        mbar_wait_bounded(&full[get_stage], get_phase, a.status, STATUS_TIMEOUT_TMA);
        get_stage = get_stage + 1 == kStages ? 0 : get_stage + 1;
        get_phase ^= get_stage == 0;
    }
}

// Items that several CTAs hold: their pieces in order.  Sequences without a token: rows of 0.
template <int D, int NT>
__global__ void __launch_bounds__(kCaThreads) cache_attention_combine_kernel(const __grid_constant__ CacheAttnArgs a)
{
    constexpr int kRows = 8 * NT;
    __shared__ long long scratch[2 * kCaWarps];
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int items = a.kv_heads * a.row_blocks, b = blockIdx.x / items, item = blockIdx.x - b * items;
    long long granules, prefix;
    ca_sums(a, b, scratch, granules, prefix);
    const CaSplit split = ca_split(a, granules);
    const int G = ca_granules(a, b);
    const long long start = prefix * items + (long long)item * G;
    int c0 = 0, c1 = 0;
    if (G) {
        c0 = (int)(start / split.quota);
        c1 = (int)((start + G - 1) / split.quota);
        if (c0 == c1)
            return;
    }
    const int slot0 = 2 * c0 + (start == c0 * split.quota ? 0 : 1);
    const int head = item / a.row_blocks, row0 = (item - head * a.row_blocks) * kRows, rows = a.n * a.group;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + (size_t)2 * a.ctas * kRows * D);
    for (int x = threadIdx.x; x < kRows * (D / 8); x += kCaThreads) {
        const int row = x / (D / 8), sub = x % (D / 8), at = row0 + row;
        if (at >= rows)
            break;
        float v[8] = {}, inv = 0.f;
        if (G) {
            float top = ml[(size_t)slot0 * kRows + row].x, lsum = 0.f;
            for (int c = c0 + 1; c <= c1; ++c)
                top = fmaxf(top, ml[(size_t)2 * c * kRows + row].x);
#pragma unroll 4
            for (int c = c0; c <= c1; ++c) {
                const size_t slot = c == c0 ? slot0 : 2 * c;
                const float2 p = ml[slot * kRows + row];
                const float f = p.x == -INFINITY ? 1.f : ex2(p.x - top);
                lsum = fmaf(f, p.y, lsum);
                const float *src = a.part + (slot * kRows + row) * D + sub * 8;
                const float4 lo = *reinterpret_cast<const float4 *>(src), hi = *reinterpret_cast<const float4 *>(src + 4);
                v[0] = fmaf(f, lo.x, v[0]), v[1] = fmaf(f, lo.y, v[1]), v[2] = fmaf(f, lo.z, v[2]), v[3] = fmaf(f, lo.w, v[3]);
                v[4] = fmaf(f, hi.x, v[4]), v[5] = fmaf(f, hi.y, v[5]), v[6] = fmaf(f, hi.z, v[6]), v[7] = fmaf(f, hi.w, v[7]);
            }
            inv = lsum == 0.f ? 0.f : 1.f / lsum;
        }
        const int i = at / a.group, hh = at - i * a.group;
        *reinterpret_cast<uint4 *>(a.out + ((long long)b * a.n + i) * a.out_stride + (long long)(head * a.group + hh) * a.out_head_stride + sub * 16) =
            make_uint4(float_pair_to_half(v[0] * inv, v[1] * inv, a.bf16), float_pair_to_half(v[2] * inv, v[3] * inv, a.bf16),
                       float_pair_to_half(v[4] * inv, v[5] * inv, a.bf16), float_pair_to_half(v[6] * inv, v[7] * inv, a.bf16));
    }
}

} // namespace abq
