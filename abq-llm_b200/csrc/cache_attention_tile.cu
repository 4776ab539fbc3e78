// Attention over the cache for more query rows than the mma.sync kernel carries well (cache_attention.cuh): trees of drafted tokens of grouped heads.
//
// The same formulas, with 128 query rows as the lanes of fifth-generation tensor-core products: S = Q C_K^T over 128 tokens, P = p vs (fp16, beside S in
// TMEM), O += P C_V.  C are centred codes, which fp16 holds exactly; they are expanded once per 128 rows from the granules (bulk copies) into
// swizzled operand tiles in shared memory.  Scale and offset of a token's key and value are applied to its column of S and of p.
//
// Roles of a CTA (one per SM; each takes an equal run of the line of tiles of all sequences, heads and row blocks):
//   warps 0-7   softmax: a row has two threads, of 64 of the tile's tokens each.  They agree on the maximum where one has to look for it and share the rest at the
//               end; each loads half of the row's queries, scales and writes half of its result
//   warps 8-15  expand codes, a granule each of a tile
//   warp 16     issues the products (S of the next tile before P of this one: S is double-buffered)
//   warp 17     bulk copies of granules, two tiles ahead
// What bounds it: softmax and expansion alike.  Four parameters per token come to every row from shared memory, whose return path takes 2048 clocks a tile for that;
// with one thread a row the softmax took 3100 (latency: 16 trees of 64 rows, heads of 64, 36 us instead of 31; four of 2000 tokens, heads of 128, 45 instead
// of 42).  Expanding a tile takes 1400, its products 512 (D = 64) or 1024.
// Measured against blocks of 16 rows on mma.sync (us; 8 bits, heads of 128, 8 key heads): rows over 4 sequences of up to 2000 tokens, over one of 8000, over 32 of up to
// 300: 64 rows 20.6 and 21.9, 21.8 and 25.9, 31.0 and 29.8; 80 rows 22.2 and 24.8, 22.8 and 29.7, 32.5 and 33.0; 96 rows 23.4 and 26.2, 23.3 and 32.8, 34.3 and
// 39.9; 160 rows 30.8 and 32.9, 33.6 and 46.3, 61.0 and 58.4; heads of 64 and 4 bits, 64 rows 18.2 and 18.0, 20.7 and 21.5, 26.6 and 21.5; 80 rows 18.7 and 19.8, 21.0
// and 24.4, 27.0 and 23.6.  So it is taken where its blocks are at least five eighths full.
//
// The maximum is looked for at a run's first tile and where the sum over a tile says that it has risen by more than 2^8; the value scales' power of two as in
// cache_attention.cuh, on the scale that p is multiplied with.  (As a part of p's exponent it saved a multiplication a score, but lost bf16 values below 2^-80 and
// overflowed in sums of value offsets above 2^50.)
#include <type_traits>

#include "attention_tmem.cuh"
#include "cache_attention_launch.cuh"
#include "umma.cuh"

namespace abq {

constexpr int kCtThreads = 640; // (18 warps have work; registers are dealt out by fours of warps)
constexpr int kCtKeys = 128;

template <int D, int BITS>
struct CtShape {
    static constexpr int RB = kv_row_bytes(D, BITS), kGranule = kv_granule_bytes(RB), kRaw = 8 * kGranule;
    static constexpr int kTile = kCtKeys * D * 2, kHalf = 128 * 128, kHalves = D / 64;
    static constexpr int kPar = 2 * 128 * 16, kMeet = 2 * 2 * 128 * 8;
    // queries, keys, two of values, two raw tiles, token parameters, what halves of a row tell each other, 1024 to align, the rest
    static constexpr int kSmem = 4 * kTile + 2 * kRaw + kPar + kMeet + 1024 + 1024;
    static constexpr int kP = 256, kO = 384; // TMEM columns: S at 0 and 128
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

template <int D, int BITS, bool BF16>
__global__ void __launch_bounds__(kCtThreads, 1) cache_attention_tile_kernel(const __grid_constant__ CacheAttnArgs a)
{
    using Sh = CtShape<D, BITS>;
    constexpr int RB = Sh::RB, kGranule = Sh::kGranule, kTile = Sh::kTile, kHalf = Sh::kHalf, kHalves = Sh::kHalves;
    constexpr float kCentre = (float)(1 << (BITS - 1));
    constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(kCtKeys >> 3) << 17) | ((128u >> 4) << 24);
    constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *sq = smem, *sk = smem + kTile, *sv = smem + 2 * kTile, *raw = smem + 4 * kTile;
    float4 *par = reinterpret_cast<float4 *>(raw + 2 * Sh::kRaw); // [2][128]: key scale and offset, value scale and offset
    float2 *slots = reinterpret_cast<float2 *>(raw + 2 * Sh::kRaw + Sh::kPar); // [2][2 halves][128 rows]
    uint64_t *bars = reinterpret_cast<uint64_t *>(raw + 2 * Sh::kRaw + Sh::kPar + Sh::kMeet);
    uint64_t *raw_full = bars, *raw_empty = bars + 2, *ready = bars + 4, *k_free = bars + 6, *slot_free = bars + 7, *s_full = bars + 9, *s_read = bars + 11,
             *p_ready = bars + 13, *o_done = bars + 14, *q_ready = bars + 15, *drain = bars + 16, *pair = bars + 17;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 22);
    uint32_t *raw_good = tmem_slot + 2;                                  // [2] which granules of a raw tile lie in the cache
    float *vmaxs = reinterpret_cast<float *>(tmem_slot + 4);             // [2][8] largest value scale of each granule
    uint8_t *gbad = reinterpret_cast<uint8_t *>(vmaxs + 16);             // [2][8] granules that are not in the cache

    // A parity that is asked for two phases late looks like one that has not come; no barrier gets that far ahead of one that waits for it: ready, s_full and s_read
    // exist twice and their next phase but one follows p_ready of the tile between; o_done, p_ready and q_ready follow one another; k_free and
    // slot_free are waited for by the warps whose next arrival their next phase needs.
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, run = blockIdx.x;
    pdl_wait_prior_grid();
    pdl_launch_dependents();
    CaRun line;
    if (!line.begin(a, run, lane))
        return; // the whole block
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&raw_full[i], 1);
            mbar_init(&raw_empty[i], 8);
            mbar_init(&ready[i], 8);
            mbar_init(&slot_free[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&s_read[i], 8);
        }
        mbar_init(k_free, 1);
        mbar_init(p_ready, 8);
        mbar_init(o_done, 1);
        mbar_init(q_ready, 8);
        for (int i = 0; i < 4; ++i)
            mbar_init(&pair[i], 2);
        mbar_init(drain, 1);
        fence_mbar_init();
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *tmem_slot;
    uint32_t T = 0;                     // tiles so far, over all pieces
    bool ok = true;
    CaPiece p;

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 128;"); // of 96 at launch: 2 * 128 + 2 * 72 + 80 = 5 * 96
        // ---------------------------------------------------------------- queries, softmax, result
        const int half = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, tp = tmem + lanes + (uint32_t)Sh::kP, to = tmem + lanes + (uint32_t)Sh::kO;
        const int rows = a.n * a.group;
        float rf = 0.f, rs = 0.f; // score = S ks rf + ko rs
        uint64_t mask = 0;
        int at = 0, ctx = 0, len = 0;
        // what the two threads of a row tell each other; both come to every meeting, in the same order.  (Slots alternate: the other one may be at the next meeting.)
        uint32_t met = 0;
        auto meet = [&](float2 mine, float2 &theirs) {
            float2 *at_meeting = slots + (met & 1) * 256;
            at_meeting[half * 128 + row] = mine;
            __syncwarp();
            if (lane == 0)
                mbar_arrive(&pair[warp & 3]);
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&pair[warp & 3], met & 1, a.status, STATUS_TIMEOUT_PIPE)) && ok;
            theirs = at_meeting[(half ^ 1) * 128 + row];
            ++met;
        };
        auto load_queries = [&](const CaPiece &w) { // half a row each
            const int head = w.item / a.row_blocks;
            at = (w.item - head * a.row_blocks) * 128 + row;
            const bool live = at < rows;
            const int i = live ? at / a.group : 0;
            const uint8_t *src = a.q + ((long long)w.b * a.n + i) * a.q_stride + (long long)(head * a.group + at - i * a.group) * a.q_head_stride;
            len = ca_tokens(a, w.b);
            ctx = len - a.n;
            mask = !live ? 0 : a.tree ? a.tree[(size_t)w.b * a.n + i] : i >= 63 ? ~0ull : (2ull << i) - 1;
            float down = 1.f, back = 1.f, sum = 0.f;
            uint4 v[D / 16]; // (all loads under way at once)
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
                v[x] = live ? *reinterpret_cast<const uint4 *>(src + half * D + x * 16) : make_uint4(0, 0, 0, 0);
            float2 other;
            if (BF16) { // to [1, 2) by a power of two
                uint32_t top = 0;
#pragma unroll
                for (int x = 0; x < D / 16; ++x)
                    top = __vmaxu2(__vmaxu2(top, v[x].x & 0x7fff7fffu), __vmaxu2(__vmaxu2(v[x].y & 0x7fff7fffu, v[x].z & 0x7fff7fffu), v[x].w & 0x7fff7fffu));
                top = max(top & 0xffffu, top >> 16);
                meet(make_float2(__uint_as_float(top), 0.f), other);
                top = max(top, __float_as_uint(other.x));
                int e = (int)(top >> 7) - 127;
                e = e > 127 || top == 0 ? 0 : max(e, -126);
                down = __int_as_float(e == 127 ? 0x00400000 : (127 - e) << 23);
                back = __int_as_float((127 + e) << 23);
            }
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
                uint32_t w4[4] = { v[x].x, v[x].y, v[x].z, v[x].w };
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    if (BF16) {
                        const float2 f = half_pair_to_float(w4[y], true);
                        w4[y] = float_pair_to_half(f.x * down, f.y * down, false);
                    }
                    const float2 f = half_pair_to_float(w4[y], false);
                    sum += f.x + f.y;
                }
                const int chunk = half * (D / 16) + x;
                *reinterpret_cast<uint4 *>(sq + (chunk >> 3) * kHalf + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) = make_uint4(w4[0], w4[1], w4[2], w4[3]);
            }
            meet(make_float2(sum, 0.f), other);
            sum += other.x;
            rf = a.scale_log2 * back;
            rs = sum * rf;
            fence_proxy_async();
            __syncwarp();
            if (lane == 0)
                mbar_arrive(q_ready);
        };
        bool more = line.next(a, p);
        if (more)
            load_queries(p);
        while (more && ok) {
            const bool live = at < rows, some = __any_sync(0xffffffffu, live); // (of a warp of rows that do not exist nothing is read)
            float m = live ? -INFINITY : 0.f, mm = 0.f, l = 0.f, bias = 0.f;   // mm: m, or 0 before the first score (no row: nothing to look for)
            float vmax = 0.f, vnorm = 1.f;                                     // 2^(L + 1), 2^(6 - L)
            int L = -121;
            const int tiles = p.g1 - p.g0;
            for (int j = 0; j < tiles; ++j, ++T) {
                const int b = T & 1, t0 = (p.g0 + j) * kCtKeys;
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&ready[b], (T >> 1) & 1, a.status, STATUS_TIMEOUT_PIPE) &&
                                                 mbar_wait_bounded(&s_full[b], (T >> 1) & 1, a.status, STATUS_TIMEOUT_MMA) &&
                                                 (j == 0 || mbar_wait_bounded(o_done, (T - 1) & 1, a.status, STATUS_TIMEOUT_MMA)));
                if (!ok)
                    break;
                tmem_fence_after();
                if (some) {
                    const uint32_t ts = tmem + lanes + (uint32_t)(b * 128);
                    const float4 *pr = par + b * 128;
                    const uint64_t bad = *reinterpret_cast<const uint64_t *>(gbad + 8 * b);
                    const bool edge = t0 + kCtKeys > ctx || bad != 0;
                    auto seen = [&](int key) -> uint32_t { // a bit for each of the 16 tokens (a granule) from `key` on
                        if (!edge)
                            return 0xffffu;
                        const int from = t0 + key, before = min(max(ctx - from, 0), 16), held = min(max(len - from, 0), 16), draft = from - ctx;
                        const uint64_t drafts = draft >= 0 ? (draft < 64 ? mask >> draft : 0) : -draft < 16 ? mask << -draft : 0;
                        return bad >> (8 * (key >> 4)) & 1 ? 0u : ((1u << before) - 1 | (uint32_t)drafts) & ((1u << held) - 1);
                    };
                    float vtop = 0.f;
                    vtop = lane < 8 ? vmaxs[8 * b + lane] : 0.f;
                    vtop = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(vtop)));
                    bool look = __any_sync(0xffffffffu, m == -INFINITY) || vtop >= vmax;
                    float tl, tb;
                    // 16 tokens at a time, their parameters four at a time and ahead of their use (a load where it is used costs its latency each)
                    auto weights = [&](auto masked) {
                        tl = tb = 0.f;
#pragma unroll 1
                        for (int x0 = half * (kCtKeys / 2); x0 < (half + 1) * (kCtKeys / 2); x0 += 16) {
                            float s[16];
                            float4 k[2][4];
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                k[0][e] = pr[x0 + e];
                            pa_ld16(ts + x0, s);
                            const uint32_t vis = decltype(masked)::value ? seen(x0) : 0xffffu;
                            uint32_t w[8];
#pragma unroll
                            for (int g = 0; g < 4; ++g) {
                                if (g < 3) {
#pragma unroll
                                    for (int e = 0; e < 4; ++e)
                                        k[(g + 1) & 1][e] = pr[x0 + 4 * g + 4 + e];
                                }
                                float pv[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float4 &q4 = k[g & 1][e];
                                    const bool see = !decltype(masked)::value || (vis >> (4 * g + e) & 1); // (what is not seen may be Inf or NaN)
                                    const float pe = see ? pa_ex2(fmaf(s[4 * g + e], q4.x * rf, fmaf(q4.y, rs, -mm))) : 0.f;
                                    tl += pe;
                                    tb = fmaf(pe, see ? q4.w : 0.f, tb);
                                    pv[e] = pe * (see ? q4.z * vnorm : 0.f);
                                }
                                w[2 * g] = float_pair_to_half(pv[0], pv[1], false);
                                w[2 * g + 1] = float_pair_to_half(pv[2], pv[3], false);
                            }
                            pa_st8(tp + (uint32_t)(x0 >> 1), w);
                        }
                    };
                    for (;;) {
                        if (look) {
                            float top = -INFINITY;
#pragma unroll 1
                            for (int x0 = half * (kCtKeys / 2); x0 < (half + 1) * (kCtKeys / 2); x0 += 16) {
                                float s[16];
                                pa_ld16(ts + x0, s);
                                const uint32_t vis = seen(x0);
#pragma unroll
                                for (int g = 0; g < 16; g += 8) {
                                    float2 k[8];
#pragma unroll
                                    for (int e = 0; e < 8; ++e)
                                        k[e] = *reinterpret_cast<const float2 *>(pr + x0 + g + e);
#pragma unroll
                                    for (int e = 0; e < 8; ++e) {
                                        const float sc = fmaf(s[g + e], k[e].x * rf, k[e].y * rs), see = vis >> (g + e) & 1 ? sc : -INFINITY;
                                        top = pa_max3(top, see, see);
                                    }
                                }
                            }
                            float2 other;
                            meet(make_float2(top, 0.f), other);
                            top = pa_max3(top, other.x, other.x);
                            if (!(top < INFINITY)) // NaN (or an overflow): the row's result
                                l = NAN;
                            const float before = mm;
                            float down = 1.f;
                            const bool first = m == -INFINITY; // (before the first score of a row its sums are 0, whatever they are multiplied by)
                            if (top > m + 8.f)
                                m = top;
                            if (vtop >= vmax) {
                                const int Ln = max(L, max((int)(__float_as_uint(vtop) >> 23) - 127, -120));
                                down = pa_ex2((float)(L - Ln));
                                L = Ln;
                                vmax = __int_as_float(min(128 + L, 255) << 23);
                                vnorm = __int_as_float((133 - L) << 23);
                            }
                            mm = m == -INFINITY ? 0.f : m;
                            const float f = first ? 1.f : pa_ex2(before - mm);
                            down *= f; // of O
                            if (__any_sync(0xffffffffu, down != 1.f)) {
                                l *= f;
                                bias *= f;
                                if (j > 0) {
#pragma unroll 1
                                    for (int x = half * (D / 2); x < (half + 1) * (D / 2); x += 32) {
                                        float o[32];
                                        pa_ld32(to + x, o);
                                        pa_ld_wait(o);
                                        uint32_t w[32];
#pragma unroll
                                        for (int e = 0; e < 32; ++e)
                                            w[e] = __float_as_uint(o[e] * down);
                                        pa_st16(to + x, w);
                                        pa_st16(to + x + 16, w + 16);
                                    }
                                }
                            }
                        }
                        if (edge)
                            weights(std::true_type());
                        else
                            weights(std::false_type());
                        // no p above 2^8, so none times a value scale above 2^15
                        if (look)
                            break;
                        look = !__all_sync(0xffffffffu, tl <= 256.f);
                        float2 other;
                        meet(make_float2(look ? 1.f : 0.f, 0.f), other);
                        look = look || other.x != 0.f;
                        if (!look || !ok)
                            break;
                    }
                    l += tl;
                    bias += tb;
                    pa_st_wait();
                }
                if (!ok) // (a meeting that did not take place)
                    break;
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&s_read[b]);
                    mbar_arrive(p_ready);
                }
            }
            if (!ok)
                break;
            // ---- the next piece's queries (all scores of this one are made), then this one's result
            const CaPiece cur = p;
            more = line.next(a, p);
            if (more)
                load_queries(p);
            ok = ok && __all_sync(0xffffffffu, mbar_wait_bounded(o_done, (T - 1) & 1, a.status, STATUS_TIMEOUT_MMA));
            float2 other;
            if (!ok)
                break;
            meet(make_float2(l, bias), other);
            l += other.x;
            bias += other.y;
            if (!ok)
                break;
            tmem_fence_after();
            const int head = cur.item / a.row_blocks, row0 = (cur.item - head * a.row_blocks) * 128;
            const bool whole = cur.g0 == 0 && cur.g1 == cur.G;
            const size_t slot = 2 * (size_t)run + (cur.first ? 0 : 1);
            auto put = [&](int to_row, int x, const float *v, float inv) { // 8 features from x on of this lane's row
                if (whole) {
                    const int i = to_row / a.group;
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        y[e] = (v[e] + bias) * inv;
                    *reinterpret_cast<uint4 *>(a.out + ((long long)cur.b * a.n + i) * a.out_stride + (long long)(head * a.group + to_row - i * a.group) * a.out_head_stride + 2 * x) =
                        make_uint4(float_pair_to_half(y[0], y[1], BF16), float_pair_to_half(y[2], y[3], BF16), float_pair_to_half(y[4], y[5], BF16),
                                   float_pair_to_half(y[6], y[7], BF16));
                } else {
                    float *dst = a.part + (slot * a.slot_rows + row) * D + x;
                    *reinterpret_cast<float4 *>(dst) = make_float4(v[0] + bias, v[1] + bias, v[2] + bias, v[3] + bias);
                    *reinterpret_cast<float4 *>(dst + 4) = make_float4(v[4] + bias, v[5] + bias, v[6] + bias, v[7] + bias);
                }
            };
            float2 *ml = reinterpret_cast<float2 *>(a.part + 2 * (size_t)a.runs * a.slot_rows * D) + slot * a.slot_rows;
            const int to_row = row0 + row;
            const float inv = l == 0.f ? 0.f : 1.f / l, undo = __int_as_float((121 + L) << 23); // 2^(L - 6); L >= -121
#pragma unroll 1
            for (int x = half * (D / 2); x < (half + 1) * (D / 2); x += 16) {
                float o[16];
                pa_ld16(to + x, o);
                if (to_row < rows) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        o[e] = l == 0.f ? 0.f : o[e] * undo; // (0: P was 0 throughout, or nothing was written to these columns)
                    put(to_row, x, o, inv);
                    put(to_row, x + 8, o + 8, inv);
                }
            }
            if (half == 0 && !whole && to_row < rows)
                ml[row] = make_float2(l == 0.f ? -INFINITY : m, l);
            tmem_fence_before(); // (O is read before the next piece's first product, which waits for this warp's p)
        }
    } else if (warp < 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        // ---------------------------------------------------------------- codes -> operand tiles
        const int w = warp - 8, t = lane & 15, h = lane >> 4, key = 16 * w + t;
        constexpr int kBytes = RB / 2; // of a lane: half a row of keys, half a row of values
        auto expand = [&](const uint8_t *src, uint8_t *dst) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) {
                const uint4 c4 = *reinterpret_cast<const uint4 *>(src + kv_place<RB>(t, h * kBytes + 16 * i));
                const uint32_t c[4] = { c4.x, c4.y, c4.z, c4.w };
                auto put = [&](int chunk, uint32_t x, uint32_t y, uint32_t z, uint32_t u) { // 8 features
                    *reinterpret_cast<uint4 *>(dst + (chunk >> 3) * kHalf + key * 128 + (((chunk & 7) ^ (key & 7)) << 4)) = make_uint4(x, y, z, u);
                };
                if (BITS == 8) {
                    const int chunk = h * (D / 16) + 2 * i;
                    put(chunk, bytes_lo(c[0]), bytes_hi(c[0]), bytes_lo(c[1]), bytes_hi(c[1]));
                    put(chunk + 1, bytes_lo(c[2]), bytes_hi(c[2]), bytes_lo(c[3]), bytes_hi(c[3]));
                } else {
#pragma unroll
                    for (int y = 0; y < 4; ++y) { // a word: 8 codes, as the pairs (0, 4), (1, 5), (2, 6), (3, 7)
                        const uint32_t n0 = nibbles_lo(c[y]), n1 = nibbles_hi(c[y]), n2 = nibbles_lo(c[y] >> 8), n3 = nibbles_hi(c[y] >> 8);
                        put(h * (D / 16) + 4 * i + y, __byte_perm(n0, n1, 0x5410), __byte_perm(n2, n3, 0x5410), __byte_perm(n0, n1, 0x7632), __byte_perm(n2, n3, 0x7632));
                    }
                }
            }
        };
        while (ok && line.next(a, p)) {
            const int len = ca_tokens(a, p.b);
            for (int j = p.g0; j < p.g1; ++j, ++T) {
                const int b = T & 1;
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&raw_full[b], (T >> 1) & 1, a.status, STATUS_TIMEOUT_TMA) &&
                                                 (T < 2 || mbar_wait_bounded(&slot_free[b], ((T >> 1) - 1) & 1, a.status, STATUS_TIMEOUT_MMA)));
                if (!ok)
                    break;
                const uint8_t *g = raw + b * Sh::kRaw + w * kGranule;
                const bool good = raw_good[b] >> w & 1;
                const float2 pp = half_pair_to_float(*reinterpret_cast<const uint32_t *>(g + kv_param_offset(RB, h) + 4 * t), BF16);
                reinterpret_cast<float2 *>(par + b * 128 + key)[h] = make_float2(pp.x, fmaf(kCentre, pp.x, pp.y));
                const bool counts = h && good && j * kCtKeys + key < len && pp.x < INFINITY;
                const uint32_t top = __reduce_max_sync(0xffffffffu, counts ? __float_as_uint(pp.x) : 0u); // scales are not negative: ordered like their bits
                if (lane == 0) {
                    vmaxs[8 * b + w] = __uint_as_float(top);
                    gbad[8 * b + w] = !good;
                }
                expand(g + 16 * RB, sv + b * kTile);
                // the one tile of keys is free when the scores before are made: they are, while the values are expanded
                ok = __all_sync(0xffffffffu, T < 1 || mbar_wait_bounded(k_free, (T - 1) & 1, a.status, STATUS_TIMEOUT_MMA));
                if (!ok)
                    break;
                expand(g, sk);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&raw_empty[b]);
                    mbar_arrive(&ready[b]);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    }
    if (warp == 16) {
        // ---------------------------------------------------------------- products
        uint32_t pieces = 0;
        while (ok && line.next(a, p)) {
            const int tiles = p.g1 - p.g0;
            bool fine = true;
            if (elect_one()) {
                auto scores = [&](uint32_t tile) {
                    const int b = tile & 1;
                    fine = mbar_wait_bounded(&ready[b], (tile >> 1) & 1, a.status, STATUS_TIMEOUT_PIPE) &&
                           (tile < 2 || mbar_wait_bounded(&s_read[b], ((tile >> 1) - 1) & 1, a.status, STATUS_TIMEOUT_PIPE));
                    if (!fine)
                        return;
                    tmem_fence_after();
#pragma unroll
                    for (int h = 0; h < kHalves; ++h) {
                        const uint64_t dq = make_smem_desc_sw128(smem_u32(sq + h * kHalf)), dk = make_smem_desc_sw128(smem_u32(sk + h * kHalf));
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            umma_f16(tmem + (uint32_t)(b * 128), dq + (uint64_t)(2 * x), dk + (uint64_t)(2 * x), kIdescS, (h | x) != 0);
                    }
                    umma_commit(&s_full[b]);
                    umma_commit(k_free);
                };
                fine = mbar_wait_bounded(q_ready, pieces & 1, a.status, STATUS_TIMEOUT_PIPE);
                if (fine)
                    scores(T);
                for (int j = 0; j < tiles && fine; ++j) {
                    if (j + 1 < tiles)
                        scores(T + j + 1);
                    fine = fine && mbar_wait_bounded(p_ready, (T + j) & 1, a.status, STATUS_TIMEOUT_PIPE);
                    if (!fine)
                        break;
                    tmem_fence_after();
                    const int b = (T + j) & 1;
                    const uint64_t dv = make_smem_desc_sw128_mn(smem_u32(sv + b * kTile), kHalf);
#pragma unroll
                    for (int x = 0; x < kCtKeys / 16; ++x)
                        umma_f16_ts(tmem + (uint32_t)Sh::kO, tmem + (uint32_t)(Sh::kP + 8 * x), dv + (uint64_t)(x * 2048 >> 4), kIdescO, (j | x) != 0);
                    umma_commit(o_done);
                    umma_commit(&slot_free[b]);
                }
            }
            __syncwarp();
            ok = __all_sync(0xffffffffu, fine);
            T += tiles;
            ++pieces;
        }
        if (elect_one()) { // every product, and every arrival that one of them still owes, before the block ends
            umma_commit(drain);
            mbar_wait_bounded(drain, 0, a.status, STATUS_TIMEOUT_MMA);
        }
        __syncwarp();
    } else if (warp == 17) {
        // ---------------------------------------------------------------- copies
        while (ok && line.next(a, p)) {
            const int granules = (int)(((long long)ca_tokens(a, p.b) + 15) >> 4), head = p.item / a.row_blocks;
            uint32_t place = ~0u;
            for (int j = p.g0; j < p.g1; ++j, ++T) {
                if (((j - p.g0) & 3) == 0) { // lane i: granule i of the next four tiles
                    const int g = 8 * j + lane;
                    place = ~0u;
                    if (g < granules && g < 8 * p.g1) {
                        const int entry = ca_entry(a, g), page = a.table[(size_t)p.b * a.table_stride + entry];
                        if (page >= 0 && page < a.num_pages)
                            place = ((uint32_t)page * a.kv_heads + head) * a.page_granules + (g - entry * a.page_granules);
                        else if (a.status)
                            atomicOr(a.status, ABQ_STATUS_BAD_PAGE);
                    }
                }
                const int b = T & 1, first = 8 * ((j - p.g0) & 3);
                const uint32_t good = __ballot_sync(0xffffffffu, place != ~0u) >> first & 255u;
                ok = __all_sync(0xffffffffu, T < 2 || mbar_wait_bounded(&raw_empty[b], ((T >> 1) - 1) & 1, a.status, STATUS_TIMEOUT_PIPE));
                if (!ok)
                    break;
                if (lane == 0) {
                    raw_good[b] = good;
                    mbar_arrive_expect_tx(&raw_full[b], __popc(good) * kGranule);
                }
                __syncwarp();
                if (lane >= first && lane < first + 8 && place != ~0u)
                    bulk_load(raw + b * Sh::kRaw + (lane - first) * kGranule, a.data + (size_t)place * kGranule, kGranule, &raw_full[b]);
            }
        }
        for (uint32_t t = T < 2 ? 0 : T - 2; !ok && t < T; ++t) // a wait ran out: what has been asked for arrives before the block ends
            mbar_wait_bounded(&raw_full[t & 1], (t >> 1) & 1, a.status, STATUS_TIMEOUT_TMA);
    }

    tmem_fence_before();
    __syncthreads();
    if (warp == 16) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int D, int BITS, bool BF16>
static cudaError_t launch_tile(const CacheAttnArgs &args, cudaStream_t stream)
{
    static thread_local SmemOptIn opted;
    constexpr int smem = CtShape<D, BITS>::kSmem;
    auto kern = cache_attention_tile_kernel<D, BITS, BF16>;
    const cudaError_t e = opted.ensure(kern, smem);
    if (e != cudaSuccess)
        return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(args.runs);
    cfg.blockDim = dim3(kCtThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e2 = cudaLaunchKernelEx(&cfg, kern, args);
    return e2 != cudaSuccess ? e2 : launch_cache_attention_combine<D, BF16>(args, 128, stream);
}

cudaError_t launch_cache_attention_tile(const CacheAttnArgs &args, int head_dim, int bits, bool bf16, cudaStream_t stream)
{
    if (head_dim == 128) {
        if (bits == 8)
            return bf16 ? launch_tile<128, 8, true>(args, stream) : launch_tile<128, 8, false>(args, stream);
        return bf16 ? launch_tile<128, 4, true>(args, stream) : launch_tile<128, 4, false>(args, stream);
    }
    if (bits == 8)
        return bf16 ? launch_tile<64, 8, true>(args, stream) : launch_tile<64, 8, false>(args, stream);
    return bf16 ? launch_tile<64, 4, true>(args, stream) : launch_tile<64, 4, false>(args, stream);
}

} // namespace abq
