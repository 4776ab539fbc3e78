// Causal attention of packed prompts (abq_prompt_attention) on the fifth-generation tensor cores.
//
// Per block of 256 query rows of one key head: S = Q K^T over 128 keys at a time, p = 2^(scale log2(e) s - m) with the running row maximum m,
// O = O 2^(m_old - m) + P V, at the end O / sum(p).  Operands never leave the chip between the two products: S and O are TMEM accumulators, P replaces S
// in TMEM as the first operand of the second product, K and V tiles come by TMA.
//
// A row of a block is a (token, query head) pair: the largest power of two of heads that share a key head lie behind one another in a tile (TMA
// gathers them as a box), so that short prompts fill tiles and the heads of a group share the K and V tiles.
//
// Roles of a CTA (one per SM, persistent over blocks, the longest of a sequence first and dealt to and fro so that long and short ones add up):
//   warps 0-3, 4-7  softmax of the two 128-row tiles, a thread per row; they also scale O (only when the maximum has grown by more than 2^8: the
//                   exponent stays bounded without it) and write the result
//   warp 8          TMA: Q of a block, K and V tiles in the order of their use through one ring
//   warp 9          issues the products: while one tile's softmax runs, the tensor cores work for the other (D = 64: for the next keys, too)
//   warps 10, 11    look through the V tiles that some row of the block does not see to the end: 0 times Inf or NaN is no 0, so such values are set to 0 in
//                   shared memory and added by the rows that see them when they write their result
// What bounds it: the tensor cores (4 * 128 * 128 * D operations a tile pair) and, as long for D = 128 and twice as long for D = 64, one exponential per score on
// the special-function units.  So part of the exponentials of a tile (kPaPoly of 8 pairs) is computed on the multiply-add pipes, two at a time: 2^x =
// 2^n 2^f with n = rint(x), a minimax polynomial for 2^f on [-1/2, 1/2] (Remez, relative error 2^-18.5 with five coefficients for fp16, 2^-13.7 with four for
// bf16), n added to the exponent.  Tiles with masked scores take the units' function for all (it gives the 0 that they need).  A share of one in eight measured best for
// heads of 64 (none 137.5 us, one 133.1, two 134.4); more costs more issue slots than the units save.
//
// Measured: a prompt of 2048, 32 heads of 128, bf16: 44 to 46 us in a graph (0.75 PFLOP/s), 49 in a loop of calls; of 8192, 32 heads on 8: 460 to 485 us in short bursts (1.15
// PFLOP/s), 524 to 540 sustained, where the power limit lowers the clock; heads of 64, 16 prompts of up to 1023 behind a prefix of 517 each, 32 heads on 4: 113 to 122 us (0.42).
// In clocks: a pair of tiles over 128 keys 3100 to 3550 (D = 128: softmax 1750 and the products 1100 that it waits for); a block 2400 to 3900 until its first scores and about
// 4000 for its result.  Two threads a row (16 softmax warps), the product of P started on half of its columns, and no maximum per tile were no faster.
//
// P is rounded to the 16-bit type (tensor-core operands); fp16 holds p times 2^6, so that weights down to 2^-20 of the maximum keep all bits.  The sum of p is
// that of the unrounded values.
#include <cuda.h>
#include <algorithm>
#include <type_traits>

#include "abq_kernels.h"
#include "attention_tmem.cuh"
#include "kv_cache.cuh"
#include "umma.cuh"

namespace abq {

constexpr int kPaThreads = 384;
constexpr int kPaKeys = 128; // keys of a tile
constexpr int kPaPoly = 1;   // pairs of 8 whose exponentials are polynomials

struct PaArgs {
    const int *cu_q, *cu_k;
    const uint8_t *v;
    uint8_t *out;
    long long v_stride, v_head_stride, out_stride, out_head_stride; // bytes
    int total_q, total_k, batch, head_groups, pack_log2, group;
    int sorted; // blocks by the key tiles they see (several rounds of blocks, 2 to 32 sequences)
    float scale_log2;
    int *status;
};

template <int D>
struct PaShape {
    static constexpr int kTile = 128 * D * 2, kHalf = 128 * 128, kHalves = D / 64; // a 128-byte-swizzled half holds 64 features
    // D = 64 leaves TMEM for P beside S, and shared memory for the next block's Q: S of the next keys is made while the softmax of these ones runs
    static constexpr bool kApart = D == 64;
    static constexpr int kQBlocks = kApart ? 2 : 1, kStages = kApart ? 9 : 5;
    static constexpr int kSmem = (2 * kQBlocks + kStages) * kTile + 1024 + 512;
    // TMEM columns: S of the tiles at 0 and 128, with P over their first half or from 256; then O
    static constexpr int kP = kApart ? 256 : 0, kPStep = kApart ? 64 : 128, kO = kApart ? 384 : 256;
};

struct PaItem {
    int q0, nq, k0, nk, off; // rows of q and of k, keys that a row sees beyond its own index
    int tok0, hg;            // first token of the block, group of heads
    int n[2], most, edge;    // key tiles per row tile, the larger, the first that some row does not see to its end
    bool valid;
};

// Rows of sequence b and of its keys, cut to what the arrays hold.
struct PaSeq {
    int q0, nq, k0, nk;
};
__device__ __forceinline__ PaSeq pa_seq(const PaArgs &a, int b)
{
    PaSeq s = { 0, 0, 0, 0 };
    if (b < a.batch) {
        s.q0 = min(max(a.cu_q[b], 0), a.total_q);
        s.nq = min(max(a.cu_q[b + 1], s.q0), a.total_q) - s.q0;
        s.k0 = min(max(a.cu_k[b], 0), a.total_k);
        s.nk = min(max(a.cu_k[b + 1], s.k0), a.total_k) - s.k0;
    }
    return s;
}
__device__ __forceinline__ int pa_scan(int x, int lane) // sum of this and the lanes before
{
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        x += lane >= o ? y : 0;
    }
    return x;
}

// Block number `idx`, found by all lanes of a warp.  Sorted (up to 32 sequences, a lane looks at one): blocks of all sequences by the key tiles they see,
// most first, so that dealing them to and fro leaves no CTA with much more than the others (16 prompts of 200 to 1023 tokens: 57 tiles on one, 38 on another
// in the order of the sequences).  Otherwise one sequence after the other, the last block, which sees most, first.
__device__ __forceinline__ PaItem pa_item(const PaArgs &a, int idx, int lane)
{
    PaItem it;
    const int shift = 8 - a.pack_log2, tokens = 1 << shift; // of a block
    int slot = idx / a.head_groups, block = 0, at = 0;
    it.hg = idx - slot * a.head_groups;
    it.valid = false;
    PaSeq s;
    if (a.sorted) {
        s = pa_seq(a, lane);
        const int blocks = (s.nq + tokens - 1) >> shift, off = s.nk - s.nq;
        auto first = [&](int x) { return min(blocks, max(0, (kPaKeys * (x - 1) - off) >> shift)); };                  // block that sees x tiles or more (x > 0)
        auto count = [&](int x) { return x == 0 ? blocks : s.nk > kPaKeys * (x - 1) ? blocks - first(x) : 0; };       // and how many do
        int lo = 0, hi = (__reduce_max_sync(0xffffffffu, s.nk) + kPaKeys - 1) / kPaKeys;
        it.valid = slot < __reduce_add_sync(0xffffffffu, blocks);
        while (lo < hi) { // the most tiles that more than `slot` blocks see
            const int mid = (lo + hi + 1) >> 1;
            if (__reduce_add_sync(0xffffffffu, count(mid)) > slot)
                lo = mid;
            else
                hi = mid - 1;
        }
        const int more = count(lo + 1), here = count(lo) - more;
        slot -= __reduce_add_sync(0xffffffffu, more);
        const int end = pa_scan(here, lane);
        at = __ffs(__ballot_sync(0xffffffffu, slot < end)) - 1;
        block = __shfl_sync(0xffffffffu, (lo ? first(lo) : 0) + slot - (end - here), at & 31);
    } else {
        for (int b0 = 0; b0 < a.batch; b0 += 32) {
            s = pa_seq(a, b0 + lane);
            const int end = pa_scan((s.nq + tokens - 1) >> shift, lane);
            const uint32_t behind = __ballot_sync(0xffffffffu, slot < end);
            if (behind) {
                at = __ffs(behind) - 1;
                block = __shfl_sync(0xffffffffu, end, at) - 1 - slot;
                it.valid = true;
                break;
            }
            slot -= __shfl_sync(0xffffffffu, end, 31);
        }
    }
    if (!it.valid)
        return it;
    it.q0 = __shfl_sync(0xffffffffu, s.q0, at);
    it.nq = __shfl_sync(0xffffffffu, s.nq, at);
    it.k0 = __shfl_sync(0xffffffffu, s.k0, at);
    it.nk = __shfl_sync(0xffffffffu, s.nk, at);
    it.tok0 = block << shift;
    it.off = it.nk - it.nq;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int first = it.tok0 + t * (tokens >> 1), last = min(it.nq, first + (tokens >> 1)) - 1;
        it.n[t] = first >= it.nq ? 0 : (max(0, min(it.nk, last + it.off + 1)) + kPaKeys - 1) / kPaKeys;
    }
    it.most = max(it.n[0], it.n[1]);
    it.edge = max(0, min(it.nk, it.tok0 + it.off + 1)) / kPaKeys;
    return it;
}

// Place of a tile in the ring, counted from the block's first: K0, K1, V0, K2, V1, .. , V(n - 1)
__device__ __forceinline__ int pa_k_place(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int pa_v_place(int j, int n) { return j == n - 1 ? 2 * n - 1 : 2 * j + 2; }

// 2^x of two numbers of at most 2^14; below 2^-125 it stays there.  NaN is lost: the caller looks for it.
template <bool BF16>
__device__ __forceinline__ void pa_ex2_poly(uint64_t x2, float &lo, float &hi)
{
    constexpr float kMagic = 12582912.f; // 1.5 * 2^23: the sum's low bits are rint(x)
    pa_unpack(x2, lo, hi);
    const uint64_t x = pa_pack(fmaxf(lo, -125.f), fmaxf(hi, -125.f));
    const uint64_t t = pa_add2(x, pa_pack(kMagic, kMagic));
    const uint64_t f = pa_add2(x, pa_fma2(t, pa_pack(-1.f, -1.f), pa_pack(kMagic, kMagic)));
    uint64_t y;
    auto c = [](float v) { return pa_pack(v, v); };
    if (BF16) {
        y = pa_fma2(f, c(0.0551716685295105f), c(0.2426111251115799f));
        y = pa_fma2(f, y, c(0.6932609677314758f));
        y = pa_fma2(f, y, c(0.9999280571937561f));
    } else {
        y = pa_fma2(f, c(0.009570102207362652f), c(0.05591785907745361f));
        y = pa_fma2(f, y, c(0.240247443318367f));
        y = pa_fma2(f, y, c(0.6931217908859253f));
        y = pa_fma2(f, y, c(0.9999992847442627f));
    }
    float n0, n1;
    pa_unpack(y, lo, hi);
    pa_unpack(t, n0, n1);
    lo = __int_as_float(__float_as_int(lo) + (__float_as_int(n0) << 23));
    hi = __int_as_float(__float_as_int(hi) + (__float_as_int(n1) << 23));
}

// 16-byte pieces w[0..3] of four neighbouring lanes: lane b of them ends with piece b of lane k in w[k]
__device__ __forceinline__ void transpose4(uint32_t (&w)[4][4], int lane)
{
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k & o)
                continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) { // keep the piece on the diagonal, trade the other
                const uint32_t give = up ? w[k][e] : w[k | o][e], got = __shfl_xor_sync(0xffffffffu, give, o);
                w[k][e] = up ? got : w[k][e];
                w[k | o][e] = up ? w[k | o][e] : got;
            }
        }
    }
}

// The rows of a block whose last V tiles held Inf or NaN, once more: the product's part from TMEM, and those values where a row sees them (they were left out of
// the product).  Rare, and apart so that the usual path stays short.
template <int D, bool BF16>
__device__ __noinline__ void add_foul_values(const PaArgs &a, uint32_t to, int q_row, bool live, int head, int k0, int first, int sees, float inv)
{
    const uint8_t *v = a.v + (long long)k0 * a.v_stride + (long long)(head / a.group) * a.v_head_stride;
    uint8_t *dst = a.out + (long long)q_row * a.out_stride + (long long)head * a.out_head_stride;
#pragma unroll 1
    for (int x = 0; x < D; x += 16) {
        float o[16];
        pa_ld16(to + x, o);
#pragma unroll
        for (int e = 0; e < 16; ++e)
            o[e] *= inv;
        for (int k = first; k < sees; ++k) {
            const unsigned short *vr = reinterpret_cast<const unsigned short *>(v + (long long)k * a.v_stride) + x;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float f = half_bits_to_float(vr[e], BF16);
                if (!(fabsf(f) <= 3.402823466e38f))
                    o[e] += f;
            }
        }
        if (live) {
#pragma unroll
            for (int e = 0; e < 16; e += 8)
                *reinterpret_cast<uint4 *>(dst + 2 * (x + e)) =
                    make_uint4(float_pair_to_half(o[e], o[e + 1], BF16), float_pair_to_half(o[e + 2], o[e + 3], BF16),
                               float_pair_to_half(o[e + 4], o[e + 5], BF16), float_pair_to_half(o[e + 6], o[e + 7], BF16));
        }
    }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kPaThreads, 1)
prompt_attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                        const __grid_constant__ PaArgs a)
{
    using Sh = PaShape<D>;
    constexpr int kStages = Sh::kStages, kTile = Sh::kTile, kHalf = Sh::kHalf, kHalves = Sh::kHalves;
    constexpr uint32_t kType = BF16 ? 1u : 0u;
    constexpr uint32_t kIdescS = (1u << 4) | (kType << 7) | (kType << 10) | ((uint32_t)(kPaKeys >> 3) << 17) | ((128u >> 4) << 24);
    constexpr uint32_t kIdescO = (1u << 4) | (kType << 7) | (kType << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    constexpr bool kApart = Sh::kApart;
    constexpr int kQBlocks = Sh::kQBlocks;
    uint8_t *sq = smem, *ring = smem + 2 * kQBlocks * kTile;
    uint64_t *bars = reinterpret_cast<uint64_t *>(ring + kStages * kTile);
    uint64_t *q_full = bars, *q_empty = bars + 2, *s_full = bars + 4, *p_ready = bars + 6, *s_read = bars + 8, *o_done = bars + 10, *drain = bars + 12, *half_way = bars + 13;
    uint64_t *kv_full = bars + 15, *kv_empty = kv_full + kStages, *edge_full = kv_empty + kStages;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(edge_full + kStages);
    // [2 row tiles][4][2 warps]: the V tiles that this row tile's rows do not all see to the end held Inf or NaN.  Slots go round over the blocks in which the row tile
    // has such V tiles: only these are written for it and read by it.  A slot is read before it is written again, four such blocks later: that block's V comes
    // behind its Q, whose place is free when the scores of the block one or two before (kQBlocks) are made; by then the row tile's scores of the third of these blocks
    // have been asked for (D = 64) or its p's of it used, and both wait for its softmax to be in the second or later, past the first one's flag.
    int *poison = reinterpret_cast<int *>(tmem_slot + 2);

    // No barrier completes a phase before everybody who waits for the one before has seen that: a parity that is asked for two phases late looks like one
    // that has not come.  s_full: the scores of the next keys follow p_ready (or s_read), which follows the wait for these.  o_done: the next product it
    // stands for follows a p_ready behind the wait.  p_ready and s_read: their next arrival follows an s_full that the MMA warp sends after its wait.
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(drain, 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(&q_full[t], 1);
            mbar_init(&q_empty[t], 1);
            mbar_init(&s_full[t], 1);
            mbar_init(&p_ready[t], 4);
            mbar_init(&s_read[t], 4);
            mbar_init(&o_done[t], 1);
            mbar_init(&half_way[t], 4);
        }
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&kv_full[s], 2); // the producer twice, or the two warps that looked through the tile
            mbar_init(&kv_empty[s], 1);
            mbar_init(&edge_full[s], 1);
        }
        fence_mbar_init();
        prefetch_tmap(&tmap_q);
        prefetch_tmap(&tmap_k);
        prefetch_tmap(&tmap_v);
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    pdl_wait_prior_grid();

    // The pool is what the block was launched with: 384 threads x 168 registers = 256 x 208 + 128 x 88
    const int G = gridDim.x, c = blockIdx.x;
    auto number = [&](int round) { return round * G + (round & 1 ? G - 1 - c : c); };

    if (warp >= 8)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < 8) {
        // ---------------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + (uint32_t)(t * 128), tp = tmem + lanes + (uint32_t)(Sh::kP + t * Sh::kPStep), to = tmem + lanes + (uint32_t)(Sh::kO + t * D);
        const int pack = 1 << a.pack_log2;
        uint32_t phase = 0, done = 0, others = 0; // of s_full; of o_done (a product with V each, or with S and P in one place a block); key tiles of the other row tile so far
        uint32_t flags = 0;           // flags read
        bool ok = true;
        PaItem next = pa_item(a, number(0), lane);
        for (int round = 0; ok; ++round) {
            const PaItem it = next;
            if (!it.valid)
                break;
            const int token = it.tok0 + t * (128 >> a.pack_log2) + (row >> a.pack_log2);
            const int sees = min(it.nk, token + it.off + 1);
            float m = -INFINITY;
            uint64_t sum2 = 0;
            float l = 0.f;
            const int n = t ? it.n[1] : it.n[0];
            for (int j = 0; j < n; ++j) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_full[t], phase & 1, a.status, STATUS_TIMEOUT_MMA));
                if (!ok)
                    break;
                ++phase;
                tmem_fence_after();
                float s[128];
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    pa_ld32(ts + 32 * x, s + 32 * x);
                pa_ld_wait(s);
                pa_ld_tie(s + 32);
                pa_ld_tie(s + 64);
                pa_ld_tie(s + 96);
                if (kApart) { // these scores are in registers: their columns may take the next ones
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(&s_read[t]);
                }
                const int lim = sees - j * kPaKeys;
                const bool masked = __any_sync(0xffffffffu, lim < kPaKeys);
                if (masked) {
#pragma unroll
                    for (int x = 0; x < 128; ++x)
                        s[x] = x < lim ? s[x] : -INFINITY;
                }
                float top[4] = { s[0], s[1], s[2], s[3] };
#pragma unroll
                for (int x = 4; x < 128; x += 8) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        top[e] = x + 4 + e < 128 ? pa_max3(top[e], s[x + e], s[x + 4 + e]) : pa_max3(top[e], s[x + e], s[x + e]);
                }
                const float peak = pa_max3(pa_max3(top[0], top[1], top[2]), top[3], top[3]) * a.scale_log2;
                if (!(peak < INFINITY)) // NaN (or an overflow) among the scores: the row's result
                    l = NAN;
                if (kApart && j > 0) { // the product with the P before: its columns and O are free
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&o_done[t], (done + j - 1) & 1, a.status, STATUS_TIMEOUT_MMA));
                    if (!ok)
                        break;
                    tmem_fence_after();
                }
                const bool raise = peak > m + 8.f;
                if (__any_sync(0xffffffffu, raise)) {
                    const float f = raise ? pa_ex2(m - peak) : 1.f;
                    m = raise ? peak : m;
                    float lo, hi;
                    pa_unpack(sum2, lo, hi);
                    l = (l + lo + hi) * f;
                    sum2 = 0;
                    if (j > 0) { // (the first product of a block overwrites O)
#pragma unroll 1
                        for (int x = 0; x < D; x += 32) {
                            float o[32];
                            pa_ld32(to + x, o);
                            pa_ld_wait(o);
                            uint32_t w[32];
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                w[e] = __float_as_uint(o[e] * f);
                            pa_st16(to + x, w);
                            pa_st16(to + x + 16, w + 16);
                        }
                    }
                }
                const float base = (BF16 ? 0.f : 6.f) - (m == -INFINITY ? 0.f : m);
                const uint64_t scale2 = pa_pack(a.scale_log2, a.scale_log2), base2 = pa_pack(base, base);
                // D = 64: the two tiles' softmaxes would fall into step and take turns at leaving the special-function units idle and fighting for them.  Each starts its
                // exponentials when the other is half way through its own: tile 0 after tile 1's of the keys before, tile 1 after tile 0's of the same
                // keys.  Only a matter of time: nothing depends on it, and the wait is given up after a few microseconds.
                if (kApart) {
                    const int theirs = t ? j : j - 1;
                    if (theirs >= 0 && theirs < (t ? it.n[0] : it.n[1])) {
#pragma unroll 1
                        for (int i = 0; i < 64 && !mbar_try_wait(&half_way[t ^ 1], (others + theirs) & 1); ++i)
                            ;
                        __syncwarp();
                    }
                }
                auto weights = [&](auto poly) {
#pragma unroll
                    for (int x = 0; x < 128; x += 32) {
                        uint32_t w[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float lo, hi;
                            if (decltype(poly)::value && (e >> 1) * kPaPoly % 8 < kPaPoly) { // (spread over the 8)
                                pa_ex2_poly<BF16>(pa_fma2(pa_pack(s[x + e], s[x + e + 1]), scale2, base2), lo, hi);
                            } else {
                                lo = pa_ex2(fmaf(s[x + e], a.scale_log2, base));
                                hi = pa_ex2(fmaf(s[x + e + 1], a.scale_log2, base));
                            }
                            sum2 = pa_add2(sum2, pa_pack(lo, hi));
                            w[e >> 1] = float_pair_to_half(lo, hi, BF16);
                        }
                        pa_st16(tp + (x >> 1), w);
                        if (kApart && x == 32) {
                            __syncwarp();
                            if (lane == 0)
                                mbar_arrive(&half_way[t]);
                        }
                    }
                };
                if (masked)
                    weights(std::false_type());
                else
                    weights(std::true_type());
                pa_st_wait();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&p_ready[t]);
            }
            if (!ok)
                break;
            next = pa_item(a, number(round + 1), lane); // (while the last product runs)
            float inv = 0.f;
            bool foul = false;
            if (n > 0) {
                done += kApart ? n : 1;
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&o_done[t], (done - 1) & 1, a.status, STATUS_TIMEOUT_MMA));
                if (!ok)
                    break;
                tmem_fence_after();
                float lo, hi;
                pa_unpack(sum2, lo, hi);
                l += lo + hi;
                inv = l == 0.f ? 0.f : 1.f / l;
                if (it.edge < n) { // (its V tiles have been looked through by now; the other row tile's may not)
                    const int slot = 4 * t + (flags & 3);
                    foul = *reinterpret_cast<volatile int *>(&poison[2 * slot]) | *reinterpret_cast<volatile int *>(&poison[2 * slot + 1]);
                    ++flags;
                }
            }
            others += t ? it.n[0] : it.n[1];
            // Four lanes exchange their 16-byte pieces, so that a store covers 64 bytes of 8 rows and not 16 of 32: lane 4 a + b gets piece b of rows 4 a ..
            uint8_t *dst[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int r2 = (row & ~3) + k, token2 = it.tok0 + t * (128 >> a.pack_log2) + (r2 >> a.pack_log2);
                dst[k] = token2 >= it.nq ? nullptr
                                         : a.out + (long long)(it.q0 + token2) * a.out_stride + (long long)(it.hg * pack + (r2 & (pack - 1))) * a.out_head_stride + (lane & 3) * 16;
            }
#pragma unroll 1
            for (int x = 0; x < D; x += 32) {
                float o[32];
                if (n > 0) {
                    pa_ld32(to + x, o);
                    pa_ld_wait(o);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        o[e] = 0.f;
                }
                uint32_t w[4][4];
#pragma unroll
                for (int e = 0; e < 32; e += 2) // (a row that saw nothing: P and O are 0)
                    w[e >> 3][(e >> 1) & 3] = float_pair_to_half(o[e] * inv, o[e + 1] * inv, BF16);
                transpose4(w, lane);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (dst[k])
                        *reinterpret_cast<uint4 *>(dst[k] + 2 * x) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
            }
            if (foul) { // (the same for the whole warp)
                __syncwarp(); // what other lanes have written of this row comes first
                add_foul_values<D, BF16>(a, to, it.q0 + token, token < it.nq, it.hg * pack + (row & (pack - 1)), it.k0, it.edge * kPaKeys, sees, inv);
            }
            tmem_fence_before(); // (O is read before the next block's first product, which waits for this tile's p)
        }
    } else if (warp == 8) {
        // ---------------------------------------------------------------- copies
        int place = 0, blocks = 0, asked = 0, queries = 0; // tiles and blocks of queries asked for
        uint32_t edges = 0, last_edge = 0;                 // a bit per stage: parity of edge_full; whether the last tile went there
        bool ok = true;
        for (int round = 0; ok; ++round) {
            const PaItem it = pa_item(a, number(round), lane);
            if (!it.valid)
                break;
            if (it.most == 0)
                continue;
            const int pack = 1 << a.pack_log2, kv_head = (it.hg << a.pack_log2) / a.group, total = 2 * it.most;
            bool fine = true, leader = false;
            if (elect_one()) {
                leader = true;
                for (int i = 0; i < total; ++i) {
                    if (i == 1) { // Q behind the first K tile: its place is free when the S of the block before (or the one before that) are done
                        const int qb = blocks % kQBlocks, use = blocks / kQBlocks;
                        if (use && !mbar_wait_bounded(&q_empty[qb], (use - 1) & 1, a.status, STATUS_TIMEOUT_PIPE)) {
                            fine = false;
                            break;
                        }
                        mbar_arrive_expect_tx(&q_full[qb], (uint32_t)kTile * ((it.n[0] > 0) + (it.n[1] > 0)));
                        ++queries;
#pragma unroll
                        for (int t = 0; t < 2; ++t)
                            if (it.n[t] > 0)
                                for (int h = 0; h < kHalves; ++h)
                                    tma_load_3d(sq + (2 * qb + t) * kTile + h * kHalf, &tmap_q, h * 128, it.hg * pack, it.q0 + it.tok0 + t * (128 >> a.pack_log2), &q_full[qb]);
                    }
                    const int at = place + i, s = at % kStages;
                    if (at >= kStages && !mbar_wait_bounded(&kv_empty[s], ((at / kStages) - 1) & 1, a.status, STATUS_TIMEOUT_PIPE)) {
                        fine = false;
                        break;
                    }
                    const bool value = i == total - 1 || (i > 0 && (i & 1) == 0);
                    const int j = i == total - 1 ? it.most - 1 : value ? (i - 2) / 2 : (i + 1) / 2;
                    uint64_t *bar = &kv_full[s];
                    last_edge &= ~(1u << s);
                    if (value && j >= it.edge) {
                        bar = &edge_full[s];
                        edges ^= 1u << s;
                        last_edge |= 1u << s;
                    } else {
                        mbar_arrive(bar);
                    }
                    mbar_arrive_expect_tx(bar, kTile);
                    asked = at + 1;
                    for (int h = 0; h < kHalves; ++h)
                        tma_load_3d(ring + s * kTile + h * kHalf, value ? &tmap_v : &tmap_k, h * 128, kv_head, it.k0 + j * kPaKeys, bar);
                }
            }
            __syncwarp();
            const int from = __ffs(__ballot_sync(0xffffffffu, leader)) - 1;
            ok = __shfl_sync(0xffffffffu, (int)fine, from);
            asked = __shfl_sync(0xffffffffu, asked, from);
            queries = __shfl_sync(0xffffffffu, queries, from);
            edges = __shfl_sync(0xffffffffu, edges, from);
            last_edge = __shfl_sync(0xffffffffu, last_edge, from);
            place += total;
            ++blocks;
        }
        if (!ok) { // a wait ran out: what has been asked for arrives before the block ends, whether or not it is used
            for (int at = max(0, asked - kStages); at < asked; ++at) {
                const int s = at % kStages;
                if (last_edge >> s & 1)
                    mbar_wait_bounded(&edge_full[s], (edges >> s & 1) ^ 1, a.status, STATUS_TIMEOUT_TMA);
                else
                    mbar_wait_bounded(&kv_full[s], (at / kStages) & 1, a.status, STATUS_TIMEOUT_TMA);
            }
            for (int q = max(0, queries - kQBlocks); q < queries; ++q)
                mbar_wait_bounded(&q_full[q % kQBlocks], (q / kQBlocks) & 1, a.status, STATUS_TIMEOUT_TMA);
        }
    } else if (warp == 9) {
        // ---------------------------------------------------------------- products
        int place = 0, blocks = 0;
        uint32_t p_phase[2] = { 0, 0 };
        bool ok = true;
        for (int round = 0; ok; ++round) {
            const PaItem it = pa_item(a, number(round), lane);
            if (!it.valid)
                break;
            if (it.most == 0)
                continue;
            bool fine = true;
            if (elect_one()) {
                auto wait_kv = [&](int at) { return mbar_wait_bounded(&kv_full[at % kStages], (at / kStages) & 1, a.status, STATUS_TIMEOUT_TMA); };
                const int qb = blocks % kQBlocks;
                auto scores = [&](int t, int at) {
                    const uint32_t qa = smem_u32(sq + (2 * qb + t) * kTile), ka = smem_u32(ring + (at % kStages) * kTile);
#pragma unroll
                    for (int h = 0; h < kHalves; ++h) {
                        const uint64_t dq = make_smem_desc_sw128(qa + h * kHalf), dk = make_smem_desc_sw128(ka + h * kHalf);
#pragma unroll
                        for (int x = 0; x < 4; ++x) // 16 features of 2 bytes a step
                            umma_f16(tmem + (uint32_t)(t * 128), dq + (uint64_t)(2 * x), dk + (uint64_t)(2 * x), kIdescS, (h | x) != 0);
                    }
                    umma_commit(&s_full[t]);
                };
                auto values = [&](int t, int j, int at) {
                    const uint64_t dv = make_smem_desc_sw128_mn(smem_u32(ring + (at % kStages) * kTile), kHalf);
#pragma unroll
                    for (int x = 0; x < kPaKeys / 16; ++x) // 16 keys a step: 16 rows of V, 8 columns of P
                        umma_f16_ts(tmem + (uint32_t)(Sh::kO + t * D), tmem + (uint32_t)(Sh::kP + t * Sh::kPStep + 8 * x), dv + (uint64_t)(x * 2048 >> 4), kIdescO, (j | x) != 0);
                };
                // scores of key tile j; where P lies beside S they only wait until the softmax has read those before them
                auto free_scores = [&](int t, int j) {
                    const uint32_t before = p_phase[t] + j; // tiles of scores so far
                    return !kApart || before == 0 || mbar_wait_bounded(&s_read[t], (before - 1) & 1, a.status, STATUS_TIMEOUT_PIPE);
                };
                fine = mbar_wait_bounded(&q_full[qb], (blocks / kQBlocks) & 1, a.status, STATUS_TIMEOUT_TMA) && wait_kv(place);
                if (fine) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        if (it.n[t] > 0 && fine) {
                            fine = free_scores(t, 0);
                            tmem_fence_after();
                            if (fine)
                                scores(t, place);
                        }
                    umma_commit(&kv_empty[place % kStages]);
                    if (it.most == 1)
                        umma_commit(&q_empty[qb]);
                }
                for (int j = 0; j < it.most && fine; ++j) {
                    const int vat = place + pa_v_place(j, it.most), kat = place + pa_k_place(j + 1);
                    if (kApart) {
                        if (j + 1 < it.most) {
                            fine = wait_kv(kat);
#pragma unroll
                            for (int t = 0; t < 2; ++t)
                                if (j + 1 < it.n[t] && fine) {
                                    fine = free_scores(t, j + 1);
                                    tmem_fence_after();
                                    if (fine)
                                        scores(t, kat);
                                }
                            umma_commit(&kv_empty[kat % kStages]);
                            if (j + 2 == it.most)
                                umma_commit(&q_empty[qb]);
                        }
                        fine = fine && wait_kv(vat);
#pragma unroll
                        for (int t = 0; t < 2; ++t)
                            if (j < it.n[t] && fine) {
                                fine = mbar_wait_bounded(&p_ready[t], (p_phase[t] + j) & 1, a.status, STATUS_TIMEOUT_PIPE);
                                tmem_fence_after();
                                if (fine) {
                                    values(t, j, vat);
                                    umma_commit(&o_done[t]);
                                }
                            }
                        umma_commit(&kv_empty[vat % kStages]);
                        continue;
                    }
                    bool have_v = false, have_k = false;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (j >= it.n[t] || !fine)
                            continue;
                        fine = mbar_wait_bounded(&p_ready[t], (p_phase[t] + j) & 1, a.status, STATUS_TIMEOUT_PIPE) && (have_v || wait_kv(vat));
                        if (!fine)
                            continue;
                        have_v = true;
                        tmem_fence_after();
                        values(t, j, vat);
                        if (j == it.n[t] - 1) {
                            umma_commit(&o_done[t]); // O is complete (a barrier of its own: the next block's scores may be done before anybody has looked)
                        } else {
                            fine = have_k || wait_kv(kat);
                            if (!fine)
                                continue;
                            have_k = true;
                            tmem_fence_after();
                            scores(t, kat);
                        }
                    }
                    umma_commit(&kv_empty[vat % kStages]);
                    if (j + 1 < it.most)
                        umma_commit(&kv_empty[kat % kStages]);
                    if (j + 2 == it.most)
                        umma_commit(&q_empty[qb]);
                }
            }
            __syncwarp();
            ok = __all_sync(0xffffffffu, fine);
            p_phase[0] += it.n[0];
            p_phase[1] += it.n[1];
            place += 2 * it.most;
            ++blocks;
        }
        if (elect_one()) { // every product, and every arrival that one of them still owes, before the block ends
            umma_commit(drain);
            mbar_wait_bounded(drain, 0, a.status, STATUS_TIMEOUT_MMA);
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- V tiles that are not seen to the end
        const int half = warp - 10;
        int place = 0;
        uint32_t edges = 0, flags[2] = { 0, 0 }; // flags written, per row tile
        bool ok = true;
        for (int round = 0; ok; ++round) {
            const PaItem it = pa_item(a, number(round), lane);
            if (!it.valid)
                break;
            if (it.most == 0)
                continue;
            int bad = 0;
            for (int j = it.edge; j < it.most; ++j) {
                const int s = (place + pa_v_place(j, it.most)) % kStages;
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&edge_full[s], edges >> s & 1, a.status, STATUS_TIMEOUT_TMA));
                if (!ok)
                    break;
                edges ^= 1u << s;
                uint8_t *tile = ring + s * kTile + half * 64 * 128;
#pragma unroll 1
                for (int h = 0; h < kHalves; ++h) {
#pragma unroll 4
                    for (int i = 0; i < 64 * 128 / (32 * 16); ++i) {
                        uint4 *p = reinterpret_cast<uint4 *>(tile + h * kHalf + (i * 32 + lane) * 16);
                        uint4 x = *p;
                        uint32_t w[4] = { x.x, x.y, x.z, x.w }, top = 0;
                        constexpr uint32_t kOne = BF16 ? 0x00800080u : 0x04000400u; // the exponent's lowest bit: a full exponent carries into bit 15
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            top |= ((w[e] & 0x7fff7fffu) + kOne) & 0x80008000u;
                        if (top) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t f = ((w[e] & 0x7fff7fffu) + kOne) & 0x80008000u;
                                w[e] &= ~((f >> 15) * 0xffffu);
                            }
                            *p = make_uint4(w[0], w[1], w[2], w[3]);
                            const int key = j * kPaKeys + half * 64 + ((i * 32 + lane) >> 3);
                            bad |= key < it.nk;
                        }
                    }
                }
                bad = __any_sync(0xffffffffu, bad);
                if (lane == 0) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        if (j < it.n[t])
                            poison[2 * (4 * t + (flags[t] & 3)) + half] = bad;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&kv_full[s]);
            }
            place += 2 * it.most;
            flags[0] += it.edge < it.n[0];
            flags[1] += it.edge < it.n[1];
        }
    }

    tmem_fence_before();
    __syncthreads();
    if (warp == 9) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

static int pack_log2_of(int group) // the largest power of two that divides the group, at most 16
{
    int p = 0;
    while (p < 4 && group % (2 << p) == 0)
        ++p;
    return p;
}

static bool map_rows(CUtensorMap *m, const void *base, int D, int heads, int rows, long long head_stride, long long stride, int box_heads, int box_rows)
{
    const uint64_t dims[3] = { (uint64_t)D * 2, (uint64_t)heads, (uint64_t)rows };
    // (a dimension of one may come with any stride)
    const uint64_t strides[2] = { (uint64_t)(heads > 1 ? 2 * head_stride : 2 * D), (uint64_t)(rows > 1 ? 2 * stride : 2 * D) };
    const uint32_t box[3] = { 128, (uint32_t)box_heads, (uint32_t)box_rows };
    return encode_tmap(m, TMAP_U8, 3, base, dims, strides, box, TMAP_SWIZZLE_128B);
}

template <int D, bool BF16>
static cudaError_t launch_prompt(const CUtensorMap *m, const PaArgs &a, unsigned grid, cudaStream_t stream)
{
    static thread_local SmemOptIn opted;
    auto kern = prompt_attention_kernel<D, BF16>;
    const cudaError_t e = opted.ensure(kern, PaShape<D>::kSmem);
    if (e != cudaSuccess)
        return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kPaThreads);
    cfg.dynamicSmemBytes = PaShape<D>::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, m[0], m[1], m[2], a);
}

static bool strides_positive(int rows, int heads, long long stride, long long head_stride)
{
    return (rows <= 1 || (stride > 0 && stride < (1ll << 38))) && (heads <= 1 || (head_stride > 0 && head_stride < (1ll << 38)));
}

} // namespace abq

extern "C" abq_status abq_prompt_attention(const abq_prompt_attention_params *p, abq_stream_t stream)
{
    using namespace abq;
    if (!p || p->total_q < 0 || p->total_k < 0 || p->batch < 0 || p->kv_heads <= 0 || p->q_heads <= 0 || p->q_heads % p->kv_heads || p->q_heads > 65536 ||
        (p->head_dim != 64 && p->head_dim != 128) || (p->half_type != ABQ_HALF_FP16 && p->half_type != ABQ_HALF_BF16) || p->max_q < 0 ||
        !(p->scale > 0.f && p->scale <= 2e38f) || (reinterpret_cast<uintptr_t>(p->status_word) & 3))
        return ABQ_ERR_INVALID_ARG;
    if (p->total_q == 0 || p->batch == 0)
        return ABQ_OK;
    if (!half_rows_valid(p->q, p->q_stride, p->q_head_stride) || !half_rows_valid(p->out, p->out_stride, p->out_head_stride) ||
        !strides_positive(p->total_q, p->q_heads, p->q_stride, p->q_head_stride) || !strides_positive(p->total_q, p->q_heads, p->out_stride, p->out_head_stride) ||
        !p->cu_q || !p->cu_k || ((reinterpret_cast<uintptr_t>(p->cu_q) | reinterpret_cast<uintptr_t>(p->cu_k)) & 3))
        return ABQ_ERR_INVALID_ARG;
    if (p->total_k > 0 && (!half_rows_valid(p->k, p->k_stride, p->k_head_stride) || !half_rows_valid(p->v, p->v_stride, p->v_head_stride) ||
                           !strides_positive(p->total_k, p->kv_heads, p->k_stride, p->k_head_stride) || !strides_positive(p->total_k, p->kv_heads, p->v_stride, p->v_head_stride)))
        return ABQ_ERR_INVALID_ARG;
    if (p->out == p->q && (p->out_stride != p->q_stride || p->out_head_stride != p->q_head_stride))
        return ABQ_ERR_INVALID_ARG;
    const int group = p->q_heads / p->kv_heads, pl = pack_log2_of(group), D = p->head_dim;
    const long long head_groups = p->q_heads >> pl, tokens = 256 >> pl;
    long long slots = p->total_q / tokens + p->batch; // each sequence at most one block that is not full
    if (p->max_q)
        slots = std::min<long long>(slots, p->batch * ((p->max_q + tokens - 1) / tokens));
    if (slots * head_groups + 2048 >= (1ll << 31))
        return ABQ_ERR_INVALID_ARG;
    CUtensorMap m[3];
    const void *k = p->total_k ? p->k : p->q, *v = p->total_k ? p->v : p->q; // (without a key nothing is read)
    const int rows_k = p->total_k ? p->total_k : 1, heads_k = p->total_k ? p->kv_heads : 1;
    if (!map_rows(&m[0], p->q, D, p->q_heads, p->total_q, p->q_head_stride, p->q_stride, 1 << pl, 128 >> pl) ||
        !map_rows(&m[1], k, D, heads_k, rows_k, p->k_head_stride, p->k_stride, 1, kPaKeys) || !map_rows(&m[2], v, D, heads_k, rows_k, p->v_head_stride, p->v_stride, 1, kPaKeys))
        return ABQ_ERR_CUDA;
    PaArgs a = {};
    a.cu_q = p->cu_q, a.cu_k = p->cu_k, a.v = reinterpret_cast<const uint8_t *>(p->v), a.out = reinterpret_cast<uint8_t *>(p->out);
    a.v_stride = 2 * p->v_stride, a.v_head_stride = 2 * p->v_head_stride, a.out_stride = 2 * p->out_stride, a.out_head_stride = 2 * p->out_head_stride;
    a.total_q = p->total_q, a.total_k = p->total_k, a.batch = p->batch, a.head_groups = (int)head_groups, a.pack_log2 = pl, a.group = group;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.sorted = p->batch > 1 && p->batch <= 32 && slots * head_groups > 148;
    a.status = p->status_word;
    const unsigned grid = (unsigned)std::max<long long>(1, std::min<long long>(148, slots * head_groups));
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const bool bf16 = p->half_type == ABQ_HALF_BF16;
    const cudaError_t e = D == 128 ? (bf16 ? launch_prompt<128, true>(m, a, grid, s) : launch_prompt<128, false>(m, a, grid, s))
                                   : (bf16 ? launch_prompt<64, true>(m, a, grid, s) : launch_prompt<64, false>(m, a, grid, s));
    if (e != cudaSuccess) {
        set_last_cuda_error(e);
        return ABQ_ERR_CUDA;
    }
    return ABQ_OK;
}
