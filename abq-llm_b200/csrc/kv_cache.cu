// Quantising a cache as it is written, and reading it back (abq_kv_cache_write, abq_kv_cache_read).
//
// Both move each value once: 2 bytes of fp16 / bf16 on one side, bits / 8 of codes and 4 / head_dim of parameters on the other.  What bounds them is
// HBM.  A group of head_dim / 8 lanes owns one token's row of one head: a lane holds 8 values (one 16-byte access), the row's range meets by
// shuffles on a packed (min, -max) pair.  A CTA takes 16 consecutive tokens, so that the rows of a granule and its 64-byte parameter lines are
// touched by one CTA, and several heads one after the other, keys and values of one head in flight together.
//
// Quantiser: code = rint((x - min) / scale), a correctly rounded fp32 division.  It is taken twice as a product with the reciprocal, made 2^-20 too small and
// too large, in one multiply-add that rounds to an integer: where both give the same code the division does too; a row part where they do not (a quotient
// close to the middle between two codes), or whose scale is below the normal range, is divided.  The scale is rounded up to 16 bits, so max never passes the
// last code.
//
// Measured: 16001 tokens of 32 heads of 128, fp16 and 4 bits (332 MB either way): written in 76 to 81 us (4.1 to 4.4 TB/s; bound by instructions: 135 before the arithmetic was
// packed and the divisions taken out, 90 with every lane working out both rows' parameters), read back in 62 us (5.4 TB/s, 82 % of a copy's rate), 55 behind the write, part
// of the cache still in L2; 8 bits (398 MB) written in 78 us (5.1 TB/s), read in 70 (5.7).
#include <type_traits>

#include "abq_kernels.h"
#include "kv_cache.cuh"

namespace abq {

constexpr int kKvThreads = 256;
constexpr int kKvMostRows = 0x7fffff00; // a CTA's last row has a 32-bit number

struct KvShape {
    uint8_t *data;
    long long capacity; // places: num_pages * page_size
    int num_pages, page_size, kv_heads;
};

__device__ __forceinline__ uint8_t *kv_granule(const KvShape &c, int page, int place, int head, int granule_bytes)
{
    return c.data + (((size_t)page * c.kv_heads + head) * (c.page_size >> 4) + (place >> 4)) * granule_bytes;
}

// The lesser and the larger of two packed pairs; NaN stays
template <bool BF16>
__device__ __forceinline__ uint32_t pair_min(uint32_t a, uint32_t b)
{
    uint32_t r;
    if (BF16)
        asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
        asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b)
{
    uint32_t r;
    if (BF16)
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint64_t pack_floats(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack_bits(uint64_t v, uint32_t &lo, uint32_t &hi) { asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t add_floats(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma_floats(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// (min, -max) of a lane's eight values
template <bool BF16>
__device__ __forceinline__ uint32_t range8(const uint4 &x)
{
    const uint32_t lo = pair_min<BF16>(pair_min<BF16>(x.x, x.y), pair_min<BF16>(x.z, x.w));
    const uint32_t hi = pair_max<BF16>(pair_max<BF16>(x.x, x.y), pair_max<BF16>(x.z, x.w)) ^ 0x80008000u;
    return pair_min<BF16>(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
}

// A row's parameters from its range: the 32 bits (scale, min) that are stored, and the scale's reciprocal, or 0 where that is no use (a scale of 0, or one whose
// reciprocal is not a normal number)
template <int BITS, bool BF16>
__device__ __forceinline__ uint32_t row_params(uint32_t range, float &inv)
{
    const float2 mm = half_pair_to_float(range, BF16);
    const float spread = -mm.y - mm.x, fine = spread / (float)((1 << BITS) - 1);
    uint32_t sbits = float_pair_to_half(fine, 0.f, BF16) & 0xffffu;
    if (half_bits_to_float(sbits, BF16) < fine)
        ++sbits; // up to the next 16-bit value (positive values are ordered like their bits)
    const float s = half_bits_to_float(sbits, BF16);
    asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(s)); // at most 1 ulp off
    inv = s >= 1.17549435e-38f && s <= 8.5e37f ? inv : 0.f;
    return spread <= 3.402823466e38f ? sbits | range << 16 : BF16 ? 0x7fc07fc0u : 0x7e007e00u; // (not for Inf or NaN among the values)
}

template <int D, int BITS, bool BF16>
__device__ __forceinline__ void quantise_row(const uint4 &x, uint32_t params, float inv, int at, uint8_t *rows, bool kept)
{
    const uint32_t w[4] = { x.x, x.y, x.z, x.w };
    const float2 sm = half_pair_to_float(params, BF16);
    const float s = sm.x, mn = sm.y;
    const float less = inv * (1.f - 9.5367432e-7f), more = inv * (1.f + 9.5367432e-7f);
    const uint64_t less2 = pack_floats(less, less), more2 = pack_floats(more, more), mn2 = pack_floats(-mn, -mn);
    const uint64_t magic2 = pack_floats(12582912.f, 12582912.f); // 1.5 * 2^23: the sum's low bits are the rounded value
    uint32_t code[8], differ = s > 0.f && inv == 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = half_pair_to_float(w[i], BF16);
        const uint64_t d = add_floats(pack_floats(f.x, f.y), mn2);
        uint32_t m0, m1;
        unpack_bits(fma_floats(d, less2, magic2), code[2 * i], code[2 * i + 1]);
        unpack_bits(fma_floats(d, more2, magic2), m0, m1);
        differ |= (code[2 * i] ^ m0) | (code[2 * i + 1] ^ m1);
    }
    if (differ) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = half_pair_to_float(w[i], BF16);
            code[2 * i] = s > 0.f ? (uint32_t)__float2int_rn((f.x - mn) / s) : 0u;
            code[2 * i + 1] = s > 0.f ? (uint32_t)__float2int_rn((f.y - mn) / s) : 0u;
        }
    }
    if (s != s) { // NaN stands for the row
#pragma unroll
        for (int i = 0; i < 8; ++i)
            code[i] = 0;
    }
    if (!kept)
        return;
    if (BITS == 8) {
        uint2 o;
        o.x = __byte_perm(__byte_perm(code[0], code[1], 0x0040), __byte_perm(code[2], code[3], 0x0040), 0x5410);
        o.y = __byte_perm(__byte_perm(code[4], code[5], 0x0040), __byte_perm(code[6], code[7], 0x0040), 0x5410);
        *reinterpret_cast<uint2 *>(rows + at) = o;
    } else {
        uint32_t two[4]; // the low byte: two codes
#pragma unroll
        for (int i = 0; i < 4; ++i)
            two[i] = code[2 * i] + (code[2 * i + 1] << 4);
        const uint32_t o = __byte_perm(__byte_perm(two[0], two[1], 0x0040), __byte_perm(two[2], two[3], 0x0040), 0x5410);
        *reinterpret_cast<uint32_t *>(rows + at) = o;
    }
}

// A token's rows of keys and values of one head.  The lower half of the lanes takes the keys' range and parameters, the upper half the values': what is the same for a
// whole row is worked out by half as many instructions.
template <int D, int BITS, bool BF16>
__device__ __forceinline__ void quantise_token(const uint4 &x, const uint4 &y, int sub, int place, uint8_t *granule, bool kept)
{
    constexpr int RB = kv_row_bytes(D, BITS), kLanes = D / 8, kHalf = kLanes / 2;
    const bool upper = sub >= kHalf;
    const uint32_t rx = range8<BF16>(x), ry = range8<BF16>(y);
    uint32_t range = pair_min<BF16>(upper ? ry : rx, __shfl_xor_sync(0xffffffffu, upper ? rx : ry, kHalf));
#pragma unroll
    for (int o = 1; o < kHalf; o <<= 1)
        range = pair_min<BF16>(range, __shfl_xor_sync(0xffffffffu, range, o));
    float inv;
    const uint32_t params = row_params<BITS, BF16>(range, inv);
    const uint32_t other = __shfl_xor_sync(0xffffffffu, params, kHalf);
    const float other_inv = __shfl_xor_sync(0xffffffffu, inv, kHalf);
    const int t = place & 15, at = kv_place<RB>(t, sub * BITS);
    quantise_row<D, BITS, BF16>(x, upper ? other : params, upper ? other_inv : inv, at, granule, kept);
    quantise_row<D, BITS, BF16>(y, upper ? params : other, upper ? inv : other_inv, at, granule + 16 * RB, kept);
    if (kept && (sub & (kHalf - 1)) == 0)
        *reinterpret_cast<uint32_t *>(granule + (upper ? kv_param_offset(RB, 1) : kv_param_offset(RB, 0)) + 4 * t) = params;
}

struct KvWriteArgs {
    KvShape c;
    const uint8_t *k, *v;
    long long k_stride, k_head_stride, v_stride, v_head_stride; // bytes
    const int64_t *slots;
    int tokens, heads_per_cta;
};

template <int D, int BITS, bool BF16>
__global__ void __launch_bounds__(kKvThreads) kv_write_kernel(const KvWriteArgs a)
{
    constexpr int kLanes = D / 8, kTokens = kKvThreads / kLanes, kGranule = kv_granule_bytes(kv_row_bytes(D, BITS));
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int sub = threadIdx.x % kLanes, token = blockIdx.x * kTokens + threadIdx.x / kLanes;
    // lanes of rows that are left out stay for the shuffles; what they work out is not stored
    const int h0 = blockIdx.y * a.heads_per_cta, h1 = min(a.c.kv_heads, h0 + a.heads_per_cta);
    const bool exists = token < a.tokens;
    const uint8_t *ks = a.k + (exists ? token * a.k_stride : 0) + sub * 16, *vs = a.v + (exists ? token * a.v_stride : 0) + sub * 16;
    uint4 x = make_uint4(0, 0, 0, 0), y = x;
    int64_t slot = -1;
    if (exists) { // the first head's rows with the slot, not behind it: one latency less
        x = *reinterpret_cast<const uint4 *>(ks + h0 * a.k_head_stride);
        y = *reinterpret_cast<const uint4 *>(vs + h0 * a.v_head_stride);
        slot = a.slots[token];
    }
    const bool kept = slot >= 0 && slot < a.c.capacity;
    const int page = kept ? (int)(slot / a.c.page_size) : 0, place = kept ? (int)(slot - (int64_t)page * a.c.page_size) : 0;
    if (!__any_sync(0xffffffffu, kept))
        return;
    uint8_t *granule = kv_granule(a.c, page, place, h0, kGranule);
    const size_t head_step = (size_t)(a.c.page_size >> 4) * kGranule;
    for (int h = h0; h < h1; ++h, granule += head_step) {
        uint4 nx = x, ny = y; // the next head's rows are under way while this one's are quantised
        if (kept && h + 1 < h1) {
            nx = *reinterpret_cast<const uint4 *>(ks + (h + 1) * a.k_head_stride);
            ny = *reinterpret_cast<const uint4 *>(vs + (h + 1) * a.v_head_stride);
        }
        quantise_token<D, BITS, BF16>(x, y, sub, place, granule, kept);
        x = nx;
        y = ny;
    }
}

// eight codes of a row -> eight 16-bit values: 0x4b000000 | c is the number 2^23 + c; code * scale is exact in 24 bits, so the multiply-add rounds like the sum
template <int BITS, bool BF16>
__device__ __forceinline__ uint4 restore8(uint2 codes, float2 p)
{
    const uint64_t scale2 = pack_floats(p.x, p.x), min2 = pack_floats(p.y, p.y), off2 = pack_floats(-8388608.f, -8388608.f);
    uint32_t half[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t a, b;
        if (BITS == 8) {
            const uint32_t w = i < 2 ? codes.x : codes.y;
            a = __byte_perm(w, 0x4b000000u, (i & 1) ? 0x7442 : 0x7440);
            b = __byte_perm(w, 0x4b000000u, (i & 1) ? 0x7443 : 0x7441);
        } else {
            a = ((codes.x >> (8 * i)) & 15u) | 0x4b000000u;
            b = ((codes.x >> (8 * i + 4)) & 15u) | 0x4b000000u;
        }
        uint32_t lo, hi;
        unpack_bits(fma_floats(add_floats(pack_floats(__uint_as_float(a), __uint_as_float(b)), off2), scale2, min2), lo, hi);
        half[i] = float_pair_to_half(__uint_as_float(lo), __uint_as_float(hi), BF16);
    }
    return make_uint4(half[0], half[1], half[2], half[3]);
}

struct KvReadArgs {
    KvShape c;
    uint8_t *k, *v;
    long long k_stride, k_head_stride, v_stride, v_head_stride; // bytes
    const int *block_table, *cu_seqlens;
    int rows, batch, table_stride, heads_per_cta;
};

template <int D, int BITS, bool BF16>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(const KvReadArgs a)
{
    constexpr int kLanes = D / 8, kTokens = kKvThreads / kLanes, RB = kv_row_bytes(D, BITS), kGranule = kv_granule_bytes(RB);
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int sub = threadIdx.x % kLanes, row = blockIdx.x * kTokens + threadIdx.x / kLanes;
    int lo = 0, start, end; // the sequence with cu[lo] <= row < cu[lo + 1]
    if (a.batch < 32) {     // one load, a place a lane
        const int lane = threadIdx.x & 31, mine = a.cu_seqlens[min(lane, a.batch)], first = row - lane / kLanes;
#pragma unroll
        for (int j = 0; j < 32 / kLanes; ++j) {
            const uint32_t before = __ballot_sync(0xffffffffu, lane < a.batch && mine <= first + j);
            if (lane / kLanes == j)
                lo = max(0, 31 - __clz((int)before));
        }
        start = __shfl_sync(0xffffffffu, mine, lo);
        end = __shfl_sync(0xffffffffu, mine, a.batch);
    } else {
        int hi = a.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.cu_seqlens[mid] <= row)
                lo = mid;
            else
                hi = mid;
        }
        start = a.cu_seqlens[lo];
        end = a.cu_seqlens[a.batch];
    }
    start = max(start, 0);
    if (row >= a.rows || row >= end || row < start) // (rows before the first sequence have no position: a negative one would lie in front of its page)
        return;
    const int pos = row - start, entry = pos / a.c.page_size, place = pos - entry * a.c.page_size;
    const int page = entry < a.table_stride ? a.block_table[(size_t)lo * a.table_stride + entry] : -1;
    const bool held = page >= 0 && page < a.c.num_pages;
    const int h0 = blockIdx.y * a.heads_per_cta, h1 = min(a.c.kv_heads, h0 + a.heads_per_cta), t = place & 15;
    const int at = kv_place<RB>(t, sub * BITS);
    uint8_t *ko = a.k + row * a.k_stride + sub * 16, *vo = a.v + row * a.v_stride + sub * 16;
    struct Item {
        uint2 kc, vc;
        uint32_t kp, vp;
    };
    auto load = [&](int h) {
        Item i = {};
        if (held) {
            const uint8_t *g = kv_granule(a.c, page, place, h, kGranule);
            if (BITS == 8) {
                i.kc = *reinterpret_cast<const uint2 *>(g + at);
                i.vc = *reinterpret_cast<const uint2 *>(g + 16 * RB + at);
            } else {
                i.kc.x = *reinterpret_cast<const uint32_t *>(g + at);
                i.vc.x = *reinterpret_cast<const uint32_t *>(g + 16 * RB + at);
            }
            i.kp = *reinterpret_cast<const uint32_t *>(g + kv_param_offset(RB, 0) + 4 * t);
            i.vp = *reinterpret_cast<const uint32_t *>(g + kv_param_offset(RB, 1) + 4 * t);
        }
        return i;
    };
    Item i = load(h0);
    for (int h = h0; h < h1; ++h) {
        const Item next = h + 1 < h1 ? load(h + 1) : i; // under way while this head's values are written
        *reinterpret_cast<uint4 *>(ko + h * a.k_head_stride) = restore8<BITS, BF16>(i.kc, half_pair_to_float(i.kp, BF16));
        *reinterpret_cast<uint4 *>(vo + h * a.v_head_stride) = restore8<BITS, BF16>(i.vc, half_pair_to_float(i.vp, BF16));
        i = next;
    }
}

bool kv_cache_valid(const abq_kv_cache &c)
{
    return c.num_pages > 0 && c.page_size > 0 && c.page_size % 16 == 0 && c.page_size <= 1024 && c.kv_heads > 0 && c.kv_heads <= 65535 &&
           (c.head_dim == 64 || c.head_dim == 128) && (c.bits == 8 || c.bits == 4) && (c.half_type == ABQ_HALF_FP16 || c.half_type == ABQ_HALF_BF16);
}

// rows of head_dim values, 16 bytes at a time: alignment of the pointer and strides
bool half_rows_valid(const void *p, long long stride, long long head_stride)
{
    return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0 && head_stride % 8 == 0;
}

static KvShape kv_shape(const abq_kv_cache &c)
{
    return { reinterpret_cast<uint8_t *>(c.data), (long long)c.num_pages * c.page_size, c.num_pages, c.page_size, c.kv_heads };
}

// Heads that a CTA takes one after the other: as many as leave the GPU a few thousand CTAs (a CTA is 16 or 32 tokens), at most 8
static int heads_per_cta(int row_blocks, int heads)
{
    const long long ctas = (long long)row_blocks * heads;
    return ctas >= 8 * 2368 ? 8 : ctas >= 4 * 2368 ? 4 : ctas >= 2 * 2368 ? 2 : 1;
}

template <typename Kernel, typename Args>
static abq_status launch_kv(Kernel kern, dim3 grid, const Args &args, abq_stream_t stream)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kKvThreads);
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args);
    if (e != cudaSuccess) {
        set_last_cuda_error(e);
        return ABQ_ERR_CUDA;
    }
    return ABQ_OK;
}

// The kernel's template arguments from a cache's description
template <typename F>
static abq_status with_shape(const abq_kv_cache &c, F f)
{
    using std::integral_constant;
    auto typed = [&](auto dim, auto bits) {
        return c.half_type == ABQ_HALF_BF16 ? f(dim, bits, std::true_type()) : f(dim, bits, std::false_type());
    };
    auto sized = [&](auto dim) { return c.bits == 8 ? typed(dim, integral_constant<int, 8>()) : typed(dim, integral_constant<int, 4>()); };
    return c.head_dim == 128 ? sized(integral_constant<int, 128>()) : sized(integral_constant<int, 64>());
}

} // namespace abq

extern "C" size_t abq_kv_cache_bytes(const abq_kv_cache *cache)
{
    if (!cache || !abq::kv_cache_valid(*cache))
        return 0;
    return (size_t)cache->num_pages * cache->kv_heads * (cache->page_size / 16) * abq::kv_granule_bytes(abq::kv_row_bytes(cache->head_dim, cache->bits));
}

extern "C" abq_status abq_kv_cache_write(const abq_kv_write_params *p, abq_stream_t stream)
{
    using namespace abq;
    if (!p || !kv_cache_valid(p->cache) || !p->cache.data || (reinterpret_cast<uintptr_t>(p->cache.data) & 15) || p->tokens < 0 || p->tokens > kKvMostRows)
        return ABQ_ERR_INVALID_ARG;
    if (p->tokens == 0)
        return ABQ_OK;
    if (!half_rows_valid(p->k, p->k_stride, p->k_head_stride) || !half_rows_valid(p->v, p->v_stride, p->v_head_stride) || !p->slots ||
        (reinterpret_cast<uintptr_t>(p->slots) & 7))
        return ABQ_ERR_INVALID_ARG;
    const int D = p->cache.head_dim, H = p->cache.kv_heads, per = kKvThreads / (D / 8), blocks = (p->tokens - 1) / per + 1, hpc = heads_per_cta(blocks, H);
    const KvWriteArgs a = { kv_shape(p->cache), reinterpret_cast<const uint8_t *>(p->k), reinterpret_cast<const uint8_t *>(p->v), 2 * p->k_stride,
                            2 * p->k_head_stride, 2 * p->v_stride, 2 * p->v_head_stride, p->slots, p->tokens, hpc };
    const dim3 grid(blocks, (H + hpc - 1) / hpc);
    return with_shape(p->cache, [&](auto dim, auto bits, auto bf16) {
        return launch_kv(kv_write_kernel<decltype(dim)::value, decltype(bits)::value, decltype(bf16)::value>, grid, a, stream);
    });
}

extern "C" abq_status abq_kv_cache_read(const abq_kv_read_params *p, abq_stream_t stream)
{
    using namespace abq;
    if (!p || !kv_cache_valid(p->cache) || !p->cache.data || (reinterpret_cast<uintptr_t>(p->cache.data) & 15) || p->rows < 0 || p->rows > kKvMostRows || p->batch < 0)
        return ABQ_ERR_INVALID_ARG;
    if (p->rows == 0 || p->batch == 0)
        return ABQ_OK;
    if (!half_rows_valid(p->k, p->k_stride, p->k_head_stride) || !half_rows_valid(p->v, p->v_stride, p->v_head_stride) || !p->block_table || p->table_stride <= 0 ||
        !p->cu_seqlens || ((reinterpret_cast<uintptr_t>(p->block_table) | reinterpret_cast<uintptr_t>(p->cu_seqlens)) & 3))
        return ABQ_ERR_INVALID_ARG;
    const int D = p->cache.head_dim, H = p->cache.kv_heads, per = kKvThreads / (D / 8), blocks = (p->rows - 1) / per + 1, hpc = heads_per_cta(blocks, H);
    const KvReadArgs a = { kv_shape(p->cache), reinterpret_cast<uint8_t *>(p->k), reinterpret_cast<uint8_t *>(p->v), 2 * p->k_stride, 2 * p->k_head_stride,
                           2 * p->v_stride, 2 * p->v_head_stride, p->block_table, p->cu_seqlens, p->rows, p->batch, p->table_stride, hpc };
    const dim3 grid(blocks, (H + hpc - 1) / hpc);
    return with_shape(p->cache, [&](auto dim, auto bits, auto bf16) {
        return launch_kv(kv_read_kernel<decltype(dim)::value, decltype(bits)::value, decltype(bf16)::value>, grid, a, stream);
    });
}
