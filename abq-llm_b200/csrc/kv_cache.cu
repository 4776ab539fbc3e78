// Quantising a cache as it is written, and reading it back (abq_kv_cache_write, abq_kv_cache_read).
//
// Both move each value once: 2 bytes of fp16 / bf16 on one side, bits / 8 of codes and 4 / head_dim of parameters on the other.  What bounds them is
// HBM.  A group of head_dim / 8 lanes owns one token's row of one head: a lane holds 8 values (one 16-byte access), the row's range meets by
// shuffles on a packed (min, -max) pair.  A CTA takes 16 consecutive tokens, so that the rows of a granule and its 64-byte parameter lines are
// touched by one CTA, and several heads one after the other, keys and values of one head in flight together.
//
// Quantiser: code = rint((x - min) / scale), a correctly rounded fp32 division.  It is taken as a product with the reciprocal: that is off by at most
// 2^-23 of a quotient of at most 255.5, 3.1e-5, so a quotient further than 2^-14 from the middle between two codes rounds to the same one;
// the others (and rows whose scale is below the normal range) are divided.  The scale is rounded up to 16 bits, so max never passes the last code.
#include "abq_kernels.h"
#include "kv_cache.cuh"

namespace abq {

constexpr int kKvThreads = 256;

struct KvShape {
    uint8_t *data;
    long long capacity; // places: num_pages * page_size
    int num_pages, page_size, kv_heads;
    bool bf16;
};

__device__ __forceinline__ uint8_t *kv_granule(const KvShape &c, int page, int place, int head, int granule_bytes)
{
    return c.data + (((size_t)page * c.kv_heads + head) * (c.page_size >> 4) + (place >> 4)) * granule_bytes;
}

// The lesser (min, -max) of two packed pairs, NaN ignored
__device__ __forceinline__ uint32_t range_min(uint32_t a, uint32_t b, bool bf16)
{
    if (bf16) {
        const __nv_bfloat162 r = __hmin2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    const __half2 r = __hmin2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}

template <int D, int BITS>
__device__ __forceinline__ void quantise_row(const uint4 &x, int sub, int place, uint8_t *granule, int part, bool bf16, bool kept)
{
    constexpr int RB = kv_row_bytes(D, BITS), kLanes = D / 8;
    const uint32_t w[4] = { x.x, x.y, x.z, x.w };
    uint32_t lo = w[0], neg = w[0] ^ 0x80008000u, mag = w[0] & 0x7fff7fffu; // lo: mins of even and odd values, neg: mins of their negatives
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        lo = range_min(lo, w[i], bf16);
        neg = range_min(neg, w[i] ^ 0x80008000u, bf16);
        mag = __vmaxu2(mag, w[i] & 0x7fff7fffu);
    }
    // (min of all, min of negatives) in one word, and the largest magnitude's bits for the check on Inf and NaN
    uint32_t range = range_min(__byte_perm(lo, neg, 0x5410), __byte_perm(lo, neg, 0x7632), bf16);
    uint32_t top = max(mag & 0xffffu, mag >> 16);
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) {
        range = range_min(range, __shfl_xor_sync(0xffffffffu, range, o), bf16);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    const float2 mm = half_pair_to_float(range, bf16);
    const float mn = mm.x, spread = -mm.y - mm.x;
    const bool finite = top < (bf16 ? 0x7f80u : 0x7c00u) && spread <= 3.402823466e38f;
    const float fine = spread / (float)((1 << BITS) - 1);
    uint32_t sbits = float_pair_to_half(fine, 0.f, bf16) & 0xffffu;
    if (half_bits_to_float(sbits, bf16) < fine)
        ++sbits; // up to the next 16-bit value (positive values are ordered like their bits)
    const float s = half_bits_to_float(sbits, bf16);
    const bool usual = s >= 1.17549435e-38f; // the reciprocal of a normal number is finite
    const float inv = usual ? 1.f / s : 0.f;
    uint32_t code[8];
    bool close = s > 0.f && !usual;
    const float magic = 12582912.f; // 1.5 * 2^23: the sum's low bits are the rounded value
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = half_pair_to_float(w[i], bf16);
        const float t0 = (f.x - mn) * inv, t1 = (f.y - mn) * inv;
        const float r0 = t0 + magic, r1 = t1 + magic;
        close |= fabsf(t0 - (r0 - magic)) > 0.5f - 6.1035156e-5f;
        close |= fabsf(t1 - (r1 - magic)) > 0.5f - 6.1035156e-5f;
        code[2 * i] = __float_as_uint(r0);
        code[2 * i + 1] = __float_as_uint(r1);
    }
    if (close) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = half_pair_to_float(w[i], bf16);
            code[2 * i] = (uint32_t)__float2int_rn((f.x - mn) / s);
            code[2 * i + 1] = (uint32_t)__float2int_rn((f.y - mn) / s);
        }
    }
    if (!finite) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            code[i] = 0;
    }
    if (!kept)
        return;
    uint8_t *rows = granule + part * 16 * RB;
    const int t = place & 15;
    if (BITS == 8) {
        uint2 o;
        o.x = __byte_perm(__byte_perm(code[0], code[1], 0x0040), __byte_perm(code[2], code[3], 0x0040), 0x5410);
        o.y = __byte_perm(__byte_perm(code[4], code[5], 0x0040), __byte_perm(code[6], code[7], 0x0040), 0x5410);
        *reinterpret_cast<uint2 *>(rows + kv_place<RB>(t, sub * 8)) = o;
    } else {
        uint32_t o = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            o |= (code[i] & 15u) << (4 * i);
        *reinterpret_cast<uint32_t *>(rows + kv_place<RB>(t, sub * 4)) = o;
    }
    if (sub == 0) {
        const uint32_t pair = finite ? sbits | range << 16 : (bf16 ? 0x7fc07fc0u : 0x7e007e00u);
        *reinterpret_cast<uint32_t *>(granule + kv_param_offset(RB, part) + 4 * t) = pair;
    }
}

struct KvWriteArgs {
    KvShape c;
    const uint8_t *k, *v;
    long long k_stride, k_head_stride, v_stride, v_head_stride; // bytes
    const int64_t *slots;
    int tokens, heads_per_cta;
};

template <int D, int BITS>
__global__ void __launch_bounds__(kKvThreads) kv_write_kernel(const KvWriteArgs a)
{
    constexpr int kLanes = D / 8, kTokens = kKvThreads / kLanes, kGranule = kv_granule_bytes(kv_row_bytes(D, BITS));
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int sub = threadIdx.x % kLanes, token = blockIdx.x * kTokens + threadIdx.x / kLanes;
    // lanes of rows that are left out stay for the shuffles, with a row of zeros that is not stored
    const int64_t slot = token < a.tokens ? a.slots[token] : -1;
    const bool kept = slot >= 0 && slot < a.c.capacity;
    const int page = kept ? (int)(slot / a.c.page_size) : 0, place = kept ? (int)(slot - (int64_t)page * a.c.page_size) : 0;
    const int h0 = blockIdx.y * a.heads_per_cta, h1 = min(a.c.kv_heads, h0 + a.heads_per_cta);
    const uint8_t *ks = a.k + (kept ? token * a.k_stride : 0) + sub * 16, *vs = a.v + (kept ? token * a.v_stride : 0) + sub * 16;
    if (!__any_sync(0xffffffffu, kept))
        return;
    uint4 x = make_uint4(0, 0, 0, 0), y = x;
    if (kept) {
        x = *reinterpret_cast<const uint4 *>(ks + h0 * a.k_head_stride);
        y = *reinterpret_cast<const uint4 *>(vs + h0 * a.v_head_stride);
    }
    for (int h = h0; h < h1; ++h) {
        uint4 nx = x, ny = y; // the next head's rows are under way while this one's are quantised
        if (kept && h + 1 < h1) {
            nx = *reinterpret_cast<const uint4 *>(ks + (h + 1) * a.k_head_stride);
            ny = *reinterpret_cast<const uint4 *>(vs + (h + 1) * a.v_head_stride);
        }
        uint8_t *granule = kv_granule(a.c, page, place, h, kGranule);
        quantise_row<D, BITS>(x, sub, place, granule, 0, a.c.bf16, kept);
        quantise_row<D, BITS>(y, sub, place, granule, 1, a.c.bf16, kept);
        x = nx;
        y = ny;
    }
}

// eight codes of a row -> eight 16-bit values
template <int BITS>
__device__ __forceinline__ uint4 restore8(uint2 codes, float2 p, bool bf16)
{
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t c = BITS == 8 ? ((i < 4 ? codes.x : codes.y) >> (8 * (i & 3))) & 255u : (codes.x >> (4 * i)) & 15u;
        f[i] = fmaf((float)c, p.x, p.y); // one rounding: code * scale is exact in 24 bits, so this is the sum's
    }
    return make_uint4(float_pair_to_half(f[0], f[1], bf16), float_pair_to_half(f[2], f[3], bf16), float_pair_to_half(f[4], f[5], bf16),
                      float_pair_to_half(f[6], f[7], bf16));
}

struct KvReadArgs {
    KvShape c;
    uint8_t *k, *v;
    long long k_stride, k_head_stride, v_stride, v_head_stride; // bytes
    const int *block_table, *cu_seqlens;
    int rows, batch, table_stride, heads_per_cta;
};

template <int D, int BITS>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(const KvReadArgs a)
{
    constexpr int kLanes = D / 8, kTokens = kKvThreads / kLanes, RB = kv_row_bytes(D, BITS), kGranule = kv_granule_bytes(RB);
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int sub = threadIdx.x % kLanes, row = blockIdx.x * kTokens + threadIdx.x / kLanes;
    if (row >= a.rows || row >= a.cu_seqlens[a.batch])
        return;
    int lo = 0, hi = a.batch; // the sequence with cu[lo] <= row < cu[lo + 1]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu_seqlens[mid] <= row)
            lo = mid;
        else
            hi = mid;
    }
    const int pos = row - a.cu_seqlens[lo], entry = pos / a.c.page_size, place = pos - entry * a.c.page_size;
    const int page = entry >= 0 && entry < a.table_stride ? a.block_table[(size_t)lo * a.table_stride + entry] : -1;
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
        *reinterpret_cast<uint4 *>(ko + h * a.k_head_stride) = restore8<BITS>(i.kc, half_pair_to_float(i.kp, a.c.bf16), a.c.bf16);
        *reinterpret_cast<uint4 *>(vo + h * a.v_head_stride) = restore8<BITS>(i.vc, half_pair_to_float(i.vp, a.c.bf16), a.c.bf16);
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
    return { reinterpret_cast<uint8_t *>(c.data), (long long)c.num_pages * c.page_size, c.num_pages, c.page_size, c.kv_heads, c.half_type == ABQ_HALF_BF16 };
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
    if (!p || !kv_cache_valid(p->cache) || !p->cache.data || (reinterpret_cast<uintptr_t>(p->cache.data) & 15) || p->tokens < 0)
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
    if (D == 128)
        return p->cache.bits == 8 ? launch_kv(kv_write_kernel<128, 8>, grid, a, stream) : launch_kv(kv_write_kernel<128, 4>, grid, a, stream);
    return p->cache.bits == 8 ? launch_kv(kv_write_kernel<64, 8>, grid, a, stream) : launch_kv(kv_write_kernel<64, 4>, grid, a, stream);
}

extern "C" abq_status abq_kv_cache_read(const abq_kv_read_params *p, abq_stream_t stream)
{
    using namespace abq;
    if (!p || !kv_cache_valid(p->cache) || !p->cache.data || (reinterpret_cast<uintptr_t>(p->cache.data) & 15) || p->rows < 0 || p->batch < 0)
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
    if (D == 128)
        return p->cache.bits == 8 ? launch_kv(kv_read_kernel<128, 8>, grid, a, stream) : launch_kv(kv_read_kernel<128, 4>, grid, a, stream);
    return p->cache.bits == 8 ? launch_kv(kv_read_kernel<64, 8>, grid, a, stream) : launch_kv(kv_read_kernel<64, 4>, grid, a, stream);
}
