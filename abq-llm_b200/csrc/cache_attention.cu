// C entry of the attention over the quantised cache: checks, row blocks and grid (the kernels are in cache_attention.cuh).
#include <algorithm>

#include "cache_attention.cuh"

namespace abq {

template <int NT>
cudaError_t launch_cache_attention(const CacheAttnArgs &args, int head_dim, int bits, bool bf16, cudaStream_t stream);
extern template cudaError_t launch_cache_attention<1>(const CacheAttnArgs &, int, int, bool, cudaStream_t);
extern template cudaError_t launch_cache_attention<2>(const CacheAttnArgs &, int, int, bool, cudaStream_t);

// Tiles of 8 query rows that a block of the mma.sync kernel holds.  One conversion of the codes serves them all, but with more rows fewer warps fit: blocks of 16
// measured faster than of 32 for 26 rows over 40 heads of 128, 8 bits (36.8 and 43.5 us; blocks of 8: 41.8).
static int row_tiles(int rows) { return rows <= 8 ? 1 : 2; }

cudaError_t launch_cache_attention_tile(const CacheAttnArgs &args, int head_dim, int bits, bool bf16, cudaStream_t stream);

// What a call of so many query rows a head runs on.
struct CaPlan {
    bool tile;              // the kernel of 128 rows (cache_attention_tile.cu)
    int block, most_runs;   // rows of a block; runs the line is cut into at most
    int unit_log2, extra, min_quota;
};
static CaPlan ca_plan(int rows, int head_dim)
{
    const int blocks = (rows + 127) / 128;
    if (rows >= 80 * blocks) // (measured: see there)
        return { true, 128, kCaSms, 7, 2, 1 }; // (an item counts for two tiles more; with 1, 2, 3: 31.0, 29.8, 31.1 us for 16 trees of 64 rows, 41.7, 38.5, 41.2 for four; at least one tile a CTA: with two 18.3 instead of 16.7 for 1000 tokens)
    const int tiles = row_tiles(rows);
    return { false, 8 * tiles, kCaSms * ca_ctas_per_sm(head_dim, tiles) * kCaWarps, 4, kCaExtra, ca_min_quota(tiles) };
}

static bool attention_shape_valid(const abq_kv_cache &c, int batch, int n, int q_heads)
{
    // the grid of the joining kernel and 32-bit indexes of granules bound the sizes
    return kv_cache_valid(c) && batch >= 0 && n >= 1 && n <= 64 && q_heads > 0 && q_heads % c.kv_heads == 0 && q_heads <= 65536 &&
           (long long)c.num_pages * c.kv_heads * (c.page_size / 16) < (1ll << 31) && (long long)batch * n * q_heads < (1ll << 31);
}

} // namespace abq

extern "C" size_t abq_cache_attention_workspace_bytes(const abq_kv_cache *cache, int batch, int rows_per_seq, int q_heads)
{
    using namespace abq;
    if (!cache || !attention_shape_valid(*cache, batch, rows_per_seq, q_heads))
        return 0;
    const int rows = rows_per_seq * (q_heads / cache->kv_heads);
    const CaPlan plan = ca_plan(rows, cache->head_dim);
    return (size_t)2 * plan.most_runs * std::min(rows, plan.block) * (cache->head_dim + 2) * sizeof(float);
}

extern "C" abq_status abq_cache_attention(const abq_cache_attention_params *p, abq_stream_t stream)
{
    using namespace abq;
    if (!p || !attention_shape_valid(p->cache, p->batch, p->rows_per_seq, p->q_heads) || !p->cache.data || (reinterpret_cast<uintptr_t>(p->cache.data) & 15))
        return ABQ_ERR_INVALID_ARG;
    if (p->batch == 0)
        return ABQ_OK;
    if (!half_rows_valid(p->q, p->q_stride, p->q_head_stride) || !half_rows_valid(p->out, p->out_stride, p->out_head_stride) || !p->block_table || p->table_stride <= 0 ||
        !p->seq_lens || ((reinterpret_cast<uintptr_t>(p->block_table) | reinterpret_cast<uintptr_t>(p->seq_lens) | reinterpret_cast<uintptr_t>(p->status_word)) & 3) ||
        (reinterpret_cast<uintptr_t>(p->tree) & 7) || !(p->scale - p->scale == 0.f))
        return ABQ_ERR_INVALID_ARG;
    if (p->out == p->q && (p->out_stride != p->q_stride || p->out_head_stride != p->q_head_stride))
        return ABQ_ERR_INVALID_ARG;
    if (!p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 15) ||
        p->workspace_bytes < abq_cache_attention_workspace_bytes(&p->cache, p->batch, p->rows_per_seq, p->q_heads))
        return ABQ_ERR_WORKSPACE;
    CacheAttnArgs a = {};
    a.data = reinterpret_cast<const uint8_t *>(p->cache.data);
    a.q = reinterpret_cast<const uint8_t *>(p->q);
    a.out = reinterpret_cast<uint8_t *>(p->out);
    a.q_stride = 2 * p->q_stride, a.q_head_stride = 2 * p->q_head_stride, a.out_stride = 2 * p->out_stride, a.out_head_stride = 2 * p->out_head_stride;
    a.table = p->block_table, a.seq_lens = p->seq_lens, a.tree = p->tree, a.part = reinterpret_cast<float *>(p->workspace), a.status = p->status_word;
    a.num_pages = p->cache.num_pages, a.page_granules = p->cache.page_size / 16, a.kv_heads = p->cache.kv_heads, a.batch = p->batch, a.n = p->rows_per_seq;
    a.group = p->q_heads / p->cache.kv_heads, a.table_stride = p->table_stride;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.page_magic = ((1ull << 34) + a.page_granules - 1) / a.page_granules;
    const int rows = a.n * a.group;
    const CaPlan plan = ca_plan(rows, p->cache.head_dim);
    a.row_blocks = (rows + plan.block - 1) / plan.block;
    a.slot_rows = std::min(rows, plan.block);
    a.unit_log2 = plan.unit_log2, a.extra = plan.extra, a.min_quota = plan.min_quota;
    // the longest sequences that the tables can hold bound the work; real lengths are read on the device
    const long long units = (((long long)a.table_stride * p->cache.page_size + (1 << a.unit_log2) - 1) >> a.unit_log2) + a.extra;
    const long long most = (long long)a.batch * a.kv_heads * a.row_blocks * units;
    a.runs = (int)std::min<long long>((most + a.min_quota - 1) / a.min_quota, plan.most_runs);
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int D = p->cache.head_dim, bits = p->cache.bits;
    const bool bf16 = p->cache.half_type == ABQ_HALF_BF16;
    const cudaError_t e = plan.tile        ? launch_cache_attention_tile(a, D, bits, bf16, s)
                          : plan.block == 8 ? launch_cache_attention<1>(a, D, bits, bf16, s)
                                            : launch_cache_attention<2>(a, D, bits, bf16, s);
    if (e != cudaSuccess) {
        set_last_cuda_error(e);
        return ABQ_ERR_CUDA;
    }
    return ABQ_OK;
}
