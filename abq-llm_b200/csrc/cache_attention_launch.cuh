// Launches of the attention over the cache and of the kernel that joins its pieces.
#pragma once
#include "cache_attention.cuh"

namespace abq {

template <typename Kernel, typename... Args>
cudaError_t launch_chained(Kernel kern, dim3 grid, size_t smem, cudaStream_t stream, const Args &...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kCaThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <int D, bool BF16>
cudaError_t launch_cache_attention_combine(const CacheAttnArgs &args, int block_rows, cudaStream_t stream)
{
    constexpr int kGroups = kCaThreads / (D / 8);
    // rows of a block at a time: few (the other groups of threads take pieces in turn) where the items alone do not fill the GPU
    const long long items = (long long)args.batch * args.kv_heads * args.row_blocks;
    int rows = 1;
    while (rows < args.slot_rows && rows < kGroups && items * args.slot_rows / rows > 4 * kCaSms)
        rows *= 2;
    return launch_chained(cache_attention_combine_kernel<D, BF16>, dim3((unsigned)items, (args.slot_rows + rows - 1) / rows), 0, stream, args, block_rows, rows);
}

template <int D, int BITS, int NT, bool BF16>
cudaError_t launch_cache_attention_as(const CacheAttnArgs &args, cudaStream_t stream)
{
    static thread_local SmemOptIn opted;
    constexpr int smem = CaShape<D, BITS, NT>::kSmem;
    auto kern = cache_attention_kernel<D, BITS, NT, BF16>;
    cudaError_t e = opted.ensure(kern, smem);
    if (e == cudaSuccess)
        e = launch_chained(kern, dim3((args.runs + kCaWarps - 1) / kCaWarps), smem, stream, args);
    return e != cudaSuccess ? e : launch_cache_attention_combine<D, BF16>(args, 8 * NT, stream);
}

template <int NT>
cudaError_t launch_cache_attention(const CacheAttnArgs &args, int head_dim, int bits, bool bf16, cudaStream_t stream)
{
    if (head_dim == 128) {
        if (bits == 8)
            return bf16 ? launch_cache_attention_as<128, 8, NT, true>(args, stream) : launch_cache_attention_as<128, 8, NT, false>(args, stream);
        return bf16 ? launch_cache_attention_as<128, 4, NT, true>(args, stream) : launch_cache_attention_as<128, 4, NT, false>(args, stream);
    }
    if (bits == 8)
        return bf16 ? launch_cache_attention_as<64, 8, NT, true>(args, stream) : launch_cache_attention_as<64, 8, NT, false>(args, stream);
    return bf16 ? launch_cache_attention_as<64, 4, NT, true>(args, stream) : launch_cache_attention_as<64, 4, NT, false>(args, stream);
}

} // namespace abq
