// Launches of the attention over the cache and of the kernel that joins its pieces.
#pragma once
#include "cache_attention.cuh"

namespace abq {

template <typename Kernel>
cudaError_t launch_chained(Kernel kern, unsigned grid, unsigned block, size_t smem, cudaStream_t stream, const CacheAttnArgs &args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args);
}

template <int D, int BITS, int NT>
cudaError_t launch_cache_attention_as(const CacheAttnArgs &args, cudaStream_t stream)
{
    static thread_local SmemOptIn opted;
    constexpr int smem = CaShape<D, BITS, NT>::kSmem;
    auto kern = cache_attention_kernel<D, BITS, NT>;
    cudaError_t e = opted.ensure(kern, smem);
    if (e == cudaSuccess)
        e = launch_chained(kern, args.ctas, kCaThreads, smem, stream, args);
    if (e == cudaSuccess)
        e = launch_chained(cache_attention_combine_kernel<D, NT>, (unsigned)(args.batch * args.kv_heads * args.row_blocks), kCaThreads, 0, stream, args);
    return e;
}

template <int NT>
cudaError_t launch_cache_attention(const CacheAttnArgs &args, int head_dim, int bits, cudaStream_t stream)
{
    if (head_dim == 128)
        return bits == 8 ? launch_cache_attention_as<128, 8, NT>(args, stream) : launch_cache_attention_as<128, 4, NT>(args, stream);
    return bits == 8 ? launch_cache_attention_as<64, 8, NT>(args, stream) : launch_cache_attention_as<64, 4, NT>(args, stream);
}

} // namespace abq
