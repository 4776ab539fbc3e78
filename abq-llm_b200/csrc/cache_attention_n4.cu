// cache_attention kernels for 32 query rows a block (see cache_attention.cuh)
#include "cache_attention_launch.cuh"

namespace abq {
template cudaError_t launch_cache_attention<4>(const CacheAttnArgs &, int head_dim, int bits, bool bf16, cudaStream_t stream);
}
