// The quantised key/value cache: where a token's codes and parameters lie (include/abq_b200.h describes the layout), and the 16-bit types.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "abq_common.cuh"

namespace abq {

constexpr int kGranuleTokens = 16;

__host__ __device__ constexpr int kv_row_bytes(int head_dim, int bits) { return head_dim * bits / 8; }
__host__ __device__ constexpr int kv_granule_bytes(int row_bytes) { return 32 * row_bytes + 128; }
__host__ __device__ constexpr int kv_param_offset(int row_bytes, int part) { return 32 * row_bytes + 64 * part; } // part 0: keys, 1: values

// Offset of byte `byte` of token t's row inside the 16 rows of a part.  A 128-byte line holds 1, 2 or 4 rows; its 16-byte pieces are
// exchanged so that the eight (LDS.128) or sixteen (LDS.64) lanes of a shared-memory phase, which read the same pieces of tokens one or four
// apart, touch all 32 banks once.
template <int RB>
__host__ __device__ __forceinline__ int kv_place(int t, int byte)
{
    static_assert(RB == 128 || RB == 64 || RB == 32, "row bytes");
    const int at = t * RB + byte, line = at >> 7;
    const int turn = RB == 128 ? ((line & 3) * 2) ^ ((line >> 2 & 1) * 4) : RB == 64 ? (line & 3) * 2 : (line & 1) * 4;
    return at ^ (turn << 4);
}

__device__ __forceinline__ float half_bits_to_float(uint32_t bits, bool bf16)
{
    return bf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((unsigned short)bits));
}
__device__ __forceinline__ float2 half_pair_to_float(uint32_t pair, bool bf16)
{
    if (bf16)
        return make_float2(__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2 *>(&pair));
}
__device__ __forceinline__ uint32_t float_pair_to_half(float a, float b, bool bf16)
{
    if (bf16) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
}

} // namespace abq
