// Layout of the paged cache held in 4 bits, shared by the kernels that write it and those that read it, and what the latter share besides.
//
// The cache is [pages][kv_heads][page_size][40 G] bytes, G = ceil(head_dim / 32) groups of 32 values, page_size a multiple
// of 16.  The bytes of one (page, head) are page_size / 16 tiles of 16 tokens (a tile is what one warp feeds to the matrix
// instructions at a time), each of 640 G bytes:
//   key codes    [16 tokens][4 t][G g] 32-bit words     nibble n (0..7) of word (t, g) is dim 32 g + 8 t + n
//   value codes  [2 h][8 c][4 t][G g] 32-bit words      low half token 8 h + 2 t, high half token 8 h + 2 t + 1;
//                                                       nibble n (0..3) of a half is dim 32 g + 4 c + n
//   parameters   [16 tokens][key scales G | key minima G | value scales G | value minima G] fp16
// A value is code * scale + minimum, code 0..15.  Lane (4 c + t) of a warp finds in these words exactly the operands that
// it has to hold for mma.m16n8k16, in 16-byte pieces that the warp reads without gaps; and a token's codes are whole
// 16-bit halves, so that tokens can be written one by one, by different warps, without reading first.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace cfb {

constexpr int KV4_TILE = 16;       // tokens
constexpr int KV4_GROUP = 32;      // values that share a scale and a minimum
constexpr int KV4_MAX_DIM = 128;

__host__ __device__ constexpr int kv4_groups(int dim) { return (dim + KV4_GROUP - 1) / KV4_GROUP; }
__host__ __device__ constexpr int kv4_tile_bytes(int G) { return 640 * G; }

// byte offsets inside a tile
__host__ __device__ constexpr int kv4_key_half(int G, int token, int dim) {  // the 16-bit half that holds dims dim .. dim + 3 (dim a multiple of 4)
    const int g = dim / 32, e = dim % 32;
    return token * 16 * G + (e / 8) * 4 * G + g * 4 + (e % 8) / 2;
}
__host__ __device__ constexpr int kv4_value_half(int G, int token, int dim) {
    const int g = dim / 32, c = (dim % 32) / 4, h = token / 8, t = (token % 8) / 2;
    return 256 * G + (((h * 8 + c) * 4 + t) * G + g) * 4 + (token & 1) * 2;
}
__host__ __device__ constexpr int kv4_param(int G, int token, int which, int g) {  // which: 0 key scale, 1 key minimum, 2 value scale, 3 value minimum
    return 512 * G + token * 8 * G + (which * G + g) * 2;
}

// ---- queries, as both attention kernels take them
template <class T> __device__ __forceinline__ float2 to_float2(uint32_t v);
template <> __device__ __forceinline__ float2 to_float2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
template <> __device__ __forceinline__ float2 to_float2<__nv_bfloat16>(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // e in -126 .. 127
// A row of queries whose largest is `top` becomes fp16 numbers of at most 2^10 by the power of two query_scaling(e): 2^e <= top < 2^(e + 1)
__device__ __forceinline__ int query_exponent(float top) { return max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100); }
__device__ __forceinline__ float query_scaling(int e) { return power_of_two(min(9 - e, 127)); }

// status word of this unit on the current device (CF status 8: a page or slot outside the cache)
constexpr int ST_BAD_SLOT = 8;

}  // namespace cfb
