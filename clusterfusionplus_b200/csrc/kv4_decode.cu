// Attention over the 4-bit cache for few query rows a request: single tokens, grouped heads, a few drafted tokens.
//
// What bounds it is reading the cache: 1.25 bytes a (key, value) pair of elements against 4 flops for each query row, so
// every byte is loaded once for up to 8 (or 16) query rows and everything else has to fit under the load: at 6.5 TB/s an SM
// receives a tile of 16 tokens (2560 bytes at head_dim 128) every ~110 clocks, in which its four schedulers issue ~450
// warp instructions.  Unpacking 4096 codes to fp16 the usual way would take most of them, so no code is ever converted:
//  - a code masked out of its word, w & 0x000f000f or w & 0x00f000f0, IS a pair of fp16 numbers, code * 2^-24 or code *
//    2^-20 (subnormals, which the matrix instructions take at full rate).  The factor of 16 between the two is put
//    into the query (exactly, below) and into the result; 2^24 goes into the fp32 factor of the softmax.
//  - keys: S^T = K Q^T with the codes as the 16-row operand, 32 dims (one group) at a time from a zero accumulator, then one fp32
//    multiply-add by the group's scale.  The minima contribute sum_g m_g (sum of q over group g): one more matrix instruction, the
//    query sums as two fp16 numbers each (hi + lo, 22 bits).  Scores are exact to fp32's rounding.
//  - values: O^T = V^T P^T, again codes as the 16-row operand (two tokens in one word's halves, so no re-pairing).  P is rounded to
//    fp16, transposed, and multiplied by the groups' scales two tokens at a time (a second rounding).  One more instruction takes the
//    minima and a row of ones times the same P: sum p m of every group and the softmax's denominator, fp32 sums of the P that the
//    numerators use.
// Queries are scaled by a power of two to at most 2^10 before they become fp16: exact for fp16 and bf16 inputs of any size
// down to 2^-20 of their row's largest, off by less than 2^-30 of it below.  Probabilities are kept within (0, 4] (the running maximum is
// two binary steps low) so that their product with a scale of up to 8734 (the widest fp16 range / 15) fits fp16 and small
// scales keep their bits.
//
// The work of one (request, cached head) is dealt out tile by tile to the warps of a cluster of up to 8 CTAs, each warp streaming its tiles
// through its own ring of shared memory by cp.async.  The partial results meet in distributed shared memory in a fixed
// order: no workspace, one launch, the same bits every time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kv4_attention.h"
#include "kv4_layout.cuh"
#include "mma.cuh"

namespace cfb {
namespace {

constexpr int W = 4;                 // warps of a CTA
constexpr int STAGES = 4;            // tiles of a warp's ring
constexpr float LOWEST = -3.0e38f;   // reference of a result without tokens: finite, so that no difference of infinities is formed

template <class T> __device__ __forceinline__ float2 to_float2(uint32_t v);
template <> __device__ __forceinline__ float2 to_float2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
template <> __device__ __forceinline__ float2 to_float2<__nv_bfloat16>(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // e in -126 .. 127

// N consecutive 32-bit words of shared memory (4 N-byte aligned for N = 1, 2, 4)
template <int N> __device__ __forceinline__ void load_words(uint32_t (&x)[N], const uint8_t* p) {
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        x[0] = v.x, x[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
    }
}

// N consecutive fp16 numbers as floats (2 N-byte aligned for even N)
template <int N> __device__ __forceinline__ void load_halves(float (&x)[N], const uint8_t* p) {
    if constexpr (N % 2 == 0) {
        uint32_t w[N / 2];
        load_words<N / 2>(w, p);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = __half2float(*reinterpret_cast<const __half*>(p + 2 * i));
    }
}

// word i: the i-th fp16 numbers at a (low half) and at b
template <int N> __device__ __forceinline__ void pair_halves(uint32_t (&x)[N], const uint8_t* a, const uint8_t* b) {
    if constexpr (N % 2 == 0) {
        uint32_t u[N / 2], v[N / 2];
        load_words<N / 2>(u, a);
        load_words<N / 2>(v, b);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            x[2 * i] = __byte_perm(u[i], v[i], 0x5410);
            x[2 * i + 1] = __byte_perm(u[i], v[i], 0x7632);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = *reinterpret_cast<const uint16_t*>(a + 2 * i) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(b + 2 * i)) << 16;
    }
}

__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
    const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&y);
}

// 0xffff in each half that holds a finite fp16 number, else 0
__device__ __forceinline__ uint32_t finite_halves(uint32_t x) {
    const uint32_t over = (((x & 0x7fff7fffu) + 0x04000400u) >> 15) & 0x00010001u;  // 1: exponent all ones
    return ~(over * 0xffffu);
}

// G groups of 32 dims, NT tiles of 8 query rows
template <class T, int G, int NT>
__global__ void __launch_bounds__(32 * W) kv4_few_kernel(const Kv4AttnArgs a, int cluster) {
    constexpr int TB = kv4_tile_bytes(G), DP = 32 * G, COLS = 8 * NT, LINE = DP + 4;
    constexpr int PAIRS = (G + 1) / 2;
    extern __shared__ __align__(16) uint8_t smem[];  // the rings, later the warps' partial results
    __shared__ float part[COLS][LINE];               // this CTA's partial result: DP numerators, maximum, denominator

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g8 = lane >> 2, t = lane & 3;
    const int rank = cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const long long item = blockIdx.x / cluster;
    const int b = static_cast<int>(item / a.kv_heads), kvh = static_cast<int>(item % a.kv_heads);
    const int per = a.heads / a.kv_heads, tiles_a_page = a.page / KV4_TILE;
    int first = b, n = 1;
    if (a.qo_indptr) {
        first = a.qo_indptr[b];
        n = first < 0 ? 0 : min(a.qo_indptr[b + 1], static_cast<int>(a.rows)) - first;
    }
    const int rows = n > 0 ? n * per : 0;  // at most rows * heads of the call: fits
    const long long cap = a.table_width * a.page;
    const long long before = static_cast<long long>(a.kv_lens[b]) - n;  // tokens ahead of the request's queries
    const int* table = a.table + b * a.table_stride;

    for (int r0 = blockIdx.y * COLS; r0 < rows; r0 += gridDim.y * COLS) {
        // ---- queries: B operands, and what the columns of S^T need
        uint32_t qa[NT][G][2], qb[NT][G][2], qm[NT];
        float factor[NT][2];
        int last[NT][2];  // the last token that a column's query sees (before the cap), -1 for none
        int all_see = 0x7fffffff, most = -1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = r0 + nt * 8 + g8;
            const bool real = r < rows;
            float q[G][8], top = 0.f;
            if (real) {
                const T* src = static_cast<const T*>(a.query) + static_cast<long long>(first + r / per) * a.q_ts + (kvh * per + r % per) * a.q_hs;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const int dim = 32 * g + 8 * t;
                    uint4 raw = make_uint4(0, 0, 0, 0);
                    if (dim < a.D) raw = *reinterpret_cast<const uint4*>(src + dim);
                    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 f = to_float2<T>(words[i]);
                        q[g][2 * i] = f.x, q[g][2 * i + 1] = f.y;
                        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                }
            } else {
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int i = 0; i < 8; ++i) q[g][i] = 0.f;
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100);  // 2^e <= top < 2^(e + 1)
            const float up = power_of_two(min(9 - e, 127));
            float sums[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                sums[g] = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    q[g][i] *= up;
                    sums[g] += q[g][i];
                }
                qa[nt][g][0] = pack_half2(q[g][0], q[g][4]);
                qa[nt][g][1] = pack_half2(q[g][2], q[g][6]);
                qb[nt][g][0] = pack_half2(q[g][1] * 0.0625f, q[g][5] * 0.0625f);
                qb[nt][g][1] = pack_half2(q[g][3] * 0.0625f, q[g][7] * 0.0625f);
                sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 1);
                sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 2);
            }
            qm[nt] = 0;  // row pair t of the minima's product: sums of groups 2 j, 2 j + 1 rounded (t = j), and what the rounding left (t = j + PAIRS)
#pragma unroll
            for (int j = 0; j < PAIRS; ++j) {
                const float x = sums[2 * j], y = 2 * j + 1 < G ? sums[2 * j + 1] : 0.f;
                const float xh = __half2float(__float2half_rn(x)), yh = __half2float(__float2half_rn(y));
                if (t == j) qm[nt] = pack_half2(x, y);
                if (t == j + PAIRS) qm[nt] = pack_half2(x - xh, y - yh);
            }
            // fp32 factor of a column's scores: 2^24 of the codes, the query's power of two, the softmax scale in binary logarithms
            const float f = fminf(fmaxf(a.scale_log2 * 16777216.f * power_of_two(e - 9), -3.4e38f), 3.4e38f);
            const long long see = before + r / per;
            const int end = real ? static_cast<int>(min(see, cap - 1)) : -1;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                factor[nt][c] = __shfl_sync(0xffffffffu, f, (2 * t + c) * 4);
                last[nt][c] = __shfl_sync(0xffffffffu, end < 0 ? -1 : end, (2 * t + c) * 4);
            }
            if (real) {
                most = max(most, end);
                all_see = min(all_see, end);
            }
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            all_see = min(all_see, __shfl_xor_sync(0xffffffffu, all_see, o));
        }

        // ---- this warp's tiles: unit, unit + units, ...
        const int units = cluster * W, unit = rank * W + warp;
        const int tiles = most < 0 ? 0 : most / KV4_TILE + 1;
        const int mine = tiles > unit ? (tiles - unit + units - 1) / units : 0;
        uint8_t* ring = smem + warp * STAGES * TB;
        int col = unit / tiles_a_page, in_page = unit % tiles_a_page, issued = 0;
        const int step_col = units / tiles_a_page, step_in = units % tiles_a_page;
        int held = mine > 0 ? table[col] : -1;
        unsigned there = 0;  // bit s: the tile in stage s exists (its page lies in the cache)
        auto issue = [&] {
            if (issued < mine) {
                const int stage = issued % STAGES;
                const bool ok = held >= 0 && held < a.pages;
                there = (there & ~(1u << stage)) | (static_cast<unsigned>(ok) << stage);
                if (ok) {
                    const uint8_t* src = a.cache + ((static_cast<long long>(held) * a.kv_heads + kvh) * tiles_a_page + in_page) * TB;
                    const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(ring + stage * TB));
#pragma unroll
                    for (int i = 0; i < (TB / 16 + 31) / 32; ++i)
                        if (i * 32 + lane < TB / 16) cp_async_16(dst + (i * 32 + lane) * 16, src + (i * 32 + lane) * 16);
                } else if (lane == 0) {
                    atomicCAS(a.status, 0, ST_BAD_SLOT);
                }
                ++issued;
                col += step_col, in_page += step_in;
                if (in_page >= tiles_a_page) in_page -= tiles_a_page, ++col;
                held = issued < mine ? table[col] : -1;
            }
            cp_async_commit();
        };
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) issue();

        // numerators in units of 2^-24 and 2^-20; rows of `low`: group g's sum of p times the minimum (row g), the sum of p (row G)
        float o[NT][2 * G][4], low[NT][4], m[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 2 * G; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[nt][i][j] = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) low[nt][j] = 0.f;
            m[nt][0] = m[nt][1] = 0.f;
        }
        bool first_tile = true;

        for (int i = 0; i < mine; ++i) {
            cp_async_wait<STAGES - 2>();
            __syncwarp();
            const int stage = i % STAGES, token = (unit + i * units) * KV4_TILE;
            const bool ok = (there >> stage) & 1;
            issue();  // into the stage that the whole warp is done with
            if (!ok) continue;
            const uint8_t* tile = ring + stage * TB;
            const uint8_t* par0 = tile + 512 * G + g8 * 8 * G;  // parameters of tokens g8 and g8 + 8
            const uint8_t* par1 = par0 + 64 * G;

            // ---- scores
            float x[NT][4];
            {
                uint32_t low0 = 0, low1 = 0;
                if constexpr (G % 2 == 0) {
                    low0 = *reinterpret_cast<const uint32_t*>(par0 + 2 * G + 4 * (t % PAIRS));
                    low1 = *reinterpret_cast<const uint32_t*>(par1 + 2 * G + 4 * (t % PAIRS));
                } else {
                    const int j = t % PAIRS;
                    low0 = *reinterpret_cast<const uint16_t*>(par0 + 2 * G + 4 * j);
                    low1 = *reinterpret_cast<const uint16_t*>(par1 + 2 * G + 4 * j);
                    if (2 * j + 1 < G) {
                        low0 |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(par0 + 2 * G + 4 * j + 2)) << 16;
                        low1 |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(par1 + 2 * G + 4 * j + 2)) << 16;
                    }
                }
                if (2 * PAIRS < 4 && t >= 2 * PAIRS) low0 = low1 = 0;
                uint32_t k0[G], k1[G];
                float s0[G], s1[G];
                load_words<G>(k0, tile + g8 * 16 * G + t * 4 * G);
                load_words<G>(k1, tile + (g8 + 8) * 16 * G + t * 4 * G);
                load_halves<G>(s0, par0);
                load_halves<G>(s1, par1);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma_16816_zero(x[nt], low0, low1, 0u, 0u, qm[nt], 0u);
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[nt][j] *= 5.9604644775390625e-08f;  // 2^-24: the codes' unit
                }
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const uint32_t h0 = k0[g] >> 8, h1 = k1[g] >> 8;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float c[4];
                        mma_16816_zero(c, k0[g] & 0x000f000fu, k1[g] & 0x000f000fu, h0 & 0x000f000fu, h1 & 0x000f000fu, qa[nt][g][0], qa[nt][g][1]);
                        mma_16816(c, k0[g] & 0x00f000f0u, k1[g] & 0x00f000f0u, h0 & 0x00f000f0u, h1 & 0x00f000f0u, qb[nt][g][0], qb[nt][g][1]);
                        x[nt][0] = fmaf(s0[g], c[0], x[nt][0]);
                        x[nt][1] = fmaf(s0[g], c[1], x[nt][1]);
                        x[nt][2] = fmaf(s1[g], c[2], x[nt][2]);
                        x[nt][3] = fmaf(s1[g], c[3], x[nt][3]);
                    }
                }
            }
            // ---- softmax: x becomes the binary logarithm of p, at most 2 above the running reference m
            const bool whole = token + KV4_TILE - 1 <= all_see;
            bool rise = first_tile;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[nt][j] = fmaf(x[nt][j], factor[nt][j & 1], -m[nt][j & 1]);
                    if (!whole && token + g8 + (j >> 1) * 8 > last[nt][j & 1]) x[nt][j] = -INFINITY;
                }
                rise |= fmaxf(fmaxf(x[nt][0], x[nt][2]), fmaxf(x[nt][1], x[nt][3])) > 2.f;
            }
            if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float top = fmaxf(x[nt][c], x[nt][c + 2]);
#pragma unroll
                        for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                        // a column's first tile sets its reference; one that sees nothing of its first tile sees nothing of later ones
                        const float up = first_tile ? (top == -INFINITY ? 0.f : top - 2.f) : fmaxf(top - 2.f, 0.f);
                        m[nt][c] += up;
                        x[nt][c] -= up;
                        x[nt][c + 2] -= up;
                        const float keep = first_tile ? 1.f : ex2(-up);
                        low[nt][c] *= keep;
#pragma unroll
                        for (int q = 0; q < 2 * G; ++q) o[nt][q][c] *= keep, o[nt][q][c + 2] *= keep;
                    }
                first_tile = false;
            }
            // ---- values: scales of tokens 2 t, 2 t + 1 (sa) and 2 t + 8, 2 t + 9 (sb), group by group; minima likewise, of group g8
            const uint8_t* pv = tile + 512 * G + 2 * t * 8 * G + 4 * G;
            uint32_t sa[G], sb[G], ma = 0, mb = 0;
            pair_halves<G>(sa, pv, pv + 8 * G);
            pair_halves<G>(sb, pv + 64 * G, pv + 72 * G);
            if (g8 < G) {
                const uint8_t* pm = pv + 2 * G + 2 * g8;
                ma = *reinterpret_cast<const uint16_t*>(pm) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(pm + 8 * G)) << 16;
                mb = *reinterpret_cast<const uint16_t*>(pm + 64 * G) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(pm + 72 * G)) << 16;
            } else if (g8 == G) ma = mb = 0x3c003c00u;  // ones
            uint32_t v0[G], v1[G];
            load_words<G>(v0, tile + 256 * G + lane * 4 * G);
            load_words<G>(v1, tile + 384 * G + lane * 4 * G);
            if (!whole) {
                // What a query does not see must not reach its sums, not even times 0: a token with a parameter that is not finite is taken
                // out here, and the sums of those that do see it become NaN in that group.
                const uint32_t ra = finite_halves(ma), rb = finite_halves(mb);
                uint32_t bad = 0;  // of group g8: tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const uint32_t fa = finite_halves(sa[g]), fb = finite_halves(sb[g]);
                    // the lanes of column t that hold group g's minima say whether those are finite
                    const uint32_t ga = __shfl_sync(0xffffffffu, ra, g * 4 + t) & fa, gb = __shfl_sync(0xffffffffu, rb, g * 4 + t) & fb;
                    sa[g] &= ga, sb[g] &= gb;
                    if (g8 == g) bad = (~ga & 1u) | (~(ga >> 16) & 1u) << 1 | (~gb & 1u) << 8 | (~(gb >> 16) & 1u) << 9;
                }
                if (g8 < G) ma &= ra, mb &= rb;
                if (__any_sync(0xffffffffu, bad != 0)) {
                    uint32_t tokens = bad << (2 * t);  // bit k: token k of the tile, over the four lanes of a row
                    tokens |= __shfl_xor_sync(0xffffffffu, tokens, 1);
                    tokens |= __shfl_xor_sync(0xffffffffu, tokens, 2);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int see = last[nt][c] - token;  // tokens 0 .. see of the tile
                            const uint32_t seen = see < 0 ? 0u : see >= 15 ? 0xffffu : (2u << see) - 1u;
                            if (g8 < G && (tokens & seen)) low[nt][c] = __int_as_float(0x7fffffff);
                        }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint32_t p0 = transpose_8x8(pack_half2(ex2(x[nt][0]), ex2(x[nt][1]))), p1 = transpose_8x8(pack_half2(ex2(x[nt][2]), ex2(x[nt][3])));
                mma_16816(low[nt], ma, 0u, mb, 0u, p0, p1);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const uint32_t h0 = v0[g] >> 8, h1 = v1[g] >> 8, q0 = mul_half2(p0, sa[g]), q1 = mul_half2(p1, sb[g]);
                    mma_16816(o[nt][2 * g], v0[g] & 0x000f000fu, h0 & 0x000f000fu, v1[g] & 0x000f000fu, h1 & 0x000f000fu, q0, q1);
                    mma_16816(o[nt][2 * g + 1], v0[g] & 0x00f000f0u, h0 & 0x00f000f0u, v1[g] & 0x00f000f0u, h1 & 0x00f000f0u, q0, q1);
                }
            }
        }
        cp_async_wait<0>();

        // ---- the warps' results, then the CTAs': columns of numerators, maximum and denominator
        __syncthreads();  // the rings are free
        float* merge = reinterpret_cast<float*>(smem) + warp * COLS * LINE;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float* line = merge + (nt * 8 + 2 * t + c) * LINE;
                const float sum = __shfl_sync(0xffffffffu, low[nt][c], G * 4 + t);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const float least = __shfl_sync(0xffffffffu, low[nt][c], g * 4 + t);
                    float4 y;
                    y.x = fmaf(o[nt][2 * g][c], 16777216.f, least);
                    y.y = fmaf(o[nt][2 * g + 1][c], 1048576.f, least);
                    y.z = fmaf(o[nt][2 * g][c + 2], 16777216.f, least);
                    y.w = fmaf(o[nt][2 * g + 1][c + 2], 1048576.f, least);
                    *reinterpret_cast<float4*>(line + 32 * g + 4 * g8) = y;
                }
                if (g8 == 0) line[DP] = sum == 0.f ? LOWEST : m[nt][c], line[DP + 1] = sum;  // nothing seen: no reference either
            }
        __syncthreads();
        const int cols = min(COLS, rows - r0);
        const float* all = reinterpret_cast<const float*>(smem);
        for (int e = threadIdx.x; e < cols * DP; e += 32 * W) {
            const int c = e / DP, d = e % DP;
            float top = LOWEST, num = 0.f, den = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) top = fmaxf(top, all[(w * COLS + c) * LINE + DP]);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float* line = all + (w * COLS + c) * LINE;
                const float k = ex2(line[DP] - top);
                num = fmaf(k, line[d], num);
                den = fmaf(k, line[DP + 1], den);
            }
            part[c][d] = num;
            if (d == 0) part[c][DP] = top, part[c][DP + 1] = den;
        }
        if (cluster > 1) cluster_sync_all();
        else __syncthreads();
        for (int e = rank * 32 * W + threadIdx.x; e < cols * DP; e += cluster * 32 * W) {
            const int c = e / DP, d = e % DP;
            float num, den;
            if (cluster == 1) {
                num = part[c][d];
                den = part[c][DP + 1];
            } else {
                float top = LOWEST;
                num = den = 0.f;
                for (int k = 0; k < cluster; ++k) top = fmaxf(top, cluster_ld_float(cluster_map(&part[c][DP], k)));
                for (int k = 0; k < cluster; ++k) {
                    const float f = ex2(cluster_ld_float(cluster_map(&part[c][DP], k)) - top);
                    num = fmaf(f, cluster_ld_float(cluster_map(&part[c][d], k)), num);
                    den = fmaf(f, cluster_ld_float(cluster_map(&part[c][DP + 1], k)), den);
                }
            }
            if (d < a.D) {
                const int r = r0 + c;
                // no token seen: zeros; a NaN stays one
                static_cast<T*>(a.out)[(static_cast<long long>(first + r / per) * a.heads + kvh * per + r % per) * a.D + d] = from_float<T>(den == 0.f ? 0.f : num / den);
            }
        }
        if (cluster > 1) cluster_sync_all();  // until here the other CTAs read this one's part
        else __syncthreads();
    }
}

template <class T, int G, int NT> cudaError_t launch(const Kv4AttnArgs& a, long long max_q_len, cudaStream_t st) {
    constexpr int COLS = 8 * NT;
    constexpr int ring = W * STAGES * kv4_tile_bytes(G), merge = W * COLS * (32 * G + 4) * 4;
    constexpr int smem = ring > merge ? ring : merge;
    const long long items = static_cast<long long>(a.batch) * a.kv_heads;
    const long long q_tiles = (max_q_len * (a.heads / a.kv_heads) + COLS - 1) / COLS;
    const long long tiles = (a.table_width * a.page + KV4_TILE - 1) / KV4_TILE;
    // as many CTAs to a (request, head) as fill the GPU (4 to an SM), but at least four tiles to a warp
    int cluster = 1;
    while (cluster < 8 && items * q_tiles * cluster < 4 * 148 && tiles >= 8 * W * cluster) cluster *= 2;
    auto kernel = kv4_few_kernel<T, G, NT>;
    if (smem + merge / W > 48 * 1024) {  // with the static part
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(items * cluster), static_cast<unsigned>(q_tiles < 65535 ? q_tiles : 65535));
    cfg.blockDim = dim3(32 * W);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a, cluster);
}

template <class T, int G> cudaError_t by_rows(const Kv4AttnArgs& a, long long max_q_len, cudaStream_t st) {
    return max_q_len * (a.heads / a.kv_heads) <= 8 ? launch<T, G, 1>(a, max_q_len, st) : launch<T, G, 2>(a, max_q_len, st);
}

template <class T> cudaError_t by_groups(const Kv4AttnArgs& a, long long max_q_len, cudaStream_t st) {
    switch (kv4_groups(a.D)) {
        case 1: return by_rows<T, 1>(a, max_q_len, st);
        case 2: return by_rows<T, 2>(a, max_q_len, st);
        case 3: return by_rows<T, 3>(a, max_q_len, st);
        default: return by_rows<T, 4>(a, max_q_len, st);
    }
}

}  // namespace

cudaError_t kv4_attention_few(const Kv4AttnArgs& a, bool bf16, long long max_q_len, cudaStream_t st) {
    return bf16 ? by_groups<__nv_bfloat16>(a, max_q_len, st) : by_groups<__half>(a, max_q_len, st);
}

}  // namespace cfb
