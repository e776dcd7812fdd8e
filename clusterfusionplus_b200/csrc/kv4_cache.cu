// The paged cache held in 4 bits (layout: kv4_layout.cuh): rows written at their slots and read back, and the C entry
// points.  Asymmetric 4-bit codes over groups of 32 values of one token and head:
//   m = fp16(min x), s = fp16((max x - m) / 15), code = clamp(rint((x - m) / s), 0, 15), value = code * s + m
// x in fp32 (clamped to fp16's range, which bf16 exceeds); the codes are computed against the rounded s and m, so the rounding of
// the parameters costs no accuracy but the last step's.  A group that is constant has s = 0 and code 0; one that holds a
// NaN or whose extremes are not finite in the input stores NaN as its scale: it comes back as NaN instead of as numbers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../include/clusterfusion_b200.h"
#include "host_common.h"
#include "kv4_attention.h"
#include "kv4_layout.cuh"

namespace {

using namespace cfb;

__device__ int g_kv4_status = 0;

__device__ __forceinline__ void report_bad_slot() { atomicCAS(&g_kv4_status, 0, ST_BAD_SLOT); }


// Both kernels: half a warp for a (token, head), lane l of the half holds dims 8 l .. 8 l + 7 (16 bytes) of the key and the
// value, four lanes a group.  A warp then moves 2 KB of keys and values with two loads a lane, and the index arithmetic, the
// group reductions (two shuffles) and the parameters' divisions are paid once for 64 values.
constexpr int CT = 256;          // threads of a CTA
constexpr int ITEMS = CT / 16;   // (token, head) pairs of a CTA

// pairs of the 16-bit types
template <class T> struct Two;
template <> struct Two<__half> {
    using P = __half2;
    static constexpr uint32_t INF = 0x04000400u;  // what carries an exponent of all ones into bit 15
    static __device__ __forceinline__ float2 floats(P v) { return __half22float2(v); }
};
template <> struct Two<__nv_bfloat16> {
    using P = __nv_bfloat162;
    static constexpr uint32_t INF = 0x00800080u;
    static __device__ __forceinline__ float2 floats(P v) { return __bfloat1622float2(v); }
};

// Codes of this lane's eight values (raw words, nibble i: value i), scale and minimum of its group of four lanes.  Extremes and the test
// for NaN and infinities work on the 16-bit pairs; codes are rounded by adding 1.5 * 2^23, which leaves them in the low mantissa
// bits (conversions run at a quarter of the rate), and put together by multiply-adds.
template <class T> __device__ __forceinline__ unsigned quantise8(const uint32_t (&raw)[4], bool real, __half* scale, __half* low) {
    using P = typename Two<T>::P;
    const P* p = reinterpret_cast<const P*>(raw);
    const float2 hi2 = Two<T>::floats(__hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]))), lo2 = Two<T>::floats(__hmin2(__hmin2(p[0], p[1]), __hmin2(p[2], p[3])));
    float hi = real ? fminf(fmaxf(hi2.x, hi2.y), 65504.f) : -65504.f, lo = real ? fmaxf(fminf(lo2.x, lo2.y), -65504.f) : 65504.f;
    uint32_t over = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) over |= (raw[i] & 0x7fff7fffu) + Two<T>::INF;
    unsigned bad = real && (over & 0x80008000u);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad |= __shfl_xor_sync(0xffffffffu, bad, o);
    }
    lo = fminf(lo, 65504.f), hi = fmaxf(hi, -65504.f);  // bf16 beyond fp16 on one side only
    const __half m = __float2half_rn(lo);
    const float mf = __half2float(m);
    const __half s = __float2half_rn((hi - mf) / 15.f);
    const float sf = __half2float(s);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(sf));
    unsigned codes = 0;
    if (real && sf > 0.f && !bad) {
        // rint((v - m) / s) by the reciprocal: off by a few 2^-24 of at most 22, which matters only next to a half; there it is divided
        constexpr float MAGIC = 12582912.f;
        const bool wide = sizeof(T) == 2 && Two<T>::INF == 0x00800080u && (lo <= -65504.f || hi >= 65504.f);  // bf16 beyond fp16
        float t[8], off = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 v = Two<T>::floats(p[i]);
            if (wide) v.x = fminf(fmaxf(v.x, -65504.f), 65504.f), v.y = fminf(fmaxf(v.y, -65504.f), 65504.f);
            const float x = (v.x - mf) * r, y = (v.y - mf) * r;
            t[2 * i] = x + MAGIC, t[2 * i + 1] = y + MAGIC;
            off = fmaxf(off, fmaxf(fabsf(x - (t[2 * i] - MAGIC)), fabsf(y - (t[2 * i + 1] - MAGIC))));
        }
        if (off > 0.49999f) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 v = Two<T>::floats(p[i]);
                t[2 * i] = (fminf(fmaxf(v.x, -65504.f), 65504.f) - mf) / sf + MAGIC;
                t[2 * i + 1] = (fminf(fmaxf(v.y, -65504.f), 65504.f) - mf) / sf + MAGIC;
            }
        }
        // (no value is more than half a step below the minimum; a scale that was rounded down to one of fp16's last steps reaches beyond 15)
#pragma unroll
        for (int i = 7; i >= 0; --i) codes = codes * 16 + __float_as_uint(fminf(t[i], MAGIC + 15.f));
        codes -= 0x4b400000u * 0x11111111u;
    }
    *scale = bad ? __ushort_as_half(0x7fff) : s;
    *low = m;
    return codes;
}

// the tile that holds a row, and the row in it
__device__ __forceinline__ long long tile_of(int slot, int head, int heads, int tiles_a_page) {
    const unsigned tile = static_cast<unsigned>(slot) / KV4_TILE, page = tile / tiles_a_page;
    return (static_cast<long long>(page) * heads + head) * tiles_a_page + (tile - page * tiles_a_page);
}

template <class T, int G>
__global__ void __launch_bounds__(CT) kv4_append_kernel(const T* __restrict__ key, const T* __restrict__ value, const int* __restrict__ slot_map,
                                                        uint8_t* __restrict__ cache, unsigned items, int heads, int D, int tiles_a_page, long long slots,
                                                        long long k_ts, long long k_hs, long long v_ts, long long v_hs) {
    const int l = threadIdx.x & 15;
    const unsigned item = blockIdx.x * ITEMS + threadIdx.x / 16;
    const bool there = item < items;
    const unsigned tok = there ? item / heads : 0;
    const int head = there ? static_cast<int>(item - tok * heads) : 0;
    const int slot = there ? slot_map[tok] : -1;
    if (slot >= slots && l == 0) report_bad_slot();
    const bool kept = slot >= 0 && slot < slots;  // a padded row is skipped
    const int dim = 8 * l;
    const bool real = kept && dim < D;
    uint2 k0 = make_uint2(0, 0), k1 = k0, v0 = k0, v1 = k0;  // rows are 8-byte aligned
    if (real) {
        const uint2* kp = reinterpret_cast<const uint2*>(key + tok * k_ts + head * k_hs + dim);
        const uint2* vp = reinterpret_cast<const uint2*>(value + tok * v_ts + head * v_hs + dim);
        k0 = kp[0], k1 = kp[1], v0 = vp[0], v1 = vp[1];
    }
    const uint32_t xk[4] = {k0.x, k0.y, k1.x, k1.y}, xv[4] = {v0.x, v0.y, v1.x, v1.y};
    __half ks, km, vs, vm;
    const unsigned kc = quantise8<T>(xk, real, &ks, &km), vc = quantise8<T>(xv, real, &vs, &vm);
    if (!kept || dim >= 32 * G) return;
    const int row = slot % KV4_TILE, which = l & 3;
    uint8_t* tile = cache + tile_of(slot, head, heads, tiles_a_page) * kv4_tile_bytes(G);
    *reinterpret_cast<uint32_t*>(tile + kv4_key_half(G, row, dim)) = kc;
    *reinterpret_cast<uint16_t*>(tile + kv4_value_half(G, row, dim)) = static_cast<uint16_t>(vc);
    *reinterpret_cast<uint16_t*>(tile + kv4_value_half(G, row, dim + 4)) = static_cast<uint16_t>(vc >> 16);
    *reinterpret_cast<__half*>(tile + kv4_param(G, row, which, l >> 2)) = which == 0 ? ks : which == 1 ? km : which == 2 ? vs : vm;
}

// Eight values: the codes as fp16 numbers 1024 + code two at a time (codes i and i + 4), back to 0 .. 15 exactly, times the scale plus
// the minimum with one rounding (fp16: fused in fp16; bf16: fused in fp32, then rounded)
template <class T> __device__ __forceinline__ uint4 unpack8(unsigned codes, __half s, __half m);
__device__ __forceinline__ void codes_as_halves(unsigned codes, __half2 (&c)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = ((codes >> (4 * i)) & 0x000f000fu) | 0x64006400u;
        c[i] = __hsub2(*reinterpret_cast<const __half2*>(&w), __floats2half2_rn(1024.f, 1024.f));
    }
}
template <> __device__ __forceinline__ uint4 unpack8<__half>(unsigned codes, __half s, __half m) {
    __half2 c[4];
    codes_as_halves(codes, c);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 v = __hfma2(c[i], __half2half2(s), __half2half2(m));
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return make_uint4(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410), __byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632));
}
template <> __device__ __forceinline__ uint4 unpack8<__nv_bfloat16>(unsigned codes, __half s, __half m) {
    __half2 c[4];
    codes_as_halves(codes, c);
    const float sf = __half2float(s), mf = __half2float(m);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(c[i]);
        v[i] = fmaf(f.x, sf, mf);
        v[i + 4] = fmaf(f.y, sf, mf);
    }
    __align__(16) __nv_bfloat162 e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    return *reinterpret_cast<const uint4*>(e);
}

template <class T, int G>
__global__ void __launch_bounds__(CT) kv4_read_kernel(const uint8_t* __restrict__ cache, const int* __restrict__ slot_map, T* __restrict__ key,
                                                      T* __restrict__ value, unsigned items, int heads, int D, int tiles_a_page, long long slots) {
    const int l = threadIdx.x & 15, dim = 8 * l;
    const unsigned item = blockIdx.x * ITEMS + threadIdx.x / 16;
    if (item >= items || dim >= D) return;
    const unsigned tok = item / heads;
    const int head = static_cast<int>(item - tok * heads), slot = slot_map[tok];
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (slot >= 0 && slot < slots) {
        const int row = slot % KV4_TILE, g = l >> 2;
        const uint8_t* tile = cache + tile_of(slot, head, heads, tiles_a_page) * kv4_tile_bytes(G);
        auto par = [&](int which) { return *reinterpret_cast<const __half*>(tile + kv4_param(G, row, which, g)); };
        const unsigned kc = *reinterpret_cast<const uint32_t*>(tile + kv4_key_half(G, row, dim));
        const unsigned vc = *reinterpret_cast<const uint16_t*>(tile + kv4_value_half(G, row, dim)) |
                            static_cast<unsigned>(*reinterpret_cast<const uint16_t*>(tile + kv4_value_half(G, row, dim + 4))) << 16;
        k = unpack8<T>(kc, par(0), par(1));
        v = unpack8<T>(vc, par(2), par(3));
    } else if (slot >= slots && l == 0) {
        report_bad_slot();
    }
    const long long at = static_cast<long long>(item) * D + dim;
    *reinterpret_cast<uint4*>(key + at) = k;
    *reinterpret_cast<uint4*>(value + at) = v;
}

int check_cache(int64_t pages, int64_t kv_heads, int64_t page, int64_t D) {
    if (D < 16 || D > KV4_MAX_DIM || D % 8 != 0) return cf_host_fail(CF_ERR_INVALID, "head_dim %lld must be a multiple of 8 in 16..%d", (long long)D, KV4_MAX_DIM);
    if (page < KV4_TILE || page % KV4_TILE != 0 || page > 65536) return cf_host_fail(CF_ERR_INVALID, "page size %lld must be a multiple of %d, at most 65536", (long long)page, KV4_TILE);
    if (pages < 1 || kv_heads < 1 || kv_heads > 1024 || pages > 0x7fffffff / page)
        return cf_host_fail(CF_ERR_INVALID, "cache of %lld pages of %lld rows, %lld heads (at most 2^31 - 1 rows)", (long long)pages, (long long)page, (long long)kv_heads);
    return CF_OK;
}

template <class F> void with_groups(int D, F f) {
    switch (kv4_groups(D)) {
        case 1: return f(std::integral_constant<int, 1>());
        case 2: return f(std::integral_constant<int, 2>());
        case 3: return f(std::integral_constant<int, 3>());
        default: return f(std::integral_constant<int, 4>());
    }
}

int check_launch(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cf_host_fail(CF_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
    return CF_OK;
}

// Whether 128 query rows of a (request, cached head) shall share each unpacked tile (kv4_prompt.cu) or 16 at a time read the cache for
// themselves (kv4_decode.cu).  The first takes 2.3 us for 128 tokens in each of 148 CTAs and does not divide the tokens among CTAs; the second
// divides them evenly and takes 2 ns for 16 rows x 16 tokens, 8 us at least.  Measured (rows of a (request, head); the second against the
// first): 32 pairs of 2048 tokens 48 rows 44 : 40 us, 24 rows 24 : 39; 256 pairs of 1000 tokens 24 rows 65 : 47; 8 pairs of 8192 tokens
// 128 rows 44 : 136; 32 pairs of 4000 tokens 64 rows 68 : 72, 128 rows 89 : 74.
bool prompt_sized(int64_t batch, int64_t heads, int64_t kv_heads, int64_t tokens, int64_t max_q_len) {
    const int64_t rows = max_q_len * (heads / kv_heads);
    if (rows <= 16) return false;
    const double pairs = static_cast<double>(batch) * kv_heads;
    const double turns = ceil(pairs * ((rows + 127) / 128) / 148);
    return 8 + 0.002 * pairs * ((rows + 15) / 16) * ((tokens + 15) / 16) > 4 + 2.3 * turns * ((tokens + 127) / 128);
}

bool aligned(const void* p, int to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace

int cf_host_kv4_probe_status(int* status) {
    *status = 0;
    const int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(status, g_kv4_status, sizeof(int));
    if (e == cudaSuccess && *status != 0) e = cudaMemcpyToSymbol(g_kv4_status, &zero, sizeof(int));
    if (e != cudaSuccess) return cf_host_fail(CF_ERR_CUDA, "4-bit cache status: %s", cudaGetErrorString(e));
    return CF_OK;
}

extern "C" {

int cf_kv4_append(const void* key, const void* value, int dtype, int64_t tokens, int64_t kv_heads, int64_t head_dim, int64_t key_token_stride,
                  int64_t key_head_stride, int64_t value_token_stride, int64_t value_head_stride, const int* slot_map, void* cache, int64_t pages,
                  int64_t page_size, void* stream) {
    if (int rc = check_cache(pages, kv_heads, page_size, head_dim)) return rc;
    if (dtype != CF_DTYPE_FP16 && dtype != CF_DTYPE_BF16) return cf_host_fail(CF_ERR_INVALID, "dtype %d is neither fp16 nor bf16", dtype);
    if (tokens < 0 || tokens > 0x7fffffff) return cf_host_fail(CF_ERR_INVALID, "tokens %lld", (long long)tokens);
    if (tokens == 0) return CF_OK;
    if (!key || !value || !slot_map || !cache) return cf_host_fail(CF_ERR_INVALID, "null pointer");
    if (!aligned(key, 8) || !aligned(value, 8) || !aligned(cache, 16) || (key_token_stride | key_head_stride | value_token_stride | value_head_stride) % 4 != 0)
        return cf_host_fail(CF_ERR_INVALID, "keys and values need 8-byte aligned rows (strides in multiples of 4 elements), the cache 16 bytes");
    const int64_t items = tokens * kv_heads, grid = (items + ITEMS - 1) / ITEMS;
    if (items > 0x7fffffff) return cf_host_fail(CF_ERR_INVALID, "%lld tokens of %lld heads in one call", (long long)tokens, (long long)kv_heads);
    auto go = [&](auto* k, auto kernel) {
        kernel<<<static_cast<unsigned>(grid), CT, 0, static_cast<cudaStream_t>(stream)>>>(
            k, static_cast<decltype(k)>(value), slot_map, static_cast<uint8_t*>(cache), static_cast<unsigned>(items), static_cast<int>(kv_heads), static_cast<int>(head_dim),
            static_cast<int>(page_size / KV4_TILE), pages * page_size, key_token_stride, key_head_stride, value_token_stride, value_head_stride);
    };
    with_groups(static_cast<int>(head_dim), [&](auto g) {
        if (dtype == CF_DTYPE_FP16) go(static_cast<const __half*>(key), kv4_append_kernel<__half, g.value>);
        else go(static_cast<const __nv_bfloat16*>(key), kv4_append_kernel<__nv_bfloat16, g.value>);
    });
    return check_launch("4-bit append");
}

int cf_kv4_read(const void* cache, int64_t pages, int64_t page_size, int64_t kv_heads, int64_t head_dim, const int* slot_map, int64_t tokens, void* key,
                void* value, int dtype, void* stream) {
    if (int rc = check_cache(pages, kv_heads, page_size, head_dim)) return rc;
    if (dtype != CF_DTYPE_FP16 && dtype != CF_DTYPE_BF16) return cf_host_fail(CF_ERR_INVALID, "dtype %d is neither fp16 nor bf16", dtype);
    if (tokens < 0 || tokens > 0x7fffffff) return cf_host_fail(CF_ERR_INVALID, "tokens %lld", (long long)tokens);
    if (tokens == 0) return CF_OK;
    if (!key || !value || !slot_map || !cache) return cf_host_fail(CF_ERR_INVALID, "null pointer");
    if (!aligned(key, 16) || !aligned(value, 16) || !aligned(cache, 16)) return cf_host_fail(CF_ERR_INVALID, "storage must be 16-byte aligned");
    const int64_t items = tokens * kv_heads, grid = (items + ITEMS - 1) / ITEMS;
    if (items > 0x7fffffff) return cf_host_fail(CF_ERR_INVALID, "%lld tokens of %lld heads in one call", (long long)tokens, (long long)kv_heads);
    auto go = [&](auto* k, auto kernel) {
        kernel<<<static_cast<unsigned>(grid), CT, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const uint8_t*>(cache), slot_map, k, static_cast<decltype(k)>(value), static_cast<unsigned>(items), static_cast<int>(kv_heads), static_cast<int>(head_dim),
            static_cast<int>(page_size / KV4_TILE), pages * page_size);
    };
    with_groups(static_cast<int>(head_dim), [&](auto g) {
        if (dtype == CF_DTYPE_FP16) go(static_cast<__half*>(key), kv4_read_kernel<__half, g.value>);
        else go(static_cast<__nv_bfloat16*>(key), kv4_read_kernel<__nv_bfloat16, g.value>);
    });
    return check_launch("4-bit read");
}

int64_t cf_kv4_attention_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_tokens, int64_t max_q_len) {
    if (batch < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads != 0 || head_dim < 1 || head_dim > KV4_MAX_DIM || max_tokens < 1 || max_q_len < 1) return 0;
    if (prompt_sized(batch, heads, kv_heads, max_tokens, max_q_len)) return 0;
    return kv4_few_uses_workspace(batch, heads, kv_heads, max_tokens, max_q_len) ? kv4_few_workspace(heads, kv_heads, static_cast<int>(head_dim), max_q_len) : 0;
}

int cf_kv4_attention(const void* query, int dtype, int64_t rows, int64_t heads, int64_t head_dim, int64_t query_token_stride, int64_t query_head_stride,
                     const void* cache, int64_t pages, int64_t page_size, int64_t kv_heads, const int* block_table, int64_t table_width,
                     int64_t table_stride, const int* kv_lens, const int* qo_indptr, int64_t batch, int64_t max_q_len, float scale, void* workspace,
                     int64_t workspace_bytes, void* out, void* stream) {
    if (int rc = check_cache(pages, kv_heads, page_size, head_dim)) return rc;
    if (dtype != CF_DTYPE_FP16 && dtype != CF_DTYPE_BF16) return cf_host_fail(CF_ERR_INVALID, "dtype %d is neither fp16 nor bf16", dtype);
    if (heads < kv_heads || heads % kv_heads != 0) return cf_host_fail(CF_ERR_INVALID, "%lld query heads over %lld cached heads", (long long)heads, (long long)kv_heads);
    if (rows < 0 || rows > 0x7fffffff || batch < 1 || batch > 0x7fffffff || max_q_len < 1)
        return cf_host_fail(CF_ERR_INVALID, "rows %lld, batch %lld, max_q_len %lld", (long long)rows, (long long)batch, (long long)max_q_len);
    if (!qo_indptr && rows < batch) return cf_host_fail(CF_ERR_INVALID, "%lld query rows for %lld requests", (long long)rows, (long long)batch);
    if (table_width < 1 || table_stride < table_width || table_width > 0x7fffffff) return cf_host_fail(CF_ERR_INVALID, "block table of %lld columns, %lld entries apart", (long long)table_width, (long long)table_stride);
    if (rows == 0) return CF_OK;
    if (!query || !cache || !block_table || !kv_lens || !out) return cf_host_fail(CF_ERR_INVALID, "null pointer");
    if (!aligned(query, 16) || !aligned(out, 16) || !aligned(cache, 16) || (query_token_stride | query_head_stride) % 8 != 0)
        return cf_host_fail(CF_ERR_INVALID, "queries need 16-byte aligned rows (strides in multiples of 8 elements), cache and output 16 bytes");
    if (rows > 0x3fffffff / heads) return cf_host_fail(CF_ERR_INVALID, "%lld query rows of %lld heads in one call", (long long)rows, (long long)heads);
    if (batch * kv_heads > 0x7fffffff / 8) return cf_host_fail(CF_ERR_INVALID, "%lld requests of %lld cached heads in one call", (long long)batch, (long long)kv_heads);
    const int64_t needed = kv4_few_workspace(heads, kv_heads, static_cast<int>(head_dim), max_q_len);
    const bool prompt = prompt_sized(batch, heads, kv_heads, table_width * page_size, max_q_len);
    if (workspace && !prompt && (workspace_bytes < needed || !aligned(workspace, 16)))
        return cf_host_fail(CF_ERR_INVALID, "workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)workspace_bytes, (long long)needed);
    // rows of one request, and its heads, are written while others are still read
    const int64_t to_row = (rows - 1) * query_token_stride, to_head = (heads - 1) * query_head_stride;
    const char *q_from = static_cast<const char*>(query) + 2 * (std::min<int64_t>(to_row, 0) + std::min<int64_t>(to_head, 0));
    const char *q_to = static_cast<const char*>(query) + 2 * (std::max<int64_t>(to_row, 0) + std::max<int64_t>(to_head, 0) + head_dim), *o_from = static_cast<const char*>(out);
    if (o_from < q_to && q_from < o_from + 2 * rows * heads * head_dim) return cf_host_fail(CF_ERR_INVALID, "out overlaps the queries");
    static std::atomic<int*> status_word[64];  // address of the device status word, by device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= 64)) return cf_host_fail(CF_ERR_UNSUPPORTED, "device index %d", dev);
    if (e == cudaSuccess && !status_word[dev]) {
        void* p = nullptr;
        e = cudaGetSymbolAddress(&p, g_kv4_status);
        if (e == cudaSuccess) status_word[dev] = static_cast<int*>(p);
    }
    if (e != cudaSuccess) return cf_host_fail(CF_ERR_CUDA, "4-bit attention: %s", cudaGetErrorString(e));
    const Kv4AttnArgs a{query, static_cast<const uint8_t*>(cache), block_table, kv_lens, qo_indptr, out, query_token_stride, query_head_stride, table_stride, table_width, rows,
                        static_cast<int>(batch), static_cast<int>(heads), static_cast<int>(kv_heads), static_cast<int>(head_dim), static_cast<int>(page_size),
                        static_cast<int>(pages), scale * 1.4426950408889634f, status_word[dev], workspace};
    e = prompt ? kv4_attention_prompt(a, dtype == CF_DTYPE_BF16, max_q_len, static_cast<cudaStream_t>(stream))
               : kv4_attention_few(a, dtype == CF_DTYPE_BF16, max_q_len, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cf_host_fail(CF_ERR_CUDA, "4-bit attention launch failed: %s", cudaGetErrorString(e));
    return CF_OK;
}

}  // extern "C"
