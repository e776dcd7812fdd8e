// The paged cache held in 4 bits (layout: kv4_layout.cuh): rows written at their slots and read back, and the C entry
// points.  Asymmetric 4-bit codes over groups of 32 values of one token and head:
//   m = fp16(min x), s = fp16((max x - m) / 15), code = clamp(rint((x - m) / s), 0, 15), value = code * s + m
// x in fp32 (clamped to fp16's range, which bf16 exceeds); the codes are computed against the rounded s and m, so the rounding of
// the parameters costs no accuracy but the last step's.  A group that is constant has s = 0 and code 0; one that holds a
// NaN or whose extremes are not finite in the input stores NaN as its scale: it comes back as NaN instead of as numbers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/clusterfusion_b200.h"
#include "host_common.h"
#include "kv4_attention.h"
#include "kv4_layout.cuh"

namespace {

using namespace cfb;

__device__ int g_kv4_status = 0;

__device__ __forceinline__ void report_bad_slot() { atomicCAS(&g_kv4_status, 0, ST_BAD_SLOT); }

template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Both kernels: half a warp for a (token, head), lane l of the half holds dims 8 l .. 8 l + 7 (16 bytes) of the key and the
// value, four lanes a group.  A warp then moves 2 KB of keys and values with two loads a lane, and the index arithmetic, the
// group reductions (two shuffles) and the parameters' divisions are paid once for 64 values.
constexpr int CT = 256;          // threads of a CTA
constexpr int ITEMS = CT / 16;   // (token, head) pairs of a CTA

template <class T> __device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    const uint2 raw[2] = {*reinterpret_cast<const uint2*>(p), *reinterpret_cast<const uint2*>(p + 4)};  // rows are 8-byte aligned
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float<T>(e[i]);
}

// Codes of this lane's eight values (nibble i: value i), scale and minimum of its group of four lanes.
__device__ __forceinline__ unsigned quantise8(const float (&x)[8], bool real, __half* scale, __half* low) {
    float lo = 65504.f, hi = -65504.f, v[8];
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        bad |= !(fabsf(x[i]) <= 3.4028234663852886e38f);  // NaN and the infinities
        v[i] = fminf(fmaxf(x[i], -65504.f), 65504.f);
        lo = fminf(lo, v[i]);
        hi = fmaxf(hi, v[i]);
    }
    if (!real) lo = 65504.f, hi = -65504.f, bad = 0;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad |= __shfl_xor_sync(0xffffffffu, bad, o);
    }
    const __half m = __float2half_rn(lo);
    const float mf = __half2float(m);
    const __half s = __float2half_rn((hi - mf) / 15.f);
    const float sf = __half2float(s), r = 1.f / sf;
    unsigned codes = 0;
    if (real && sf > 0.f) {
        // rint((v - m) / s) by the reciprocal: off by a few 2^-24 of at most 16, which matters only next to a half; there it is divided
        float q[8];
        bool near_half = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            q[i] = (v[i] - mf) * r;
            near_half |= fabsf(fabsf(q[i] - rintf(q[i])) - 0.5f) < 1e-5f;
        }
        if (near_half)
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = (v[i] - mf) / sf;
#pragma unroll
        for (int i = 0; i < 8; ++i) codes |= static_cast<unsigned>(__float2int_rn(fminf(fmaxf(q[i], 0.f), 15.f))) << (4 * i);
    }
    *scale = bad ? __ushort_as_half(0x7fff) : s;
    *low = m;
    return bad ? 0u : codes;
}

// the tile that holds a row, and the row in it
__device__ __forceinline__ long long tile_of(int slot, int head, int heads, int tiles_a_page) {
    const unsigned tile = static_cast<unsigned>(slot) / KV4_TILE, page = tile / tiles_a_page;
    return (static_cast<long long>(page) * heads + head) * tiles_a_page + (tile - page * tiles_a_page);
}

template <class T>
__global__ void __launch_bounds__(CT) kv4_append_kernel(const T* __restrict__ key, const T* __restrict__ value, const int* __restrict__ slot_map,
                                                        uint8_t* __restrict__ cache, unsigned items, int heads, int D, int tiles_a_page, long long slots,
                                                        long long k_ts, long long k_hs, long long v_ts, long long v_hs) {
    const int G = kv4_groups(D), l = threadIdx.x & 15;
    const unsigned item = blockIdx.x * ITEMS + threadIdx.x / 16;
    const bool there = item < items;
    const unsigned tok = there ? item / heads : 0;
    const int head = there ? static_cast<int>(item - tok * heads) : 0;
    const int slot = there ? slot_map[tok] : -1;
    if (slot >= slots && l == 0) report_bad_slot();
    const bool kept = slot >= 0 && slot < slots;  // a padded row is skipped
    const int dim = 8 * l;
    const bool real = kept && dim < D;
    float xk[8], xv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) xk[i] = xv[i] = 0.f;
    if (real) {
        load8(key + tok * k_ts + head * k_hs + dim, xk);
        load8(value + tok * v_ts + head * v_hs + dim, xv);
    }
    __half ks, km, vs, vm;
    const unsigned kc = quantise8(xk, real, &ks, &km), vc = quantise8(xv, real, &vs, &vm);
    if (!kept || dim >= 32 * G) return;
    const int row = slot % KV4_TILE, which = l & 3;
    uint8_t* tile = cache + tile_of(slot, head, heads, tiles_a_page) * kv4_tile_bytes(G);
    *reinterpret_cast<uint32_t*>(tile + kv4_key_half(G, row, dim)) = kc;
    *reinterpret_cast<uint16_t*>(tile + kv4_value_half(G, row, dim)) = static_cast<uint16_t>(vc);
    *reinterpret_cast<uint16_t*>(tile + kv4_value_half(G, row, dim + 4)) = static_cast<uint16_t>(vc >> 16);
    *reinterpret_cast<__half*>(tile + kv4_param(G, row, which, l >> 2)) = which == 0 ? ks : which == 1 ? km : which == 2 ? vs : vm;
}

template <class T> __device__ __forceinline__ uint4 unpack8(unsigned codes, float s, float m) {
    __align__(16) T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_float<T>(fmaf(static_cast<float>((codes >> (4 * i)) & 15u), s, m));
    return *reinterpret_cast<const uint4*>(e);
}

template <class T>
__global__ void __launch_bounds__(CT) kv4_read_kernel(const uint8_t* __restrict__ cache, const int* __restrict__ slot_map, T* __restrict__ key,
                                                      T* __restrict__ value, unsigned items, int heads, int D, int tiles_a_page, long long slots) {
    const int G = kv4_groups(D), l = threadIdx.x & 15, dim = 8 * l;
    const unsigned item = blockIdx.x * ITEMS + threadIdx.x / 16;
    if (item >= items || dim >= D) return;
    const unsigned tok = item / heads;
    const int head = static_cast<int>(item - tok * heads), slot = slot_map[tok];
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (slot >= 0 && slot < slots) {
        const int row = slot % KV4_TILE, g = l >> 2;
        const uint8_t* tile = cache + tile_of(slot, head, heads, tiles_a_page) * kv4_tile_bytes(G);
        auto par = [&](int which) { return __half2float(*reinterpret_cast<const __half*>(tile + kv4_param(G, row, which, g))); };
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

int check_launch(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cf_host_fail(CF_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
    return CF_OK;
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
    if (dtype == CF_DTYPE_FP16) go(static_cast<const __half*>(key), kv4_append_kernel<__half>);
    else go(static_cast<const __nv_bfloat16*>(key), kv4_append_kernel<__nv_bfloat16>);
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
    if (dtype == CF_DTYPE_FP16) go(static_cast<__half*>(key), kv4_read_kernel<__half>);
    else go(static_cast<__nv_bfloat16*>(key), kv4_read_kernel<__nv_bfloat16>);
    return check_launch("4-bit read");
}

int64_t cf_kv4_attention_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_tokens, int64_t max_q_len) {
    if (batch < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads != 0 || head_dim < 1 || head_dim > KV4_MAX_DIM || max_tokens < 1 || max_q_len < 1) return 0;
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
    if (workspace && (workspace_bytes < needed || !aligned(workspace, 16)))
        return cf_host_fail(CF_ERR_INVALID, "workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)workspace_bytes, (long long)needed);
    static int* status_word[64] = {};  // address of the device status word, by device
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
    e = kv4_attention_few(a, dtype == CF_DTYPE_BF16, max_q_len, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cf_host_fail(CF_ERR_CUDA, "4-bit attention launch failed: %s", cudaGetErrorString(e));
    return CF_OK;
}

}  // extern "C"
