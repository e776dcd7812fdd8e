// The paged cache held in 4 bits (layout: kv4_layout.cuh): rows written at their slots and read back, and the C entry
// points.  Asymmetric 4-bit codes over groups of 32 values of one token and head:
//   m = fp16(min x), s = fp16((max x - m) / 15), code = clamp(rint((x - m) / s), 0, 15), value = code * s + m
// A scale that was rounded up so far that m + 15 s would lie beyond fp16's largest number is stored one step lower: whatever reads
// the row, in fp16 or not, gets the same finite values.  x in fp32 (clamped to fp16's range, which bf16 exceeds); the codes are computed against the rounded s and m, so the rounding of
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
#include "f32x2.cuh"
#include "host_common.h"
#include "kv4_attention.h"
#include "kv4_layout.cuh"

namespace {

using namespace cfb;

__device__ int g_kv4_status = 0;

__device__ __forceinline__ void report_bad_slot() { atomicCAS(&g_kv4_status, 0, ST_BAD_SLOT); }


// Both kernels: half a warp for a (token, head), lane l of the half holds dims 8 l .. 8 l + 7 (16 bytes) of the key and the
// value, four lanes a group.  A warp then moves 2 KB of keys and values with two loads a lane, and the index arithmetic, the
// group reductions (two shuffles) and the parameters' divisions are paid once for 64 values.  Both are bound by integer and
// comparison instructions, not by memory: 8191 tokens of 8 heads of 128 in bf16, 88 MB both ways and 13.6 us at the copy bandwidth,
// take 28.7 us together on the GPU, 20.4 and 8.7 alone (append: ALU 61 % of its rate, issue slots 70 %; read: 58 %, 69 %).  740 resident CTAs that go through
// their items with the next one's loads in flight took 5 % more.
constexpr int CT = 256;          // threads of a CTA
constexpr int ITEMS = CT / 16;   // (token, head) pairs of a CTA

// pairs of the 16-bit types
template <class T> struct Two;
template <> struct Two<__half> {
    using P = __half2;
    static constexpr bool BEYOND = false;         // whether finite numbers reach beyond fp16
    static constexpr uint32_t INF = 0x04000400u;  // what carries an exponent of all ones into bit 15
    static constexpr uint32_t LEAST = 0xfbfffbffu;
    static __device__ __forceinline__ float2 floats(P v) { return __half22float2(v); }
};
template <> struct Two<__nv_bfloat16> {
    using P = __nv_bfloat162;
    static constexpr bool BEYOND = true;
    static constexpr uint32_t INF = 0x00800080u, LEAST = 0xff7fff7fu;
    static __device__ __forceinline__ float2 floats(P v) { return __bfloat1622float2(v); }
};
template <class P> __device__ __forceinline__ uint32_t bits_of(P v) { return *reinterpret_cast<const uint32_t*>(&v); }
template <class P> __device__ __forceinline__ P pair_of(uint32_t w) { return *reinterpret_cast<const P*>(&w); }

// n / d for n < 2^31 by a multiplication (T. Granlund and P. Montgomery, Division by Invariant Integers using Multiplication, 1994): with
// 2^(l - 1) < d <= 2^l, (n (floor(2^(31 + l) / d) + 1)) >> (31 + l) is exact
struct Divisor {
    unsigned times, shift;
    explicit Divisor(unsigned d) {
        unsigned l = 0;
        while ((1ull << l) < d) ++l;
        times = static_cast<unsigned>((1ull << (31 + l)) / d + 1);
        shift = 31 + l;
    }
    __device__ __forceinline__ unsigned operator()(unsigned n) const { return static_cast<unsigned>((static_cast<unsigned long long>(n) * times) >> shift); }
};

// Codes of this lane's eight values (raw words, nibble i: value i), scale and minimum of its group of four lanes.  Extremes stay in the 16-bit
// type, the greatest value and the greatest negated one as a pair, and carry a NaN or an infinity along.  A code is rounded by adding
// 1.5 * 2^23 and taking it off (conversions run at a quarter of the rate); four codes are put together as one fp32 number below 2^16.
template <class T> __device__ __forceinline__ unsigned quantise8(const uint32_t (&raw)[4], bool real, __half* scale, __half* low) {
    using P = typename Two<T>::P;
    auto p = [&](int i) { return pair_of<P>(raw[i]); };
    const uint32_t hi2 = bits_of(__hmax2_nan(__hmax2_nan(p(0), p(1)), __hmax2_nan(p(2), p(3))));
    const uint32_t lo2 = bits_of(__hmin2_nan(__hmin2_nan(p(0), p(1)), __hmin2_nan(p(2), p(3)))) ^ 0x80008000u;
    uint32_t ends = bits_of(__hmax2_nan(pair_of<P>(__byte_perm(hi2, lo2, 0x5410)), pair_of<P>(__byte_perm(hi2, lo2, 0x7632))));
    if (!real) ends = Two<T>::LEAST;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) ends = bits_of(__hmax2_nan(pair_of<P>(ends), pair_of<P>(__shfl_xor_sync(0xffffffffu, ends, o))));
    const bool bad = ((ends & 0x7fff7fffu) + Two<T>::INF) & 0x80008000u;
    float2 end = Two<T>::floats(pair_of<P>(ends));
    end.y = -end.y;
    bool wide = false;
    if constexpr (Two<T>::BEYOND) {
        wide = end.y < -65504.f || end.x > 65504.f;
        end.x = fminf(fmaxf(end.x, -65504.f), 65504.f), end.y = fminf(fmaxf(end.y, -65504.f), 65504.f);
    }
    const __half m = __float2half_rn(end.y);
    const float mf = __half2float(m);
    // x / 15 correctly rounded (P. Markstein, Computation of Elementary Functions on the IBM RISC System/6000 Processor, 1990): the product with the
    // rounded 1 / 15, corrected by its residual, which is exact in a fused multiply-add (where that would fall below fp32's range the quotient is far
    // below fp16's)
    const float x15 = end.x - mf, near = x15 * (1.f / 15.f);
    __half s = __float2half_rn(fmaf(fmaf(-15.f, near, x15), 1.f / 15.f, near));
    if (fmaf(15.f, __half2float(s), mf) > 65504.f) s = __ushort_as_half(static_cast<unsigned short>(__half_as_ushort(s) - 1));
    const float sf = __half2float(s);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(sf));
    unsigned codes = 0;
    if (real && sf > 0.f && !bad) {
        // rint((v - m) / s) by the reciprocal: off by a few 2^-24 of at most 22, which matters only next to a half; there it is divided
        constexpr float MAGIC = 12582912.f;
        const Pair magic(MAGIC, MAGIC), less(-MAGIC, -MAGIC), lowest(-mf, -mf), times(r, r), minus(-1.f, -1.f);
        Pair c[4];
        float off = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 v = Two<T>::floats(p(i));
            if (Two<T>::BEYOND && wide) v.x = fminf(fmaxf(v.x, -65504.f), 65504.f), v.y = fminf(fmaxf(v.y, -65504.f), 65504.f);
            const Pair x = (Pair(v.x, v.y) + lowest) * times;
            c[i] = (x + magic) + less;
            const float2 e = fma2(c[i], minus, x).both();
            off = fmaxf(off, fmaxf(fabsf(e.x), fabsf(e.y)));
        }
        if (off > 0.49999f) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 v = Two<T>::floats(p(i));
                c[i] = Pair(rintf((fminf(fmaxf(v.x, -65504.f), 65504.f) - mf) / sf), rintf((fminf(fmaxf(v.y, -65504.f), 65504.f) - mf) / sf));
            }
        }
        // No value is more than half a step below the minimum.  Above, a normal scale is at most 2^-10 too small (15.015 steps); one rounded to
        // fp16's last steps reaches beyond 15.
        if (sf < 6.103515625e-5f) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = c[i].both();
                c[i] = Pair(fminf(f.x, 15.f), fminf(f.y, 15.f));
            }
        }
        const Pair step(256.f, 256.f);
        const float2 a = fma2(c[1], step, c[0]).both(), b = fma2(c[3], step, c[2]).both();
        codes = __byte_perm(__float_as_uint(fmaf(a.y, 16.f, a.x + 8388608.f)), __float_as_uint(fmaf(b.y, 16.f, b.x + 8388608.f)), 0x5410);
    }
    *scale = bad ? __ushort_as_half(0x7fff) : s;
    *low = m;
    return codes;
}

// the tile that holds a row, and the row in it
__device__ __forceinline__ long long tile_of(int slot, int head, int heads, int tiles_a_page, Divisor by_page) {
    const unsigned tile = static_cast<unsigned>(slot) / KV4_TILE, page = by_page(tile);
    return (static_cast<long long>(page) * heads + head) * tiles_a_page + (tile - page * tiles_a_page);
}

template <class T, int G>
__global__ void __launch_bounds__(CT) kv4_append_kernel(const T* __restrict__ key, const T* __restrict__ value, const int* __restrict__ slot_map,
                                                        uint8_t* __restrict__ cache, unsigned items, int heads, int D, int tiles_a_page, Divisor by_heads, Divisor by_page, long long slots,
                                                        long long k_ts, long long k_hs, long long v_ts, long long v_hs) {
    const int l = threadIdx.x & 15;
    const unsigned item = blockIdx.x * ITEMS + threadIdx.x / 16;
    const bool there = item < items;
    const unsigned tok = there ? by_heads(item) : 0;
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
    uint8_t* tile = cache + tile_of(slot, head, heads, tiles_a_page, by_page) * kv4_tile_bytes(G);
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
                                                      T* __restrict__ value, unsigned items, int heads, int D, int tiles_a_page, Divisor by_heads, Divisor by_page, long long slots) {
    const int l = threadIdx.x & 15, dim = 8 * l;
    const unsigned item = blockIdx.x * ITEMS + threadIdx.x / 16;
    if (item >= items || dim >= D) return;
    const unsigned tok = by_heads(item);
    const int head = static_cast<int>(item - tok * heads), slot = slot_map[tok];
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (slot >= 0 && slot < slots) {
        const int row = slot % KV4_TILE, g = l >> 2;
        const uint8_t* tile = cache + tile_of(slot, head, heads, tiles_a_page, by_page) * kv4_tile_bytes(G);
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
// themselves (kv4_decode.cu).  The first takes 2.2 us for 128 tokens in each of 148 CTAs, 6 us besides, and does not divide the tokens among CTAs; the
// second divides them and takes 0.88 ns for 16 rows x 16 tokens and 12 us besides.  Measured (rows of a (request, head); the second against the
// first): 32 pairs of 2048 tokens 64 rows 29 : 40 us, 128 rows 39 : 42; 256 pairs of 1000 tokens 32 rows 46 : 47, 64 rows 89 : 48; 8 pairs of
// 8192 tokens 256 rows 70 : 135; 32 pairs of 4000 tokens 128 rows 65 : 73; 64 pairs of 2000 tokens 64 rows 38 : 41, 96 rows 65 : 41.
bool prompt_sized(int64_t batch, int64_t heads, int64_t kv_heads, int64_t tokens, int64_t max_q_len) {
    const int64_t rows = max_q_len * (heads / kv_heads);
    if (rows <= 16) return false;
    const double pairs = static_cast<double>(batch) * kv_heads;
    const double turns = ceil(pairs * ((rows + 127) / 128) / 148);
    return 12 + 0.00088 * pairs * ((rows + 15) / 16) * ((tokens + 15) / 16) > turns * (6 + 2.2 * ((tokens + 127) / 128));
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
            static_cast<int>(page_size / KV4_TILE), Divisor(static_cast<unsigned>(kv_heads)), Divisor(static_cast<unsigned>(page_size / KV4_TILE)), pages * page_size, key_token_stride, key_head_stride, value_token_stride, value_head_stride);
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
            static_cast<int>(page_size / KV4_TILE), Divisor(static_cast<unsigned>(kv_heads)), Divisor(static_cast<unsigned>(page_size / KV4_TILE)), pages * page_size);
    };
    with_groups(static_cast<int>(head_dim), [&](auto g) {
        if (dtype == CF_DTYPE_FP16) go(static_cast<__half*>(key), kv4_read_kernel<__half, g.value>);
        else go(static_cast<__nv_bfloat16*>(key), kv4_read_kernel<__nv_bfloat16, g.value>);
    });
    return check_launch("4-bit read");
}

int64_t cf_kv4_attention_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_tokens, int64_t max_q_len) {
    if (batch < 1 || kv_heads < 1 || heads < kv_heads || heads % kv_heads != 0 || head_dim < 1 || head_dim > KV4_MAX_DIM || max_tokens < 1 || max_q_len < 1 || max_q_len > 0x7fffffff ||
        batch > 0x7fffffff || heads > 0x7fffffff || max_tokens > 0x7fffffffll * 65536)
        return 0;
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
    if (rows < 0 || rows > 0x7fffffff || batch < 1 || batch > 0x7fffffff || max_q_len < 1 || max_q_len > 0x7fffffff)
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
