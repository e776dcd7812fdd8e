// Attention over the 4-bit cache for many query rows a request: chunks of prompts.
//
// Here every cached token meets 128 query rows (queries times the heads of one cached head) and the work is two matrix products, 4 D flops
// for each (row, token): it goes to the 5th-generation tensor cores, S = Q K^T and O += P V with 128 x 128 tiles, operands in shared
// memory (K-major, 128-byte swizzle), accumulators in tensor memory.  At 4096 fp16 multiply-adds a clock a pair of tiles takes
// ~1000 clocks of the tensor cores and as many of the exponential unit (16 a clock), and unpacking the codes takes ~600 issue slots
// of each scheduler: three things that overlap, so each has its warps:
//  - 8 warps unpack: 16 tokens each of a 128-token tile, to fp16 value = code * scale + minimum in one fused rounding (2^-11 of a key or
//    value: the operands' type; scores and sums stay fp32).  Keys as rows of dims, values as rows of tokens, which is how the cache's
//    words hold them: two neighbouring tokens in the halves of a word are two neighbouring elements of a row of V^T.
//  - 8 warps do the softmax, two threads a query row, in one pass over a tile's scores.  The reference of a row moves only when a score
//    lies more than 8 binary steps above the greatest before it, which after a row's first tile hardly ever happens: then the accumulator in tensor
//    memory is rescaled and the pass repeated.
//  - 1 thread issues the products: S of the next tile before P V of this one, so that they run under the softmax.
// Every wait is bounded; one that runs out ends the kernel with a device status.
// Measured: chunks of 267, 723 and 985 queries over 267, 3514 and 3954 tokens, 32 heads over 8 of 128: 202 us, 465 TFLOP/s of products
// (28 % of the measured rate of large products); in fp16 205 us.  The softmax warps are the chain: 3500 clocks a tile, 2400 of them arithmetic, 450 for
// the agreement of a row's two threads, the rest waits that find their event already there; the unpacking warps need as many, and what makes
// one of them faster (a hardware barrier for the agreement, half the commits, no bank conflicts, look-ups moved) slows the others: 202 to 210.  One
// thread a row took 234 us, 256 rows a CTA (each unpacked tile used twice, at half the warps a row) 246 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "f32x2.cuh"
#include "kv4_attention.h"
#include "kv4_layout.cuh"
#include "mma.cuh"
#include "pipeline.cuh"

namespace cfb {
namespace {

constexpr int ROWS = 128;            // query rows of a CTA
constexpr int KEYS = 128;            // tokens of a tile
constexpr int SOFT = 8, UNPACK = 8;  // warps; one more issues the products
constexpr int THREADS = 32 * (SOFT + UNPACK + 1);
constexpr int BLOCK = 128 * 128;     // bytes of a K-major operand block of 128 rows x 64 elements
// A row's reference is set so that its greatest p is 2^HIGH, and moves when one exceeds 2^SLACK: p is an fp16 operand, and what lies far below the
// maximum keeps its bits (normal numbers down to 2^-14) the longer the higher the maximum stands
constexpr float HIGH = 7.f, SLACK = 15.f;

// ------------------------------------------------------------------------------------------------ tensor cores
__device__ __forceinline__ uint64_t operand(uint32_t saddr) {  // K-major, 128-byte swizzle: rows of 128 bytes, groups of 8 rows 1024 bytes apart
    return static_cast<uint64_t>((saddr & 0x3ffffu) >> 4) | static_cast<uint64_t>(1u) << 16 | static_cast<uint64_t>(1024u >> 4) << 32 |
           static_cast<uint64_t>(1u) << 46 | static_cast<uint64_t>(2u) << 61;
}
__device__ __forceinline__ constexpr uint32_t shape(int m, int n) {  // fp16 operands, fp32 accumulator, both K-major
    return (1u << 4) | static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(m >> 4) << 24;
}
__device__ __forceinline__ void product(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {  // arrives once every product issued so far is done
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }  // plain stores, for the tensor cores to read

// 16 columns of this thread's row of tensor memory; the wait belongs to the load, so that nothing uses the registers before it
__device__ __forceinline__ void tmem_load(uint32_t at, float (&x)[16]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]), "=f"(x[8]), "=f"(x[9]), "=f"(x[10]),
          "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15])
        : "r"(at)
        : "memory");
}
// the same in two steps: asked for now, there after tmem_wait (which names the registers, so that nothing uses them before it)
__device__ __forceinline__ void tmem_ask(uint32_t at, float (&x)[16]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]), "=f"(x[8]), "=f"(x[9]),
          "=f"(x[10]), "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_wait(float (&x)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]), "+f"(x[7]), "+f"(x[8]), "+f"(x[9]),
                   "+f"(x[10]), "+f"(x[11]), "+f"(x[12]), "+f"(x[13]), "+f"(x[14]), "+f"(x[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_store(uint32_t at, const float (&x)[16]) {
    __syncwarp();
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};\n\t"
        "tcgen05.wait::st.sync.aligned;" ::"r"(at), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]), "f"(x[8]),
        "f"(x[9]), "f"(x[10]), "f"(x[11]), "f"(x[12]), "f"(x[13]), "f"(x[14]), "f"(x[15])
        : "memory");
}

// ------------------------------------------------------------------------------------------------ numbers
template <class T> __device__ __forceinline__ uint32_t pack(float a, float b);
// (a result is a mean of values within fp16's range: what the sums' rounding puts beyond it is not infinity; NaN stays)
template <> __device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
    auto held = [](float x) { return x > 65504.f ? 65504.f : x < -65504.f ? -65504.f : x; };
    return pack_half2(held(a), held(b));
}
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
__device__ __forceinline__ uint32_t as_word(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }

// (w & mask) | bits in one instruction
__device__ __forceinline__ uint32_t select_or(uint32_t w, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
    return r;
}
// codes 0, 4 | 1, 5 | 2, 6 | 3, 7 of a word as pairs of fp16 numbers: 1024 + code and 64 + code by the bits, less 1024 and 64
__device__ __forceinline__ void code_pairs(uint32_t w, __half2 (&c)[4]) {
    const uint32_t h = w >> 8;
    const __half2 k1024 = as_half2(0x64006400u), k64 = as_half2(0x54005400u);
    c[0] = __hsub2(as_half2(select_or(w, 0x000f000fu, 0x64006400u)), k1024);
    c[1] = __hsub2(as_half2(select_or(w, 0x00f000f0u, 0x54005400u)), k64);
    c[2] = __hsub2(as_half2(select_or(h, 0x000f000fu, 0x64006400u)), k1024);
    c[3] = __hsub2(as_half2(select_or(h, 0x00f000f0u, 0x54005400u)), k64);
}
__device__ __forceinline__ bool finite_half(uint32_t x) { return (x & 0x7c00u) != 0x7c00u; }

// N consecutive words of global memory; two and four are aligned to all of them
template <int N> __device__ __forceinline__ void global_words(uint32_t (&x)[N], const uint8_t* p) {
    if constexpr (N == 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
        x[0] = v.x, x[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
    }
}

struct Shared {
    unsigned long long q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full, pv_done, drain;
    uint32_t tmem;
    int abort;
    unsigned there[4];          // [tile % 4] bit t: the 16 tokens t of the tile exist.  Four: keys are unpacked two tiles ahead of the softmax
    unsigned long long agreed[4], summed[4];  // of the two warps that share rows
    float high[2][2][ROWS], sums[2][ROWS];    // [tile & 1][half][row]: greatest score; [half][row]: denominator
    // [item % 8][group]: the first token that some row sees and whose value parameters are not finite.  The unpacking warps may be three tiles, so as
    // many items, ahead of the softmax; a thread of the softmax clears an item's place four items before it, when that of four items ago was read.
    int first_broken[8][4];
    __align__(16) uint16_t kpar[8][16][8];     // [unpacking warp][token][scales, minima of the keys]
    __align__(16) uint16_t vpar[8][2][4][16];  // [unpacking warp][scale, minimum of the values][group][token]
};

template <class T, int G>
__global__ void __launch_bounds__(THREADS, 1) kv4_prompt_kernel(const Kv4AttnArgs a) {
    constexpr int TB = kv4_tile_bytes(G), DP = 32 * G, DB = (DP + 63) / 64;  // blocks of 64 dims
    constexpr int VBLOCK = DP * 128;                                         // bytes of V^T, 64 tokens
    extern __shared__ uint8_t raw[];
    uint8_t* base = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;  // (by an offset: the compiler has to see that it is shared memory)
    uint8_t* s_q = base;
    uint8_t* s_k = s_q + DB * BLOCK;            // [2]
    uint8_t* s_v = s_k + 2 * DB * BLOCK;        // [2]
    uint8_t* s_p = s_v + 2 * 2 * VBLOCK;
    __shared__ Shared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    auto bar = [](unsigned long long& b) { return smem_u32(&b); };
    if (tid == 0) {
        mbar_init(bar(sh.q_full), 32 * SOFT);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(sh.k_full[i]), UNPACK);
            mbar_init(bar(sh.k_empty[i]), 1);
            mbar_init(bar(sh.v_full[i]), UNPACK);
            mbar_init(bar(sh.v_empty[i]), 1);
            mbar_init(bar(sh.s_full[i]), 1);
        }
        mbar_init(bar(sh.p_full), 32 * SOFT);
        mbar_init(bar(sh.pv_done), 1);
        mbar_init(bar(sh.drain), 1);
        mbar_fence_init();
        for (int i = 0; i < 4; ++i) {
            mbar_init(bar(sh.agreed[i]), 64);
            mbar_init(bar(sh.summed[i]), 64);
        }
        sh.abort = 0;
        for (int i = 0; i < 8 * 4; ++i) sh.first_broken[i / 4][i % 4] = 0x7fffffff;
        for (int i = 0; i < 4; ++i) sh.there[i] = 0;
    }
    if (warp == SOFT + UNPACK) {  // scores twice 128 columns, numerators 128: 512 is the next size there is
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        fence_before();
    }
    __syncthreads();
    fence_after();
    const uint32_t tm_s = sh.tmem, tm_o = sh.tmem + 2 * KEYS;  // columns: scores of two tiles, numerators
    const AbortCtl ctl{&sh.abort, a.status};
    // one answer for the whole warp, which goes on together
    auto wait_one = [&](unsigned long long& b, int phase, int code) { return mbar_wait(bar(b), phase & 1, ctl, code); };
    auto wait = [&](unsigned long long& b, int phase, int code) { return __all_sync(0xffffffffu, wait_one(b, phase, code)) != 0; };

    const int b = blockIdx.x / a.kv_heads, kvh = blockIdx.x - b * a.kv_heads, per = a.heads / a.kv_heads;
    int first = b, n_q = 1;
    if (a.qo_indptr) {
        first = a.qo_indptr[b];
        n_q = first < 0 ? 0 : min(a.qo_indptr[b + 1], static_cast<int>(a.rows)) - first;
    }
    const int rows = n_q > 0 ? n_q * per : 0, q_tiles = (rows + ROWS - 1) / ROWS;
    const long long cap = a.table_width * a.page, before = static_cast<long long>(a.kv_lens[b]) - n_q;
    const int* table = a.table + b * a.table_stride;
    const int N = (a.D + 15) / 16 * 16;

    int done = 0;   // tiles of tokens so far: the phase of every barrier follows from it
    int items = 0;  // (request, head, 128 rows) so far
    for (int y = blockIdx.y; y < q_tiles; y += gridDim.y) {
        const int r0 = (q_tiles - 1 - y) * ROWS;  // the longest first
        const long long end = min(before + (min(r0 + ROWS, rows) - 1) / per, cap - 1);  // the last token that these rows see
        const int n = end < 0 ? 0 : static_cast<int>(end / KEYS) + 1;
        bool ok = true;

        if (warp < SOFT) {
            // ================================================================ softmax: two threads a row, 64 columns of a tile each
            const int line = tid & (ROWS - 1), half = warp >> 2, pair = warp & 3, r = r0 + line;
            const bool real = r < rows;
            const int qi = real ? r / per : 0, head = kvh * per + (real ? r % per : 0);
            const T* src = static_cast<const T*>(a.query) + static_cast<long long>(first + qi) * a.q_ts + head * a.q_hs;
            T* dst = static_cast<T*>(a.out) + (static_cast<long long>(first + qi) * a.heads + head) * a.D;
            const int last = real ? static_cast<int>(max(min(before + qi, cap - 1), -1ll)) : -1;
            const int all_see = static_cast<int>(max(min(before + r0 / per, cap - 1), -1ll));  // every real row sees these
            if (n > 0) {
                if (tid < 4) sh.first_broken[(items + 4) & 7][tid] = 0x7fffffff;
                // all loads of the row at once: in turn they would take longer than a tile.  The row's two threads write half of it each.
                uint4 own[DP / 16], rest[DP / 16];
#pragma unroll
                for (int j = 0; j < DP / 16; ++j) {
                    const int d = 16 * j + 8 * half, e = 16 * j + 8 * (half ^ 1);
                    own[j] = real && d < a.D ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0, 0, 0, 0);
                    rest[j] = real && e < a.D ? *reinterpret_cast<const uint4*>(src + e) : make_uint4(0, 0, 0, 0);
                }
                float top = 0.f;
#pragma unroll
                for (int j = 0; j < DP / 16; ++j) {
                    const uint32_t w[8] = {own[j].x, own[j].y, own[j].z, own[j].w, rest[j].x, rest[j].y, rest[j].z, rest[j].w};
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 f = to_float2<T>(w[i]);
                        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                }
                // a power of two takes the row to at most 2^10 (exact; bf16 reaches beyond fp16), the scale's sign goes along
                const int e = query_exponent(top);
                const float up = copysignf(query_scaling(e), a.scale_log2);
#pragma unroll
                for (int j = 0; j < DP / 16; ++j) {
                    const int d = 16 * j + 8 * half;
                    const uint32_t w[4] = {own[j].x, own[j].y, own[j].z, own[j].w};
                    float v8[8];
                    uint32_t o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 f = to_float2<T>(w[i]);
                        v8[2 * i] = f.x * up, v8[2 * i + 1] = f.y * up;
                    }
                    // dims 0, 4, 1, 5, 2, 6, 3, 7 of each eight: the order in which the keys come out of their words
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = pack_half2(v8[i], v8[i + 4]);
                    *reinterpret_cast<uint4*>(s_q + d / 64 * BLOCK + line * 128 + ((d % 64 / 8) ^ (line & 7)) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
                }
                fence_shared();
                mbar_arrive(bar(sh.q_full));
                const float factor = fminf(fabsf(a.scale_log2) * power_of_two(e - 9), 3.4e38f);
                const uint32_t mine = static_cast<uint32_t>(pair * 32) << 16;  // this warp's lanes of tensor memory

                float m = 0.f, l = 0.f;  // reference of the row, sum of this thread's p
                bool set = false;        // the row has a reference
                for (int i = 0; ok && i < n; ++i) {
                    const int at = done + i, buf = at & 1, key0 = i * KEYS + 64 * half;
                    if (!(ok = wait(sh.s_full[buf], at >> 1, ST_TIMEOUT_FULL))) break;
                    fence_after();
                    const unsigned there = sh.there[at & 3];
                    const bool whole = i * KEYS + KEYS - 1 <= all_see && there == 0xffu;
                    // One pass: p by the reference that the row has, and the greatest score with it.  Only where that lies more than SLACK above the
                    // reference (or the row had none) the reference moves, the numerators are rescaled and the pass is done again.
                    for (bool again = false;; again = true) {
                        constexpr int C = 16, CHUNKS = 64 / C;
                        float high = -INFINITY, x[2][C];
                        Pair sum(0.f, 0.f);
                        uint32_t held[CHUNKS / 2][C / 2];
                        const uint32_t from = tm_s + buf * KEYS + 64 * half + mine;
                        tmem_ask(from, x[0]);
#pragma unroll
                        for (int q = 0; q < CHUNKS; ++q) {
                            float(&y)[C] = x[q & 1];
                            tmem_wait(y);
                            if (q + 1 < CHUNKS) tmem_ask(from + C * (q + 1), x[(q + 1) & 1]);
#pragma unroll
                            for (int j = 0; j < C; j += 2) {
                                const float2 f = fma2(Pair(y[j], y[j + 1]), Pair(factor, factor), Pair(-m, -m)).both();
                                y[j] = f.x, y[j + 1] = f.y;
                            }
                            if (!whole) {
                                const int see = there >> (4 * half + q) & 1u ? last - key0 - C * q : -1;  // columns 0 .. see of the chunk (16 tokens: one page's)
#pragma unroll
                                for (int j = 0; j < C; ++j)
                                    if (j > see) y[j] = -INFINITY;
                            }
#pragma unroll
                            for (int j = 0; j < C; ++j) high = fmaxf(high, y[j]);
                            uint32_t(&h)[C / 2] = held[q % (CHUNKS / 2)];
#pragma unroll
                            for (int j = 0; j < C; j += 2) {
                                const Pair p(ex2(y[j]), ex2(y[j + 1]));
                                sum = sum + p;
                                const float2 f = p.both();
                                h[j / 2] = pack_half2(f.x, f.y);
                            }
                            if (q + 1 < CHUNKS / 2) continue;
                            // the products of the tile before read P: the first half waits in registers for their end
                            if (q + 1 == CHUNKS / 2 && !again && i > 0) {
                                if (!(ok = wait(sh.pv_done, at - 1, ST_TIMEOUT_FULL))) {
                                    tmem_wait(x[(q + 1) & 1]);
                                    break;
                                }
                                fence_after();
                            }
#pragma unroll
                            for (int w = q + 1 == CHUNKS / 2 ? 0 : q; w <= q; ++w)
#pragma unroll
                                for (int j = 0; j < 2; ++j) {
                                    const uint32_t(&v)[C / 2] = held[w % (CHUNKS / 2)];
                                    *reinterpret_cast<uint4*>(s_p + half * BLOCK + line * 128 + ((w * 2 + j) ^ (line & 7)) * 16) =
                                        make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                                }
                        }
                        if (!ok) break;
                        if (!again) {  // the row's other thread: both have to come to the same reference
                            sh.high[at & 1][half][line] = high;
                            mbar_arrive(bar(sh.agreed[pair]));
                            if (!(ok = wait(sh.agreed[pair], at, ST_TIMEOUT_FULL))) break;
                            high = fmaxf(high, sh.high[at & 1][half ^ 1][line]);
                        }
                        const bool move = !again && (high > SLACK || (!set && high != -INFINITY));
                        if (!__any_sync(0xffffffffu, move)) {
                            const float2 both = sum.both();
                            l += both.x + both.y;
                            break;
                        }
                        const float by = move ? high - HIGH : 0.f, keep = set ? ex2(-by) : 1.f;
                        m += by;
                        l *= keep;
                        set |= move;
                        if (i > 0)
                            for (int c = 16 * half; c < N; c += 32) {
                                float o[16];
                                tmem_load(tm_o + c + mine, o);
#pragma unroll
                                for (int j = 0; j < 16; ++j) o[j] *= keep;
                                tmem_store(tm_o + c + mine, o);
                            }
                    }
                    if (!ok) break;
                    fence_before();
                    fence_shared();
                    mbar_arrive(bar(sh.p_full));
                }
                if (ok) {
                    sh.sums[half][line] = l;
                    mbar_arrive(bar(sh.summed[pair]));
                    ok = wait(sh.summed[pair], items, ST_TIMEOUT_FULL) && wait(sh.pv_done, done + n - 1, ST_TIMEOUT_FULL);
                }
                if (ok) {
                    fence_after();
                    l += sh.sums[half ^ 1][line];
                    unsigned broken = 0;  // groups in which the row sees a value that is not finite
#pragma unroll
                    for (int g = 0; g < G; ++g) broken |= (sh.first_broken[items & 7][g] <= last ? 1u : 0u) << g;
                    const float by = l == 0.f ? 0.f : 1.f / l;  // no token seen: zeros; NaN stays
                    for (int c = 16 * half; c < N; c += 32) {
                        float o[16];
                        tmem_load(tm_o + c + mine, o);
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = broken >> (c / 32) & 1u ? __int_as_float(0x7fffffff) : l == 0.f ? 0.f : o[j] * by;
#pragma unroll
                        for (int j = 0; j < 16; j += 8)
                            if (real && c + j < a.D)
                                *reinterpret_cast<uint4*>(dst + c + j) =
                                    make_uint4(pack<T>(o[j], o[j + 1]), pack<T>(o[j + 2], o[j + 3]), pack<T>(o[j + 4], o[j + 5]), pack<T>(o[j + 6], o[j + 7]));
                    }
                    fence_before();
                }
            } else if (real) {
                for (int d = 8 * half; d < a.D; d += 16) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
            }
        } else if (warp < SOFT + UNPACK) {
            // ================================================================ unpacking: warp = 16 tokens of each tile
            // What a tile needs is asked for while the tile before it is unpacked: the block table's entry first, then codes and parameters, each
            // as soon as its registers are free.  The parameters of the 16 tokens are looked over once, and handed round through shared memory in
            // the order of their use.
            const int part = warp - SOFT, tiles_a_page = a.page / KV4_TILE;
            const int step_col = (KEYS / KV4_TILE) / tiles_a_page, step_in = (KEYS / KV4_TILE) % tiles_a_page;
            int looked = 0, col = part / tiles_a_page, in = part % tiles_a_page;  // tiles looked up so far; column and place in the page of the next
            const int wanted = n > 0 && part * KV4_TILE <= end ? static_cast<int>((end - part * KV4_TILE) / KEYS) + 1 : 0;  // tiles that exist for this warp
            int held = -1, held_in = 0;  // page and place of the tile looked up last
            auto look = [&] {
                held_in = in;
                held = looked < wanted ? table[col] : -1;
                ++looked;
                col += step_col, in += step_in;
                if (in >= tiles_a_page) in -= tiles_a_page, ++col;
            };
            auto find = [&]() -> const uint8_t* {  // of the tile looked up last
                if (held >= 0 && held < a.pages) return a.cache + ((static_cast<long long>(held) * a.kv_heads + kvh) * tiles_a_page + held_in) * TB;
                if (looked <= wanted && lane == 0) atomicCAS(a.status, 0, ST_BAD_SLOT);
                return nullptr;
            };
            // keys: lane = row (16) and half of the t's; values: lane = (c, h) and half of the groups (neighbouring lanes differ in c & 1 and
            // h, which spreads their stores over the banks); parameters: lane = token (16) and half of the groups
            constexpr int GP = (G + 1) / 2;
            const int row = lane & 15, th = lane >> 4, h = lane >> 1 & 1, c8 = (lane & 1) | (lane >> 1 & 6), g0 = th * GP;
            uint32_t kw[2][G], vw[4][GP], par[4][GP];  // codes; key scale, key minimum, value scale, value minimum of token `row`, groups g0 ..
            auto load_par = [&](const uint8_t* src) {
#pragma unroll
                for (int which = 0; which < 4; ++which)
#pragma unroll
                    for (int k = 0; k < GP; ++k)
                        par[which][k] = src && g0 + k < G ? __ldg(reinterpret_cast<const unsigned short*>(src + kv4_param(G, row, which, g0)) + k) : 0u;
            };
            auto load_keys = [&](const uint8_t* src) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (src) global_words<G>(kw[j], src + (row * 4 + 2 * th + j) * 4 * G);
            };
            auto load_values = [&](const uint8_t* src) {
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    if (src) {
                        const uint8_t* w = src + kv4_value_half(G, 8 * h + 2 * t, 32 * g0 + 4 * c8);
                        if constexpr (G == 4) {
                            global_words<GP>(vw[t], w);
                        } else {
#pragma unroll
                            for (int k = 0; k < GP; ++k) vw[t][k] = g0 + k < G ? __ldg(reinterpret_cast<const uint32_t*>(w) + k) : 0u;
                        }
                    }
            };
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int g = 0; g < G; ++g) kw[j][g] = 0;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int k = 0; k < GP; ++k) vw[t][k] = 0;
            look();
            const uint8_t* src = find();
            load_par(src);
            load_keys(src);
            load_values(src);
            look();
            for (int i = 0; ok && i < n; ++i) {
                const int at = done + i, buf = at & 1;
                const long long token0 = (static_cast<long long>(i) * (KEYS / KV4_TILE) + part) * KV4_TILE;
                const uint8_t* next = find();
                look();
                // ---- parameters (those of a missing page are 0: so are its keys and values)
#pragma unroll
                for (int k = 0; k < GP; ++k) {
                    // Nothing that is not finite goes into P V, where it would reach rows that do not see the token: it is left out here, and the
                    // rows that see it become NaN in this group at the end.  Behind the last token, where anything may lie, nothing is taken.
                    if (g0 + k < G) {
                        const bool seen = token0 + row <= end, fine = finite_half(par[2][k]) && finite_half(par[3][k]);
                        if (seen && !fine) atomicMin(&sh.first_broken[items & 7][g0 + k], static_cast<int>(token0) + row);
                        sh.kpar[part][row][g0 + k] = static_cast<uint16_t>(par[0][k]);
                        sh.kpar[part][row][4 + g0 + k] = static_cast<uint16_t>(par[1][k]);
                        sh.vpar[part][0][g0 + k][row] = static_cast<uint16_t>(seen && fine ? par[2][k] : 0u);
                        sh.vpar[part][1][g0 + k][row] = static_cast<uint16_t>(seen && fine ? par[3][k] : 0u);
                    }
                }
                load_par(next);
                __syncwarp();
                // ---- keys
                if (!(ok = wait(sh.k_empty[buf], (at >> 1) + 1, ST_TIMEOUT_EMPTY))) break;
                {
                    const uint4 sm = *reinterpret_cast<const uint4*>(sh.kpar[part][row]);
                    const uint32_t pw[4] = {sm.x, sm.y, sm.z, sm.w};  // scales 0, 1 | 2, 3; minima 0, 1 | 2, 3
                    uint8_t* kd = s_k + buf * DB * BLOCK + (part * KV4_TILE + row) * 128;
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const uint32_t both = g & 1 ? 0x3232 : 0x1010;
                        const __half2 s2 = as_half2(__byte_perm(pw[g / 2], 0, both)), m2 = as_half2(__byte_perm(pw[2 + g / 2], 0, both));
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            __half2 c[4];
                            code_pairs(kw[j][g], c);
                            uint32_t v[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) v[k] = as_word(__hfma2(c[k], s2, m2));
                            const int d = 32 * g + 8 * (2 * th + j);
                            *reinterpret_cast<uint4*>(kd + d / 64 * BLOCK + ((d % 64 / 8) ^ (row & 7)) * 16) =
                                make_uint4(v[0], v[1], v[2], v[3]);  // (the queries' dims are in the same order)
                        }
                    }
                }
                if (lane == 0) {
                    if (src) atomicOr(&sh.there[at & 3], 1u << part);
                    else atomicAnd(&sh.there[at & 3], ~(1u << part));
                }
                fence_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(sh.k_full[buf]));
                load_keys(next);
                // ---- values
                if (!(ok = wait(sh.v_empty[buf], (at >> 1) + 1, ST_TIMEOUT_EMPTY))) break;
#pragma unroll
                for (int k = 0; k < GP; ++k) {
                    const int g = g0 + k;
                    if (g < G) {
                        const uint4 s8 = *reinterpret_cast<const uint4*>(&sh.vpar[part][0][g][8 * h]), m8 = *reinterpret_cast<const uint4*>(&sh.vpar[part][1][g][8 * h]);
                        const uint32_t s2[4] = {s8.x, s8.y, s8.z, s8.w}, m2[4] = {m8.x, m8.y, m8.z, m8.w};  // token pairs
                        uint32_t out[4][4];  // [dim][token pair]
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            __half2 c[4];
                            code_pairs(vw[t][k], c);  // nibble n of both tokens
#pragma unroll
                            for (int d = 0; d < 4; ++d) out[d][t] = as_word(__hfma2(c[d], as_half2(s2[t]), as_half2(m2[t])));
                        }
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            const int dim = 32 * g + 4 * c8 + d, key = part * KV4_TILE + 8 * h;
                            *reinterpret_cast<uint4*>(s_v + (buf * 2 + key / 64) * VBLOCK + dim * 128 + ((key % 64 / 8) ^ (dim & 7)) * 16) =
                                make_uint4(out[d][0], out[d][1], out[d][2], out[d][3]);
                        }
                    }
                }
                fence_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(sh.v_full[buf]));
                load_values(next);
                src = next;
            }
        } else if (lane == 0 && n > 0) {
            // ================================================================ products, one thread
            const uint32_t d_s = shape(ROWS, KEYS), d_o = shape(ROWS, N);
            const uint32_t q = smem_u32(s_q), k0 = smem_u32(s_k), v0 = smem_u32(s_v), p = smem_u32(s_p);
            auto scores = [&](int i) {
                const int at = done + i, buf = at & 1;
                if (!wait_one(sh.k_full[buf], (at >> 1) & 1, ST_TIMEOUT_FULL)) return false;
                fence_after();
                for (int s = 0; s < N / 16; ++s)
                    product(tm_s + buf * KEYS, operand(q + s / 4 * BLOCK + s % 4 * 32), operand(k0 + buf * DB * BLOCK + s / 4 * BLOCK + s % 4 * 32), d_s, s > 0);
                commit(bar(sh.s_full[buf]));
                commit(bar(sh.k_empty[buf]));
                return true;
            };
            ok = wait_one(sh.q_full, items & 1, ST_TIMEOUT_FULL) && scores(0);
            for (int i = 0; ok && i < n; ++i) {
                const int at = done + i, buf = at & 1;
                if (i + 1 < n && !(ok = scores(i + 1))) break;
                if (!(ok = wait_one(sh.v_full[buf], (at >> 1) & 1, ST_TIMEOUT_FULL) && wait_one(sh.p_full, at & 1, ST_TIMEOUT_FULL))) break;
                fence_after();
                for (int s = 0; s < KEYS / 16; ++s)
                    product(tm_o, operand(p + s / 4 * BLOCK + s % 4 * 32), operand(v0 + (buf * 2 + s / 4) * VBLOCK + s % 4 * 32), d_o, i > 0 || s > 0);
                commit(bar(sh.pv_done));
                commit(bar(sh.v_empty[buf]));
            }
        }
        if (!ok || *ctl.flag) break;
        done += n;
        items += n > 0;
    }
    // every product has ended where the last P V was waited for; after a wait that ran out, wait for what was issued (bounded) before freeing
    __syncwarp();
    if (warp == SOFT + UNPACK) {
        if (lane == 0 && *ctl.flag) {
            commit(bar(sh.drain));
            for (int spin = 0; spin < 1 << 20 && !mbar_try_wait(bar(sh.drain), 0); ++spin) {}
        }
        __syncwarp();
    }
    __syncthreads();
    if (warp == SOFT + UNPACK) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sh.tmem) : "memory");
    }
}

template <class T, int G> cudaError_t launch(const Kv4AttnArgs& a, long long max_q_len, cudaStream_t st) {
    constexpr int DB = (32 * G + 63) / 64, smem = 1024 + 3 * DB * BLOCK + 4 * 32 * G * 128 + 2 * BLOCK;
    static std::atomic<unsigned long long> allowed{0};
    const cudaError_t e = allow_shared_once(reinterpret_cast<const void*>(kv4_prompt_kernel<T, G>), smem, allowed);
    if (e != cudaSuccess) return e;
    const long long q_tiles = (max_q_len * (a.heads / a.kv_heads) + ROWS - 1) / ROWS;
    const dim3 grid(static_cast<unsigned>(a.batch * a.kv_heads), static_cast<unsigned>(q_tiles < 65535 ? q_tiles : 65535));
    kv4_prompt_kernel<T, G><<<grid, THREADS, smem, st>>>(a);
    return cudaGetLastError();
}

template <class T> cudaError_t by_groups(const Kv4AttnArgs& a, long long max_q_len, cudaStream_t st) {
    switch (kv4_groups(a.D)) {
        case 1: return launch<T, 1>(a, max_q_len, st);
        case 2: return launch<T, 2>(a, max_q_len, st);
        case 3: return launch<T, 3>(a, max_q_len, st);
        default: return launch<T, 4>(a, max_q_len, st);
    }
}

}  // namespace

cudaError_t kv4_attention_prompt(const Kv4AttnArgs& a, bool bf16, long long max_q_len, cudaStream_t st) {
    return bf16 ? by_groups<__nv_bfloat16>(a, max_q_len, st) : by_groups<__half>(a, max_q_len, st);
}

}  // namespace cfb
