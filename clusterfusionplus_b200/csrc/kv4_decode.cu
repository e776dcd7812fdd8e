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
//  - values: O^T = V^T P^T, again codes as the 16-row operand (two tokens in one word's halves, so no re-pairing).  P goes in as two fp16 numbers,
//    p = h + l, transposed, and so does its product with the groups' scales, two tokens at a time: q = h s rounded and t = (h s - q) + l s, of
//    which the first part is exact.  The minima and a row of ones times h and l: sum p m of every group and the softmax's denominator.  So
//    probabilities keep 22 bits and results are as near as 32-bit arithmetic brings them (fp16: off by 0.206e-3 of the result, of which its own
//    rounding is 0.203e-3); h and q alone, with 8 (h s - q) added to the group's sum, gave 0.26e-3 and 4 % less time.
// Queries are scaled by a power of two to at most 2^10 before they become fp16: exact for fp16 and bf16 inputs of any size
// down to 2^-20 of their row's largest, off by less than 2^-30 of it below.  Both p and q = p s have to stay among fp16's normal numbers: a
// token far below the maximum may still carry the result where the maximum's value is next to nothing, and scales of 2^-8 are usual.  So p
// is kept as large as the scales allow, up to 2^13 with scales up to 4, and lower only once a warp meets larger ones (up to 8734, the widest
// fp16 range / 15): p s <= 2^15 always.  With p <= 4 whatever the scales, values of std 0.005 beside a token 10 nats above
// them were off by 7e-3, where the rounding of bf16 results is 1.7e-3.  It costs 1 % of the line's time.
//
// Two ways to deal out the work, both without a wait between CTAs and with the same bits every time:
//  - little work: a cluster of up to 8 CTAs takes a (request, cached head), its tiles go round the warps, the partial results meet in
//    distributed shared memory.  One launch, no workspace.
//  - much work: the tiles of all requests in one line, cut into equal pieces, one for each CTA that fits on the GPU, so that requests of any
//    lengths keep every SM busy to the end; what a cut divides goes to a workspace and a second launch joins it.
// Each warp streams its tiles through its own ring of shared memory by cp.async.
//
// Measured on the GPU: one request of 4096 tokens, 32 heads of 128 (21 MB, 3.3 us of reading), 11.2 us: a CTA's queries, first loads
// and the joining take 4 us.  64 requests of up to 8192 tokens, 8 cached heads under 32 (350 MB, 54 us): line and
// join 97 us (3.6 TB/s; the join alone takes 8 us, most of them under the line's end).  No unit is full: ~390 instructions a tile fill 57 % of the
// issue slots (ALU 45 %, memory 45 %, matrix pipe 32 % of their rates), because the chain of a tile, load to last product, is waited for with 4
// warps a scheduler, which is what 128 registers leave.
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
constexpr int STAGES = 2;            // pairs of tiles in a warp's ring
constexpr int MAX_CLUSTER = 8;
constexpr int RUN = 8;               // pairs of tiles that a warp sums up before it puts the sums by (16: half the cost, twice the error)
constexpr float LOWEST = -3.0e38f;   // reference of a result without tokens: finite, so that no difference of infinities is formed

template <class T> __device__ __forceinline__ T from_float(float v);
// (a result is a mean of values within fp16's range: what the sums' rounding puts beyond it is not infinity; NaN stays)
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v > 65504.f ? 65504.f : v < -65504.f ? -65504.f : v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Shared memory by the offset in the CTA's dynamic part: a pointer that may be null loses its address space, and generic loads with 64-bit
// arithmetic cost a tenth of the instructions of a tile.
extern __shared__ __align__(16) uint8_t smem[];

template <int N> __device__ __forceinline__ void load_words(uint32_t (&x)[N], uint32_t p) {  // N 32-bit words, 4 N-byte aligned for N = 1, 2, 4
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(smem + p);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(smem + p);
        x[0] = v.x, x[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = *reinterpret_cast<const uint32_t*>(smem + p + 4 * i);
    }
}
__device__ __forceinline__ uint32_t load_word(uint32_t p) { return *reinterpret_cast<const uint32_t*>(smem + p); }
__device__ __forceinline__ uint32_t load_half(uint32_t p) { return *reinterpret_cast<const uint16_t*>(smem + p); }

// N consecutive fp16 numbers as floats (2 N-byte aligned for even N)
template <int N> __device__ __forceinline__ void load_halves(float (&x)[N], uint32_t p) {
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
        for (int i = 0; i < N; ++i) x[i] = __half2float(__ushort_as_half(static_cast<unsigned short>(load_half(p + 2 * i))));
    }
}

// word i: the i-th fp16 numbers at a (low half) and at b
template <int N> __device__ __forceinline__ void pair_halves(uint32_t (&x)[N], uint32_t a, uint32_t b) {
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
        for (int i = 0; i < N; ++i) x[i] = load_half(a + 2 * i) | load_half(b + 2 * i) << 16;
    }
}

__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
    const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&y);
}

// (a + l) b - ab, ab being the rounded product a b
__device__ __forceinline__ uint32_t rest_half2(uint32_t a, uint32_t l, uint32_t b, uint32_t ab) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b), __hneg2(*reinterpret_cast<const __half2*>(&ab)));  // exact
    const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&l), *reinterpret_cast<const __half2*>(&b), r);
    return *reinterpret_cast<const uint32_t*>(&y);
}

// 0xffff in each half that holds a finite fp16 number, else 0
__device__ __forceinline__ uint32_t finite_halves(uint32_t x) {
    const uint32_t over = (((x & 0x7fff7fffu) + 0x04000400u) >> 15) & 0x00010001u;  // 1: exponent all ones
    return ~(over * 0xffffu);
}

// what a request is made of
struct Request {
    int first, rows, per;    // first query row; query rows times heads of one cached head; heads of one cached head
    long long before, cap;   // tokens ahead of its queries; tokens that its table can name
    const int* table;

    __device__ __forceinline__ Request(const Kv4AttnArgs& a, int b) {
        int n = 1;
        first = b;
        if (a.qo_indptr) {
            first = a.qo_indptr[b];
            n = first < 0 ? 0 : min(a.qo_indptr[b + 1], static_cast<int>(a.rows)) - first;
        }
        per = a.heads / a.kv_heads;
        rows = n > 0 ? n * per : 0;  // at most rows * heads of the call: fits
        cap = a.table_width * a.page;
        before = static_cast<long long>(a.kv_lens[b]) - n;
        table = a.table + b * a.table_stride;
    }
    // tiles that the queries of the request see, at least 1
    __device__ __forceinline__ int tiles() const {
        const long long seen = min(before + rows / per, cap);
        return seen <= 0 ? 1 : static_cast<int>((seen - 1) / KV4_TILE) + 1;
    }
};

template <class T> __device__ __forceinline__ void write_out(const Kv4AttnArgs& a, int first, int per, int kvh, int r, int d, float num, float den) {
    if (d < a.D)  // no token seen: zeros; a NaN stays one
        static_cast<T*>(a.out)[(static_cast<long long>(first + r / per) * a.heads + kvh * per + r % per) * a.D + d] = from_float<T>(den == 0.f ? 0.f : num / den);
}

// ---------------------------------------------------------------------------------------------------- query rows
// Up to 8 NT rows of one (request, cached head): row r is query r / per, head kvh * per + r % per.
template <int G, int NT> struct Rows {
    uint32_t qa[NT][G][2], qb[NT][G][2], qm[NT];  // B operands: even dims, odd dims / 16, sums of the groups
    float factor[NT][2];                          // of a column's scores
    int last[NT][2];                              // the last token that a column's query sees, -1 for none
    int all_see, most;                            // tokens up to all_see are seen by every row, none after `most` by any

    template <class T> __device__ __forceinline__ void load(const Kv4AttnArgs& a, const Request& own, int kvh, int r0);
};

template <int G, int NT>
template <class T>
__device__ __forceinline__ void Rows<G, NT>::load(const Kv4AttnArgs& a, const Request& own, int kvh, int r0) {
    constexpr int PAIRS = (G + 1) / 2;
    const int lane = threadIdx.x & 31, g8 = lane >> 2, t = lane & 3, per = own.per, rows = own.rows;
    all_see = 0x7fffffff, most = -1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = r0 + nt * 8 + g8;
        const bool real = r < rows;
        float q[G][8], top = 0.f;
        if (real) {
            const T* src = static_cast<const T*>(a.query) + static_cast<long long>(own.first + r / per) * a.q_ts + (kvh * per + r % per) * a.q_hs;
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
        const int e = query_exponent(top);
        const float up = query_scaling(e);
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
        const long long see = own.before + r / per;
        const int end = real ? static_cast<int>(min(see, own.cap - 1)) : -1;
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
}

// ---------------------------------------------------------------------------------------------------- accumulators
template <int G, int NT, bool PUT_BY> struct Acc {
    static constexpr int DP = 32 * G, LINE = DP + 4;
    float o[NT][2 * G][4];  // numerators in units of 2^-24 and 2^-20
    float low[NT][4];       // row g: group g's sum of p times the minimum; row G: the sum of p
    float m[NT][2];         // reference of a column: p = 2^(score - m), at most 2^room
    float den[NT][2];       // what low's row G was before the last put_by
    uint32_t kept;          // where this lane's numerators are that were put by, in shared memory
    bool any_kept;
    float room;
    uint32_t wide;          // 2^(15 - room) twice, fp16: no scale of a token that some row sees is larger
    bool first_tile;

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 2 * G; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[nt][i][j] = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) low[nt][j] = 0.f;
        }
    }
    __device__ __forceinline__ void reset(uint32_t keep_at) {  // of this warp: keep_bytes()
        clear();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = den[nt][0] = den[nt][1] = 0.f;
        first_tile = true, any_kept = false;
        room = 13.f, wide = 0x44004400u;
        kept = keep_at + (threadIdx.x & 31) * 16;
    }
    // eight numerators of this lane, of group g: its columns 2 t and 2 t + 1 in turn, four of o[2 g] and four of o[2 g + 1]
    __device__ __forceinline__ void numerators(int nt, int g, float (&x)[8]) const {
        const int t = threadIdx.x & 3;
        const float least[2] = {__shfl_sync(0xffffffffu, low[nt][0], g * 4 + t), __shfl_sync(0xffffffffu, low[nt][1], g * 4 + t)};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = fmaf(o[nt][2 * g][j], 16777216.f, least[j & 1]);
            x[4 + j] = fmaf(o[nt][2 * g + 1][j], 1048576.f, least[j & 1]);
        }
    }
    // Numerators that are put by: of each (nt, g) two times four, a lane's next to the other lanes'
    static __host__ __device__ constexpr int keep_bytes() { return PUT_BY ? NT * G * 2 * 32 * 16 : 0; }
    __device__ __forceinline__ float4& place(int nt, int g, int half) const { return *reinterpret_cast<float4*>(smem + kept + ((nt * G + g) * 2 + half) * 512); }
    __device__ __forceinline__ void add_kept(int nt, int g, float (&x)[8]) const {
        const float4 a = place(nt, g, 0), b = place(nt, g, 1);
        x[0] += a.x, x[1] += a.y, x[2] += a.z, x[3] += a.w, x[4] += b.x, x[5] += b.y, x[6] += b.z, x[7] += b.w;
    }
    __device__ __forceinline__ void keep(int nt, int g, const float (&x)[8]) const {
        place(nt, g, 0) = make_float4(x[0], x[1], x[2], x[3]);
        place(nt, g, 1) = make_float4(x[4], x[5], x[6], x[7]);
    }
    // The matrix instructions cut their sums off, by up to 2^-23 at each step, and the codes' and the minima's sums, which nearly cancel in the
    // result, each grow to some hundred times of it: 64 requests of 8192 tokens were off by 1.4e-3, of 131072 by 4e-2 (even probabilities).  So after every
    // RUN pairs of tiles their sum is added, rounded to nearest, to numbers in shared memory: 0.3e-3 and 0.7e-3, for 2 % of the time.
    __device__ __forceinline__ void put_by() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float x[8];
                numerators(nt, g, x);
                if (any_kept) add_kept(nt, g, x);
                keep(nt, g, x);
            }
            den[nt][0] += low[nt][0], den[nt][1] += low[nt][1];
        }
        any_kept = true;
        clear();
    }
    __device__ __forceinline__ void scale_kept(const float (&by)[NT][2]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                add_kept(nt, g, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= by[nt][j & 1];
                keep(nt, g, x);
            }
            den[nt][0] *= by[nt][0], den[nt][1] *= by[nt][1];
        }
    }
    template <int K> __device__ __forceinline__ void make_room(const uint32_t (&scales)[K]);
    template <int K> __device__ __forceinline__ void step(const int (&tile)[K], int token, const Rows<G, NT>& r, int lane);
    __device__ __forceinline__ void store(float* lines) const;
};

// scales beyond `wide` among the warp's: room for the greatest of them (one that is not finite makes its group NaN anyway)
template <int G, int NT, bool PUT_BY>
template <int K>
__device__ __forceinline__ void Acc<G, NT, PUT_BY>::make_room(const uint32_t (&scales)[K]) {
    uint32_t most = 0;
#pragma unroll
    for (int u = 0; u < K; ++u) {
        const uint32_t x = scales[u] & finite_halves(scales[u]) & 0x7fff7fffu;
        most = max(most, max(x & 0xffffu, x >> 16));
    }
    const int e = static_cast<int>(__reduce_max_sync(0xffffffffu, most) >> 10) - 14;  // the greatest is below 2^e
    if (e > 15 - static_cast<int>(room)) {
        room = static_cast<float>(15 - e);
        wide = static_cast<uint32_t>(e + 15) * 0x04000400u;  // (2^16 is infinity: nothing lies beyond)
    }
}

// K tiles of 16 tokens in a row, the first token of all `token`, the tiles at these offsets of shared memory
template <int G, int NT, bool PUT_BY>
template <int K>
__device__ __forceinline__ void Acc<G, NT, PUT_BY>::step(const int (&tile)[K], int token, const Rows<G, NT>& r, int lane) {
    constexpr int PAIRS = (G + 1) / 2;
    const int g8 = lane >> 2, t = lane & 3;

    // ---- scores
    float x[K][NT][4];
#pragma unroll
    for (int u = 0; u < K; ++u) {
        const uint32_t par0 = tile[u] + 512 * G + g8 * 8 * G, par1 = par0 + 64 * G;  // parameters of tokens g8 and g8 + 8
        uint32_t low0 = 0, low1 = 0;
        const int j = t % PAIRS;
        if constexpr (G % 2 == 0) {
            low0 = load_word(par0 + 2 * G + 4 * j);
            low1 = load_word(par1 + 2 * G + 4 * j);
        } else {
            low0 = load_half(par0 + 2 * G + 4 * j);
            low1 = load_half(par1 + 2 * G + 4 * j);
            if (2 * j + 1 < G) {
                low0 |= load_half(par0 + 2 * G + 4 * j + 2) << 16;
                low1 |= load_half(par1 + 2 * G + 4 * j + 2) << 16;
            }
        }
        if (2 * PAIRS < 4 && t >= 2 * PAIRS) low0 = low1 = 0;
        uint32_t k0[G], k1[G];
        float s0[G], s1[G];
        load_words<G>(k0, tile[u] + g8 * 16 * G + t * 4 * G);
        load_words<G>(k1, tile[u] + (g8 + 8) * 16 * G + t * 4 * G);
        load_halves<G>(s0, par0);
        load_halves<G>(s1, par1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            mma_16816_zero(x[u][nt], low0, low1, 0u, 0u, r.qm[nt], 0u);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[u][nt][i] *= 5.9604644775390625e-08f;  // 2^-24: the codes' unit
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t h0 = k0[g] >> 8, h1 = k1[g] >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float c[4];
                mma_16816_zero(c, k0[g] & 0x000f000fu, k1[g] & 0x000f000fu, h0 & 0x000f000fu, h1 & 0x000f000fu, r.qa[nt][g][0], r.qa[nt][g][1]);
                mma_16816(c, k0[g] & 0x00f000f0u, k1[g] & 0x00f000f0u, h0 & 0x00f000f0u, h1 & 0x00f000f0u, r.qb[nt][g][0], r.qb[nt][g][1]);
                x[u][nt][0] = fmaf(s0[g], c[0], x[u][nt][0]);
                x[u][nt][1] = fmaf(s0[g], c[1], x[u][nt][1]);
                x[u][nt][2] = fmaf(s1[g], c[2], x[u][nt][2]);
                x[u][nt][3] = fmaf(s1[g], c[3], x[u][nt][3]);
            }
        }
    }
    // ---- softmax: x becomes the binary logarithm of p.  The reference is set so that the greatest p is a quarter of the most and moves when one
    // exceeds that: seldom after the first tiles.  Each lane looks at one token's scales (two groups of four), whose greatest decides how much
    // p may be; tokens that no row sees do not count.
    const bool whole = token + K * KV4_TILE - 1 <= r.all_see;
    bool rise = first_tile;
    uint32_t scales[K];
#pragma unroll
    for (int u = 0; u < K; ++u) {
        const int row = G == 4 ? lane >> 1 : lane & 15;
        const uint32_t at = tile[u] + 512 * G + row * 8 * G + 4 * G;
        if constexpr (G == 4) scales[u] = load_word(at + (lane & 1) * 4);
        else if constexpr (G == 1) scales[u] = load_half(at);
        else if constexpr (G == 2) scales[u] = load_word(at);
        else scales[u] = lane < 16 ? load_word(at) : load_half(at + 4);
        if (!whole && token + u * KV4_TILE + row > r.most) scales[u] = 0;
        rise |= !__hble2(__habs2(*reinterpret_cast<const __half2*>(&scales[u])), *reinterpret_cast<const __half2*>(&wide));
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < K; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[u][nt][j] = fmaf(x[u][nt][j], r.factor[nt][j & 1], -m[nt][j & 1]);
    if (!whole) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int u = 0; u < K; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (token + u * KV4_TILE + g8 + (j >> 1) * 8 > r.last[nt][j & 1]) x[u][nt][j] = -INFINITY;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float top = fmaxf(fmaxf(x[0][nt][0], x[0][nt][2]), fmaxf(x[0][nt][1], x[0][nt][3]));
        if constexpr (K == 2) top = fmaxf(top, fmaxf(fmaxf(x[K - 1][nt][0], x[K - 1][nt][2]), fmaxf(x[K - 1][nt][1], x[K - 1][nt][3])));
        rise |= top > room;
    }
    if (__any_sync(0xffffffffu, rise)) {
        make_room(scales);
        float kept_by[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float top = fmaxf(x[0][nt][c], x[0][nt][c + 2]);
                if constexpr (K == 2) top = fmaxf(top, fmaxf(x[K - 1][nt][c], x[K - 1][nt][c + 2]));
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                // a column's first tiles set its reference; one that sees nothing of them sees nothing of later ones
                const float up = (first_tile || top > room) && top != -INFINITY ? top - (room - 2.f) : 0.f;
                m[nt][c] += up;
#pragma unroll
                for (int u = 0; u < K; ++u) x[u][nt][c] -= up, x[u][nt][c + 2] -= up;
                const float keep = first_tile ? 1.f : ex2(-up);
                kept_by[nt][c] = keep;
                low[nt][c] *= keep;
#pragma unroll
                for (int q = 0; q < 2 * G; ++q) o[nt][q][c] *= keep, o[nt][q][c + 2] *= keep;
            }
        first_tile = false;
        if (PUT_BY && any_kept) scale_kept(kept_by);
    }
    // ---- values: scales of tokens 2 t, 2 t + 1 (sa) and 2 t + 8, 2 t + 9 (sb), group by group; minima likewise, of group g8
#pragma unroll
    for (int u = 0; u < K; ++u) {
        const uint32_t pv = tile[u] + 512 * G + 2 * t * 8 * G + 4 * G;
        uint32_t sa[G], sb[G], ma = 0, mb = 0;
        pair_halves<G>(sa, pv, pv + 8 * G);
        pair_halves<G>(sb, pv + 64 * G, pv + 72 * G);
        if (g8 < G) {
            const uint32_t pm = pv + 2 * G + 2 * g8;
            ma = load_half(pm) | load_half(pm + 8 * G) << 16;
            mb = load_half(pm + 64 * G) | load_half(pm + 72 * G) << 16;
        } else if (g8 == G) ma = mb = 0x3c003c00u;  // ones
        uint32_t v0[G], v1[G];
        load_words<G>(v0, tile[u] + 256 * G + lane * 4 * G);
        load_words<G>(v1, tile[u] + 384 * G + lane * 4 * G);
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
                        const int see = r.last[nt][c] - token - u * KV4_TILE;  // tokens 0 .. see of the tile
                        const uint32_t seen = see < 0 ? 0u : see >= 15 ? 0xffffu : (2u << see) - 1u;
                        if (g8 < G && (tokens & seen)) low[nt][c] = __int_as_float(0x7fffffff);
                    }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            uint32_t h[2], l[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float a = ex2(x[u][nt][2 * i]), b = ex2(x[u][nt][2 * i + 1]);
                h[i] = pack_half2(a, b);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
                l[i] = transpose_8x8(pack_half2(a - f.x, b - f.y));
                h[i] = transpose_8x8(h[i]);
            }
            const uint32_t p0 = h[0], p1 = h[1];
            mma_16816(low[nt], ma, 0u, mb, 0u, p0, p1);
            uint32_t t0[G], t1[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t h0 = v0[g] >> 8, h1 = v1[g] >> 8, q0 = mul_half2(p0, sa[g]), q1 = mul_half2(p1, sb[g]);
                mma_16816(o[nt][2 * g], v0[g] & 0x000f000fu, h0 & 0x000f000fu, v1[g] & 0x000f000fu, h1 & 0x000f000fu, q0, q1);
                mma_16816(o[nt][2 * g + 1], v0[g] & 0x00f000f0u, h0 & 0x00f000f0u, v1[g] & 0x00f000f0u, h1 & 0x00f000f0u, q0, q1);
                t0[g] = rest_half2(p0, l[0], sa[g], q0), t1[g] = rest_half2(p1, l[1], sb[g], q1);
            }
            mma_16816(low[nt], ma, 0u, mb, 0u, l[0], l[1]);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t h0 = v0[g] >> 8, h1 = v1[g] >> 8;
                mma_16816(o[nt][2 * g], v0[g] & 0x000f000fu, h0 & 0x000f000fu, v1[g] & 0x000f000fu, h1 & 0x000f000fu, t0[g], t1[g]);
                mma_16816(o[nt][2 * g + 1], v0[g] & 0x00f000f0u, h0 & 0x00f000f0u, v1[g] & 0x00f000f0u, h1 & 0x00f000f0u, t0[g], t1[g]);
            }
        }
    }
}

// this warp's result: COLS lines of DP numerators, reference and denominator
template <int G, int NT, bool PUT_BY> __device__ __forceinline__ void Acc<G, NT, PUT_BY>::store(float* lines) const {
    const int lane = threadIdx.x & 31, g8 = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float* line = lines + (nt * 8 + 2 * t + c) * LINE;
            const float sum = __shfl_sync(0xffffffffu, low[nt][c] + den[nt][c], G * 4 + t);
            if (g8 == 0) line[DP] = sum == 0.f ? LOWEST : m[nt][c], line[DP + 1] = sum;  // nothing seen: no reference either
        }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float x[8];
            numerators(nt, g, x);
            if (PUT_BY && any_kept) add_kept(nt, g, x);
#pragma unroll
            for (int c = 0; c < 2; ++c)
                *reinterpret_cast<float4*>(lines + (nt * 8 + 2 * t + c) * LINE + 32 * g + 4 * g8) = make_float4(x[c], x[4 + c], x[2 + c], x[6 + c]);
        }
}

// ---------------------------------------------------------------------------------------------------- a warp's tiles
// Tiles from .. to of a request go round the units (warps) in pairs, through each warp's ring.  Lane l looks up the l-th of 32 tiles at a
// time in the block table, 32 tiles ahead of their use.  Two tiles a step: the waits, the bookkeeping and the vote on the
// maximum are paid once for both.
template <int G> struct Feed {
    static constexpr int TB = kv4_tile_bytes(G);
    const Kv4AttnArgs& a;
    const int lane;
    const uint32_t ring;  // offset in shared memory
    const int* table;
    int kvh, start, step, count, issued, in, out;  // tiles of this warp; tiles asked for; the stages to be filled and used next
    unsigned there;       // bits 2 s, 2 s + 1: the tiles in stage s exist (their pages lie in the cache)
    long long now, next;  // this lane's tile of the present 32 and of the next: its index in the cache, -1 for none

    __device__ __forceinline__ Feed(const Kv4AttnArgs& args, int warp) : a(args), lane(threadIdx.x & 31), ring(warp * STAGES * 2 * TB) {}
    __device__ __forceinline__ long long look(int base) const {
        const int i = base + lane;
        if (i >= count) return -1;
        const int tiles_a_page = a.page / KV4_TILE, tile = start + (i >> 1) * step + (i & 1), col = tile / tiles_a_page, held = table[col];
        if (held < 0 || held >= a.pages) {
            atomicCAS(a.status, 0, ST_BAD_SLOT);
            return -1;
        }
        return (static_cast<long long>(held) * a.kv_heads + kvh) * tiles_a_page + (tile - col * tiles_a_page);
    }
    // returns the pairs of this warp; pair i begins with tile from + 2 (unit + i units)
    __device__ __forceinline__ int begin(const int* t, int head, int from, int to, int unit, int units) {
        const int pairs = (to - from + 1) / 2, mine = pairs > unit ? (pairs - unit + units - 1) / units : 0;
        table = t, kvh = head, start = from + 2 * unit, step = 2 * units, issued = in = out = 0, there = 0;
        count = 2 * mine - (mine > 0 && ((to - from) & 1) && unit + (mine - 1) * units == pairs - 1);
        now = look(0);
        next = look(32);
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) issue();
        return mine;
    }
    __device__ __forceinline__ void issue() {
        if (issued < count) {
            const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + ring + in * 2 * TB + lane * 16;
            there &= ~(3u << 2 * in);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const long long tile = __shfl_sync(0xffffffffu, now, (issued & 31) + u);  // past the last: -1
                if (tile >= 0) {
                    there |= 1u << (2 * in + u);
                    const uint8_t* src = a.cache + tile * TB + lane * 16;
#pragma unroll
                    for (int i = 0; i < (TB / 16 + 31) / 32; ++i)
                        if (i * 32 + lane < TB / 16) cp_async_16(dst + u * TB + i * 512, src + i * 512);
                }
            }
            in = in == STAGES - 1 ? 0 : in + 1;
            issued += 2;
            if ((issued & 31) == 0) {
                now = next;
                next = look(issued + 32);
            }
        }
        cp_async_commit();
    }
    // waits for the next pair and gives it to `acc`; `token`: its first
    template <int NT, bool PUT_BY> __device__ __forceinline__ void take(Acc<G, NT, PUT_BY>& acc, int token, const Rows<G, NT>& rows) {
        cp_async_wait<STAGES - 2>();
        __syncwarp();
        const int tile = static_cast<int>(ring + out * 2 * TB);
        const unsigned both = there >> 2 * out & 3u;
        out = out == STAGES - 1 ? 0 : out + 1;
        issue();  // into the stage that the whole warp is done with
        if (both == 3u) acc.template step<2>({tile, tile + TB}, token, rows, lane);
        else if (both == 1u) acc.template step<1>({tile}, token, rows, lane);
        else if (both == 2u) acc.template step<1>({tile + TB}, token + KV4_TILE, rows, lane);
    }
};

// shared memory of the rings, and in their place later the warps' results; what is put by lies behind
template <int G, int NT> __host__ __device__ constexpr int shared_bytes() {
    constexpr int ring = W * STAGES * 2 * kv4_tile_bytes(G), merge = W * 8 * NT * (32 * G + 4) * 4;
    return ring > merge ? ring : merge;
}

// The results of the CTA's warps for element e = (column, dim), joined: numerator, denominator, reference
template <int G, int NT> __device__ __forceinline__ void join_warps(const float* lines, int c, int d, float& num, float& den, float& top) {
    constexpr int DP = 32 * G, COLS = 8 * NT, LINE = DP + 4;
    top = LOWEST, num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, lines[(w * COLS + c) * LINE + DP]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float* line = lines + (w * COLS + c) * LINE;
        const float k = ex2(line[DP] - top);
        num = fmaf(k, line[d], num);
        den = fmaf(k, line[DP + 1], den);
    }
}

// ---------------------------------------------------------------------------------------------------- little work
// LONG: no cluster, and sums are put by, in the shared memory that clusters need for what they exchange
template <class T, int G, int NT, bool LONG>
__global__ void __launch_bounds__(32 * W, NT == 1 ? 4 : 2) kv4_few_kernel(const Kv4AttnArgs a, int clusters) {
    constexpr int DP = 32 * G, COLS = 8 * NT, LINE = DP + 4;
    // what the CTAs of the cluster send one another: pieces of 128 numerators go to CTA (piece % cluster), every column's reference
    // and denominator to all
    constexpr int PIECES = (COLS * DP + 32 * W - 1) / (32 * W);
    __shared__ float received[LONG ? 1 : (PIECES + MAX_CLUSTER) * 32 * W];
    __shared__ float terms[LONG ? 1 : MAX_CLUSTER][COLS][2];

    const int warp = threadIdx.x >> 5, cluster = LONG ? 1 : clusters;
    const int rank = cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int item = static_cast<int>(blockIdx.x / cluster), b = item / a.kv_heads, kvh = item - b * a.kv_heads;
    const Request own(a, b);
    const int units = cluster * W, unit = rank * W + warp;
    if (cluster > 1) cluster_arrive();  // waited for before the first store to a peer, which must have begun by then

    const int first_row = blockIdx.y * COLS;
    for (int r0 = first_row; r0 < own.rows; r0 += gridDim.y * COLS) {
        const long long end = min(own.before + (min(r0 + COLS, own.rows) - 1) / own.per, own.cap - 1);  // the last token that these rows see
        const int tiles = end < 0 ? 0 : static_cast<int>(end / KV4_TILE) + 1;
        Feed<G> feed(a, warp);
        const int pairs = feed.begin(own.table, kvh, 0, tiles, unit, units);
        Rows<G, NT> rows;
        rows.template load<T>(a, own, kvh, r0);
        Acc<G, NT, LONG> acc;
        acc.reset(shared_bytes<G, NT>() + warp * acc.keep_bytes());
        for (int i = 0; i < pairs; ++i) {
            feed.take(acc, 2 * (unit + i * units) * KV4_TILE, rows);
            if (LONG && i % RUN == RUN - 1) acc.put_by();
        }
        cp_async_wait<0>();
        __syncthreads();  // the rings are free
        float* lines = reinterpret_cast<float*>(smem);
        acc.store(lines + warp * COLS * LINE);
        __syncthreads();
        if (cluster > 1 && r0 == first_row) cluster_wait();
        const int cols = min(COLS, own.rows - r0);
        const int owned = (PIECES + cluster - 1) / cluster;  // pieces of one CTA, at most
        for (int e = threadIdx.x; e < cols * DP; e += 32 * W) {
            const int c = e / DP, d = e % DP;
            float num, den, top;
            join_warps<G, NT>(lines, c, d, num, den, top);
            if (cluster == 1) {
                write_out<T>(a, own.first, own.per, kvh, r0 + c, d, num, den);
            } else {
                const int piece = e / (32 * W), owner = piece % cluster;
                cluster_st_float(cluster_map(&received[(rank * owned + piece / cluster) * 32 * W + threadIdx.x], owner), num);
                if (d < cluster) {
                    cluster_st_float(cluster_map(&terms[rank][c][0], d), top);
                    cluster_st_float(cluster_map(&terms[rank][c][1], d), den);
                }
            }
        }
        if (cluster > 1) {
            cluster_sync_all();
            for (int piece = rank; piece * 32 * W < cols * DP; piece += cluster) {
                const int e = piece * 32 * W + threadIdx.x, c = e / DP;
                if (e >= cols * DP) break;
                float top = LOWEST, num = 0.f, den = 0.f;
                for (int k = 0; k < cluster; ++k) top = fmaxf(top, terms[k][c][0]);
                for (int k = 0; k < cluster; ++k) {
                    const float f = ex2(terms[k][c][0] - top);
                    num = fmaf(f, received[(k * owned + piece / cluster) * 32 * W + threadIdx.x], num);
                    den = fmaf(f, terms[k][c][1], den);
                }
                write_out<T>(a, own.first, own.per, kvh, r0 + c, e % DP, num, den);
            }
            if (r0 + gridDim.y * COLS < own.rows) cluster_sync_all();  // the next rows' results go to the same place
        } else {
            __syncthreads();
        }
    }
    if (cluster > 1 && first_row >= own.rows) cluster_wait();  // no rows
}

// ---------------------------------------------------------------------------------------------------- much work
// The line: request by request, cached head by cached head, 8 NT rows by 8 NT rows, AHEAD units for what each of these costs besides its
// tiles (queries, the first loads' latency, joining the warps: about 2 us, in which the CTA's warps do a dozen tiles), then
// its tiles, one unit each.  CTA c takes units c * chunk .. (c + 1) * chunk.
constexpr int AHEAD = 12;

struct Cut {  // what the CTA's first tile belongs to, for the join
    long long begin, end, chunk;  // of its tiles in the line; begin = -1: the CTA has no tiles
    int first, per, kvh, r0, cols, pad;
};

__host__ __device__ constexpr long long cuts_bytes(int ctas) { return (static_cast<long long>(ctas) * sizeof(Cut) + 15) / 16 * 16; }

__device__ __forceinline__ long long block_sum_before(long long v, long long* total, long long* buf) {  // exclusive prefix over the CTA's threads
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) buf[warp] = inc;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        if (w < warp) before += buf[w];
        all += buf[w];
    }
    *total = all;
    return before + inc - v;
}

template <class T, int G, int NT>
__global__ void __launch_bounds__(32 * W, NT == 1 ? 4 : 2) kv4_line_kernel(const Kv4AttnArgs a, int least) {
    constexpr int DP = 32 * G, COLS = 8 * NT, LINE = DP + 4;
    // all shared memory is dynamic: four CTAs with what they put by take an SM's to the last byte.  Where the rings will be:
    long long *sums = reinterpret_cast<long long*>(smem), *found = sums + W;
    const int tid = threadIdx.x, warp = tid >> 5;
    asm volatile("griddepcontrol.launch_dependents;");  // the join may be set up; it waits for this grid's end by itself

    // ---- where this CTA's piece lies
    auto weight = [&](const Request& q) { return static_cast<long long>(a.kv_heads) * ((q.rows + COLS - 1) / COLS) * (q.tiles() + AHEAD); };
    const int share = (a.batch + 32 * W - 1) / (32 * W);
    const int b0 = min(tid * share, a.batch), b1 = min(b0 + share, a.batch);
    long long mine = 0, total;
    for (int b = b0; b < b1; ++b) mine += weight(Request(a, b));
    const long long before = block_sum_before(mine, &total, sums);
    const long long chunk = max((total + gridDim.x - 1) / gridDim.x, static_cast<long long>(least));
    long long pos = blockIdx.x * chunk;
    const long long stop = min(pos + chunk, total);
    Cut* cut = static_cast<Cut*>(a.workspace) + blockIdx.x;
    if (pos >= stop) {
        if (tid == 0) cut->begin = -1;
        return;
    }
    if (before <= pos && pos < before + mine) {
        long long at = before;
        int b = b0;
        for (;; ++b) {
            const long long w = weight(Request(a, b));
            if (pos < at + w) break;
            at += w;
        }
        found[0] = b, found[1] = at;
    }
    __syncthreads();
    int b = static_cast<int>(found[0]);
    long long base = found[1];  // of request b in the line
    __syncthreads();
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + cuts_bytes(gridDim.x)) + static_cast<long long>(blockIdx.x) * 2 * COLS * LINE;
    float* lines = reinterpret_cast<float*>(smem);  // the warps' results, where the rings are

    // ---- piece by piece
    bool first_piece = true;
    if (tid == 0) cut->begin = -1;
    while (pos < stop) {
        const Request own(a, b);
        const long long w = weight(own);
        if (pos >= base + w) {
            base += w;
            ++b;
            continue;
        }
        const int nb = own.tiles(), q_tiles = (own.rows + COLS - 1) / COLS;
        const int item = static_cast<int>((pos - base) / (nb + AHEAD));
        const long long begin = base + static_cast<long long>(item) * (nb + AHEAD) + AHEAD;  // its first tile
        const int kvh = item / q_tiles, r0 = (item - kvh * q_tiles) * COLS, cols = min(COLS, own.rows - r0);
        const int from = static_cast<int>(max(pos - begin, 0ll)), to = static_cast<int>(min(static_cast<long long>(nb), stop - begin));
        const int count = to - from;
        if (to <= 0) break;  // the piece ends ahead of its tiles
        Feed<G> feed(a, warp);
        // no query of the request sees a token: its one tile is not looked at
        const int pairs = feed.begin(own.table, kvh, from, own.before + own.rows / own.per <= 0 ? from : to, warp, W);
        Rows<G, NT> rows;
        rows.template load<T>(a, own, kvh, r0);
        Acc<G, NT, true> acc;
        acc.reset(shared_bytes<G, NT>() + warp * acc.keep_bytes());
        for (int i = 0; i < pairs; ++i) {
            feed.take(acc, (from + 2 * (warp + i * W)) * KV4_TILE, rows);
            if (i % RUN == RUN - 1) acc.put_by();
        }
        cp_async_wait<0>();
        __syncthreads();  // the rings are free
        acc.store(lines + warp * COLS * LINE);
        __syncthreads();
        if (first_piece && tid == 0) *cut = Cut{begin, begin + nb, chunk, own.first, own.per, kvh, r0, cols, 0};
        const bool whole = count == nb;
        float* part = parts + (begin > blockIdx.x * chunk ? COLS * LINE : 0);  // a piece that begins here, or one begun before
        for (int e = tid; e < cols * DP; e += 32 * W) {
            const int c = e / DP, d = e % DP;
            float num, den, top;
            join_warps<G, NT>(lines, c, d, num, den, top);
            if (whole) {
                write_out<T>(a, own.first, own.per, kvh, r0 + c, d, num, den);
            } else {
                part[c * LINE + d] = num;
                if (d == 0) part[c * LINE + DP] = top, part[c * LINE + DP + 1] = den;
            }
        }
        __syncthreads();
        pos = begin + to;
        first_piece = false;
    }
}

constexpr int JT = 256;  // threads of a joining CTA

// CTA c - 1 belongs to the start of CTA c's piece of the line.  If that cuts a (request, head, rows) in two, it joins a share of its
// elements: all the cuts inside take one share each.
template <class T, int G, int NT>
__global__ void __launch_bounds__(JT) kv4_join_kernel(const Kv4AttnArgs a, int ctas) {
    constexpr int DP = 32 * G, COLS = 8 * NT, LINE = DP + 4;
    __shared__ float part[3][JT];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int c = blockIdx.x + 1, tid = threadIdx.x;
    const Cut cut = static_cast<const Cut*>(a.workspace)[c];
    if (cut.begin < 0 || cut.begin >= c * cut.chunk) return;  // no tiles, or no cut
    const int first = static_cast<int>(cut.begin / cut.chunk), n = static_cast<int>((cut.end - 1) / cut.chunk) - first + 1;  // n CTAs share it: n - 1 cuts
    const int all = cut.cols * DP, share = (all + n - 2) / (n - 1);
    const int from = min((c - first - 1) * share, all), to = min(from + share, all);
    const float* parts = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.workspace) + cuts_bytes(ctas)) + static_cast<long long>(first) * 2 * COLS * LINE;
    const int second = cut.begin > first * cut.chunk ? COLS * LINE : 0;  // the first CTA's part lies behind that of its piece's start
    int width = 1;
    while (width < to - from && width < JT) width *= 2;
    const int groups = JT / width, lane = tid % width, group = tid / width;
    for (int e0 = from; e0 < to; e0 += width) {
        const int e = e0 + lane, col = e / DP, d = e % DP;
        float top = LOWEST, num = 0.f, den = 0.f;
        if (e < to) {
#pragma unroll 4
            for (int k = group; k < n; k += groups) {
                const float* line = parts + static_cast<long long>(k) * 2 * COLS * LINE + (k == 0 ? second : 0) + col * LINE;
                const float m = line[DP], l = line[DP + 1], x = line[d], t = fmaxf(top, m), keep = ex2(top - t), f = ex2(m - t);
                num = fmaf(f, x, num * keep);
                den = fmaf(f, l, den * keep);
                top = t;
            }
        }
        for (int half = groups / 2; half > 0; half /= 2) {  // the upper half of the groups hands over to the lower
            part[0][tid] = top, part[1][tid] = num, part[2][tid] = den;
            __syncthreads();
            if (group < half) {
                const int at = tid + half * width;
                const float m = part[0][at], t = fmaxf(top, m), keep = ex2(top - t), f = ex2(m - t);
                num = fmaf(f, part[1][at], num * keep);
                den = fmaf(f, part[2][at], den * keep);
                top = t;
            }
            __syncthreads();
        }
        if (group == 0 && e < to) write_out<T>(a, cut.first, cut.per, cut.kvh, cut.r0 + col, d, num, den);
    }
}

// ---------------------------------------------------------------------------------------------------- launches
constexpr int SMS = 148;
constexpr int LEAST = 2 * W;  // tiles of a CTA's piece, at least: below that the join costs more than it saves
constexpr int DEEP = 4 * RUN;  // tiles that a warp of a cluster sums up at most
constexpr int places(int nt) { return SMS * (nt == 1 ? 4 : 2); }  // CTAs that find room on the GPU at once: __launch_bounds__ of the kernels
template <int NT> constexpr int line_ctas() { return places(NT); }

// CTAs to each of `items` (request, head, rows) of up to `tiles` tiles: as many as find room on the GPU at once (a CTA costs 4 us besides its tiles, a
// tile 0.5 us of a warp: 256 pairs of up to 2048 tokens 19.4 us with 2, 23.8 with 4; of 9 to 16 rows, where half as many find room, 37.9 with 1,
// 51.6 with 2, and 64 pairs 17.9 with 4, 26.1 with 8), but at least two tiles to a warp.
int cluster_size(long long items, long long tiles, int nt) {
    int cluster = 1;
    while (cluster < MAX_CLUSTER && items * cluster * 2 <= places(nt) && tiles >= 4 * W * cluster) cluster *= 2;
    return cluster;
}
// Sums of more tiles a warp are to be put by, for which a cluster, with what its CTAs exchange, has no shared memory
bool too_deep(int cluster, long long tiles) { return cluster > 1 && tiles > static_cast<long long>(DEEP) * W * cluster; }

template <class T, int G, int NT> cudaError_t launch(const Kv4AttnArgs& a, long long max_q_len, cudaStream_t st) {
    constexpr int COLS = 8 * NT;
    constexpr int smem = shared_bytes<G, NT>(), keep = W * Acc<G, NT, true>::keep_bytes();
    static_assert((smem + keep + 1024) * (NT == 1 ? 4 : 2) <= 228 * 1024, "the CTAs of an SM");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    cfg.blockDim = dim3(32 * W);
    cfg.stream = st;
    cfg.attrs = at;
    if (a.workspace) {
        constexpr int ctas = line_ctas<NT>();
        static std::atomic<unsigned long long> allowed{0};
        cudaError_t e = allow_shared_once(reinterpret_cast<const void*>(kv4_line_kernel<T, G, NT>), smem + keep, allowed);
        if (e != cudaSuccess) return e;
        cfg.gridDim = dim3(ctas);
        cfg.dynamicSmemBytes = smem + keep;
        e = cudaLaunchKernelEx(&cfg, kv4_line_kernel<T, G, NT>, a, LEAST);
        if (e != cudaSuccess) return e;
        cfg.gridDim = dim3(ctas - 1);
        cfg.blockDim = dim3(JT);
        cfg.dynamicSmemBytes = 0;
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, G, NT>, a, ctas);
    }
    const long long items = static_cast<long long>(a.batch) * a.kv_heads;
    const long long q_tiles = (max_q_len * (a.heads / a.kv_heads) + COLS - 1) / COLS;
    const long long tiles = (a.table_width * a.page + KV4_TILE - 1) / KV4_TILE;
    int cluster = cluster_size(items * q_tiles, tiles, NT);
    if (too_deep(cluster, tiles)) cluster = 1;  // only without a workspace
    const bool put_by = cluster == 1 && tiles > 2 * RUN * W;
    static std::atomic<unsigned long long> allowed[2] = {{0}, {0}};
    const auto kernel = put_by ? kv4_few_kernel<T, G, NT, true> : kv4_few_kernel<T, G, NT, false>;
    const cudaError_t e = allow_shared_once(reinterpret_cast<const void*>(kernel), smem + (put_by ? keep : 0), allowed[put_by]);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3(static_cast<unsigned>(items * cluster), static_cast<unsigned>(q_tiles < 65535 ? q_tiles : 65535));
    cfg.dynamicSmemBytes = smem + (put_by ? keep : 0);
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
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

long long kv4_few_workspace(long long heads, long long kv_heads, int D, long long max_q_len) {
    const int nt = max_q_len * (heads / kv_heads) <= 8 ? 1 : 2, ctas = nt == 1 ? line_ctas<1>() : line_ctas<2>();
    return cuts_bytes(ctas) + static_cast<long long>(ctas) * 2 * 8 * nt * (32 * kv4_groups(D) + 4) * 4;
}

// The line pays where requests of any length have to keep the GPU busy for long (from about 100 000 tiles of 16 tokens: 250 MB at
// head_dim 128; below, its second launch and its look at all lengths cost what the even spread gives.  Requests of mixed lengths, the line
// against clusters: 512 (request, head) pairs of up to 8192 tokens 85 : 115 us, 256 pairs 49 : 59, 128 pairs 33 : 34, 160 pairs of up to 1000
// tokens 16 : 12), and where there are too few pairs for clusters of 8 CTAs to reach half the GPU and each is long (8 heads x 32768
// tokens 21 : 34, x 16384 16 : 19, x 8192 13 : 12).  With 9 to 16 rows a pair takes twice as long and half as many CTAs find room: there more
// pairs than places keep the GPU even by themselves (1024 pairs of up to 8192 tokens 359 : 288, 512 pairs 187 : 152), and the line pays for
// fewer and long ones only (256 pairs of up to 16384 163 : 213, of up to 8192 122 : 112; 128 pairs of up to 16384 88 : 113; 16 pairs x 16384
// 31 : 37, 32 pairs 44 : 39).  And it takes what clusters must not sum up (too_deep).
bool kv4_few_uses_workspace(long long batch, long long heads, long long kv_heads, long long tokens, long long max_q_len) {
    const long long rows = max_q_len * (heads / kv_heads), cols = rows <= 8 ? 8 : 16;
    const long long items = batch * kv_heads * ((rows + cols - 1) / cols), tiles = (tokens + KV4_TILE - 1) / KV4_TILE;
    const bool few = items * MAX_CLUSTER < places(cols / 8) / 2;
    if (too_deep(cluster_size(items, tiles, static_cast<int>(cols / 8)), tiles)) return true;
    if (cols == 8) return items * tiles >= 100000 || (few && tiles >= 640);
    return tiles >= 640 && (few || (items <= places(2) && items * tiles >= 100000));
}

cudaError_t kv4_attention_few(const Kv4AttnArgs& a, bool bf16, long long max_q_len, cudaStream_t st) {
    return bf16 ? by_groups<__nv_bfloat16>(a, max_q_len, st) : by_groups<__half>(a, max_q_len, st);
}

}  // namespace cfb
