// Log probabilities of given tokens, the entropy of the distribution and its most probable tokens, from logits.
//
//   m = max_j x_j, z = sum_j e^(x_j - m), w = sum_j e^(x_j - m) (x_j - m)
//   log p_i = (x_i - m) - log z,   H = log z - w / z
//
// Nothing is formed as a difference of large numbers (no log-sum-exp is subtracted from a logit), so logits of any size keep
// fp32's relative precision.  The floor is reading the logits once; one exponential an element comes second (2047 rows of
// 50304: 32 us of reading, 23 us of MUFU).  One CTA takes a row, or a cluster of CTAs a row when there are few rows: the partial
// results meet in distributed shared memory, so there is no workspace and no second launch.  Measured on the GPU: 2047 rows of 50304 in
// fp16 with the top 20 58 us (3.55 TB/s, 55 % of the copy bandwidth; issue slots 72 %, exponentials 50 %, memory 47 %: 14 instructions an
// element; without the top k 46 us), in fp32 101 us (72); one row of 50304 in fp32 with the top 5 7.2 us.
//
// The top k (at most 32) cost a quarter more: every thread remembers its greatest element.  Of 32 or 64 groups of threads, the k-th
// greatest group maximum bounds the k-th greatest element from below (k groups hold one each), and only a thread whose own greatest
// reaches the bound can hold any of the top k.  There are a few more than k of them: their elements are looked through
// once more, what reaches the bound is kept, ranked by counting and written.  Order: greater first, equal values by the lower
// index, NaN before everything, -0 equal to +0.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>

#include "../../include/clusterfusion_b200.h"
#include "f32x2.cuh"
#include "host_common.h"
#include "mma.cuh"

namespace {

using cfb::ex2;
using cfb::fma2;
using cfb::Pair;

constexpr int LT = 256;        // threads of a CTA
constexpr int LW = LT / 32;
constexpr int MAX_TOP = 32;
constexpr int MAX_CLUSTER = 8;
constexpr int KEEP = 1024;     // candidates that are kept; more (adversarial orders only) take the slow way
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// order of the top k as an unsigned key
__device__ __forceinline__ unsigned order_key(float x) {
    if (x != x) return 0xffffffffu;
    const unsigned u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long ranked(float x, int idx) {  // greater key first, then lower index
    return static_cast<unsigned long long>(order_key(x)) << 32 | (0x7fffffffu - static_cast<unsigned>(idx));
}

__device__ __forceinline__ float key_value(unsigned key) {  // the value back (NaN for NaN)
    return __uint_as_float(key == 0xffffffffu ? 0x7fffffffu : key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// greatest and least of the 16 bytes' elements (NaN left out), the 16-bit types two at a time
__device__ __forceinline__ void extremes(const uint4& v, float& hi, float& lo, float) {
    const float a = __uint_as_float(v.x), b = __uint_as_float(v.y), c = __uint_as_float(v.z), d = __uint_as_float(v.w);
    hi = fmaxf(fmaxf(a, b), fmaxf(c, d));
    lo = fminf(fminf(a, b), fminf(c, d));
}
template <class P, class F> __device__ __forceinline__ void extremes_of_pairs(const uint4& v, float& hi, float& lo, F to_float2) {
    const P* p = reinterpret_cast<const P*>(&v);
    const float2 h = to_float2(__hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]))), l = to_float2(__hmin2(__hmin2(p[0], p[1]), __hmin2(p[2], p[3])));
    hi = fmaxf(h.x, h.y);
    lo = fminf(l.x, l.y);
}
__device__ __forceinline__ void extremes(const uint4& v, float& hi, float& lo, __half) {
    extremes_of_pairs<__half2>(v, hi, lo, [](__half2 x) { return __half22float2(x); });
}
__device__ __forceinline__ void extremes(const uint4& v, float& hi, float& lo, __nv_bfloat16) {
    extremes_of_pairs<__nv_bfloat162>(v, hi, lo, [](__nv_bfloat162 x) { return __bfloat1622float2(x); });
}

// Running statistics of a thread relative to a reference m within 4 of its greatest element (e^4 costs no precision, and the
// reference hardly ever moves).  m starts at the lowest finite number so that no difference of infinities is ever formed.
struct Stat {
    float m = -FLT_MAX;
    Pair z = Pair(0.f, 0.f), w = Pair(0.f, 0.f);
    __device__ __forceinline__ void meet(float top) {  // before elements up to `top` are added
        if (top > m + 4.f) {
            const float d = fmaxf(m - top, -150.f), r = ex2(d * LOG2E);  // e^-150 is 0 here
            w = Pair(r, r) * fma2(Pair(d, d), z, w);
            z = Pair(r, r) * z;
            m = top;
        }
    }
    // CLAMP where x - m may be -inf (0 times infinity in w); NaN goes through
    template <bool CLAMP> __device__ __forceinline__ void add(float x, float y) {
        Pair d = Pair(x, y) + Pair(-m, -m);
        if (CLAMP) {
            const float2 f = d.both();
            d = Pair(max_nan(f.x, -150.f), max_nan(f.y, -150.f));
        }
        const float2 l = (d * Pair(LOG2E, LOG2E)).both();
        const Pair e(ex2(l.x), ex2(l.y));
        z = z + e;
        w = fma2(e, d, w);
    }
};

// a sum of statistics: reference, z, w
struct Sum {
    float m = -FLT_MAX, z = 0.f, w = 0.f;
    __device__ __forceinline__ Sum() {}
    __device__ __forceinline__ Sum(float m_, float z_, float w_) : m(m_), z(z_), w(w_) {}
    __device__ __forceinline__ void refer_to(float top) {  // top >= m
        const float d = fmaxf(m - top, -150.f), r = ex2(d * LOG2E);
        w = r * fmaf(d, z, w);
        z *= r;
        m = top;
    }
    __device__ __forceinline__ void join(Sum o) {
        const float top = fmaxf(m, o.m);
        refer_to(top);
        o.refer_to(top);
        z += o.z;
        w += o.w;
    }
};

struct LogprobArgs {
    const void* logits;
    const void* tokens;
    float* logprobs;
    float* entropy;
    float* top_logprobs;
    long long* top_tokens;
    long long row_stride;
    int vocab, top, tokens64;
};

// Elements of [begin, end) of a row as one thread meets them, in index order: 16-byte vectors v = tid, tid + LT, ..., before
// them (threads below E) or after them (the next E threads) a single one of the ragged head or tail.
template <class T> struct Walk {
    static constexpr int E = 16 / sizeof(T);
    const T* row;
    int begin, head, vecs, tail_at, end;
    __device__ Walk(const T* r, int b, int e) : row(r), begin(b), end(e) {
        const int off = static_cast<int>((reinterpret_cast<uintptr_t>(r + b) & 15) / sizeof(T));
        head = off ? min(E - off, e - b) : 0;
        vecs = (e - b - head) / E;
        tail_at = b + head + vecs * E;
    }
    __device__ __forceinline__ int single(int tid) const {  // index of this thread's single element, -1 for none
        if (tid < head) return begin + tid;
        const int i = tail_at + tid - E;  // threads E .. 2 E - 1 take the tail
        return tid >= E && tid < 2 * E && i < end ? i : -1;
    }
    __device__ __forceinline__ int vec_at(int v) const { return begin + head + v * E; }
};

__device__ __forceinline__ float peer_float(uint32_t a) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ unsigned long long peer_u64(uint32_t a) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}

struct __align__(16) Shared {
    unsigned long long best[LT];
    unsigned long long group[64];
    unsigned long long keep[KEEP];
    unsigned long long top[MAX_TOP];
    unsigned long long all[MAX_CLUSTER * MAX_TOP];
    unsigned long long bound;
    float part[LW][3];
    float stat[3];
    int kept, found;
    uint16_t who[LT];
};

// For each of n <= LT / PARTS values: how many of the n are greater; PARTS neighbouring threads work on a value and all get the count
template <int PARTS> __device__ __forceinline__ int count_greater(const unsigned long long* v, int n, unsigned long long x) {
    int c = 0;
    for (int j = threadIdx.x % PARTS; j < n; j += PARTS) c += v[j] > x;
#pragma unroll
    for (int o = 1; o < PARTS; o <<= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    return c;
}

// The k greatest of [w.begin, w.end) as ranked() words in sh.top, greatest first, 0 where there are fewer.  `best`: this thread's greatest (0
// for none), its index rounded down to the start of its vector.  In this coarser order k elements reach the bound, and one
// that does not has k elements above it in the exact order too.
template <int GROUPS, class T> __device__ void block_top(const Walk<T>& w, unsigned long long best, int k, Shared& sh) {
    constexpr int E = Walk<T>::E;
    const int tid = threadIdx.x;
    sh.best[tid] = best;
    unsigned long long mine = best;
#pragma unroll
    for (int o = 1; o < LT / GROUPS; o <<= 1) {
        const unsigned long long x = __shfl_xor_sync(0xffffffffu, mine, o);
        mine = x > mine ? x : mine;
    }
    if (tid % (LT / GROUPS) == 0) sh.group[tid / (LT / GROUPS)] = mine;
    if (tid == 0) sh.kept = sh.found = 0, sh.bound = 0;
    if (tid < MAX_TOP) sh.top[tid] = 0;
    __syncthreads();
    {   // groups without elements have 0 and share a count: with fewer than k others the bound stays 0 and everything is kept
        const unsigned long long x = sh.group[tid / (LT / GROUPS)];
        if (count_greater<LT / GROUPS>(sh.group, GROUPS, x) == k - 1 && tid % (LT / GROUPS) == 0) sh.bound = x;
    }
    __syncthreads();
    const unsigned long long bound = sh.bound;
    const float bound_value = key_value(static_cast<unsigned>(bound >> 32));
    auto keep = [&](float x, int idx, int start) {
        if (!(x < bound_value) && ranked(x, start) >= bound) {
            const int at = atomicAdd(&sh.kept, 1);
            if (at < KEEP) sh.keep[at] = ranked(x, idx);
        }
    };
    // the threads that reach the bound, and their vectors (and singles, last), dealt out one by one to all threads
    if (best != 0 && best >= bound) sh.who[atomicAdd(&sh.found, 1)] = static_cast<uint16_t>(tid);
    __syncthreads();
    const int per = (w.vecs + LT - 1) / LT + 1, all = sh.found * per;
    for (int p = tid; p < all; p += LT) {
        const int nth = p / per, j = p - nth * per, o = sh.who[nth], v = o + j * LT;
        if (j == per - 1) {
            const int s = w.single(o);
            if (s >= 0) keep(to_float(w.row[s]), s, s);
        } else if (v < w.vecs) {
            const int at = w.vec_at(v);
            const uint4 raw = __ldg(reinterpret_cast<const uint4*>(w.row + at));
            const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int i = 0; i < E; ++i) keep(to_float(e[i]), at + i, at);
        }
    }
    __syncthreads();
    const int kept = sh.kept;
    if (kept <= LT / 4) {  // the usual case: four threads a value
        const unsigned long long x = tid / 4 < kept ? sh.keep[tid / 4] : 0;
        const int rank = count_greater<4>(sh.keep, kept, x);
        if (tid / 4 < kept && tid % 4 == 0 && rank < k) sh.top[rank] = x;
        __syncthreads();
        return;
    }
    if (kept <= KEEP) {
        for (int c = tid; c < kept; c += LT) {
            const unsigned long long x = sh.keep[c];
            int rank = 0;
            for (int j = 0; j < kept; ++j) rank += sh.keep[j] > x;
            if (rank < k) sh.top[rank] = x;
        }
        __syncthreads();
        return;
    }
    // an order of the row that puts very many of its greatest into few threads' shares: k passes, each finds the next
    unsigned long long last = ~0ull;
    for (int r = 0; r < k; ++r) {
        unsigned long long x = 0;
        auto look = [&](float f, int idx) {
            const unsigned long long y = ranked(f, idx);
            if (y < last && y > x) x = y;
        };
        const int s = w.single(tid);
        if (s >= 0) look(to_float(w.row[s]), s);
        for (int v = tid; v < w.vecs; v += LT)
            for (int i = 0; i < E; ++i) look(to_float(w.row[w.vec_at(v) + i]), w.vec_at(v) + i);
        __syncthreads();
        sh.best[tid] = x;
        __syncthreads();
        x = 0;
        for (int j = 0; j < LT; ++j) x = sh.best[j] > x ? sh.best[j] : x;
        if (tid == 0) sh.top[r] = x;
        if (x == 0) break;
        last = x;
    }
    __syncthreads();
}

template <class T>
__global__ void __launch_bounds__(LT, 8) token_logprobs_kernel(const LogprobArgs a, int cluster) {
    __shared__ Shared sh;
    constexpr int E = Walk<T>::E;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long r = blockIdx.x / cluster;
    const int rank = cluster > 1 ? static_cast<int>(cfb::cluster_ctarank()) : 0;
    const T* row = static_cast<const T*>(a.logits) + r * a.row_stride;
    const int share = ((a.vocab + cluster - 1) / cluster + 63) / 64 * 64;
    const int begin = min(rank * share, a.vocab), end = min(begin + share, a.vocab);
    const Walk<T> w(row, begin, end);

    float asked = -INFINITY;  // the given token's logit
    if (tid == 0 && rank == 0) {
        const long long tok = a.tokens64 ? static_cast<const long long*>(a.tokens)[r] : static_cast<const int*>(a.tokens)[r];
        if (tok >= 0 && tok < a.vocab) asked = to_float(row[tok]);
    }
    Stat st;
    float best_value = -FLT_MAX;
    int best_at = -1;  // start of the vector (or the single) that holds this thread's first maximum
    const int single = w.single(tid);
    auto meet = [&](float top, int at) {
        if (top > best_value || best_at < 0) {
            best_value = fmaxf(top, best_value);
            best_at = at;
        }
        st.meet(top);
    };
    auto take_single = [&] {
        const float x = to_float(row[single]);
        meet(x, single);
        st.template add<true>(x, -INFINITY);
    };
    if (single >= 0 && tid < E) take_single();
    auto take = [&](const uint4& raw, int at) {
        const T* e = reinterpret_cast<const T*>(&raw);
        float hi, lo;
        extremes(raw, hi, lo, T());
        meet(hi, at);
        if (lo - st.m < -1e38f) {  // masked by -inf or the lowest number, or so far below the greatest that the difference may overflow
#pragma unroll
            for (int i = 0; i < E; i += 2) st.template add<true>(to_float(e[i]), to_float(e[i + 1]));
        } else {
#pragma unroll
            for (int i = 0; i < E; i += 2) st.template add<false>(to_float(e[i]), to_float(e[i + 1]));
        }
    };
    const uint4* vec = reinterpret_cast<const uint4*>(row + w.vec_at(0));
    constexpr int UNROLL = 4;
    int v = tid;
    for (; v + (UNROLL - 1) * LT < w.vecs; v += UNROLL * LT) {
        uint4 raw[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) raw[u] = __ldg(vec + v + u * LT);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) take(raw[u], w.vec_at(v + u * LT));
    }
    for (; v < w.vecs; v += LT) take(__ldg(vec + v), w.vec_at(v));
    if (single >= 0 && tid >= E) take_single();

    Sum sum;
    {
        const float2 z = st.z.both(), ww = st.w.both();
        sum = Sum(st.m, z.x + z.y, ww.x + ww.y);
    }
    if (a.top > 0) {
        unsigned long long best = 0;
        if (best_at >= 0) {
            if (sum.z == sum.z && best_value > -FLT_MAX) {
                best = ranked(best_value, best_at);
            } else {  // a NaN, an infinity or nothing above the lowest number among them: look at each
                if (single >= 0) best = ranked(to_float(row[single]), single);
                for (int u = tid; u < w.vecs; u += LT)
                    for (int i = 0; i < E; ++i) {
                        const unsigned long long y = ranked(to_float(row[w.vec_at(u) + i]), w.vec_at(u));
                        best = y > best ? y : best;
                    }
            }
        }
        // Ranking g groups costs g squared; of g the k-th greatest has about g ln(g / (g - k)) elements above it (k = 5: 5.4 with 32, 5.2 with
        // 64; k = 20: 31 and 24).  One row of 50304 with the top 5 6.7 us by 32 groups, 7.0 by 64; 2047 rows with the top 20 57.0 and 56.4.
        // Groups without elements bound nothing, so every thread has to have some for the large groups.
        if (a.top <= 10 && w.vecs >= LT) block_top<32>(w, best, a.top, sh);
        else block_top<64>(w, best, a.top, sh);
    }

    auto join_lanes = [&](int width) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            if (o >= width) continue;
            sum.join(Sum(__shfl_xor_sync(0xffffffffu, sum.m, o), __shfl_xor_sync(0xffffffffu, sum.z, o), __shfl_xor_sync(0xffffffffu, sum.w, o)));
        }
    };
    join_lanes(32);
    if (lane == 0) sh.part[warp][0] = sum.m, sh.part[warp][1] = sum.z, sh.part[warp][2] = sum.w;
    __syncthreads();
    if (warp == 0) {
        sum = Sum(sh.part[lane % LW][0], sh.part[lane % LW][1], sh.part[lane % LW][2]);
        join_lanes(LW);
        if (lane == 0) sh.stat[0] = sum.m, sh.stat[1] = sum.z, sh.stat[2] = sum.w;
    }
    if (cluster > 1) cfb::cluster_sync_all();
    if (rank == 0) {
        if (cluster > 1 && a.top > 0) {  // the CTAs' lists, ranked by counting (at most 256 entries: one thread each)
            const int n = cluster * a.top;
            unsigned long long x = 0;
            if (tid < n) sh.all[tid] = x = peer_u64(cfb::cluster_map(&sh.top[tid % a.top], tid / a.top));
            __syncthreads();
            int at = 0;
            for (int j = 0; j < n; ++j) at += sh.all[j] > x;
            if (tid < n && x != 0 && at < a.top) sh.keep[at] = x;
            __syncthreads();
            if (tid < a.top) sh.top[tid] = sh.keep[tid];
        }
        if (warp == 0) {
            if (cluster > 1) {
                const int c = lane % cluster;
                sum = Sum(peer_float(cfb::cluster_map(&sh.stat[0], c)), peer_float(cfb::cluster_map(&sh.stat[1], c)), peer_float(cfb::cluster_map(&sh.stat[2], c)));
                join_lanes(cluster);
            }
            __syncwarp();
            const float log_z = logf(sum.z);
            if (lane == 0) {
                a.logprobs[r] = (asked - sum.m) - log_z;
                a.entropy[r] = log_z - sum.w / sum.z;
            }
            if (lane < a.top) {
                const unsigned long long x = sh.top[lane];
                a.top_tokens[r * a.top + lane] = static_cast<int>(0x7fffffffu - static_cast<unsigned>(x));
                a.top_logprobs[r * a.top + lane] = (key_value(static_cast<unsigned>(x >> 32)) - sum.m) - log_z;
            }
        }
    }
    if (cluster > 1) cfb::cluster_sync_all();  // a peer's shared memory is read until here
}

template <class T> cudaError_t launch(const LogprobArgs& a, long long rows, int cluster, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * cluster));
    cfg.blockDim = dim3(LT);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a, cluster);
}

}  // namespace

extern "C" int cf_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride, const void* tokens, int token_bytes,
                                 int64_t top_k, float* logprobs, float* entropy, float* top_logprobs, int64_t* top_tokens, void* stream) {
    if (dtype != CF_DTYPE_FP16 && dtype != CF_DTYPE_BF16 && dtype != CF_DTYPE_FP32) return cf_host_fail(CF_ERR_INVALID, "dtype %d is neither fp16, bf16 nor fp32", dtype);
    if (rows < 0 || rows > 0x7fffffff / MAX_CLUSTER) return cf_host_fail(CF_ERR_INVALID, "rows %lld", (long long)rows);
    if (vocab < 1 || vocab > (1 << 30)) return cf_host_fail(CF_ERR_INVALID, "vocabulary of %lld", (long long)vocab);
    if (top_k < 0 || top_k > MAX_TOP || top_k > vocab) return cf_host_fail(CF_ERR_INVALID, "top_k %lld outside 0..%d (and the vocabulary)", (long long)top_k, MAX_TOP);
    if (token_bytes != 4 && token_bytes != 8) return cf_host_fail(CF_ERR_INVALID, "tokens of %d bytes", token_bytes);
    if (rows == 0) return CF_OK;
    if (!logits || !tokens || !logprobs || !entropy || (top_k > 0 && (!top_logprobs || !top_tokens))) return cf_host_fail(CF_ERR_INVALID, "null pointer");
    const int size = dtype == CF_DTYPE_FP32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % size != 0) return cf_host_fail(CF_ERR_INVALID, "logits are not aligned to their elements");
    LogprobArgs a{logits, tokens, logprobs, entropy, top_logprobs, reinterpret_cast<long long*>(top_tokens), row_stride, static_cast<int>(vocab), static_cast<int>(top_k), token_bytes == 8};
    // Few rows: up to 8 CTAs share one, each with at least 16 KB, below which the exchange costs what it saves (fp16, top 5: a row of 8192 alone
    // 5.5 us, by two 6.5; 16 rows of 50304 by one CTA 9.6, by 4 7.8, by 8 8.4; fp32: a row of 50304 by one 11.2, by 4 7.4, by 8 7.1)
    int cluster = 1;
    while (cluster < MAX_CLUSTER && rows * cluster < 148 && vocab * size / (2 * cluster) >= 16384) cluster *= 2;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == CF_DTYPE_FP16   ? launch<__half>(a, rows, cluster, st)
                          : dtype == CF_DTYPE_BF16 ? launch<__nv_bfloat16>(a, rows, cluster, st)
                                                   : launch<float>(a, rows, cluster, st);
    if (e != cudaSuccess) return cf_host_fail(CF_ERR_CUDA, "token log probabilities launch failed: %s", cudaGetErrorString(e));
    return CF_OK;
}
