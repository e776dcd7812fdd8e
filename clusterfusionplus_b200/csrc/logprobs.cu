// Log probabilities of given tokens, the entropy of the distribution and its most probable tokens, from logits.
//
//   m = max_j x_j, z = sum_j e^(x_j - m), w = sum_j e^(x_j - m) (x_j - m)
//   log p_i = (x_i - m) - log z,   H = log z - w / z
//
// Nothing is formed as a difference of large numbers (no log-sum-exp is subtracted from a logit), so logits of any size keep
// fp32's relative precision.  The floor is reading the logits once.  One CTA takes a row (or a cluster of CTAs a row when
// there are few rows: the partial results meet in distributed shared memory, so no workspace and no second launch).
//
// The top k (at most 32) cost next to nothing: every thread knows the largest element it met.  The k-th largest of these
// maxima is a lower bound of the k-th largest element, and only the (at most k) threads whose maximum reaches it can hold any of
// the top k.  Their elements are looked through once more, what reaches the bound is kept (a little over k values), ranked
// and written.  Order: greater first, equal values by the lower index, NaN before everything, -0 equal to +0.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>

#include "../../include/clusterfusion_b200.h"
#include "host_common.h"

namespace {

constexpr int LT = 512;        // threads of a CTA
constexpr int LW = LT / 32;
constexpr int MAX_TOP = 32;
constexpr int MAX_CLUSTER = 8;
constexpr int KEEP = 1024;     // candidates that are kept; more (adversarial orders only) take the slow way
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
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

template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// running statistics; m starts at the lowest finite number so that no difference of infinities is ever formed
struct Stat {
    float m = -FLT_MAX, z = 0.f, w = 0.f;
    __device__ __forceinline__ void refer_to(float top) {  // top >= m
        const float d = fmaxf(m - top, -150.f), r = ex2(d * LOG2E);  // e^-150 is 0 here
        w = r * fmaf(d, z, w);
        z *= r;
        m = top;
    }
    __device__ __forceinline__ void add(float x) {  // x <= m; NaN goes through
        const float d = max_nan(x - m, -150.f), e = ex2(d * LOG2E);
        z += e;
        w = fmaf(e, d, w);
    }
    __device__ __forceinline__ void join(float m2, float z2, float w2) {
        Stat o;
        o.m = m2, o.z = z2, o.w = w2;
        const float top = fmaxf(m, m2);
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

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer(const void* p, unsigned rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
    return a;
}
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
    float part[LW][3];
    float stat[3];
    unsigned long long bests[LT];
    unsigned long long keep[KEEP];
    unsigned long long top[MAX_TOP];
    unsigned long long all[MAX_CLUSTER * MAX_TOP];
    unsigned long long bound;
    int kept;
};

// The k greatest of [w.begin, w.end) as ranked() words in sh.top, greatest first, 0 where there are fewer.  `best`: this
// thread's greatest (0 for none).
template <class T> __device__ void block_top(const Walk<T>& w, unsigned long long best, int k, Shared& sh) {
    const int tid = threadIdx.x, lane = tid & 31;
    sh.bests[tid] = best;
    if (tid == 0) sh.kept = 0;
    if (tid < MAX_TOP) sh.top[tid] = 0;
    __syncthreads();
    if (tid < 32) {  // the k-th greatest of the threads' bests
        unsigned long long mine[LW];
#pragma unroll
        for (int i = 0; i < LW; ++i) mine[i] = sh.bests[i * 32 + lane];
        unsigned long long top = 0;
        for (int r = 0; r < k; ++r) {
            unsigned long long x = 0;
#pragma unroll
            for (int i = 0; i < LW; ++i) x = mine[i] > x ? mine[i] : x;
            const unsigned hi = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(x >> 32));
            const unsigned lo = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(x >> 32) == hi ? static_cast<unsigned>(x) : 0u);
            top = static_cast<unsigned long long>(hi) << 32 | lo;
#pragma unroll
            for (int i = 0; i < LW; ++i) mine[i] = mine[i] == top ? 0 : mine[i];
        }
        if (lane == 0) sh.bound = top;
    }
    __syncthreads();
    const unsigned long long bound = sh.bound;
    auto keep = [&](float x, int idx) {
        const unsigned long long r = ranked(x, idx);
        if (r >= bound) {
            const int at = atomicAdd(&sh.kept, 1);
            if (at < KEEP) sh.keep[at] = r;
        }
    };
    // the threads that reach the bound: each one's elements are dealt out to a warp
    int nth = 0;
    for (int i = 0; i < LW; ++i) {
        const unsigned long long theirs = sh.bests[i * 32 + lane];
        unsigned who = __ballot_sync(0xffffffffu, theirs >= bound && theirs != 0);
        for (; who; who &= who - 1) {
            if (nth++ % LW != tid >> 5) continue;
            const int o = i * 32 + __ffs(who) - 1, s = w.single(o);
            if (s >= 0 && lane == 0) keep(to_float(w.row[s]), s);
            for (int v = o + lane * LT; v < w.vecs; v += 32 * LT)
#pragma unroll
                for (int j = 0; j < Walk<T>::E; ++j) keep(to_float(w.row[w.vec_at(v) + j]), w.vec_at(v) + j);
        }
    }
    __syncthreads();
    const int kept = sh.kept;
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
            for (int i = 0; i < Walk<T>::E; ++i) look(to_float(w.row[w.vec_at(v) + i]), w.vec_at(v) + i);
        __syncthreads();
        sh.bests[tid] = x;
        __syncthreads();
        x = 0;
        for (int j = 0; j < LT; ++j) x = sh.bests[j] > x ? sh.bests[j] : x;
        if (tid == 0) sh.top[r] = x;
        if (x == 0) break;
        last = x;
    }
    __syncthreads();
}

template <class T>
__global__ void __launch_bounds__(LT) token_logprobs_kernel(const LogprobArgs a, int cluster) {
    __shared__ Shared sh;
    constexpr int E = Walk<T>::E;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long r = blockIdx.x / cluster;
    const int rank = cluster > 1 ? static_cast<int>(cluster_rank()) : 0;
    const T* row = static_cast<const T*>(a.logits) + r * a.row_stride;
    const int share = ((a.vocab + cluster - 1) / cluster + 63) / 64 * 64;
    const int begin = min(rank * share, a.vocab), end = min(begin + share, a.vocab);
    const Walk<T> w(row, begin, end);

    Stat st;
    int best_at = -1;  // first index of the vector (or single) that holds this thread's first maximum
    const int single = w.single(tid);
    auto take_single = [&] {
        const float x = to_float(row[single]);
        if (x > st.m) {
            st.refer_to(x);
            best_at = single;
        } else if (best_at < 0) best_at = single;
        st.add(x);
    };
    if (single >= 0 && tid < E) take_single();
    auto take = [&](const uint4& raw, int at) {
        const T* e = reinterpret_cast<const T*>(&raw);
        float x[E], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            x[i] = to_float(e[i]);
            top = fmaxf(top, x[i]);
        }
        if (top > st.m) {
            st.refer_to(top);
            best_at = at;
        } else if (best_at < 0) best_at = at;
#pragma unroll
        for (int i = 0; i < E; ++i) st.add(x[i]);
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

    if (a.top > 0) {
        unsigned long long best = 0;
        if (best_at >= 0) {
            if (st.z == st.z) {
                const int n = best_at == single ? 1 : E;
                for (int i = 0; i < n; ++i) {
                    const unsigned long long y = ranked(to_float(row[best_at + i]), best_at + i);
                    best = y > best ? y : best;
                }
                if (st.m == -FLT_MAX) best = 0;
            }
            if (best == 0) {  // a NaN, an infinity or nothing above the lowest number among them: look at each
                if (single >= 0) best = ranked(to_float(row[single]), single);
                for (int u = tid; u < w.vecs; u += LT)
                    for (int i = 0; i < E; ++i) {
                        const unsigned long long y = ranked(to_float(row[w.vec_at(u) + i]), w.vec_at(u) + i);
                        best = y > best ? y : best;
                    }
            }
        }
        block_top(w, best, a.top, sh);
    }

#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m = __shfl_xor_sync(0xffffffffu, st.m, o), z = __shfl_xor_sync(0xffffffffu, st.z, o), ww = __shfl_xor_sync(0xffffffffu, st.w, o);
        st.join(m, z, ww);
    }
    if (lane == 0) sh.part[warp][0] = st.m, sh.part[warp][1] = st.z, sh.part[warp][2] = st.w;
    __syncthreads();
    if (tid == 0) {
        Stat all;
        for (int i = 0; i < LW; ++i) all.join(sh.part[i][0], sh.part[i][1], sh.part[i][2]);
        sh.stat[0] = all.m, sh.stat[1] = all.z, sh.stat[2] = all.w;
    }
    if (cluster > 1) cluster_sync();
    else __syncthreads();
    if (rank == 0) {
        Stat all;
        if (cluster == 1) {
            all.m = sh.stat[0], all.z = sh.stat[1], all.w = sh.stat[2];
        } else {
            for (int c = 0; c < cluster; ++c) all.join(peer_float(peer(&sh.stat[0], c)), peer_float(peer(&sh.stat[1], c)), peer_float(peer(&sh.stat[2], c)));
            if (a.top > 0) {
                const int n = cluster * a.top;
                for (int i = tid; i < n; i += LT) sh.all[i] = peer_u64(peer(&sh.top[i % a.top], i / a.top));
                __syncthreads();
                unsigned long long x = 0;
                int at = a.top;
                if (tid < n) {
                    x = sh.all[tid];
                    at = 0;
                    for (int j = 0; j < n; ++j) at += sh.all[j] > x;
                }
                if (x != 0 && at < a.top) sh.keep[at] = x;
                __syncthreads();
                if (tid < a.top) sh.top[tid] = sh.keep[tid];
            }
        }
        const float log_z = logf(all.z);
        if (tid == 0) {
            const long long tok = a.tokens64 ? static_cast<const long long*>(a.tokens)[r] : static_cast<const int*>(a.tokens)[r];
            const bool known = tok >= 0 && tok < a.vocab;
            const float x = known ? to_float(row[tok]) : -INFINITY;
            a.logprobs[r] = (x - all.m) - log_z;
            a.entropy[r] = log_z - all.w / all.z;
        }
        if (tid < a.top) {
            const int idx = static_cast<int>(0x7fffffffu - static_cast<unsigned>(sh.top[tid]));
            a.top_tokens[r * a.top + tid] = idx;
            a.top_logprobs[r * a.top + tid] = (to_float(row[idx]) - all.m) - log_z;
        }
    }
    if (cluster > 1) cluster_sync();  // a peer's shared memory is read until here
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
    // few rows: up to 8 CTAs share one, each with at least 4096 elements (below that the exchange costs more than it saves)
    int cluster = 1;
    while (cluster < MAX_CLUSTER && rows * cluster < 148 && vocab / (2 * cluster) >= 4096) cluster *= 2;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == CF_DTYPE_FP16   ? launch<__half>(a, rows, cluster, st)
                          : dtype == CF_DTYPE_BF16 ? launch<__nv_bfloat16>(a, rows, cluster, st)
                                                   : launch<float>(a, rows, cluster, st);
    if (e != cudaSuccess) return cf_host_fail(CF_ERR_CUDA, "token log probabilities launch failed: %s", cudaGetErrorString(e));
    return CF_OK;
}
