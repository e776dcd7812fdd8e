// One step of a batch over a paged cache, planned on the GPU: block tables, slot maps, positions and the row lists that
// the paged blocks read, from request lengths that never leave device memory.
//
//   have_b = ceil(cached_b / P), need_b = ceil((cached_b + new_b) / P), P = page size
//   fresh page j of request b (table column have_b + j) = free[count - 1 - (sum_{a < b} (need_a - have_a) + j)]
//   slot of position p of request b = table[b][p / P] * P + p % P
//
// What bounds it is latency: the largest lists are a few MB.  So there is one launch and no hand-over between CTAs: every CTA
// scans the lengths for itself (the batch is at most 4096), knows from the prefix sums which pages the step takes from the
// free list, and expands its share of the token and row lists; CTA 0 writes what exists once.  A CTA reads only table
// entries below have_b and CTA 0 writes only entries from have_b on, so nothing is read that another CTA writes.
// Measured on the GPU: 16 requests of up to 2048 tokens 4.8 us, 256 requests of up to 8192 with 1.0 M listed rows (4.8 MB, 0.7 us of
// writing) 8.3 us: a launch, three scans of the batch and the issue of ~5 instructions a row (63 % of the issue slots).
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/clusterfusion_b200.h"
#include "host_common.h"

namespace {

constexpr int PT = 256;            // threads of a CTA
constexpr int PLAN_MAX_BATCH = 4096;
constexpr int ROWS_PER_THREAD = 4;  // consecutive rows of one thread: one 16-byte store

struct PlanArgs {
    const int* cached;
    const int* fresh;
    int batch;
    int* table;
    long long table_width, table_stride;
    const int* free_pages;
    long long n_free;
    const int* free_count;
    int* free_count_out;
    int page;
    int* kv_lens;
    int* qo_indptr;
    long long* positions;
    int* slot_map;
    long long max_tokens;
    int* kv_indptr;
    int* kv_indices;
    long long max_rows;
    int* status;
};

struct Sums {  // of one request or of a prefix of them
    long long tokens, rows, pages;
};

__device__ __forceinline__ Sums operator+(Sums a, Sums b) { return {a.tokens + b.tokens, a.rows + b.rows, a.pages + b.pages}; }

__device__ __forceinline__ Sums shfl_up(Sums v, int o) {
    return {__shfl_up_sync(0xffffffffu, v.tokens, o), __shfl_up_sync(0xffffffffu, v.rows, o), __shfl_up_sync(0xffffffffu, v.pages, o)};
}

__device__ __forceinline__ int pages_of(long long len, int page) { return static_cast<int>((len + page - 1) / page); }

// exclusive prefix of v over the CTA's threads, and the sum over all
__device__ __forceinline__ Sums block_exclusive(Sums v, Sums* total, Sums* buf) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Sums inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Sums up = shfl_up(inc, o);
        if (lane >= o) inc = inc + up;
    }
    if (lane == 31) buf[warp] = inc;
    __syncthreads();
    Sums before = {0, 0, 0}, all = {0, 0, 0};
#pragma unroll
    for (int w = 0; w < PT / 32; ++w) {
        if (w < warp) before = before + buf[w];
        all = all + buf[w];
    }
    *total = all;
    return {before.tokens + inc.tokens - v.tokens, before.rows + inc.rows - v.rows, before.pages + inc.pages - v.pages};
}

// the request that holds element j of a list whose requests start at start[0 .. batch]
__device__ __forceinline__ int owner_of(const int* start, int batch, int j) {
    int lo = 0, hi = batch;  // start[lo] <= j < start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= j) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PT) paged_kv_plan_kernel(const PlanArgs a) {
    extern __shared__ int sm[];
    int* s_cached = sm;                        // [batch]
    int* s_tok = s_cached + a.batch;           // [batch + 1] first token of a request
    int* s_row = s_tok + a.batch + 1;          // [batch + 1] first row
    int* s_page = s_row + a.batch + 1;         // [batch + 1] first fresh page
    int* s_have = s_page + a.batch + 1;        // [batch] pages held already
    __shared__ Sums buf[PT / 32];
    __shared__ int s_bits;

    const int tid = threadIdx.x, per = (a.batch + PT - 1) / PT;
    const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    if (tid == 0) s_bits = 0;
    const long long avail = *a.free_count;
    Sums mine = {0, 0, 0};
    int bits = 0;
    for (int b = b0; b < b1; ++b) {
        const int c = a.cached[b], n = a.fresh[b];
        const long long total = static_cast<long long>(c) + n;
        if (c < 0 || n < 0 || total > 0x7fffffffll) {
            bits |= CF_PLAN_BAD_LENGTH;
            continue;
        }
        const int need = pages_of(total, a.page);
        if (need > a.table_width) bits |= CF_PLAN_TABLE_WIDTH;
        mine = mine + Sums{n, total, need - pages_of(c, a.page)};
    }
    __syncthreads();
    if (bits) atomicOr(&s_bits, bits);
    Sums all;
    const Sums before = block_exclusive(mine, &all, buf);  // its barrier also orders s_bits
    bits = s_bits;
    if (avail < 0 || avail > a.n_free || all.pages > avail) bits |= CF_PLAN_NO_PAGES;  // a count that the list cannot have says nothing about which entries are free
    if (all.tokens > a.max_tokens) bits |= CF_PLAN_MAX_TOKENS;
    if (a.max_rows > 0 ? all.rows > a.max_rows : all.rows > 0x7fffffffll) bits |= CF_PLAN_MAX_ROWS;
    const bool ok = bits == 0;  // all or nothing: a step that does not fit changes no table and deals out nothing
    const bool first = blockIdx.x == 0;
    if (ok) {
        Sums at = before;
        for (int b = b0; b < b1; ++b) {
            const int c = a.cached[b], n = a.fresh[b];
            s_cached[b] = c;
            s_tok[b] = static_cast<int>(at.tokens);
            s_row[b] = static_cast<int>(at.rows);
            s_page[b] = static_cast<int>(at.pages);
            s_have[b] = pages_of(c, a.page);
            at = at + Sums{n, static_cast<long long>(c) + n, pages_of(static_cast<long long>(c) + n, a.page) - s_have[b]};
        }
        if (tid == 0) {
            s_tok[a.batch] = static_cast<int>(all.tokens);
            s_row[a.batch] = static_cast<int>(all.rows);
            s_page[a.batch] = static_cast<int>(all.pages);
        }
        __syncthreads();
    }
    if (first) {
        for (int b = tid; b <= a.batch; b += PT) {
            a.qo_indptr[b] = ok ? s_tok[b] : 0;
            a.kv_indptr[b] = ok ? s_row[b] : 0;
            if (b < a.batch) a.kv_lens[b] = a.cached[b] + (ok ? a.fresh[b] : 0);
        }
        if (tid == 0) {
            *a.free_count_out = static_cast<int>(avail - (ok ? all.pages : 0));
            *a.status = bits;
        }
        if (ok)
            for (int e = tid; e < s_page[a.batch]; e += PT) {
                const int b = owner_of(s_page, a.batch, e);
                a.table[b * a.table_stride + s_have[b] + (e - s_page[b])] = a.free_pages[avail - 1 - e];
            }
    }
    // page of column col of request b: held pages come from the table, fresh ones from where this step takes them
    auto page_of = [&](int b, int col) -> long long {
        return col < s_have[b] ? a.table[b * a.table_stride + col] : a.free_pages[avail - 1 - (s_page[b] + col - s_have[b])];
    };
    auto slot_at = [&](long long held, int in) -> int {
        const long long slot = held * a.page + in;
        return held < 0 || slot > 0x7fffffffll ? -1 : static_cast<int>(slot);
    };
    const long long stride = static_cast<long long>(gridDim.x) * PT;
    for (long long j = static_cast<long long>(blockIdx.x) * PT + tid; j < a.max_tokens; j += stride) {
        long long pos = 0;
        int slot = -1;
        if (ok && j < all.tokens) {
            const int b = owner_of(s_tok, a.batch, static_cast<int>(j));
            pos = s_cached[b] + (j - s_tok[b]);
            const int col = static_cast<int>(pos) / a.page;
            slot = slot_at(page_of(b, col), static_cast<int>(pos) - col * a.page);
        }
        a.positions[j] = pos;
        a.slot_map[j] = slot;
    }
    const long long groups = (a.max_rows + ROWS_PER_THREAD - 1) / ROWS_PER_THREAD;
    for (long long g = static_cast<long long>(blockIdx.x) * PT + tid; g < groups; g += stride) {
        const long long j0 = g * ROWS_PER_THREAD;
        int slot[ROWS_PER_THREAD];
        int b = -1, left = 0, in = 0, col = 0;  // request; its rows from here on; place in the page; column
        long long held = 0;
#pragma unroll
        for (int i = 0; i < ROWS_PER_THREAD; ++i) {
            slot[i] = -1;
            if (ok && j0 + i < all.rows) {
                const int j = static_cast<int>(j0) + i;
                if (left == 0) {  // the first row, or the first of the next request that has any
                    if (b < 0) b = owner_of(s_row, a.batch, j);
                    while (j >= s_row[b + 1]) ++b;
                    left = s_row[b + 1] - j;
                    const int pos = j - s_row[b];
                    col = pos / a.page, in = pos - col * a.page;
                    held = page_of(b, col);
                } else if (in == a.page) {
                    in = 0;
                    held = page_of(b, ++col);
                }
                slot[i] = slot_at(held, in++);
                --left;
            }
        }
        if (j0 + ROWS_PER_THREAD <= a.max_rows) {
            *reinterpret_cast<int4*>(a.kv_indices + j0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        } else {
#pragma unroll
            for (int i = 0; i < ROWS_PER_THREAD; ++i)
                if (j0 + i < a.max_rows) a.kv_indices[j0 + i] = slot[i];
        }
    }
}

struct ReleaseArgs {
    const int* finished;
    const int* kv_lens;
    int batch;
    int* table;
    long long table_width, table_stride;
    int* free_pages;
    long long n_free;
    const int* free_count;
    int* free_count_out;
    int page;
    int* status;
};

// One CTA: the pages of the finished requests go back on top of the free list in request and column order.  Two sweeps over
// them, the first only looks (all or nothing), since an entry that names no page must not get onto the list.  51 of 256 requests of up to 8192
// tokens (3 300 pages of 64) take 15.9 us.
__global__ void __launch_bounds__(PT) paged_kv_release_kernel(const ReleaseArgs a) {
    extern __shared__ int sm[];
    int* s_page = sm;  // [batch + 1] first released page of a request
    __shared__ Sums buf[PT / 32];
    const int tid = threadIdx.x, per = (a.batch + PT - 1) / PT;
    const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    const int count = *a.free_count;
    auto held = [&](int b) -> long long { return a.finished[b] ? pages_of(max(a.kv_lens[b], 0), a.page) : 0; };
    Sums mine = {0, 0, 0};
    int bits = 0;
    for (int b = b0; b < b1; ++b) {
        const long long n = held(b);
        if (a.finished[b] && a.kv_lens[b] < 0) bits |= CF_PLAN_BAD_LENGTH;
        if (n > a.table_width) bits |= CF_PLAN_TABLE_WIDTH;
        mine.pages += n;
    }
    Sums all;
    Sums at = block_exclusive(mine, &all, buf);
    if (count < 0 || count + all.pages > a.n_free) bits |= CF_PLAN_NO_PAGES;  // the list cannot take them
    bits = __syncthreads_or(bits & CF_PLAN_BAD_LENGTH) ? bits | CF_PLAN_BAD_LENGTH : bits;
    bits = __syncthreads_or(bits & CF_PLAN_TABLE_WIDTH) ? bits | CF_PLAN_TABLE_WIDTH : bits;
    if (bits == 0) {
        for (int b = b0; b < b1; ++b) {
            s_page[b] = static_cast<int>(at.pages);
            at.pages += held(b);
        }
        if (tid == 0) s_page[a.batch] = static_cast<int>(all.pages);
        __syncthreads();
        int bad = 0;
        for (int e = tid; e < all.pages; e += PT) {
            const int b = owner_of(s_page, a.batch, e);
            bad |= a.table[b * a.table_stride + (e - s_page[b])] < 0;
        }
        if (__syncthreads_or(bad)) bits |= CF_PLAN_BAD_PAGE;
    }
    if (bits == 0)
        for (int e = tid; e < all.pages; e += PT) {
            const int b = owner_of(s_page, a.batch, e);
            int* entry = a.table + b * a.table_stride + (e - s_page[b]);
            a.free_pages[count + e] = *entry;
            *entry = -1;
        }
    if (tid == 0) {
        *a.free_count_out = count + (bits == 0 ? static_cast<int>(all.pages) : 0);
        *a.status = bits;
    }
}

int check_common(int64_t batch, int64_t table_width, int64_t table_stride, int64_t n_free, const void* count, const void* count_out, int64_t page) {
    if (batch < 1 || batch > PLAN_MAX_BATCH) return cf_host_fail(CF_ERR_INVALID, "batch %lld outside 1..%d", (long long)batch, PLAN_MAX_BATCH);
    if (page < 1 || page > 65536) return cf_host_fail(CF_ERR_INVALID, "page size %lld outside 1..65536", (long long)page);
    if (table_width < 1 || table_width > 0x7fffffff || table_stride < table_width)
        return cf_host_fail(CF_ERR_INVALID, "block table of %lld columns, %lld entries apart", (long long)table_width, (long long)table_stride);
    if (n_free < 0 || n_free > 0x7fffffff) return cf_host_fail(CF_ERR_INVALID, "free list of %lld pages", (long long)n_free);
    if (count == count_out) return cf_host_fail(CF_ERR_INVALID, "free_count_out must not alias free_count (other CTAs still read it)");
    return CF_OK;
}

}  // namespace

extern "C" {

int cf_paged_kv_plan(const int* cached_lens, const int* new_lens, int64_t batch, int* block_table, int64_t table_width, int64_t table_stride,
                     const int* free_pages, int64_t n_free_pages, const int* free_count, int* free_count_out, int64_t page_size, int* kv_lens,
                     int* qo_indptr, int64_t* positions, int* slot_map, int64_t max_tokens, int* kv_indptr, int* kv_indices, int64_t max_rows,
                     int* status, void* stream) {
    if (!cached_lens || !new_lens || !block_table || !free_count || !free_count_out || !kv_lens || !qo_indptr || !kv_indptr || !status)
        return cf_host_fail(CF_ERR_INVALID, "null pointer");
    if ((n_free_pages > 0 && !free_pages) || (max_tokens > 0 && (!positions || !slot_map)) || (max_rows > 0 && !kv_indices))
        return cf_host_fail(CF_ERR_INVALID, "null pointer");
    if (int rc = check_common(batch, table_width, table_stride, n_free_pages, free_count, free_count_out, page_size)) return rc;
    if (kv_lens == cached_lens || kv_lens == new_lens) return cf_host_fail(CF_ERR_INVALID, "kv_lens must not alias the lengths that are read");
    if (max_tokens < 0 || max_tokens > 0x7fffffff || max_rows < 0 || max_rows > 0x7fffffff)
        return cf_host_fail(CF_ERR_INVALID, "max_tokens %lld, max_rows %lld", (long long)max_tokens, (long long)max_rows);
    if (reinterpret_cast<uintptr_t>(kv_indices) % 16 != 0) return cf_host_fail(CF_ERR_INVALID, "kv_indices must be 16-byte aligned");
    const PlanArgs a{cached_lens, new_lens, static_cast<int>(batch), block_table, table_width, table_stride, free_pages, n_free_pages, free_count,
                     free_count_out, static_cast<int>(page_size), kv_lens, qo_indptr, reinterpret_cast<long long*>(positions), slot_map, max_tokens,
                     kv_indptr, kv_indices, max_rows, status};
    // a CTA for 256 tokens or 1024 rows, at most four for each SM: more would only repeat the scan
    const int64_t want = max_tokens / PT + max_rows / (PT * ROWS_PER_THREAD) + 1;
    const unsigned grid = static_cast<unsigned>(want < 4 * 148 ? want : 4 * 148);
    const size_t smem = (5 * batch + 3) * sizeof(int);
    if (smem > 47 * 1024) {  // 48 KB without being asked for, the static part among them
        const cudaError_t e = cudaFuncSetAttribute(paged_kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return cf_host_fail(CF_ERR_CUDA, "paged plan: %s", cudaGetErrorString(e));
    }
    paged_kv_plan_kernel<<<grid, PT, smem, static_cast<cudaStream_t>(stream)>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cf_host_fail(CF_ERR_CUDA, "paged plan launch failed: %s", cudaGetErrorString(e));
    return CF_OK;
}

int cf_paged_kv_release(const int* finished, const int* kv_lens, int64_t batch, int* block_table, int64_t table_width, int64_t table_stride,
                        int* free_pages, int64_t n_free_pages, const int* free_count, int* free_count_out, int64_t page_size, int* status,
                        void* stream) {
    if (!finished || !kv_lens || !block_table || !free_count || !free_count_out || !status || (n_free_pages > 0 && !free_pages))
        return cf_host_fail(CF_ERR_INVALID, "null pointer");
    if (int rc = check_common(batch, table_width, table_stride, n_free_pages, free_count, free_count_out, page_size)) return rc;
    const ReleaseArgs a{finished, kv_lens, static_cast<int>(batch), block_table, table_width, table_stride, free_pages, n_free_pages, free_count,
                        free_count_out, static_cast<int>(page_size), status};
    paged_kv_release_kernel<<<1, PT, (batch + 1) * sizeof(int), static_cast<cudaStream_t>(stream)>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cf_host_fail(CF_ERR_CUDA, "paged release launch failed: %s", cudaGetErrorString(e));
    return CF_OK;
}

}  // extern "C"
