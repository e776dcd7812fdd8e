// Internal interface between the C entry point of the 4-bit attention (kv4_cache.cu) and its kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace cfb {

// cudaFuncSetAttribute costs a microsecond of every call: once for each kernel and device is enough.  `done` is the kernel's own record.
inline cudaError_t allow_shared_once(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    const cudaError_t s = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (s == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_release);
    return s;
}

struct Kv4AttnArgs {
    const void* query;
    const uint8_t* cache;
    const int* table;
    const int* kv_lens;
    const int* qo_indptr;  // null: one query a request
    void* out;
    long long q_ts, q_hs, table_stride, table_width, rows;
    int batch, heads, kv_heads, D, page, pages;
    float scale_log2;  // of q . k, times log2(e)
    int* status;       // device status word
    void* workspace;   // null: none
};

// few query rows a request: the cache is streamed once for up to 8 or 16 of them.  The workspace (its size in bytes; whether it is of use
// where a request has at most `tokens`) spreads requests of different lengths evenly over the GPU.
long long kv4_few_workspace(long long heads, long long kv_heads, int D, long long max_q_len);
bool kv4_few_uses_workspace(long long batch, long long heads, long long kv_heads, long long tokens, long long max_q_len);
cudaError_t kv4_attention_few(const Kv4AttnArgs& a, bool bf16, long long max_q_len, cudaStream_t st);

// many query rows a request: 128 of them at a time on the tensor cores
cudaError_t kv4_attention_prompt(const Kv4AttnArgs& a, bool bf16, long long max_q_len, cudaStream_t st);

}  // namespace cfb
