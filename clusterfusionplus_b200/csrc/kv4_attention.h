// Internal interface between the C entry point of the 4-bit attention (kv4_cache.cu) and its kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace cfb {

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
