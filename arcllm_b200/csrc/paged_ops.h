// Internal interface of the paged-cache serving kernels (paged_ops.cu,
// logits_ops.cu, attention_paged.cu, attention_paged_tiles.cu).
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "arcllm_cuda_internal.h"

namespace arc {

// The kernel's limit of dynamic shared memory (and, if asked, clusters of 16) on
// the current device, set once for each device: the attribute calls cost a
// microsecond of every launch otherwise.
template <auto Kernel, bool kClusters16 = false>
cudaError_t allow_shared(int bytes) {
    static std::atomic<uint64_t> done{0};
    const int dev = device_slot();
    if (dev >= 0 && ((done.load(std::memory_order_acquire) >> dev) & 1u)) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && kClusters16)
        e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && dev >= 0) done.fetch_or(1ull << dev, std::memory_order_release);
    return e;
}

struct PagedPlan {
    const int32_t *kv_len, *new_len;
    uint32_t n_requests, page_size, n_pages;
    const int32_t *free_pages, *n_free;
    int32_t* block_table;
    uint32_t table_stride, max_rows;
    int32_t *row_start, *kv_total, *positions, *slots, *n_free_out;
};
int paged_plan(const PagedPlan& p, cudaStream_t stream);

int rope_freqs(int scaling, uint32_t rot_dim, double theta, double factor, double trained_ctx, double* freqs,
               float* attn_scale);

struct RopePaged {
    const void *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride, out_stride;
    const float *bq, *bk, *bv;
    const double* freqs;
    uint32_t rot_dim;
    int half_layout;
    float attn_scale;
    const int32_t *positions, *slots;
    uint32_t rows, q_heads;
    void* q_out;
};
int rope_kv_paged(int act_type, const RopePaged& p, const arcllm_cuda_paged_kv& kv, cudaStream_t stream);

struct LogitsProcess {
    const void* logits;
    uint64_t stride, out_stride;
    uint32_t n_rows, vocab;
    const int32_t* history;
    uint32_t history_stride;
    const int32_t *prompt_len, *total_len;
    const float *repetition, *frequency, *presence;
    const int32_t *bias_start, *bias_ids;
    const float* bias_values;
    const uint32_t* mask;
    uint32_t mask_stride;
    void* out;
    int32_t* best;
};
int logits_process(int type, const LogitsProcess& p, cudaStream_t stream);

// Whether any of the pointers is not on a multiple of n bytes (null is): an array's words have to be.
template <typename... Ptr>
bool any_off(uintptr_t n, const Ptr*... p) {
    return ((reinterpret_cast<uintptr_t>(p) | ...) & (n - 1u)) != 0u;
}

// Whether two arrays of rows share a byte (strides and widths in bytes).  Rows of one stride may lie side by side
// in one array (parts of a fused projection); with different strides any overlap of the whole ranges counts.
inline bool rows_meet(const void* a, uint64_t a_stride, uint64_t a_width, const void* b, uint64_t b_stride,
                      uint64_t b_width, uint64_t rows) {
    const uint64_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    if (x >= y + (rows - 1u) * b_stride + b_width || y >= x + (rows - 1u) * a_stride + a_width) return false;
    if (a_stride != b_stride) return true;
    const uint64_t off = y >= x ? (y - x) % a_stride : a_stride - (x - y) % a_stride;  // of b's rows in a's
    return off < a_width || off + b_width > a_stride;
}

// Checks of a cache descriptor that every user of it makes (null pointers, shape, type, the 32-bit slot range).
int check_paged_kv(const arcllm_cuda_paged_kv* kv, const char* who);

struct AttnPaged {
    const void* q;
    uint64_t q_stride, out_stride;
    const int32_t* block_table;
    uint32_t table_stride;
    const int32_t *row_start, *kv_total;
    uint32_t n_requests, max_rows, max_new, q_heads;
    float scale;
    uint32_t window, sinks;
    void* out;
    void* workspace;
    uint64_t workspace_bytes;
};
int attention_paged(const AttnPaged& p, const arcllm_cuda_paged_kv& kv, cudaStream_t stream);
int attention_paged_workspace(uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint64_t* out);

}  // namespace arc
