// Shared parts of the paged attention kernels (attention_paged.cu): the
// arguments, what a group of query rows sees, the partial results of work that
// is split between CTAs, and the tensor-core and TMA wrappers.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include <cstdint>

#include "common.cuh"
#include "paged_ops.h"

namespace arc {
namespace paged {

constexpr uint32_t kSms = 148;          // one CTA per SM in both attention kernels
constexpr uint32_t kMaxRequests = 4096; // unit offsets of the requests in shared memory

struct Args {
    const uint16_t* q;
    uint16_t* out;
    uint64_t q_stride, out_stride;
    const int32_t* table;
    uint32_t table_stride;
    const int32_t *row_start, *kv_total;
    uint32_t n_requests, max_rows, max_new, kv_heads, gq, page_size, n_pages;
    float scale_log2;  // scale * log2(e): the softmax runs on powers of two
    uint32_t window, sinks;
};

// A request's new rows and where they stand: row i of n is at position p0 + i.
struct Req {
    uint32_t row0, n, p0;
};

// False (and the error word's bounds bit) for lengths that no step can have;
// such a request's rows are left as they were.
__device__ __forceinline__ bool load_req(const Args& a, uint32_t r, Req& q, bool& bad) {
    const int32_t s = a.row_start[r], e = a.row_start[r + 1], total = a.kv_total[r];
    q.row0 = (uint32_t)s;
    q.n = (uint32_t)(e - s);
    q.p0 = (uint32_t)(total - (e - s));
    if (e == s && s >= 0) return false;
    if (s < 0 || e < s || (uint32_t)e > a.max_rows || (uint32_t)(e - s) > a.max_new || total < e - s ||
        ((uint32_t)total - 1u) / a.page_size >= a.table_stride) {
        bad = true;
        return false;
    }
    return true;
}

// Tiles of T positions that hold anything rows at positions lo .. hi see: the
// sinks' tiles, then those from the first position of row lo's window on.
struct Span {
    uint32_t sink_tiles, first, n;
    __device__ __forceinline__ uint32_t tile(uint32_t i) const { return i < sink_tiles ? i : first + i - sink_tiles; }
};
template <uint32_t T>
__device__ __forceinline__ Span span_of(const Args& a, uint32_t lo, uint32_t hi) {
    Span s;
    const uint32_t from = a.window && lo >= a.window ? lo - a.window + 1u : 0u;
    s.first = from / T;
    s.sink_tiles = a.window ? min((min(a.sinks, hi + 1u) + T - 1u) / T, s.first) : 0u;
    s.n = s.sink_tiles + hi / T - s.first + 1u;
    return s;
}

__device__ __forceinline__ bool visible(const Args& a, uint32_t pos, uint32_t at) {
    return at <= pos && (a.window == 0u || at + a.window > pos || at < a.sinks);
}

// The part of an item (a group of query rows and one KV head) that a CTA did,
// when other CTAs did the rest: rows x D sums, then (maximum, sum) of each row.
// Slot 0 of a CTA: an item that began before its share; slot 1: one that goes on after it.
struct Record {
    uint32_t valid, last_cta, row0, rows, kvh, pad[3];
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    uint32_t r;
    if constexpr (BF16)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Box of the pages' tensor (dim, token, KV head, page) into shared memory; out of range reads zero.
__device__ __forceinline__ void tma_page(void* dst, const CUtensorMap* map, int dim, int token, int head, int page,
                                         uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(dim), "r"(token), "r"(head), "r"(page), "r"(smem_addr(bar))
        : "memory");
}

}  // namespace paged
}  // namespace arc
