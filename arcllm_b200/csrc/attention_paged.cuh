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
constexpr uint32_t kTileRows = 256;     // packed rows of an item of the tile kernel
// Requests with at most so many packed rows go to the rows kernel, whose matrix operand has 16.  32 requests over
// 4096 positions of 8 heads: 16 rows there 97 us (4 rows 94), 17 rows in the tile kernel 117 to 121 us (32 rows 122); 64
// over 512: 40 and 50 to 53 us; 4 over 4096: 23 and 24 to 26 us.
constexpr uint32_t kRowMax = 16;
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

// A wait of a whole warp, false once it has taken limit_ns (then with the timeout
// bit) or `stop()` says so.  One vote decides for all lanes, so they go on or give
// up together: what follows are instructions of the whole warp, which lanes that
// decided for themselves at the end of the limit would not reach together.  The first
// tries do not read the global timer: that takes longer than most of these waits do,
// and what arrives meanwhile is seen after it.
template <typename Stop>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned int* err, Stop stop,
                                          unsigned long long limit_ns = kWaitLimitNs) {
    unsigned long long t0 = 0;
    for (uint32_t n = 0; !__all_sync(0xffffffffu, mbar_try_wait(bar, parity)); ++n) {
        if (n < 64u) continue;
        const unsigned long long t = globaltimer();
        if (n == 64u) t0 = t;
        const bool late = t - t0 > limit_ns;
        if (late) raise_error(err, ARC_DEV_ERR_TIMEOUT);
        if (__any_sync(0xffffffffu, late || stop())) return false;
    }
    return true;
}

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

// The request that unit u of the line belongs to.
__device__ __forceinline__ uint32_t request_of(const uint32_t* off, uint32_t n, uint32_t u) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) >> 1;
        if (off[mid] <= u)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// Units of every request before request r, in off[0 .. n]; all threads of the
// CTA.  Returns the total, or 0 where it does not fit 31 bits.
template <typename Units>
__device__ __forceinline__ uint32_t scan_units(const Args& a, uint32_t* off, unsigned int* err, Units units) {
    __shared__ unsigned long long s_warp[32];
    __shared__ int s_bad;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (threadIdx.x == 0) s_bad = 0, off[0] = 0;
    unsigned long long base = 0;
    for (uint32_t r0 = 0; r0 < a.n_requests; r0 += blockDim.x) {
        const uint32_t r = r0 + threadIdx.x;
        bool bad = false;
        unsigned long long v = 0;
        if (r < a.n_requests) v = units(r, bad);
        __syncthreads();
        if (bad) s_bad = 1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long x = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= (uint32_t)o) v += x;
        }
        if (lane == 31u) s_warp[warp] = v;
        __syncthreads();
        unsigned long long all = 0;
        for (uint32_t w = 0; w < warps; ++w) {
            if (w < warp) v += s_warp[w];
            all += s_warp[w];
        }
        if (r < a.n_requests) off[r + 1] = (uint32_t)(base + v);
        base += all;
    }
    __syncthreads();
    const bool too_many = base > 0x7fffffffull;
    if (threadIdx.x == 0 && blockIdx.x == 0 && (s_bad || too_many)) raise_error(err, ARC_DEV_ERR_BOUNDS);
    return too_many ? 0u : (uint32_t)base;
}

// The pages as a tensor of (64 dims, 8 tokens, 64-dim parts, groups of 8 tokens,
// pages): a box of all parts of some groups of one page arrives in shared memory
// as [group][part][8 tokens][128 bytes], one copy for what would be a copy per
// part otherwise (a copy costs about 50 clocks beside its 2.2 per 128 bytes:
// 32 KB in boxes of 16 tokens 1390 -> 963 clocks).  KV heads are a stretch of the
// parts where pages hold token after token, of the groups where they hold head
// after head.
struct PageMap {
    uint32_t part0, group0;  // what one KV head adds to the coordinates
};
// Out of range (a page number of none) reads zeros.
__device__ __forceinline__ void tma_page(void* dst, const CUtensorMap* map, int part, int group, int page,
                                         uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %3, %4, "
        "%5}], [%6];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(part), "r"(group), "r"(page), "r"(smem_addr(bar))
        : "memory");
}

// Tensor maps of K and V with boxes of `tokens` positions of one head of one page, 128-byte swizzle.
int encode_pages(CUtensorMap* k, CUtensorMap* v, PageMap* heads, const arcllm_cuda_paged_kv& kv, uint32_t tokens);

// The requests with more than kRowMax packed rows (attention_paged_tiles.cu).
template <int D, bool BF16>
int launch_tiles(const arcllm_cuda_paged_kv& kv, const Args& a, Record* recs, float* parts,
                 cudaStream_t stream);

}  // namespace paged
}  // namespace arc
