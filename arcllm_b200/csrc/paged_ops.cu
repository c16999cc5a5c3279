// Step planning and rotary store for a batch of requests over a paged KV
// cache (B200, sm_100a).
//
//   paged_plan     row offsets, cache lengths, block tables, positions and
//                  slots of one step, from the requests' lengths, on the
//                  device (nothing returns to the host, so a captured step
//                  replays with new lengths);
//   rope_kv_paged  + bias, rotary embedding of q and k (adjacent pairs or
//                  halves, all or the first part of a head), q rounded to the
//                  cache's type, k and v stored at their slots.
#include <algorithm>
#include <cmath>
#include <cstdio>

#include <cuda_bf16.h>

#include "arcllm_cuda_internal.h"
#include "common.cuh"
#include "decode_ops.h"
#include "paged_ops.h"

namespace arc {
namespace {

// ---- plan -------------------------------------------------------------------
constexpr uint32_t kPlanThreads = 256;
constexpr uint32_t kPlanMaxRequests = 8192;  // three 32-bit numbers a request in shared memory

// number of entries of the ascending v[0, n) that are <= x, minus one
__device__ __forceinline__ uint32_t last_not_above(const int32_t* v, uint32_t n, int32_t x) {
    uint32_t lo = 0, hi = n;  // v[lo] <= x < v[hi]
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) >> 1;
        if (v[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// Every CTA scans all requests by itself (a few KB out of L2) and then fills
// its share of the rows and of the new table entries, so one launch does it
// without a grid-wide wait: the call is bounded by launch and load latency (256
// requests of a token 3.6 us, 96 requests with 48 chunks of up to 1024 rows 5.3 us).
// total_r = kv_r + new_r; request r starts at row sum of new over the requests
// before it and takes ceil(total_r / page) - ceil(kv_r / page) pages from the
// end of the free list, after the requests before it.
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PagedPlan p, unsigned int* err) {
    pdl_trigger();
    pdl_wait();  // lengths come from the preceding kernels
    extern __shared__ int32_t plan_smem[];
    int32_t* s_row = plan_smem;                   // first row of request r
    int32_t* s_need = s_row + p.n_requests;       // pages taken before request r
    int32_t* s_kv = s_need + p.n_requests;        // kv_r
    __shared__ unsigned long long s_sum[2][kPlanThreads / 32];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t per = (p.n_requests + kPlanThreads - 1u) / kPlanThreads;
    const uint32_t r0 = min(tid * per, p.n_requests), r1 = min(r0 + per, p.n_requests);
    const uint32_t ps = p.page_size;
    unsigned long long rows = 0, need = 0;
    bool bad = false;
    for (uint32_t r = r0; r < r1; ++r) {
        const int32_t kv = p.kv_len[r], nw = p.new_len[r];
        const long long total = (long long)kv + nw;
        if (kv < 0 || nw < 0 || total > 0x7fffffffll) {
            bad = true;
            continue;
        }
        const uint32_t had = ((uint32_t)kv + ps - 1u) / ps, have = ((uint32_t)total + ps - 1u) / ps;
        bad |= have > p.table_stride;
        s_kv[r] = kv;
        rows += (uint32_t)nw;
        need += have - had;
    }
    unsigned long long rs = rows, ns = need;  // inclusive scans of the threads' sums
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long a = __shfl_up_sync(0xffffffffu, rs, o), b = __shfl_up_sync(0xffffffffu, ns, o);
        if (lane >= (uint32_t)o) rs += a, ns += b;
    }
    if (lane == 31u) s_sum[0][warp] = rs, s_sum[1][warp] = ns;
    bad = __syncthreads_or(bad);
    unsigned long long rows_all = 0, need_all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kPlanThreads / 32; ++w) {
        if (w < warp) rs += s_sum[0][w], ns += s_sum[1][w];
        rows_all += s_sum[0][w];
        need_all += s_sum[1][w];
    }
    const int32_t n_free = *p.n_free;
    const bool ok = !bad && rows_all <= p.max_rows && need_all <= (unsigned long long)max(n_free, 0);
    if (!ok) {  // all or nothing: an empty step
        if (blockIdx.x == 0) {
            for (uint32_t r = tid; r <= p.n_requests; r += kPlanThreads) {
                p.row_start[r] = 0;
                if (r < p.n_requests) p.kv_total[r] = p.kv_len[r];
            }
            if (tid == 0) {
                *p.n_free_out = n_free;
                raise_error(err, ARC_DEV_ERR_BOUNDS);
            }
        }
        for (uint32_t t = blockIdx.x * kPlanThreads + tid; t < p.max_rows; t += gridDim.x * kPlanThreads)
            p.positions[t] = 0, p.slots[t] = -1;
        return;
    }
    uint32_t row = (uint32_t)(rs - rows), pages = (uint32_t)(ns - need);
    for (uint32_t r = r0; r < r1; ++r) {
        const uint32_t kv = (uint32_t)s_kv[r], nw = (uint32_t)p.new_len[r];
        s_row[r] = (int32_t)row;
        s_need[r] = (int32_t)pages;
        if (blockIdx.x == 0) {
            p.row_start[r] = (int32_t)row;
            p.kv_total[r] = (int32_t)(kv + nw);
        }
        row += nw;
        pages += (kv + nw + ps - 1u) / ps - (kv + ps - 1u) / ps;
    }
    if (blockIdx.x == 0 && tid == 0) {
        p.row_start[p.n_requests] = (int32_t)rows_all;
        *p.n_free_out = n_free - (int32_t)need_all;
    }
    __syncthreads();
    bool bad_page = false;
    const uint32_t step = gridDim.x * kPlanThreads;
    for (uint32_t i = blockIdx.x * kPlanThreads + tid; i < (uint32_t)need_all; i += step) {
        const uint32_t r = last_not_above(s_need, p.n_requests, (int32_t)i);
        const uint32_t had = ((uint32_t)s_kv[r] + ps - 1u) / ps;
        const int32_t page = p.free_pages[n_free - 1 - (int32_t)i];
        bad_page |= (uint32_t)page >= p.n_pages;
        p.block_table[(uint64_t)r * p.table_stride + had + (i - (uint32_t)s_need[r])] = page;
    }
    for (uint32_t t = blockIdx.x * kPlanThreads + tid; t < p.max_rows; t += step) {
        int32_t pos = 0, slot = -1;
        if (t < (uint32_t)rows_all) {
            const uint32_t r = last_not_above(s_row, p.n_requests, (int32_t)t);
            const uint32_t kv = (uint32_t)s_kv[r], had = (kv + ps - 1u) / ps;
            const uint32_t at = kv + (t - (uint32_t)s_row[r]), b = at / ps;
            pos = (int32_t)at;
            const int32_t page = b < had ? p.block_table[(uint64_t)r * p.table_stride + b]
                                         : p.free_pages[n_free - 1 - (s_need[r] + (int32_t)(b - had))];
            if ((uint32_t)page < p.n_pages)
                slot = page * (int32_t)ps + (int32_t)(at - b * ps);
            else
                bad_page = true;  // the row has no place: -1, as behind the last one
        }
        p.positions[t] = pos;
        p.slots[t] = slot;
    }
    if (bad_page) raise_error(err, ARC_DEV_ERR_BOUNDS);
}

// ---- rotary store -----------------------------------------------------------
template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

template <typename T, int V>
struct alignas(V * sizeof(T) >= 16 ? 16 : alignof(T)) Raw {  // V elements as they lie in memory
    T v[V];
    __device__ __forceinline__ void load(const T* src) {
        if constexpr (V * sizeof(T) >= 16) {
#pragma unroll
            for (uint32_t i = 0; i < V * sizeof(T) / 16; ++i)
                reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = src[i];
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return Elem<T>::get(v[i]); }
};

template <int V, typename T>
__device__ __forceinline__ void store_vec(T* dst, const float (&x)[V]) {
    if constexpr (V * sizeof(T) == 16) {
        uint4 w;
#pragma unroll
        for (int j = 0; j < V; ++j) reinterpret_cast<T*>(&w)[j] = Elem<T>::put(x[j]);
        *reinterpret_cast<uint4*>(dst) = w;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) dst[i] = Elem<T>::put(x[i]);
    }
}

// A unit is 2V elements of one head as two V-wide vectors: the two sides of V
// rotated pairs in the half layout, 2V neighbours otherwise; it is read and
// written by one thread, so q may be rotated in place.  Units of a head: rotated
// ones first.  A thread keeps its unit and walks over rows (a CTA has part
// blockIdx % parts of them); the next row is read before it turns to the current
// one, for which the angles are in shared memory after one barrier.
// Angles pos * freq are formed and reduced to a fraction of a turn in 64 bits
// (at 16384 an fp32 product is already 1e-3 off), then sin and cos in fp32.
// Bounded by HBM traffic for many rows and by latency for few: 8192 rows of 32 / 8
// heads of 128, bf16, 44 us (4.6 TB/s; 64 us with a row per CTA and none read
// ahead, 48 with the unit worked out anew for each row), fp32 52 us (5.8 TB/s); 48
// rows 3.3 us.  Two or three rows ahead, 3 or 4 CTAs' worth of threads per SM, or
// units of 32 elements were 0 to 40 % slower, and without the angles it takes the same.
constexpr uint32_t kRopeThreads = 512;
template <typename TA, typename TC, int V>
__global__ void __launch_bounds__(kRopeThreads) rope_kv_paged_kernel(RopePaged p, arcllm_cuda_paged_kv kv,
                                                                     uint32_t parts, unsigned int* err) {
    pdl_trigger();
    pdl_wait();  // q, k, v come from the preceding kernels
    extern __shared__ float2 rope_smem[];  // (cos, sin) * attn_scale of rot_dim / 2 pairs, twice
    const uint32_t d = kv.head_dim, half = p.rot_dim / 2u;
    const uint32_t per_head = d / (2u * V), rot_units = half / V, rot_heads = p.q_heads + kv.kv_heads;
    const uint32_t u = blockIdx.x % parts * blockDim.x + threadIdx.x;
    const bool live = u < (rot_heads + kv.kv_heads) * per_head;
    const uint32_t head = u / per_head, at = u - head * per_head;  // head of q, k, v in a row; its unit
    const bool is_q = head < p.q_heads, turned = at < rot_units && head < rot_heads;
    const bool halves = p.half_layout && turned;
    const uint32_t oa = halves ? at * V : 2u * at * V;  // places of the vectors in the head
    const uint32_t ob = halves ? half + at * V : oa + V;
    const uint32_t in_part = is_q ? head : head < rot_heads ? head - p.q_heads : head - rot_heads;
    const TA* src = static_cast<const TA*>(is_q ? p.q : head < rot_heads ? p.k : p.v) + in_part * d;
    const uint64_t src_stride = is_q ? p.q_stride : head < rot_heads ? p.k_stride : p.v_stride;
    const float* bias = is_q ? p.bq : head < rot_heads ? p.bk : p.bv;
    struct Item {
        int32_t slot, pos;
        Raw<TA, V> a, b;
    };
    auto fetch = [&](uint32_t row, Item& x) {
        x.slot = __ldg(p.slots + row);
        x.pos = __ldg(p.positions + row);
        if (!live) return;
        x.a.load(src + row * src_stride + oa);
        x.b.load(src + row * src_stride + ob);
    };
    const uint32_t step = gridDim.x / parts;
    Item next;
    fetch(blockIdx.x / parts, next);
    float2* angles = rope_smem;
    for (uint32_t row = blockIdx.x / parts; row < p.rows; row += step) {
        const Item x = next;
        if (p.rows - row > step) fetch(row + step, next);
        if (x.slot < 0) continue;  // a row without a request (the same for all threads)
        if ((uint32_t)x.slot >= kv.n_pages * kv.page_size || x.pos < 0) {
            if (threadIdx.x == 0) raise_error(err, ARC_DEV_ERR_BOUNDS);
            continue;
        }
        angles = angles == rope_smem ? rope_smem + half : rope_smem;  // others may still read the last row's
        for (uint32_t i = threadIdx.x; i < half; i += blockDim.x) {
            const double turns = (double)x.pos * p.freqs[i] * 0.15915494309189533577;  // 1 / (2 pi)
            float s, c;
            sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
            angles[i] = make_float2(c * p.attn_scale, s * p.attn_scale);
        }
        __syncthreads();
        if (!live) continue;
        float za[V], zb[V];
#pragma unroll
        for (int i = 0; i < V; ++i) za[i] = x.a[i], zb[i] = x.b[i];
        if (bias) {
            Raw<float, V> ba, bb;
            ba.load(bias + in_part * d + oa);
            bb.load(bias + in_part * d + ob);
#pragma unroll
            for (int i = 0; i < V; ++i) za[i] += ba[i], zb[i] += bb[i];
        }
        if (turned) {
            const float2* cs = angles + at * V;
            if (p.half_layout) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float s = za[i], t = zb[i];
                    za[i] = s * cs[i].x - t * cs[i].y;
                    zb[i] = s * cs[i].y + t * cs[i].x;
                }
            } else {
                float z[2 * V];
#pragma unroll
                for (int i = 0; i < V; ++i) z[i] = za[i], z[V + i] = zb[i];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float s = z[2 * i], t = z[2 * i + 1];
                    z[2 * i] = s * cs[i].x - t * cs[i].y;
                    z[2 * i + 1] = s * cs[i].y + t * cs[i].x;
                }
#pragma unroll
                for (int i = 0; i < V; ++i) za[i] = z[i], zb[i] = z[V + i];
            }
        }
        TC* dst;
        if (is_q) {
            dst = static_cast<TC*>(p.q_out) + (uint64_t)row * p.out_stride + head * d;
        } else {
            const uint32_t page = (uint32_t)x.slot / kv.page_size, token = (uint32_t)x.slot - page * kv.page_size;
            dst = static_cast<TC*>(head < rot_heads ? kv.k_pages : kv.v_pages) + (uint64_t)page * kv.page_stride +
                  (uint64_t)token * kv.token_stride + (uint64_t)in_part * kv.head_stride;
        }
        store_vec<V>(dst + oa, za);
        store_vec<V>(dst + ob, zb);
    }
}

template <typename TA, typename TC>
cudaError_t launch_rope(const RopePaged& p, const arcllm_cuda_paged_kv& kv, bool vec, cudaStream_t stream) {
    const uint32_t units = (p.q_heads + 2u * kv.kv_heads) * (kv.head_dim / (vec ? 16u : 2u));
    const uint32_t threads = std::min(kRopeThreads, (units + 31u) / 32u * 32u);
    const uint32_t parts = (units + threads - 1u) / threads;
    const uint64_t items = (uint64_t)p.rows * parts;
    const size_t smem = (size_t)p.rot_dim * sizeof(float2);
    auto go = [&](auto kernel) {
        // as many CTAs as fit the card (1024 threads an SM; 1152 of 384 would leave a second wave: 43 -> 55 us), in whole
        // sets of parts, each with its share of the rows
        const uint32_t fit = std::max(148u * std::max(1u, 1024u / threads) / parts, 1u) * parts;
        return launch_kernel(kernel, dim3((uint32_t)std::min<uint64_t>(items, fit)), dim3(threads), smem, stream, p, kv,
                             parts, dev_error_word());
    };
    return vec ? go(rope_kv_paged_kernel<TA, TC, 8>) : go(rope_kv_paged_kernel<TA, TC, 1>);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0u; }

bool overlap(const void* a, uint64_t na, const void* b, uint64_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

// One level of the places of a cache's elements: n steps of `stride` elements.
struct Level {
    uint64_t n, stride;
};

// Page, token and head levels (those of one step left out), widest first; how many, or -1 where they do not
// nest: where a step is shorter than all that the levels within it span, two places can be one.
int cache_levels(const arcllm_cuda_paged_kv& kv, Level (&lv)[3]) {
    const Level all[3] = {{kv.n_pages, kv.page_stride}, {kv.page_size, kv.token_stride}, {kv.kv_heads, kv.head_stride}};
    int n = 0;
    for (const Level& l : all)
        if (l.n > 1u) lv[n++] = l;
    std::sort(lv, lv + n, [](const Level& x, const Level& y) { return x.stride > y.stride; });
    unsigned __int128 extent = kv.head_dim;
    for (int i = n - 1; i >= 0; --i) {
        if (lv[i].stride < extent) return -1;
        extent += (unsigned __int128)lv[i].stride * (lv[i].n - 1u);
    }
    return n;
}

// Whether an element at sum of i * stride + dim, with i and dim in range, can equal one of another cache of the same
// levels that begins `off` elements after it: with nested levels the difference of i is one of two at each level.
bool caches_meet(const Level* lv, int n, __int128 off, uint32_t dim) {
    if (n == 0) return off < (__int128)dim && -off < (__int128)dim;
    const __int128 s = lv->stride, lo = off >= 0 ? off / s : -((-off + s - 1) / s), last = (__int128)lv->n - 1;
    for (__int128 d = lo; d <= lo + 1; ++d)
        if (d <= last && -d <= last && caches_meet(lv + 1, n - 1, off - d * s, dim)) return true;
    return false;
}

}  // namespace

int paged_plan(const PagedPlan& p, cudaStream_t stream) {
    if (!p.kv_len || !p.new_len || !p.free_pages || !p.n_free || !p.block_table || !p.row_start || !p.kv_total ||
        !p.positions || !p.slots || !p.n_free_out)
        return set_error(ARC_E_INVALID_ARGUMENT, "paged plan: null pointer");
    if (any_off(4u, p.kv_len, p.new_len, p.free_pages, p.n_free, p.block_table, p.row_start, p.kv_total, p.positions,
                p.slots, p.n_free_out))
        return set_error(ARC_E_ALIGNMENT, "paged plan: arrays of 32-bit words");
    if (p.n_requests == 0 || p.page_size == 0 || p.n_pages == 0 || p.table_stride == 0 || p.max_rows == 0 ||
        p.max_rows > 0x7fffffffu)
        return set_error(ARC_E_INVALID_ARGUMENT, "paged plan: zero size, or rows past 2^31");
    if ((uint64_t)p.n_pages * p.page_size > 0x7fffffffull)
        return set_error(ARC_E_UNSUPPORTED_SHAPE, "paged plan: more than 2^31 - 1 slots");
    if (p.n_requests > kPlanMaxRequests)
        return set_error(ARC_E_UNSUPPORTED_SHAPE, "paged plan: at most 8192 requests");
    // every CTA reads the inputs and old table entries while others write, and each output is written by itself (how
    // long the free list is only the device knows)
    const uint64_t n4 = 4ull * p.n_requests, m4 = 4ull * p.max_rows;
    const struct {
        const void* at;
        uint64_t bytes;
    } array[] = {{p.row_start, n4 + 4u}, {p.kv_total, n4}, {p.positions, m4}, {p.slots, m4}, {p.n_free_out, 4u},
                 {p.block_table, n4 * p.table_stride}, {p.kv_len, n4}, {p.new_len, n4}, {p.n_free, 4u}};
    for (int i = 0; i < 6; ++i)
        for (int j = i + 1; j < 9; ++j)
            if (overlap(array[i].at, array[i].bytes, array[j].at, array[j].bytes))
                return set_error(ARC_E_INVALID_ARGUMENT, "paged plan: an output overlaps another array");
    const uint32_t smem = 12u * p.n_requests;
    if (smem > 48u * 1024u - 1024u) {
        const cudaError_t e = allow_shared<paged_plan_kernel>(12 * kPlanMaxRequests);
        if (e != cudaSuccess) return set_cuda_error(e, "paged plan");
    }
    const uint32_t grid = std::min(148u, (p.max_rows + 4u * kPlanThreads - 1u) / (4u * kPlanThreads));
    return launch_checked(
        launch_kernel(paged_plan_kernel, dim3(grid), dim3(kPlanThreads), smem, stream, p, dev_error_word()),
        "paged plan launch");
}

int rope_freqs(int scaling, uint32_t rot_dim, double theta, double factor, double trained_ctx, double* freqs,
               float* attn_scale) {
    if (!freqs || !attn_scale) return set_error(ARC_E_INVALID_ARGUMENT, "rope freqs: null pointer");
    if (rot_dim == 0 || rot_dim % 2u || !(theta > 0.0) || !std::isfinite(theta))
        return set_error(ARC_E_INVALID_ARGUMENT, "rope freqs: even rot_dim and theta > 0");
    if (scaling < ARC_ROPE_NONE || scaling > ARC_ROPE_YARN)
        return set_error(ARC_E_INVALID_ARGUMENT, "rope freqs: unknown scaling");
    if (scaling != ARC_ROPE_NONE && !(factor >= 1.0 && std::isfinite(factor)))
        return set_error(ARC_E_INVALID_ARGUMENT, "rope freqs: factor below 1");
    if (scaling == ARC_ROPE_YARN && !(trained_ctx > 0.0 && std::isfinite(trained_ctx) && theta > 1.0))
        return set_error(ARC_E_INVALID_ARGUMENT, "rope freqs: YaRN needs the trained context and theta > 1");
    const double d = rot_dim;
    const double base =
        scaling == ARC_ROPE_NTK && rot_dim > 2u ? theta * std::pow(factor, d / (d - 2.0)) : theta;
    // the pair that turns `turns` times over the trained context
    auto turns_at = [&](double turns) {
        return d * std::log(trained_ctx / (turns * 6.283185307179586477)) / (2.0 * std::log(theta));
    };
    double low = 0.0, high = 1.0;
    if (scaling == ARC_ROPE_YARN) {
        low = std::max(0.0, std::floor(turns_at(32.0)));
        high = std::min(d - 1.0, std::ceil(turns_at(1.0)));
    }
    for (uint32_t i = 0; i < rot_dim / 2u; ++i) {
        double f = std::pow(base, -2.0 * i / d);
        if (scaling == ARC_ROPE_LINEAR) f /= factor;
        if (scaling == ARC_ROPE_YARN) {
            const double keep = 1.0 - std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 0.001)));
            f = f / factor * (1.0 - keep) + f * keep;
        }
        freqs[i] = f;
    }
    *attn_scale = scaling == ARC_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return ARC_OK;
}

int check_paged_kv(const arcllm_cuda_paged_kv* kv, const char* who) {
    char msg[160];
    auto fail = [&](int status, const char* what) {
        std::snprintf(msg, sizeof msg, "%s: %s", who, what);
        return set_error(status, msg);
    };
    if (!kv || !kv->k_pages || !kv->v_pages) return fail(ARC_E_INVALID_ARGUMENT, "null cache");
    if (kv->type != ARC_GGML_F16 && kv->type != ARC_GGML_BF16)
        return fail(ARC_E_INVALID_ARGUMENT, "the cache is F16 or BF16");
    if (kv->n_pages == 0 || kv->page_size == 0 || kv->kv_heads == 0 || kv->head_dim == 0)
        return fail(ARC_E_INVALID_ARGUMENT, "zero cache size");
    if ((uint64_t)kv->n_pages * kv->page_size > 0x7fffffffull)
        return fail(ARC_E_UNSUPPORTED_SHAPE, "more than 2^31 - 1 slots");
    if (kv->token_stride < kv->head_dim || kv->head_stride < kv->head_dim || kv->page_stride < kv->head_dim)
        return fail(ARC_E_INVALID_ARGUMENT, "a stride shorter than a head");
    return ARC_OK;
}

int rope_kv_paged(int act_type, const RopePaged& p, const arcllm_cuda_paged_kv& kv, cudaStream_t stream) {
    if (p.rows == 0) return ARC_OK;
    if (!p.q || !p.k || !p.v || !p.freqs || !p.positions || !p.slots || !p.q_out)
        return set_error(ARC_E_INVALID_ARGUMENT, "rope paged: null pointer");
    if (act_type != ARC_GGML_F32 && act_type != ARC_GGML_F16 && act_type != ARC_GGML_BF16)
        return set_error(ARC_E_INVALID_ARGUMENT, "rope paged: activations are F32, F16 or BF16");
    if (kv.head_dim % 2u || p.rot_dim % 2u || p.rot_dim > kv.head_dim || p.rot_dim == 0 || p.q_heads == 0 ||
        p.rows > 0x7fffffffu || kv.head_dim > 4096u || p.q_heads > 65536u || kv.kv_heads > 65536u)
        return set_error(ARC_E_INVALID_ARGUMENT, "rope paged: bad shape");
    if (p.half_layout != ARC_ROPE_INTERLEAVED && p.half_layout != ARC_ROPE_HALVES)
        return set_error(ARC_E_INVALID_ARGUMENT, "rope paged: unknown layout");
    const uint64_t qn = (uint64_t)p.q_heads * kv.head_dim, kn = (uint64_t)kv.kv_heads * kv.head_dim;
    if (p.q_stride < qn || p.out_stride < qn || p.k_stride < kn || p.v_stride < kn)
        return set_error(ARC_E_INVALID_ARGUMENT, "rope paged: a row stride shorter than the row");
    const uint64_t as = act_type == ARC_GGML_F32 ? 4u : 2u;
    if (any_off(as, p.q, p.k, p.v) || any_off(2u, p.q_out, kv.k_pages, kv.v_pages) ||
        any_off(4u, p.bq, p.bk, p.bv, p.positions, p.slots) || any_off(8u, p.freqs))
        return set_error(ARC_E_ALIGNMENT, "rope paged: pointers aligned to their type");
    // in place (the same rows of the same type) or apart
    auto meets_out = [&](const void* x, uint64_t stride, uint64_t width) {
        return rows_meet(x, stride * as, width * as, p.q_out, p.out_stride * 2u, qn * 2u, p.rows);
    };
    if (p.q == p.q_out ? act_type != kv.type || p.q_stride != p.out_stride : meets_out(p.q, p.q_stride, qn))
        return set_error(ARC_E_INVALID_ARGUMENT, "rope paged: q_out overlaps q without being the same rows");
    if (meets_out(p.k, p.k_stride, kn) || meets_out(p.v, p.v_stride, kn))
        return set_error(ARC_E_INVALID_ARGUMENT, "rope paged: q_out overlaps k or v");
    // Two threads would write one element (attention, which only reads, takes such a cache).
    Level lv[3];
    const int levels = cache_levels(kv, lv);
    if (levels < 0)
        return set_error(ARC_E_INVALID_ARGUMENT, "rope paged: strides that lay places of the cache over one another");
    const int64_t between =
        (int64_t)(reinterpret_cast<uintptr_t>(kv.v_pages) - reinterpret_cast<uintptr_t>(kv.k_pages));
    if (caches_meet(lv, levels, between / 2, kv.head_dim))
        return set_error(ARC_E_INVALID_ARGUMENT, "rope paged: K and V of the cache share places");
    // 16-byte vectors where every vector starts on 16 bytes and no unit is part rotated (8192 rows of 32 / 8 heads 44 us);
    // else element by element (132 us)
    const bool vec = p.rot_dim % 16u == 0u && kv.head_dim % 16u == 0u && aligned16(p.q) && aligned16(p.k) &&
                     aligned16(p.v) && aligned16(p.q_out) && aligned16(kv.k_pages) && aligned16(kv.v_pages) &&
                     ((p.q_stride | p.k_stride | p.v_stride) * as) % 16u == 0u && p.out_stride % 8u == 0u &&
                     kv.page_stride % 8u == 0u && kv.token_stride % 8u == 0u && kv.head_stride % 8u == 0u &&
                     (!p.bq || aligned16(p.bq)) && (!p.bk || aligned16(p.bk)) && (!p.bv || aligned16(p.bv));
    const bool bf = kv.type == ARC_GGML_BF16;
    cudaError_t e;
    if (act_type == ARC_GGML_F32)
        e = bf ? launch_rope<float, __nv_bfloat16>(p, kv, vec, stream) : launch_rope<float, __half>(p, kv, vec, stream);
    else if (act_type == ARC_GGML_F16)
        e = bf ? launch_rope<__half, __nv_bfloat16>(p, kv, vec, stream)
               : launch_rope<__half, __half>(p, kv, vec, stream);
    else
        e = bf ? launch_rope<__nv_bfloat16, __nv_bfloat16>(p, kv, vec, stream)
               : launch_rope<__nv_bfloat16, __half>(p, kv, vec, stream);
    return launch_checked(e, "rope paged launch");
}

}  // namespace arc
