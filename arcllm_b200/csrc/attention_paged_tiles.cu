// Paged attention of requests with many new rows on the 5th-generation tensor
// cores (B200, sm_100a).
//
// An item is one KV head and up to 2 x 128 packed rows ((row, head of the
// group) pairs, whole rows); a unit is a tile of positions.  Per item and tile,
// for each half s of the rows:
//   S_s = Q_s K^T        tcgen05.mma, both operands in shared memory
//   P_s = exp2(S_s - m)  one thread per row: S out of tensor memory, the row's
//                        maximum and sum in registers, P in 16 bits
//   O_s += P_s V         tcgen05.mma, P in tensor memory, V in shared memory
//   warps 0..3, 4..7  softmax of half 0, 1, and its output
//   warp 8            TMA: pages' K and V rows into a ring of tiles
//   warps 9, 10       issue the MMAs of half 0, 1
//   warp 11           TMA: the next item's queries, as soon as the last S of the
//                     item before is there
// Tensor memory (512 columns of 128 rows) decides the tile: with O in 2 x D of
// them, S and P of both halves fit side by side for 80 positions at D = 128, so S
// of the next tile is formed as soon as a softmax has S in its registers; over a
// tile of 128, P has to lie over S, and S of the next tile waits for the product.
// At D = 128 that is not shown to pay: 493 us for the 12000 rows below with tiles of
// 128, 475 to 500 with 80.  At D = 64 a tile is 96 positions, what a thread's
// registers hold, and there is room for two P of each half: P then needs no wait
// for the product before (12 requests, 16 heads, window 1024: 105.2 -> 103.2 us).
// Two P at D = 128 would leave tiles of 64 (12000 rows: 470 -> 504 us).
// O is scaled only when a row's maximum has grown by more than 2^8 since the
// last time (the sums carry the same factor, so the result is the same).
// K and V tiles are built from boxes of positions that divide the page and the
// tile, so tiles and pages need not match.
// All waits are bounded: on a timeout the roles leave their loops, drain what
// they started and the error word is set.
// Measured: 12000 new rows of 2 requests, 28 / 4 heads of 128, contexts of 2048
// before them (0.50 TFLOP): 483 to 492 us one after another in a graph, 1.02 to 1.04
// PFLOP/s, 0.62 of the measured matrix rate; called from Python with pauses between
// 534 to 555 us, 0.55 to 0.57 (the clock follows the power).  The bound is the softmax's
// chain: 2350 clocks per tile of 80 (2580 per tile of 96 at D = 64 with a window) and
// 4700 per item, where the exponentials (16 per clock and SM) of both halves are 1280
// and both halves' products 1460 beside them; the rest is issue and hand-over (a wait
// that is over costs 100 clocks, and the chain has three).  Starting the halves half a
// tile apart changed nothing, nor did a quarter of the exponentials as polynomials on
// the FMA units (0.4 %; half of them 3 % slower).
#include <algorithm>

#include "arcllm_cuda_internal.h"
#include "attention_paged.cuh"
#include "tmem.cuh"

namespace arc {
namespace paged {
namespace {

constexpr uint32_t kThreads = 384;
constexpr float kGrow = 8.f;  // log2 of the growth of a row's maximum that is let pass

template <int D>
struct Layout {
    static constexpr uint32_t kTile = D == 128 ? 80u : 96u;  // positions
    static constexpr uint32_t kMaxBox = D == 128 ? 16u : 32u;  // positions of a copy: divides the tile
    static constexpr uint32_t kParts = D / 64;           // 64-dim parts: a row of one is 128 bytes
    static constexpr uint32_t kGroup = kParts * 1024u;   // 8 positions: [part][8][128 bytes], as the pages' boxes arrive
    static constexpr uint32_t kBytes = kTile / 8u * kGroup;   // a K or V tile
    static constexpr uint32_t kStages = D == 128 ? 6u : 10u;  // K and V tiles in the ring: 120 KB
    static constexpr uint32_t kQPart = 128u * 128u;      // Q: [part][128 rows][128 bytes]
    static constexpr uint32_t kQBytes = kParts * kQPart;
    static constexpr uint32_t kRing = 2u * kQBytes;      // after the two Q halves
    static constexpr uint32_t kOff = kRing + kStages * kBytes;  // unit offsets of the requests
    // columns of tensor memory of half s
    static __device__ __forceinline__ uint32_t s_col(uint32_t s) { return s * kTile; }
    static constexpr uint32_t kPs = D == 128 ? 1u : 2u;  // P of a half: one, or of even and of odd tiles
    static __device__ __forceinline__ uint32_t p_col(uint32_t s, uint32_t n) {  // for the half's tile n
        return 2u * kTile + (s * kPs + n % kPs) * (kTile / 2u);
    }
    static __device__ __forceinline__ uint32_t o_col(uint32_t s) { return 512u - 2u * D + s * D; }
    static_assert((2u + kPs) * kTile <= 512u - 2u * D, "S and P of both halves beside O");
};

// An item costs about this many tiles beside its own (queries in, first S, last
// product, output): they count when the CTAs' stretches are made equal, or one
// that gets many short items takes half as long again.
constexpr uint32_t kItemCost = 2;

// The item that a role is at, and the part of its tiles that this CTA does: of
// the item's units [0, kItemCost + tiles), from v on, as many as are left.
template <uint32_t T>
struct Walk {
    uint32_t r, kvh, mt, v, left;
    uint32_t n_items;  // of the request
    Req q;
    uint32_t first, rows;  // query rows [first, first + rows) of the request
    uint32_t lo, hi;       // their positions
    Span s;
    __device__ __forceinline__ void enter(const Args& a, uint32_t per_item) {
        bool bad = false;
        load_req(a, r, q, bad);
        // the same for all lanes, and known to be
        q.row0 = __shfl_sync(0xffffffffu, q.row0, 0);
        q.n = __shfl_sync(0xffffffffu, q.n, 0);
        q.p0 = __shfl_sync(0xffffffffu, q.p0, 0);
        n_items = (q.n + per_item - 1u) / per_item;
    }
    __device__ __forceinline__ void item(const Args& a, uint32_t per_item) {
        first = mt * per_item;
        rows = min(per_item, q.n - first);
        lo = q.p0 + first;
        hi = lo + rows - 1u;
        s = span_of<T>(a, lo, hi);
    }
    __device__ __forceinline__ uint32_t stop() const { return min(s.n + kItemCost, v + left); }
    __device__ __forceinline__ uint32_t begin() const { return max(v, kItemCost) - kItemCost; }
    __device__ __forceinline__ uint32_t end() const { return max(stop(), kItemCost) - kItemCost; }
    // The next item with tiles for this CTA; false at the stretch's end.
    __device__ __forceinline__ bool next(const Args& a, const uint32_t* off, uint32_t per_item) {
        do {
            left -= stop() - v;
            if (left == 0) return false;
            v = 0;
            if (++mt == n_items) {
                mt = 0;
                if (++kvh == a.kv_heads) {
                    kvh = 0;
                    const uint32_t e = off[r + 1];
                    do ++r;
                    while (off[r + 1] == e);  // units are left, so a request with units follows
                    enter(a, per_item);
                }
            }
            item(a, per_item);
        } while (begin() == end());
        return true;
    }
};

template <uint32_t T>
__device__ __forceinline__ uint32_t item_units(const Args& a, const Req& q, uint32_t mt, uint32_t per_item) {
    const uint32_t first = mt * per_item, rows = min(per_item, q.n - first);
    return kItemCost + span_of<T>(a, q.p0 + first, q.p0 + first + rows - 1u).n;
}

// A role's wait: false once any role has given up.  One vote for the warp also is
// the faster form: a wait that is over costs 96 clocks this way, 215 with a branch
// of its own for each lane (and the MMA warp waits six times per tile).
__device__ __forceinline__ bool role_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, unsigned int* err) {
    return warp_wait(bar, parity, err, [&] { return *abort_flag != 0; });
}

// The 4 x 4 blocks of 16 bytes of four neighbouring lanes, transposed: v[k] of lane j becomes v[j] of lane k.
__device__ __forceinline__ void transpose4(uint4 (&v)[4], uint32_t lane) {
#pragma unroll
    for (uint32_t d = 1; d <= 2u; d <<= 1) {
        const bool up = lane & d;
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
            if (k & d) continue;
            uint4& a = v[k];
            uint4& b = v[k | d];
            const uint4 give = up ? a : b;
            uint4 get;
            get.x = __shfl_xor_sync(0xffffffffu, give.x, d);
            get.y = __shfl_xor_sync(0xffffffffu, give.y, d);
            get.z = __shfl_xor_sync(0xffffffffu, give.z, d);
            get.w = __shfl_xor_sync(0xffffffffu, give.w, d);
            if (up)
                a = get;
            else
                b = get;
        }
    }
}

// Box of the queries' tensor (64 dims, 64-dim parts, heads, rows): packed rows of one part.
__device__ __forceinline__ void tma_queries(void* dst, const CUtensorMap* map, int part, int head, int row,
                                            uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(part), "r"(head), "r"(row), "r"(smem_addr(bar))
        : "memory");
}

// ---- packed pairs of fp32 ------------------------------------------------------
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// largest of the values, NaN if one is
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    attn_paged_tiles_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                            const __grid_constant__ CUtensorMap qmap, PageMap heads, Args a,
                            uint32_t box, Record* __restrict__ recs, float* __restrict__ parts,
                            unsigned int* err) {
    using L = Layout<D>;
    constexpr uint32_t kTile = L::kTile;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_align_up<1024>(smem_raw, 0);
    uint32_t* off = reinterpret_cast<uint32_t*>(smem + L::kOff);
    __shared__ uint64_t kv_full[L::kStages], kv_empty[L::kStages], q_full[2], q_empty[2], s_full[2], s_empty[2],
        p_full[2][L::kPs], p_empty[2][L::kPs], o_full[2], done;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int abort_flag;
    __shared__ uint32_t start[4];
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31u;
    if (tid == 0) {
        for (uint32_t s = 0; s < L::kStages; ++s) mbar_init(&kv_full[s], 1), mbar_init(&kv_empty[s], 2);
        for (uint32_t s = 0; s < 2; ++s) {
            mbar_init(&q_full[s], 1);
            mbar_init(&q_empty[s], 1);
            mbar_init(&s_full[s], 1);
            mbar_init(&s_empty[s], 4);
            for (uint32_t k = 0; k < L::kPs; ++k) mbar_init(&p_full[s][k], 4), mbar_init(&p_empty[s][k], 1);
            mbar_init(&o_full[s], 1);
        }
        mbar_init(&done, 2);
        abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_base)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    pdl_trigger();
    pdl_wait();  // lengths, queries and pages come from the preceding kernels

    // The CTA's stretch.  Units of every request: by its thread where it has few items, by a warp otherwise.
    const uint32_t half_rows = 128u / a.gq, per_item = 2u * half_rows;
    constexpr uint32_t kAlone = 8, kMany = 0xffffffffu;
    bool any_bad = false;
    for (uint32_t r = tid; r < a.n_requests; r += kThreads) {
        Req q;
        unsigned long long u = 0;
        if (load_req(a, r, q, any_bad) && q.n * a.gq > kRowMax) {
            const uint32_t items = (q.n + per_item - 1u) / per_item;
            if (items <= kAlone) {
                for (uint32_t mt = 0; mt < items; ++mt) u += item_units<kTile>(a, q, mt, per_item);
                u = min(u * a.kv_heads, 0xfffffffeull);
            } else {
                u = kMany;
            }
        }
        off[r + 1] = (uint32_t)u;
    }
    __syncthreads();
    for (uint32_t r = warp; r < a.n_requests; r += kThreads / 32u) {
        if (off[r + 1] != kMany) continue;
        Req q;
        bool bad = false;
        load_req(a, r, q, bad);
        const uint32_t items = (q.n + per_item - 1u) / per_item;
        unsigned long long u = 0;
        for (uint32_t mt = lane; mt < items; mt += 32u) u += item_units<kTile>(a, q, mt, per_item);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
        if (lane == 0) off[r + 1] = (uint32_t)min(u * a.kv_heads, 0xfffffffeull);
    }
    __syncthreads();
    const uint32_t total = scan_units(a, off, err, [&](uint32_t r, bool& bad) -> unsigned long long {
        bad = any_bad;
        return off[r + 1];
    });
    const uint32_t per = max((total + gridDim.x - 1u) / gridDim.x, 1u);
    const uint32_t U0 = (uint32_t)min((unsigned long long)blockIdx.x * per, (unsigned long long)total);
    const uint32_t n_units = __shfl_sync(0xffffffffu, min(per, total - U0), 0);
    if (tid == 0) recs[blockIdx.x].valid = 0;
    if (n_units != 0 && warp == 11) {
        const uint32_t r = request_of(off, a.n_requests, U0);
        Req q;
        bool bad = false;
        load_req(a, r, q, bad);
        const uint32_t head = (off[r + 1] - off[r]) / a.kv_heads, kvh = (U0 - off[r]) / head;
        uint32_t rem = U0 - off[r] - kvh * head, mt = 0;
        const uint32_t items = (q.n + per_item - 1u) / per_item;
        for (uint32_t m0 = 0; m0 < items; m0 += 32u) {  // the item that unit rem of the head lies in
            uint32_t v = m0 + lane < items ? item_units<kTile>(a, q, m0 + lane, per_item) : 0u;
            const uint32_t mine = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= (uint32_t)o) v += x;
            }
            const uint32_t over = __ballot_sync(0xffffffffu, v > rem);
            if (over) {
                const int at = __ffs(over) - 1;
                mt = m0 + (uint32_t)at;
                rem -= __shfl_sync(0xffffffffu, v - mine, at);
                break;
            }
            rem -= __shfl_sync(0xffffffffu, v, 31);
        }
        if (lane == 0) start[0] = r, start[1] = kvh, start[2] = mt, start[3] = rem;
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);

    Walk<kTile> w;
    bool any = n_units != 0;
    if (any) {
        w.r = __shfl_sync(0xffffffffu, start[0], 0), w.kvh = __shfl_sync(0xffffffffu, start[1], 0);
        w.mt = __shfl_sync(0xffffffffu, start[2], 0), w.v = __shfl_sync(0xffffffffu, start[3], 0);
        w.left = n_units;
        w.enter(a, per_item);
        w.item(a, per_item);
        if (w.begin() == w.end()) any = w.next(a, off, per_item);
    }
    if (warp >= 8) {
      if (!any) {
        // nothing to do; the tensor memory is given back below
      } else if (warp == 8) {
        // ---------------- TMA: K, V, K, V ... tile by tile ----------------
        const uint32_t boxes = kTile / box;
        uint32_t stage = 0, phase = 0, issued = 0;
        bool bad_page = false, ok = true;
        // lane b: box b of a tile; it is loaded when it holds anything that is seen
        uint32_t i = w.begin(), end = w.end();
        auto entry = [&](const Walk<kTile>& x) -> int {
            const uint32_t p = x.s.tile(i) * kTile + lane * box;
            const uint32_t from = a.window && x.lo >= a.window ? x.lo - a.window + 1u : 0u;
            if (lane >= boxes || p > x.hi || (p + box <= from && p >= a.sinks)) return -1;
            const int page = a.table[(uint64_t)x.r * a.table_stride + p / a.page_size];
            if ((uint32_t)page < a.n_pages) return page;
            bad_page = true;
            return (int)a.n_pages;  // reads zeros
        };
        int page = entry(w);
        for (bool more = true; ok && more;) {
            const uint32_t kvh = w.kvh, token = (w.s.tile(i) * kTile + lane * box) % a.page_size;
            const int now = page;
            if (++i == end) {
                more = w.next(a, off, per_item);
                i = w.begin(), end = w.end();
            }
            if (more) page = entry(w);  // while this tile waits for its places
            const uint32_t n_need = __popc(__ballot_sync(0xffffffffu, now >= 0));
            const int part = (int)(kvh * heads.part0), group = (int)(kvh * heads.group0 + token / 8u);
#pragma unroll
            for (uint32_t kv = 0; kv < 2; ++kv) {
                if (issued >= L::kStages) ok = role_wait(&kv_empty[stage], phase ^ 1u, &abort_flag, err);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(&kv_full[stage], n_need * (box / 8u) * L::kGroup);
                __syncwarp();
                if (now >= 0)
                    tma_page(smem + L::kRing + stage * L::kBytes + lane * (box / 8u) * L::kGroup, kv ? &vmap : &kmap,
                             part, group, now, &kv_full[stage]);
                ++issued;
                if (++stage == L::kStages) stage = 0, phase ^= 1u;
            }
        }
        if (!ok) abort_flag = 1;
        // No copy may still be landing at the end.  That is also waited for when all were issued: another role may have
        // given up before it used the last ones (otherwise this is over long before the output is).
        for (uint32_t k = issued > L::kStages ? issued - L::kStages : 0u; k < issued; ++k)
            warp_wait(&kv_full[k % L::kStages], (k / L::kStages) & 1u, err, [] { return false; });
        if (__any_sync(0xffffffffu, bad_page) && lane == 0) raise_error(err, ARC_DEV_ERR_BOUNDS);
      } else if (warp < 11) {
        // ---------------- MMA of half s ----------------
        constexpr uint32_t kQk = instr_desc<BF16>(kTile, false), kPv = instr_desc<BF16>(D, true);
        const uint32_t s = warp - 9u, leader = lane == 0, ring = smem_addr(smem + L::kRing);
        const uint32_t ts = tmem + L::s_col(s), to = tmem + L::o_col(s);
        const uint64_t qa = operand_desc(smem_addr(smem) + s * L::kQBytes, 16u, 1024u);
        // Tiles come as K, V, K, V ...; K of the next one is used before V of this one.
        struct At {
            uint32_t stage, phase;
            __device__ __forceinline__ void advance() {
                stage += 2u;
                if (stage >= L::kStages) stage -= L::kStages, phase ^= 1u;
            }
        } at_k{0, 0}, at_v{1, 0};
        uint32_t n_item = 0, n_s = 0, n_p = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) { return ok = role_wait(bar, parity, &abort_flag, err); };
        auto qk = [&](bool live) {  // S = Q K^T of the tile at at_k, once the softmax has the last S
            if (!wait(&kv_full[at_k.stage], at_k.phase)) return false;
            if (live) {
                if (n_s != 0u && !wait(&s_empty[s], (n_s - 1u) & 1u)) return false;
                ++n_s;
                tmem_fence_after();
                const uint64_t kb = operand_desc(ring + at_k.stage * L::kBytes, 16u, L::kGroup);
#pragma unroll
                for (uint32_t kk = 0; kk < D / 16u; ++kk)  // addresses count 16 bytes
                    mma_smem(ts, qa + (((kk >> 2) * L::kQPart + (kk & 3u) * 32u) >> 4),
                             kb + (((kk >> 2) * 1024u + (kk & 3u) * 32u) >> 4), kQk, kk != 0u, leader);
                mma_commit(&s_full[s], leader);
            }
            mma_commit(&kv_empty[at_k.stage], leader);
            at_k.advance();
            return true;
        };
        do {
            const uint32_t i0 = w.begin(), i1 = w.end();
            const bool live = s == 0u || w.rows > half_rows;  // otherwise the tiles pass by
            if (live && !wait(&q_full[s], n_item++ & 1u)) break;
            if (!qk(live)) break;
            if (live && i0 + 1u == i1) mma_commit(&q_empty[s], leader);
            for (uint32_t i = i0; i < i1; ++i) {
                if (i + 1u < i1) {
                    if (!qk(live)) break;
                    if (live && i + 2u == i1) mma_commit(&q_empty[s], leader);  // that was the last S
                }
                if (!wait(&kv_full[at_v.stage], at_v.phase)) break;
                // V rows of positions that no row of the item sees are zeroed (by both warps): what lies there may be
                // anything, and the weight 0 does not stop a NaN.
                const uint32_t p0 = w.s.tile(i) * kTile;
                const uint32_t from = a.window && w.lo >= a.window ? w.lo - a.window + 1u : 0u;
                const bool tail = p0 + kTile - 1u > w.hi, gap = p0 < from && p0 + kTile > a.sinks;
                if (tail || gap) {
                    uint8_t* v = smem + L::kRing + at_v.stage * L::kBytes + (lane & 7u) * 16u;
                    auto clear = [&](uint32_t r0, uint32_t r1) {  // rows [r0, r1): 8 lanes a row of 128 bytes
#pragma unroll 2
                        for (uint32_t r = r0 + (lane >> 3); r < r1; r += 4u)
#pragma unroll
                            for (uint32_t c = 0; c < L::kParts; ++c)
                                *reinterpret_cast<uint4*>(v + (r >> 3) * L::kGroup + c * 1024u + (r & 7u) * 128u) =
                                    make_uint4(0, 0, 0, 0);
                    };
                    if (gap) clear(max(a.sinks, p0) - p0, min(from - p0, kTile));
                    if (tail) clear(w.hi + 1u - p0, kTile);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                if (live) {
                    if (!wait(&p_full[s][n_p % L::kPs], n_p / L::kPs & 1u)) break;
                    const uint32_t tp = tmem + L::p_col(s, n_p);
                    tmem_fence_after();
                    const uint64_t vb = operand_desc(ring + at_v.stage * L::kBytes, 1024u, L::kGroup);
#pragma unroll
                    for (uint32_t kk = 0; kk < kTile / 16u; ++kk)
                        mma_tmem(to, tp + kk * 8u, vb + kk * (2u * L::kGroup >> 4), kPv, i != i0 || kk != 0u, leader);
                    mma_commit(&p_empty[s][n_p++ % L::kPs], leader);
                    if (i + 1u == i1) mma_commit(&o_full[s], leader);
                }
                mma_commit(&kv_empty[at_v.stage], leader);
                at_v.advance();
            }
        } while (ok && w.next(a, off, per_item));
        if (!ok) abort_flag = 1;
        mma_commit(&done, leader);
        __syncwarp();
        warp_wait(&done, 0, err, [] { return false; });  // nothing of this CTA runs on the tensor core any more
      } else {
        // ---------------- TMA: queries ----------------
        uint32_t n[2] = {0, 0};
        bool ok = true;
        do {
#pragma unroll
            for (uint32_t s = 0; s < 2u; ++s) {
                if (s * half_rows >= w.rows) continue;
                if (n[s] != 0u) ok = ok && role_wait(&q_empty[s], (n[s] - 1u) & 1u, &abort_flag, err);
                if (!ok) continue;
                ++n[s];
                if (lane == 0) {  // rows past the request's are other requests' or zeros: computed, not stored
                    mbar_arrive_expect_tx(&q_full[s], L::kParts * half_rows * a.gq * 128u);
#pragma unroll
                    for (uint32_t c = 0; c < L::kParts; ++c)
                        tma_queries(smem + s * L::kQBytes + c * L::kQPart, &qmap, (int)c, (int)(w.kvh * a.gq),
                                    (int)(w.q.row0 + w.first + s * half_rows), &q_full[s]);
                }
                __syncwarp();
            }
        } while (ok && w.next(a, off, per_item));
        if (!ok) abort_flag = 1;
#pragma unroll
        for (uint32_t s = 0; s < 2u; ++s)  // no copy may still be landing at the end
            if (n[s] != 0u) warp_wait(&q_full[s], (n[s] - 1u) & 1u, err, [] { return false; });
      }
    } else {
      if (any) {
        // ---------------- softmax of half s: thread t has packed row t ----------------
        const uint32_t s = warp >> 2, t = tid & 127u;
        const uint32_t lanes = ((warp & 3u) * 32u) << 16;
        const uint32_t ts = tmem + lanes + L::s_col(s), to = tmem + lanes + L::o_col(s);
        uint32_t n_s = 0, n_o = 0;  // tiles, items so far
        const uint32_t t_row = t / a.gq;
        bool ok = true;
        for (bool more = true; more;) {
            const uint32_t i0 = w.begin(), i1 = w.end();
            if (s * half_rows >= w.rows) {  // this half has no rows (uniform over its warps)
                more = w.next(a, off, per_item);
                continue;
            }
            const uint32_t sub_rows = min(half_rows, w.rows - s * half_rows);
            const uint32_t p_lo = w.lo + s * half_rows, p_hi = p_lo + sub_rows - 1u;
            const bool live = t_row < sub_rows;
            const uint32_t pos = p_lo + min(t_row, sub_rows - 1u);
            float m = -INFINITY, l = 0.f;
            for (uint32_t i = i0; i < i1; ++i) {
                ok = role_wait(&s_full[s], n_s & 1u, &abort_flag, err);
                if (!ok) break;
                tmem_fence_after();
                float x[kTile];
                tmem_ld(ts, x);
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_empty[s]);  // the next S may come
                const uint32_t p0 = w.s.tile(i) * kTile;
                // not all rows see all of it: behind a row's position, before its window and past the sinks
                const bool past = p0 + kTile - 1u > p_lo;
                const bool before = a.window && p0 + a.window <= p_hi && p0 + kTile > a.sinks;
                if (__builtin_expect(past || before, 0)) {
                    const int last = (int)(pos - p0);
                    if (before) {
                        int first = 0, sinks = 0;
                        if (pos + 1u >= a.window) first = (int)(pos + 1u - a.window - p0), sinks = (int)(a.sinks - p0);
#pragma unroll
                        for (int c = 0; c < (int)kTile; ++c)
                            if (c < first && c >= sinks) x[c] = -INFINITY;
                    }
#pragma unroll
                    for (int c = 0; c < (int)kTile; ++c)
                        if (c > last) x[c] = -INFINITY;
                }
                float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (uint32_t c = 4; c + 8u <= kTile; c += 8u)
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k) mx[k] = max_nan(mx[k], x[c + k], x[c + 4u + k]);
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) mx[k] = max_nan(mx[k], x[kTile - 4u + k]);
                // An infinite score has no softmax: NaN for the row, as for a NaN score.
                float mn = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3])) * a.scale_log2;
                if (mn == INFINITY) mn = NAN;
                bool waited = n_s == 0u;  // for the product before: O, and P's columns where the half has one P
                auto product = [&]() {
                    const uint32_t n = n_s - 1u;
                    if (!waited) ok = role_wait(&p_empty[s][n % L::kPs], n / L::kPs & 1u, &abort_flag, err);
                    waited = true;
                    tmem_fence_after();
                    return ok;
                };
                if (i == i0) {
                    m = mn;  // O is written afresh
                } else if (__builtin_expect(__any_sync(0xffffffffu, live && !(mn <= m + kGrow)), 0)) {
                    const float to_m = max_nan(m, mn);
                    const float f = ex2(m - (to_m == -INFINITY ? 0.f : to_m));
                    l *= f;
                    m = to_m;
                    if (!product()) break;
#pragma unroll 1
                    for (uint32_t c = 0; c < (uint32_t)D; c += 32u) {
                        float o[32];
                        tmem_ld(to + c, o);
                        uint32_t ob[32];
#pragma unroll
                        for (uint32_t k = 0; k < 32u; ++k) ob[k] = __float_as_uint(o[k] * f);
                        tmem_st(to + c, ob);
                    }
                }
                const float ref = m == -INFINITY ? 0.f : m;
                const uint64_t c2 = pair(a.scale_log2, a.scale_log2), r2 = pair(-ref, -ref);
                uint64_t sum[2] = {0ull, 0ull};
                // columns between two stores: beside 96 scores a thread's registers hold the weights of 32
                constexpr uint32_t kAtOnce = kTile == 80u ? 80u : 32u;
#pragma unroll
                for (uint32_t c0 = 0; c0 < kTile; c0 += kAtOnce) {
                    uint32_t pk[kAtOnce / 2u];
#pragma unroll
                    for (uint32_t c = 0; c < kAtOnce; c += 2u) {
                        const float2 y = unpair(fma2(pair(x[c0 + c], x[c0 + c + 1u]), c2, r2));
                        const float2 e = make_float2(ex2(y.x), ex2(y.y));
                        sum[(c >> 1) & 1u] = add2(sum[(c >> 1) & 1u], pair(e.x, e.y));
                        // the product takes weights of the cache's type: half a step of it each, as the output
                        pk[c / 2u] = pack16<BF16>(e.x, e.y);
                    }
                    // Of two Ps this one's last product came before this S on the tensor core: it is over.  A warp may
                    // then be one tile ahead of another of its half, so each P has a barrier of its own, too.
                    if (L::kPs == 1u && c0 == 0u && !product()) break;
                    tmem_st(tmem + lanes + L::p_col(s, n_s) + c0 / 2u, pk);
                }
                if (!ok) break;
                const float2 sm = unpair(add2(sum[0], sum[1]));
                l += sm.x + sm.y;
                tmem_wait_st();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[s][n_s % L::kPs]);
                ++n_s;
            }
            if (ok) ok = role_wait(&o_full[s], n_o & 1u, &abort_flag, err);
            if (!ok) break;
            ++n_o;
            tmem_fence_after();
            const bool whole = i0 == 0 && i1 == w.s.n;
            const uint32_t slot = i0 != 0 ? 0u : 1u;  // began before this stretch, or goes on after it
            float* part = parts + (uint64_t)(blockIdx.x * 2u + slot) * (kTileRows * (D + 2u));
            const uint32_t ri = s * half_rows * a.gq + t;
            uint16_t* out_of[4];  // rows of this thread and its three neighbours
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                const uint32_t tk = (t & ~3u) + k, row = tk / a.gq;
                out_of[k] = row < sub_rows
                                ? a.out + (uint64_t)(w.q.row0 + w.first + s * half_rows + row) * a.out_stride +
                                      (w.kvh * a.gq + tk - row * a.gq) * D
                                : nullptr;
            }
            const float inv = 1.f / l;
#pragma unroll 1
            for (uint32_t c = 0; c < (uint32_t)D; c += 32u) {
                float o[32];
                tmem_ld(to + c, o);
                if (whole) {
                    // 16 bytes of each of four neighbours' rows instead of 64 of its own: a store then touches 8 rows
                    // of 64 bytes rather than 32 of 16
                    uint4 v[4];
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k)
                        v[k] = make_uint4(pack16<BF16>(o[8 * k] * inv, o[8 * k + 1] * inv),
                                          pack16<BF16>(o[8 * k + 2] * inv, o[8 * k + 3] * inv),
                                          pack16<BF16>(o[8 * k + 4] * inv, o[8 * k + 5] * inv),
                                          pack16<BF16>(o[8 * k + 6] * inv, o[8 * k + 7] * inv));
                    transpose4(v, lane);
#pragma unroll
                    for (uint32_t k = 0; k < 4u; ++k)
                        if (out_of[k] != nullptr) *reinterpret_cast<uint4*>(out_of[k] + c + (lane & 3u) * 8u) = v[k];
                } else if (live) {
                    float4* dst = reinterpret_cast<float4*>(part + (uint64_t)ri * D + c);
#pragma unroll
                    for (uint32_t k = 0; k < 8u; ++k)
                        dst[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                }
                __syncwarp();
            }
            tmem_fence_before();  // O has been read
            if (!whole) {
                if (live) *reinterpret_cast<float2*>(part + kTileRows * D + 2u * ri) = make_float2(m, l);
                if (slot == 1u && tid == 0)
                    recs[blockIdx.x] = {1u, (U0 + n_units - w.left - w.v + kItemCost + w.s.n - 1u) / per, w.q.row0 + w.first, w.rows * a.gq, w.kvh,
                                        {0, 0, 0}};
            }
            more = w.next(a, off, per_item);
        }
        if (!ok) abort_flag = 1;
      }
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace

template <int D, bool BF16>
int launch_tiles(const arcllm_cuda_paged_kv& kv, const Args& a, Record* recs, float* parts, cudaStream_t stream) {
    using L = Layout<D>;
    uint32_t box = 16;  // the largest power of two that divides the page, and the tile
    while (box < L::kMaxBox && kv.page_size % (2u * box) == 0u) box *= 2u;
    CUtensorMap kmap, vmap;
    PageMap heads;
    const int st = encode_pages(&kmap, &vmap, &heads, kv, box);
    if (st != ARC_OK) return st;
    CUtensorMap qmap;
    {
        const uint32_t q_heads = a.kv_heads * a.gq;
        const cuuint64_t dims[4] = {64, L::kParts, q_heads, a.max_rows};
        const cuuint64_t strides[3] = {128, 2ull * D, 2ull * a.q_stride};
        const cuuint32_t shape[4] = {64, 1, a.gq, 128u / a.gq}, one[4] = {1, 1, 1, 1};
        const CUresult rc = encode_tiled_fn()(
            &qmap, BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<uint16_t*>(a.q), dims, strides, shape, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (rc != CUDA_SUCCESS) return set_error(ARC_E_CUDA, "attention paged: tensor map of the queries");
    }
    const uint32_t smem = 1024u + L::kOff + 4u * (a.n_requests + 1u);
    cudaError_t e = allow_shared<attn_paged_tiles_kernel<D, BF16>>((int)(1024u + L::kOff + 4u * (kMaxRequests + 1u)));
    if (e == cudaSuccess)
        e = launch_kernel(attn_paged_tiles_kernel<D, BF16>, dim3(kSms), dim3(kThreads), smem, stream, kmap, vmap,
                          qmap, heads, a, box, recs, parts, dev_error_word());
    return e == cudaSuccess ? ARC_OK : set_cuda_error(e, "attention paged tiles launch");
}

template int launch_tiles<64, false>(const arcllm_cuda_paged_kv&, const Args&, Record*, float*, cudaStream_t);
template int launch_tiles<64, true>(const arcllm_cuda_paged_kv&, const Args&, Record*, float*, cudaStream_t);
template int launch_tiles<128, false>(const arcllm_cuda_paged_kv&, const Args&, Record*, float*, cudaStream_t);
template int launch_tiles<128, true>(const arcllm_cuda_paged_kv&, const Args&, Record*, float*, cudaStream_t);

}  // namespace paged
}  // namespace arc
