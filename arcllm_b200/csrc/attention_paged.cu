// Attention of a batch's new rows over a paged KV cache (B200, sm_100a).
//
// o_i = sum_j softmax_j(scale q_i . k_j) v_j over the positions j that row i
// sees: j <= p_i, and with a window j > p_i - window or j < sinks.  The query
// heads of one KV head share its keys and values, so (row, head of the group)
// pairs are packed into the rows of one matrix operand.  Work is counted in
// units (an item's tile of positions), the units of all requests stand in one
// line, and every CTA takes an equal stretch of it: contexts of any mixture of
// lengths keep all SMs equally busy.  What is split between CTAs is joined by
// a second, small launch.
#include <algorithm>
#include <cmath>

#include "arcllm_cuda_internal.h"
#include "attention_paged.cuh"
#include "decode_ops.h"

namespace arc {
namespace {

using namespace paged;

// ---- few rows: one warp per stretch ------------------------------------------
// A unit is a tile of 16 positions of a request and KV head; each warp has a
// stretch of the line and a ring of tiles that TMA fills ahead of it, and its
// scores, weights and sums stay in registers (m16n8k16 instructions; a row of the
// operand is a (row, head of the group) pair).  Parts of an item that lie in one
// CTA are joined here, what CTAs share by the join kernel.
// HBM bound: 64 requests of 1 row over up to 8192 positions, 8 heads of 128 (1.07
// GB) 177 us with the join, 6.1 TB/s, 0.93 of the measured copy rate, replayed in a
// graph (180 to 194 us called from Python); 4 requests over up to 79508 positions (1.12
// GB) 181 us.  One request over 1027 positions 11 us, a third of it the join's launch.
constexpr uint32_t kRowWarps = 8, kRowTile = 16;

struct Segment {  // an unfinished item of a warp
    uint32_t valid, u0, u1, r, kvh;
};

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// Position in the line of units: request, KV head, tile.
struct Cursor {
    uint32_t r, kvh, i;
    Req q;
    Span s;
    __device__ __forceinline__ void enter(const Args& a) {  // request r's sizes
        bool bad = false;
        load_req(a, r, q, bad);
        s = span_of<kRowTile>(a, q.p0, q.p0 + q.n - 1u);
    }
    __device__ __forceinline__ void seek(const Args& a, const uint32_t* off, uint32_t u) {
        r = request_of(off, a.n_requests, u);
        enter(a);
        kvh = (u - off[r]) / s.n;
        i = u - off[r] - kvh * s.n;
    }
    __device__ __forceinline__ void next(const Args& a, const uint32_t* off) {
        if (++i < s.n) return;
        i = 0;
        if (++kvh < a.kv_heads) return;
        kvh = 0;
        const uint32_t end = off[r + 1];
        do ++r;
        while (r < a.n_requests && off[r + 1] == end);  // requests without units
        if (r < a.n_requests) enter(a);
    }
};

template <int D, bool BF16>
__global__ void __launch_bounds__(kRowWarps * 32, 1)
    attn_paged_rows_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                           PageMap heads, Args a, uint32_t slot_rows, uint32_t stages,
                           Record* __restrict__ recs, float* __restrict__ parts, unsigned int* err) {
    constexpr uint32_t GB = D / 64 * 1024u;  // 8 positions: [64-dim part][8][128 bytes]
    constexpr uint32_t TILE = kRowTile / 8u * GB, STAGE = 2u * TILE;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_align_up<1024>(smem_raw, 0);
    const uint32_t slot_floats = slot_rows * (D + 2u);
    uint8_t* rings = smem;
    float* firsts = reinterpret_cast<float*>(smem + kRowWarps * stages * STAGE);
    uint32_t* off = reinterpret_cast<uint32_t*>(firsts + kRowWarps * slot_floats);
    __shared__ uint64_t bars[kRowWarps][4];
    __shared__ Segment segs[kRowWarps][2];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
    if (lane < stages) mbar_init(&bars[warp][lane], 1);
    if (lane < 2) segs[warp][lane].valid = 0;
    fence_mbar_init();
    pdl_trigger();
    pdl_wait();  // lengths, queries and pages come from the preceding kernels
    const uint32_t total = scan_units(a, off, err, [&](uint32_t r, bool& bad) -> unsigned long long {
        Req q;
        if (!load_req(a, r, q, bad) || q.n * a.gq > kRowMax) return 0;
        return (unsigned long long)a.kv_heads * span_of<kRowTile>(a, q.p0, q.p0 + q.n - 1u).n;
    });
    // equal shares of whole rounds of the CTA's warps
    const uint32_t per = max(((total + gridDim.x - 1u) / gridDim.x + kRowWarps - 1u) / kRowWarps, 1u) * kRowWarps;
    const uint32_t U0 = min(blockIdx.x * per, total), U1 = min(U0 + per, total);
    if (tid == 0) recs[blockIdx.x].valid = 0;
    if (U0 == U1) return;
    const uint32_t pw = per / kRowWarps;
    const uint32_t u0 = min(U0 + warp * pw, U1), n_units = min(u0 + pw, U1) - u0;

    uint8_t* ring = rings + warp * stages * STAGE;
    bool bad_page = false;
    if (n_units) {
        Cursor ci, cc;
        ci.seek(a, off, u0);
        cc = ci;
        auto entry = [&](const Cursor& c) -> int {  // the page of a cursor's tile
            return __ldg(a.table + (uint64_t)c.r * a.table_stride + c.s.tile(c.i) * kRowTile / a.page_size);
        };
        int page = entry(ci);
        uint32_t issued = 0, si = 0;
        auto issue = [&]() {
            const uint32_t pos = ci.s.tile(ci.i) * kRowTile;
            uint64_t* bar = &bars[warp][si];
            uint8_t* st = ring + si * STAGE;
            if ((uint32_t)page >= a.n_pages) {
                bad_page = true;
                page = (int)a.n_pages;  // reads zeros
            }
            if (lane == 0) {
                mbar_arrive_expect_tx(bar, STAGE);
                const int part = (int)(ci.kvh * heads.part0);
                const int group = (int)(ci.kvh * heads.group0 + pos % a.page_size / 8u);
                tma_page(st, &kmap, part, group, page, bar);
                tma_page(st + TILE, &vmap, part, group, page, bar);
            }
            si = si + 1u == stages ? 0u : si + 1u;
            ++issued;
            if (issued < n_units) {
                ci.next(a, off);
                page = entry(ci);  // used one tile later
            }
        };
        for (uint32_t s = 0; s < stages && s < n_units; ++s) issue();

        uint32_t qa[D / 16][4];
        float o[D / 8][4];
        float m[2], l[2];
        uint32_t pos_of[2];
        uint32_t s_cons = 0, parity = 0, seg_u0 = u0;
        uint32_t item_rows = 0, item_row0 = 0;
        bool first_seg = true, ok = true;
        uint32_t it = 0;
        for (; it < n_units; ++it) {
            if (it == 0 || cc.i == 0) {  // a new item: its queries into A fragments
                seg_u0 = u0 + it;
                first_seg = it == 0;
                item_rows = cc.q.n * a.gq;
                item_row0 = cc.q.row0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t ri = min(g + 8u * h, item_rows - 1u), qr = ri / a.gq;
                    pos_of[h] = cc.q.p0 + qr;
                    const uint16_t* src = a.q + (uint64_t)(item_row0 + qr) * a.q_stride +
                                          (cc.kvh * a.gq + ri - qr * a.gq) * D + 2u * t;
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        qa[kk][h] = *reinterpret_cast<const uint32_t*>(src + 16 * kk);
                        qa[kk][h + 2] = *reinterpret_cast<const uint32_t*>(src + 16 * kk + 8);
                    }
                    m[h] = -INFINITY, l[h] = 0.f;
                }
#pragma unroll
                for (int nt = 0; nt < D / 8; ++nt) o[nt][0] = o[nt][1] = o[nt][2] = o[nt][3] = 0.f;
            }
            if (!warp_wait(&bars[warp][s_cons], parity, err, [] { return false; })) {
                ok = false;
                break;
            }
            const uint32_t ks = smem_addr(ring + s_cons * STAGE), vs = ks + TILE;
            const uint32_t mi = lane >> 3, mr = lane & 7u;
            const uint32_t p_tile = cc.s.tile(cc.i) * kRowTile;
            float sc[2][4];
#pragma unroll
            for (int pb = 0; pb < 2; ++pb) {
                sc[pb][0] = sc[pb][1] = sc[pb][2] = sc[pb][3] = 0.f;
#pragma unroll
                for (int kk = 0; kk < D / 16; kk += 2) {
                    uint32_t b[4];
                    const uint32_t ch = 2u * (kk & 3) + mi;  // 16-byte column of the 128-byte row
                    ldmatrix4(b, ks + pb * GB + (kk >> 2) * 1024u + mr * 128u + ((ch ^ mr) << 4));
                    mma_16816<BF16>(sc[pb], qa[kk], b[0], b[1]);
                    mma_16816<BF16>(sc[pb], qa[kk + 1], b[2], b[3]);
                }
            }
            // positions that row g + 8(c >> 1) does not see
#pragma unroll
            for (int pb = 0; pb < 2; ++pb)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    sc[pb][c] = visible(a, pos_of[c >> 1], p_tile + 8u * pb + 2u * t + (c & 1)) ? sc[pb][c] * a.scale_log2
                                                                                                 : -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float mx = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[h], mx);
                const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen so far: all weights 0
                const float alpha = ex2(m[h] - ref);
                m[h] = mn;
                float ps = 0.f;
#pragma unroll
                for (int pb = 0; pb < 2; ++pb)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        sc[pb][2 * h + c] = ex2(sc[pb][2 * h + c] - ref);
                        ps += sc[pb][2 * h + c];
                    }
                l[h] = fmaf(l[h], alpha, ps);  // this lane's columns; the quad's are added at the end
#pragma unroll
                for (int nt = 0; nt < D / 8; ++nt) o[nt][2 * h] *= alpha, o[nt][2 * h + 1] *= alpha;
            }
            // Weights in the cache's type for the matrix product: half a step of it each, as the output's own rounding.
            const uint32_t pa[4] = {pack16<BF16>(sc[0][0], sc[0][1]), pack16<BF16>(sc[0][2], sc[0][3]),
                                    pack16<BF16>(sc[1][0], sc[1][1]), pack16<BF16>(sc[1][2], sc[1][3])};
            // What no row of the item sees (behind the last position, before the window) may hold anything, and
            // 0 * NaN would reach the sums: such values are read as zero.  A fragment register holds positions
            // 8(j & 1) + 2t, + 1.
            const uint32_t p_last = cc.q.p0 + cc.q.n - 1u;
            const uint32_t p_from = a.window && cc.q.p0 >= a.window ? cc.q.p0 - a.window + 1u : 0u;
            const bool edge = p_tile + kRowTile - 1u > p_last || (p_tile < p_from && p_tile + kRowTile > a.sinks);
            uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
            if (edge) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t p = p_tile + 8u * j + 2u * t;
                    const bool k0 = p <= p_last && (p >= p_from || p < a.sinks);
                    const bool k1 = p + 1u <= p_last && (p + 1u >= p_from || p + 1u < a.sinks);
                    keep[j] = (k0 ? 0xffffu : 0u) | (k1 ? 0xffff0000u : 0u);
                }
            }
#pragma unroll
            for (int nt = 0; nt < D / 8; nt += 2) {
                uint32_t v[4];
                const uint32_t ch = (nt & 7) + (mi >> 1);
                ldmatrix4_trans(v, vs + (mi & 1u) * GB + (nt >> 3) * 1024u + mr * 128u + ((ch ^ mr) << 4));
                mma_16816<BF16>(o[nt], pa, v[0] & keep[0], v[1] & keep[1]);
                mma_16816<BF16>(o[nt + 1], pa, v[2] & keep[0], v[3] & keep[1]);
            }
            __syncwarp();
            s_cons = s_cons + 1u == stages ? 0u : s_cons + 1u;
            if (s_cons == 0) parity ^= 1u;
            const bool ends = cc.i + 1u == cc.s.n;
            if (issued < n_units) issue();
            if (ends || it + 1u == n_units) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                }
                const uint32_t item_u0 = u0 + it - cc.i;  // may lie before this warp's stretch
                if (ends && seg_u0 == item_u0) {  // all of the item: its output
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t ri = g + 8u * h, qr = ri / a.gq;
                        if (ri >= item_rows) continue;
                        uint16_t* dst = a.out + (uint64_t)(item_row0 + qr) * a.out_stride +
                                        (cc.kvh * a.gq + ri - qr * a.gq) * D + 2u * t;
                        const float inv = 1.f / l[h];
#pragma unroll
                        for (int nt = 0; nt < D / 8; ++nt)
                            *reinterpret_cast<uint32_t*>(dst + 8 * nt) =
                                pack16<BF16>(o[nt][2 * h] * inv, o[nt][2 * h + 1] * inv);
                    }
                } else {  // a part: into shared memory (the last one over the ring, which nothing fills any more)
                    float* slot = first_seg ? firsts + warp * slot_floats : reinterpret_cast<float*>(ring);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t ri = g + 8u * h;
                        if (ri >= item_rows) continue;
#pragma unroll
                        for (int nt = 0; nt < D / 8; ++nt)
                            *reinterpret_cast<float2*>(slot + ri * D + 8 * nt + 2u * t) =
                                make_float2(o[nt][2 * h], o[nt][2 * h + 1]);
                        if (t == 0)
                            *reinterpret_cast<float2*>(slot + slot_rows * D + 2u * ri) = make_float2(m[h], l[h]);
                    }
                    if (lane == 0) segs[warp][first_seg ? 0 : 1] = {1u, item_u0, item_u0 + cc.s.n, cc.r, cc.kvh};
                }
            }
            if (it + 1u < n_units) cc.next(a, off);
        }
        if (!ok) {  // a copy did not arrive: wait (bounded) for the others before the CTA may end
            for (uint32_t k = it + 1u; k < issued; ++k) {
                s_cons = s_cons + 1u == stages ? 0u : s_cons + 1u;
                if (s_cons == 0) parity ^= 1u;
                mbar_wait(&bars[warp][s_cons], parity, err);
            }
        }
        if (bad_page && lane == 0) raise_error(err, ARC_DEV_ERR_BOUNDS);
    }
    __syncthreads();
    // Runs of parts of one item, warp by warp; an item that lies within this CTA's stretch is done here.
    for (uint32_t k = 0; k < 2u * kRowWarps;) {
        const Segment sg = segs[k >> 1][k & 1u];
        if (!sg.valid) {
            ++k;
            continue;
        }
        uint32_t e = k + 1u;
        while (e < 2u * kRowWarps && (!segs[e >> 1][e & 1u].valid || segs[e >> 1][e & 1u].u0 == sg.u0)) ++e;
        Req q;
        bool bad = false;
        load_req(a, sg.r, q, bad);
        const uint32_t rows = q.n * a.gq;
        const bool whole = sg.u0 >= U0 && sg.u1 <= U1;
        const uint32_t slot_no = sg.u0 < U0 ? 0u : 1u;
        float* part = parts + (uint64_t)(blockIdx.x * 2u + slot_no) * (kRowMax * (D + 2u));
        if (!whole && slot_no == 1u && tid == 0)
            recs[blockIdx.x] = {1u, (sg.u1 - 1u) / per, q.row0, rows, sg.kvh, {0, 0, 0}};
        for (uint32_t x = tid; x < rows * (D / 4u); x += kRowWarps * 32u) {
            const uint32_t ri = x / (D / 4u), c = (x - ri * (D / 4u)) * 4u;
            float M = -INFINITY;
            for (uint32_t j = k; j < e; ++j)
                if (segs[j >> 1][j & 1u].valid) {
                    const float* slot = (j & 1u) ? reinterpret_cast<const float*>(rings + (j >> 1) * stages * STAGE)
                                                 : firsts + (j >> 1) * slot_floats;
                    M = fmaxf(M, slot[slot_rows * D + 2u * ri]);
                }
            const float ref = M == -INFINITY ? 0.f : M;
            float L = 0.f;
            float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
            for (uint32_t j = k; j < e; ++j)
                if (segs[j >> 1][j & 1u].valid) {
                    const float* slot = (j & 1u) ? reinterpret_cast<const float*>(rings + (j >> 1) * stages * STAGE)
                                                 : firsts + (j >> 1) * slot_floats;
                    const float2 ml = *reinterpret_cast<const float2*>(slot + slot_rows * D + 2u * ri);
                    const float4 v = *reinterpret_cast<const float4*>(slot + ri * D + c);
                    const float f = ex2(ml.x - ref);
                    L = fmaf(ml.y, f, L);
                    A.x = fmaf(v.x, f, A.x), A.y = fmaf(v.y, f, A.y);
                    A.z = fmaf(v.z, f, A.z), A.w = fmaf(v.w, f, A.w);
                }
            if (whole) {
                const uint32_t qr = ri / a.gq;
                const float inv = 1.f / L;
                *reinterpret_cast<uint2*>(a.out + (uint64_t)(q.row0 + qr) * a.out_stride +
                                          (sg.kvh * a.gq + ri - qr * a.gq) * D + c) =
                    make_uint2(pack16<BF16>(A.x * inv, A.y * inv), pack16<BF16>(A.z * inv, A.w * inv));
            } else {
                *reinterpret_cast<float4*>(part + ri * D + c) = A;
                if (c == 0) *reinterpret_cast<float2*>(part + kRowMax * D + 2u * ri) = make_float2(M, L);
            }
        }
        k = e;
    }
}

// ---- join ---------------------------------------------------------------------
// Block (c, part): the item that CTA c began and later CTAs went on with.  The
// first kSms records are the rows kernel's, the others the tile kernel's.  Nearly
// always two CTAs share an item: then a thread has four pairs of loads on their
// way; a longer row of parts is walked eight at a time.  6.5 us for 148 shared
// tile items of 256 rows (12 us one pair of loads at a time).
template <int D, bool BF16>
__global__ void __launch_bounds__(256) attn_paged_join_kernel(Args a, const Record* __restrict__ recs,
                                                              const float* __restrict__ row_parts,
                                                              const float* __restrict__ tile_parts, uint32_t rec0) {
    pdl_trigger();
    pdl_wait();
    const Record rc = recs[rec0 + blockIdx.x];
    if (!rc.valid) return;
    const bool tiles = rec0 + blockIdx.x >= kSms;
    const uint32_t cta = rec0 + blockIdx.x - (tiles ? kSms : 0u);
    const uint32_t max_rows = tiles ? kTileRows : kRowMax, stride = max_rows * (D + 2u);
    const float* first = (tiles ? tile_parts : row_parts) + (uint64_t)(cta * 2u + 1u) * stride;
    const float* later = first + stride;  // slot 0 of the next CTA; those after it 2 * stride apart
    const uint32_t n = rc.last_cta - cta, total = rc.rows * (D / 4u);
    auto write = [&](uint32_t ri, uint32_t c, float4 A, float L) {
        const uint32_t qr = ri / a.gq;
        const float inv = 1.f / L;
        *reinterpret_cast<uint2*>(a.out + (uint64_t)(rc.row0 + qr) * a.out_stride +
                                  (rc.kvh * a.gq + ri - qr * a.gq) * D + c) =
            make_uint2(pack16<BF16>(A.x * inv, A.y * inv), pack16<BF16>(A.z * inv, A.w * inv));
    };
    const uint32_t step = gridDim.y * 256u;
    if (n == 1u) {
        constexpr uint32_t U = 4;
        for (uint32_t x0 = blockIdx.y * 256u + threadIdx.x; x0 < total; x0 += U * step) {
            float4 v[U], y[U];
            float2 mv[U], my[U];
#pragma unroll
            for (uint32_t j = 0; j < U; ++j) {
                const uint32_t x = min(x0 + j * step, total - 1u), ri = x / (D / 4u);
                v[j] = reinterpret_cast<const float4*>(first)[x];
                y[j] = reinterpret_cast<const float4*>(later)[x];
                mv[j] = *reinterpret_cast<const float2*>(first + max_rows * D + 2u * ri);
                my[j] = *reinterpret_cast<const float2*>(later + max_rows * D + 2u * ri);
            }
#pragma unroll
            for (uint32_t j = 0; j < U; ++j) {
                const uint32_t x = x0 + j * step;
                if (x >= total) break;
                const float M = fmaxf(mv[j].x, my[j].x), f = ex2(mv[j].x - M), g = ex2(my[j].x - M);
                write(x / (D / 4u), x % (D / 4u) * 4u,
                      make_float4(fmaf(v[j].x, f, y[j].x * g), fmaf(v[j].y, f, y[j].y * g),
                                  fmaf(v[j].z, f, y[j].z * g), fmaf(v[j].w, f, y[j].w * g)),
                      fmaf(mv[j].y, f, my[j].y * g));
            }
        }
        return;
    }
    for (uint32_t x = blockIdx.y * 256u + threadIdx.x; x < total; x += step) {
        const uint32_t ri = x / (D / 4u), c = x % (D / 4u) * 4u;
        constexpr uint32_t CH = 8;  // parts whose loads are in flight together
        float M = -INFINITY, L = 0.f;
        float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t j0 = 0; j0 <= n; j0 += CH) {
            float2 ml[CH];
            float4 v[CH];
#pragma unroll
            for (uint32_t j = 0; j < CH; ++j) {
                ml[j] = make_float2(-INFINITY, 0.f);
                v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (j0 + j <= n) {
                    const float* p = j0 + j == 0u ? first : later + (uint64_t)(j0 + j - 1u) * 2u * stride;
                    ml[j] = *reinterpret_cast<const float2*>(p + max_rows * D + 2u * ri);
                    v[j] = *reinterpret_cast<const float4*>(p + ri * D + c);
                }
            }
            float mn = M;
#pragma unroll
            for (uint32_t j = 0; j < CH; ++j) mn = fmaxf(mn, ml[j].x);
            const float ref = mn == -INFINITY ? 0.f : mn;
            const float f0 = ex2(M - ref);
            L *= f0, A.x *= f0, A.y *= f0, A.z *= f0, A.w *= f0;
#pragma unroll
            for (uint32_t j = 0; j < CH; ++j) {
                const float f = ex2(ml[j].x - ref);
                L = fmaf(ml[j].y, f, L);
                A.x = fmaf(v[j].x, f, A.x), A.y = fmaf(v[j].y, f, A.y);
                A.z = fmaf(v[j].z, f, A.z), A.w = fmaf(v[j].w, f, A.w);
            }
            M = mn;
        }
        write(ri, c, A, L);
    }
}

// ---- host ---------------------------------------------------------------------
// Workspace: the records of both kernels, then their parts.
constexpr uint64_t kRecBytes = (sizeof(Record) * 2u * kSms + 255u) / 256u * 256u;
constexpr uint64_t rows_part_bytes(uint32_t d) { return 4ull * kSms * 2u * kRowMax * (d + 2u); }

template <int D, bool BF16>
int launch_paged(const AttnPaged& p, const arcllm_cuda_paged_kv& kv, const Args& a, cudaStream_t stream) {
    constexpr uint32_t kStage = 4u * kRowTile * D, kMost = 232448u - 2048u;  // 227 KB less the static arrays
    uint8_t* ws = static_cast<uint8_t*>(p.workspace);
    Record* recs = reinterpret_cast<Record*>(ws);
    float* parts = reinterpret_cast<float*>(ws + kRecBytes);
    float* tile_parts = reinterpret_cast<float*>(ws + kRecBytes + rows_part_bytes(D));
    // the requests with few rows, if any can have; then those with many
    const bool few = a.gq <= kRowMax, many = (uint64_t)a.max_new * a.gq > kRowMax;
    cudaError_t e = cudaSuccess;
    if (few) {
        CUtensorMap kmap, vmap;
        PageMap heads;
        const int st = encode_pages(&kmap, &vmap, &heads, kv, kRowTile);
        if (st != ARC_OK) return st;
        const uint32_t slot_rows = !many && a.max_new * a.gq <= 8u ? 8u : 16u;
        const uint32_t fixed = 1024u + kRowWarps * slot_rows * (D + 2u) * 4u + 4u * (a.n_requests + 1u);
        const uint32_t stages = std::min(4u, (kMost - fixed) / (kRowWarps * kStage));
        e = allow_shared<attn_paged_rows_kernel<D, BF16>>((int)kMost);
        if (e == cudaSuccess)
            e = launch_kernel(attn_paged_rows_kernel<D, BF16>, dim3(kSms), dim3(kRowWarps * 32u),
                              fixed + kRowWarps * stages * kStage, stream, kmap, vmap, heads, a, slot_rows, stages, recs,
                              parts, dev_error_word());
    }
    if (e == cudaSuccess && many) {
        const int st = launch_tiles<D, BF16>(kv, a, recs + kSms, tile_parts, stream);
        if (st != ARC_OK) return st;
    }
    // blocks of the records that were written
    if (e == cudaSuccess)
        e = launch_kernel(attn_paged_join_kernel<D, BF16>, dim3((few ? kSms : 0u) + (many ? kSms : 0u), many ? 4 : 2),
                          dim3(256), 0, stream, a, recs, parts, tile_parts, few ? 0u : kSms);
    return launch_checked(e, "attention paged launch");
}

}  // namespace

int paged::encode_pages(CUtensorMap* k, CUtensorMap* v, PageMap* heads, const arcllm_cuda_paged_kv& kv,
                        uint32_t tokens) {
    const EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return set_error(ARC_E_CUDA, "attention paged: cuTensorMapEncodeTiled is not available");
    const cuuint32_t parts = kv.head_dim / 64u, groups = kv.page_size / 8u;
    const bool by_token = kv.kv_heads == 1u || kv.head_stride == kv.head_dim;
    *heads = by_token ? PageMap{parts, 0u} : PageMap{0u, groups};
    const cuuint64_t dims[5] = {64, 8, by_token ? (cuuint64_t)kv.kv_heads * parts : parts,
                                by_token ? groups : (cuuint64_t)kv.kv_heads * groups, kv.n_pages};
    const cuuint64_t strides[4] = {2ull * kv.token_stride, 128, 16ull * kv.token_stride, 2ull * kv.page_stride};
    const cuuint32_t box[5] = {64, 8, parts, tokens / 8u, 1}, one[5] = {1, 1, 1, 1, 1};
    for (int i = 0; i < 2; ++i) {
        const CUresult rc =
            fn(i ? v : k,
               kv.type == ARC_GGML_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
               i ? kv.v_pages : kv.k_pages, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (rc != CUDA_SUCCESS) return set_error(ARC_E_CUDA, "attention paged: tensor map of the pages");
    }
    return ARC_OK;
}

int attention_paged_workspace(uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint64_t* out) {
    if (!out) return set_error(ARC_E_INVALID_ARGUMENT, "attention paged workspace: null out");
    if (kv_heads == 0 || q_heads == 0 || q_heads % kv_heads)
        return set_error(ARC_E_UNSUPPORTED_SHAPE, "attention paged workspace: q_heads % kv_heads");
    if (head_dim != 64u && head_dim != 128u)
        return set_error(ARC_E_UNSUPPORTED_SHAPE, "attention paged workspace: head_dim must be 64 or 128");
    *out = kRecBytes + rows_part_bytes(head_dim) + 4ull * kSms * 2u * kTileRows * (head_dim + 2u);
    return ARC_OK;
}

int attention_paged(const AttnPaged& p, const arcllm_cuda_paged_kv& kv, cudaStream_t stream) {
    if (p.n_requests == 0 || p.max_rows == 0 || p.max_new == 0) return ARC_OK;
    if (!p.q || !p.block_table || !p.row_start || !p.kv_total || !p.out || !p.workspace)
        return set_error(ARC_E_INVALID_ARGUMENT, "attention paged: null pointer");
    uint64_t need = 0;
    const int st = attention_paged_workspace(p.q_heads, kv.kv_heads, kv.head_dim, &need);
    if (st != ARC_OK) return st;
    const uint32_t gq = p.q_heads / kv.kv_heads;
    if (gq > 128u) return set_error(ARC_E_UNSUPPORTED_SHAPE, "attention paged: at most 128 query heads per KV head");
    if (kv.page_size % 16u) return set_error(ARC_E_UNSUPPORTED_SHAPE, "attention paged: page_size must be a multiple of 16");
    if (p.n_requests > kMaxRequests)
        return set_error(ARC_E_UNSUPPORTED_SHAPE, "attention paged: at most 4096 requests");
    if (p.max_rows > 0x7fffffffu || p.table_stride == 0)
        return set_error(ARC_E_INVALID_ARGUMENT, "attention paged: bad shape");
    const float scale_log2 = (float)((double)p.scale * 1.4426950408889634074);
    if (!(p.scale > 0.f) || !std::isfinite(scale_log2))
        return set_error(ARC_E_INVALID_ARGUMENT, "attention paged: scale must be positive, and finite in units of log 2");
    const uint64_t width = (uint64_t)p.q_heads * kv.head_dim;
    if (p.q_stride < width || p.out_stride < width)
        return set_error(ARC_E_INVALID_ARGUMENT, "attention paged: a row stride shorter than the row");
    if (any_off(16u, p.q, p.out, kv.k_pages, kv.v_pages, p.workspace) || p.q_stride % 8u || p.out_stride % 8u ||
        kv.page_stride % 8u || kv.token_stride % 8u || kv.head_stride % 8u)
        return set_error(ARC_E_ALIGNMENT, "attention paged: pointers and strides of 16 bytes");
    if (any_off(4u, p.block_table, p.row_start, p.kv_total))
        return set_error(ARC_E_ALIGNMENT, "attention paged: arrays of 32-bit words");
    if (kv.kv_heads > 1u && kv.head_stride != kv.head_dim && kv.head_stride != (uint64_t)kv.page_size * kv.token_stride)
        return set_error(ARC_E_UNSUPPORTED_SHAPE, "attention paged: heads side by side in a token, or one after another");
    if (kv.page_stride >= (1ull << 39) || kv.token_stride >= (1u << 31) || p.q_stride >= (1ull << 39) ||
        p.out_stride >= (1ull << 39))
        return set_error(ARC_E_UNSUPPORTED_SHAPE, "attention paged: a stride past 2^40 bytes");
    if (rows_meet(p.q, 2u * p.q_stride, 2u * width, p.out, 2u * p.out_stride, 2u * width, p.max_rows))
        return set_error(ARC_E_INVALID_ARGUMENT, "attention paged: out overlaps q");
    if (p.workspace_bytes < need) return set_error(ARC_E_INVALID_ARGUMENT, "attention paged: workspace too small");
    Args a{};
    a.q = static_cast<const uint16_t*>(p.q);
    a.out = static_cast<uint16_t*>(p.out);
    a.q_stride = p.q_stride, a.out_stride = p.out_stride;
    a.table = p.block_table, a.table_stride = p.table_stride;
    a.row_start = p.row_start, a.kv_total = p.kv_total;
    a.n_requests = p.n_requests, a.max_rows = p.max_rows, a.max_new = p.max_new;
    a.kv_heads = kv.kv_heads, a.gq = gq, a.page_size = kv.page_size, a.n_pages = kv.n_pages;
    a.scale_log2 = scale_log2;
    a.window = std::min(p.window, 0x7fffffffu);  // positions are below 2^31: sums stay within 32 bits
    a.sinks = p.window ? std::min(p.sinks, 0x7fffffffu) : 0u;
    const bool bf = kv.type == ARC_GGML_BF16;
    if (kv.head_dim == 128u)
        return bf ? launch_paged<128, true>(p, kv, a, stream) : launch_paged<128, false>(p, kv, a, stream);
    return bf ? launch_paged<64, true>(p, kv, a, stream) : launch_paged<64, false>(p, kv, a, stream);
}

}  // namespace arc
