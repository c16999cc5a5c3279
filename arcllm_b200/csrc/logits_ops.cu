// Sampling constraints on a batch of logits (B200, sm_100a): penalties for
// tokens that already stand in a request, biases of single tokens, a grammar's
// mask of allowed tokens, and the greedy choice among what is left -- the step
// between the LM head and the next token when requests carry such settings
// (arcllm_cuda_argmax is the choice without them).
#include <algorithm>

#include <cuda_bf16.h>

#include "arcllm_cuda_internal.h"
#include "common.cuh"
#include "decode_ops.h"
#include "paged_ops.h"

namespace arc {
namespace {

constexpr uint32_t kLogitsThreads = 512;
constexpr uint32_t kChunk = 131072;  // most tokens a CTA takes at a time: two words of shared memory for 32
constexpr uint32_t kNamed = 4096;    // most named tokens whose words are held at a time
constexpr uint32_t kList = 4096;     // history entries of the chunk that are kept in shared memory
constexpr uint32_t kPromptSeen = 0x80000000u;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

// a value of the type in a word of shared memory
__device__ __forceinline__ uint32_t to_bits(float v) { return __float_as_uint(v); }
__device__ __forceinline__ uint32_t to_bits(__half v) { return __half_as_ushort(v); }
__device__ __forceinline__ uint32_t to_bits(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
__device__ __forceinline__ void from_bits(uint32_t w, float& o) { o = __uint_as_float(w); }
__device__ __forceinline__ void from_bits(uint32_t w, __half& o) { o = __ushort_as_half((unsigned short)w); }
__device__ __forceinline__ void from_bits(uint32_t w, __nv_bfloat16& o) {
    o = __ushort_as_bfloat16((unsigned short)w);
}

// larger float -> larger unsigned, -0 as +0 (the order of arcllm_cuda_argmax)
__device__ __forceinline__ uint32_t ordered(float f) {
    uint32_t u = __float_as_uint(f);
    if (u == 0x80000000u) u = 0u;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct RowParams {
    float rep, freq, pres;
    bool has_rep, has_freq, has_pres;
};

// One logit.  Each step rounds by itself (no contraction), so the result is
// that of the same steps in any fp32 arithmetic.
__device__ __forceinline__ float constrained(float x, uint32_t word, const RowParams& rp) {
    const uint32_t count = word & ~kPromptSeen;
    if (word) {
        if (rp.has_rep) x = x > 0.f ? __fdiv_rn(x, rp.rep) : __fmul_rn(x, rp.rep);
        if (rp.has_freq) x = __fsub_rn(x, __fmul_rn(rp.freq, (float)count));
        if (rp.has_pres && count) x = __fsub_rn(x, rp.pres);
    }
    return x;
}

struct Best {
    float v = -INFINITY;
    uint32_t at = 0xffffffffu;
};

// One 64-bit word into another CTA's shared memory, counted by a barrier there.
__device__ __forceinline__ void st_async_u64(uint32_t addr, unsigned long long v, uint32_t bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(addr), "l"(v), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ uint32_t shared_of(const void* p, uint32_t rank) {  // the same place in CTA `rank`
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
    return r;
}

// A cluster of 1 to 16 CTAs per row, each over a contiguous part of the
// vocabulary.  The tokens that the row's history or biases name are few: they are
// marked by one bit each, and the number of bits before a token's own is the
// place of its words (generated count, top bit: in the prompt; with biases 1 +
// the index of its last entry), so shared memory holds words for the named tokens
// only and a CTA's part can be long.  The history is read once, its entries of
// the part kept in a list.  The named tokens' new values are worked out by place,
// a thread for each, from logits gathered while they are counted.  Then one stream
// over the logits reads, puts these values in, masks and writes, and keeps the
// first vector with the largest finite value.  The CTAs' bests go to CTA 0's
// shared memory by asynchronous stores (a cluster barrier would first drain every
// store: 4000 clocks), so no workspace, no atomics on global memory and no order
// of arrival is involved.
// Rows need not start on 16 bytes: token t is numbered t + a, a the elements
// between the last 16-byte boundary and the row's first, so that vectors of V
// numbers are aligned (the first and the last may be partly outside the row).
// Without Shift every row starts on 16 bytes and a is 0: what Shift needs costs 58
// instead of 47 us for 128 rows of 152064 fp32 (single numbers, as where logits and
// out lie differently to 16 bytes, 116 us).
// 128 rows of 152064 fp32 with histories of 4096, biases and masks: 47 us, 3.4
// TB/s, of which counting is about 8 us with little traffic; without constraints
// 32 us, 4.9 TB/s.  fp16 and bf16: 35 and 36 us, without constraints 18 (4.4 TB/s).  A
// row by itself with a history of 301: 8.4 us, latency.  With one set of inputs over and
// over, part of it in L2, the first of these is 41 us; in that measure forming the named
// tokens in the stream took 56 (a warp nearly always has one, and then all of it waits
// for the division), a choice token by token 47, mask words loaded where they are used
// 43; bulk copies into shared memory ahead of the stream, or each register loaded again
// as soon as its vector is written, were slower than this.
template <typename T, int V, bool Shift>
__global__ void __launch_bounds__(kLogitsThreads, 2)
    logits_process_kernel(LogitsProcess p, uint32_t slice, uint32_t chunk, unsigned int* err) {
    extern __shared__ uint32_t smem[];  // named bits, bits before each word's, list; counts, numbers, last bias entries
    __shared__ unsigned long long s_best[kLogitsThreads / 32], s_keys[16];
    __shared__ uint64_t keys_in;
    __shared__ uint32_t s_sum[kLogitsThreads / 32], s_listed;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, row = blockIdx.y;
    if (tid == 0) {
        mbar_init(&keys_in, 1);
        mbar_arrive_expect_tx(&keys_in, 8u * (gridDim.x - 1u));
        fence_mbar_init();
    }
    if (gridDim.x > 1u) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    pdl_trigger();
    pdl_wait();  // logits come from the preceding kernels
    const T* first_in = static_cast<const T*>(p.logits) + (uint64_t)row * p.stride;
    const uint32_t a = Shift ? (uint32_t)(reinterpret_cast<uintptr_t>(first_in) / sizeof(T)) % V : 0u;
    const T* in = first_in - a;  // by numbers
    T* out = static_cast<T*>(p.out) + (uint64_t)row * p.out_stride - a;
    const uint32_t row_end = a + p.vocab;
    const uint32_t v_begin = min(blockIdx.x * slice, row_end), v_end = min(v_begin + slice, row_end);
    constexpr uint32_t U = V > 1 ? 4 : 16;  // vectors, or single values, in flight per thread
    T x[U][V];
    auto load = [&](uint32_t i0, uint32_t i1) {  // of the numbers [i0, i1)
#pragma unroll
        for (uint32_t j = 0; j < U; ++j) {
            const uint32_t i = i0 + (j * kLogitsThreads + tid) * V;
            if (i >= a && i + V <= i1) {
                if constexpr (V > 1)
                    *reinterpret_cast<uint4*>(x[j]) = __ldcs(reinterpret_cast<const uint4*>(in + i));
                else
                    x[j][0] = in[i];
            } else {
#pragma unroll
                for (uint32_t k = 0; k < V; ++k)
                    if (i + k >= a && i + k < i1) x[j][k] = in[i + k];
            }
        }
    };
    load(v_begin, v_end);  // on their way while the tokens are counted
    RowParams rp;
    rp.has_rep = p.repetition != nullptr, rp.has_freq = p.frequency != nullptr, rp.has_pres = p.presence != nullptr;
    const bool penalties = p.history && (rp.has_rep || rp.has_freq || rp.has_pres);
    const int32_t* hist = p.history + (uint64_t)row * p.history_stride;
    const uint32_t* mask = p.mask ? p.mask + (uint64_t)row * p.mask_stride : nullptr;
    rp.rep = rp.has_rep ? p.repetition[row] : 1.f;
    rp.freq = rp.has_freq ? p.frequency[row] : 0.f;
    rp.pres = rp.has_pres ? p.presence[row] : 0.f;
    uint32_t n_hist = 0, n_prompt = 0, b0 = 0, b1 = 0;
    if (penalties) {
        n_hist = (uint32_t)min(max(p.total_len[row], 0), (int32_t)p.history_stride);
        n_prompt = p.prompt_len ? (uint32_t)max(p.prompt_len[row], 0) : 0u;
    }
    if (p.bias_start) {
        b0 = (uint32_t)max(p.bias_start[row], 0);
        b1 = (uint32_t)max(p.bias_start[row + 1], (int32_t)b0);
    }
    const uint32_t n_words = (chunk + 31u) / 32u;
    uint32_t* named = smem;
    uint32_t* before = named + n_words;
    uint32_t* list = before + n_words + 1u;  // number - chunk's first, top bit: of the prompt
    uint32_t* count = list + kList;
    uint32_t* which = count + kNamed;  // numbers (less the chunk's first) of the named tokens, by place
    uint32_t* last = which + kNamed;   // only with biases
    const bool any = n_hist != 0u || b1 != b0;
    Best best;
    for (uint32_t c0 = v_begin; c0 < v_end; c0 += chunk) {
        const uint32_t n = min(chunk, v_end - c0);
        // a token's place in the chunk; n or more when it is of another chunk, or no token at all
        auto number = [&](int32_t id) { return (uint32_t)id < p.vocab ? (uint32_t)id + a - c0 : n; };
        uint32_t n_named = 0, n_listed = 0;
        if (any) {
#pragma unroll 1
            for (uint32_t i = tid; i < n_words; i += kLogitsThreads) named[i] = 0u;
            if (tid == 0) s_listed = 0u;
            __syncthreads();
            auto name = [&](uint32_t i) {
                const uint32_t bit = 1u << (i & 31u);
                if (!(*(volatile uint32_t*)&named[i >> 5] & bit)) atomicOr(&named[i >> 5], bit);
            };
            constexpr uint32_t E = 4;  // entries on their way together
#pragma unroll 1
            for (uint32_t e0 = 0; e0 < n_hist; e0 += kLogitsThreads * E) {
                uint32_t id[E];
#pragma unroll
                for (uint32_t k = 0; k < E; ++k) {
                    const uint32_t e = e0 + k * kLogitsThreads + tid;
                    id[k] = e < n_hist ? number(__ldg(hist + e)) : n;
                }
#pragma unroll
                for (uint32_t k = 0; k < E; ++k) {
                    const uint32_t e = e0 + k * kLogitsThreads + tid, here = __ballot_sync(0xffffffffu, id[k] < n);
                    uint32_t at = 0;
                    if (here && lane == 0) at = atomicAdd(&s_listed, (uint32_t)__popc(here));
                    at = __shfl_sync(0xffffffffu, at, 0) + __popc(here & ((1u << lane) - 1u));
                    if (id[k] >= n) continue;
                    name(id[k]);
                    if (at < kList) list[at] = id[k] | (e < n_prompt ? kPromptSeen : 0u);
                }
            }
#pragma unroll 1
            for (uint32_t e = b0 + tid; e < b1; e += kLogitsThreads)
                if (const uint32_t i = number(p.bias_ids[e]); i < n) name(i);
            __syncthreads();
            n_listed = s_listed;
            const uint32_t per = (n_words + kLogitsThreads - 1u) / kLogitsThreads;
            const uint32_t w0 = min(tid * per, n_words), w1 = min(w0 + per, n_words);
            uint32_t mine = 0;
#pragma unroll 1
            for (uint32_t i = w0; i < w1; ++i) mine += __popc(named[i]);
            uint32_t sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= (uint32_t)o) sum += y;
            }
            if (lane == 31u) s_sum[warp] = sum;
            __syncthreads();
            sum -= mine;
#pragma unroll
            for (uint32_t w = 0; w < kLogitsThreads / 32; ++w) {
                if (w < warp) sum += s_sum[w];
                n_named += s_sum[w];
            }
#pragma unroll 1
            for (uint32_t i = w0; i < w1; ++i) {
                before[i] = sum;
                sum += __popc(named[i]);
            }
        }
        if (any && tid == 0) before[n_words] = n_named;
        // As many words of bits at a time as name kNamed tokens at most (nearly always all of them).
        for (uint32_t w0 = 0; w0 * 32u < n;) {
            uint32_t w1 = n_words, first = 0, held = 0;
            if (n_named) {
                __syncthreads();  // `before` is complete; the words of the round before are done with
                first = before[w0];
                if (n_named - first > kNamed) {
                    uint32_t lo = w0;  // before[lo] <= first + kNamed < before[w1]
                    while (w1 - lo > 1u) {
                        const uint32_t mid = (lo + w1) / 2u;
                        if (before[mid] <= first + kNamed)
                            lo = mid;
                        else
                            w1 = mid;
                    }
                    w1 = lo;
                }
                held = before[w1] - first;
                for (uint32_t i = tid; i < held; i += kLogitsThreads) {
                    count[i] = 0u;
                    if (p.bias_start) last[i] = 0u;
                }
#pragma unroll 1
                for (uint32_t w = w0 + tid; w < w1; w += kLogitsThreads) {
                    uint32_t bits = named[w], r = before[w] - first;
                    for (; bits; bits &= bits - 1u) which[r++] = w * 32u + (uint32_t)__ffs(bits) - 1u;
                }
                __syncthreads();
            }
            auto place = [&](uint32_t i) {  // of a named token of these words
                const uint32_t w = i >> 5;
                return before[w] + __popc(named[w] & ((1u << (i & 31u)) - 1u)) - first;
            };
            const uint32_t s0 = w0 * 32u, s1 = min(w1 * 32u, n);
            if (n_named) {
                constexpr uint32_t G = kNamed / kLogitsThreads;
                T own[G];  // logits of the named tokens, on their way while these are counted
#pragma unroll
                for (uint32_t k = 0; k < G; ++k)
                    if (const uint32_t r = tid + k * kLogitsThreads; r < held) own[k] = in[c0 + which[r]];
                const bool listed = n_listed <= kList;  // otherwise the history is read again
                const uint32_t entries = listed ? n_listed : n_hist;
#pragma unroll 1
                for (uint32_t e = tid; e < entries; e += kLogitsThreads) {
                    const uint32_t entry = listed ? list[e] : number(__ldg(hist + e));
                    const bool prompt = listed ? (entry & kPromptSeen) != 0u : e < n_prompt;
                    const uint32_t i = listed ? entry & ~kPromptSeen : entry;
                    if (i < s0 || i >= s1) continue;
                    uint32_t* word = &count[place(i)];
                    if (!prompt)
                        atomicAdd(word, 1u);
                    else if (!(*(volatile uint32_t*)word & kPromptSeen))
                        atomicOr(word, kPromptSeen);
                }
#pragma unroll 1
                for (uint32_t e = b0 + tid; e < b1; e += kLogitsThreads)
                    if (const uint32_t i = number(p.bias_ids[e]); i >= s0 && i < s1)
                        atomicMax(&last[place(i)], e - b0 + 1u);
                __syncthreads();
#pragma unroll
                for (uint32_t k = 0; k < G; ++k)
                    if (const uint32_t r = tid + k * kLogitsThreads; r < held) {
                        float v = constrained(to_f32(own[k]), count[r], rp);
                        if (p.bias_start && last[r]) v = __fadd_rn(v, p.bias_values[b0 + last[r] - 1u]);
                        from_f32(v, own[k]);
                        count[r] = to_bits(own[k]);  // what the stream puts in the token's place
                    }
                __syncthreads();
            }
#pragma unroll 1
            for (uint32_t i0 = s0; i0 < s1; i0 += kLogitsThreads * V * U) {
                if (c0 + i0 != v_begin) load(c0 + i0, c0 + s1);
                uint32_t allow[U];  // bit k: token k of the vector
#pragma unroll
                for (uint32_t j = 0; j < U; ++j) {
                    const uint32_t at = c0 + i0 + (j * kLogitsThreads + tid) * V;
                    allow[j] = 0xffffffffu;
                    if (!mask || at >= c0 + s1) continue;
                    const uint32_t t = max(at, a) - a, sh = t & 31u;
                    allow[j] = __ldg(mask + (t >> 5)) >> sh;
                    if (Shift && sh + V > 32u && (t >> 5) < (p.vocab - 1u) / 32u)  // reaches into the next word
                        allow[j] |= __ldg(mask + (t >> 5) + 1u) << (32u - sh);
                    allow[j] <<= max(at, a) - at;
                }
#pragma unroll
                for (uint32_t j = 0; j < U; ++j) {
                    const uint32_t i = i0 + (j * kLogitsThreads + tid) * V;
                    if (i >= s1) continue;
                    // V consecutive numbers start on a multiple of V, so their bits lie in one word
                    const uint32_t here = n_named ? (named[i >> 5] >> (i & 31u)) & ((1u << V) - 1u) : 0u;
                    if (here) {
                        uint32_t r = place(i);
#pragma unroll
                        for (uint32_t k = 0; k < V; ++k) {
                            if (!((here >> k) & 1u)) continue;
                            from_bits(count[r++], x[j][k]);
                        }
                    }
                    const uint32_t at = c0 + i, allowed = allow[j];
                    if (at >= a && i + V <= s1) {
                        float top = -INFINITY;
#pragma unroll
                        for (uint32_t k = 0; k < V; ++k) {
                            if (!((allowed >> k) & 1u)) from_f32(-INFINITY, x[j][k]);
                            top = fmaxf(top, to_f32(x[j][k]));  // passes over NaN
                        }
                        if (top == INFINITY) {  // not a choice: the largest of the others
                            top = -INFINITY;
#pragma unroll
                            for (uint32_t k = 0; k < V; ++k)
                                if (const float v = to_f32(x[j][k]); v < INFINITY) top = fmaxf(top, v);
                        }
                        if (top > best.v) best.v = top, best.at = at;  // numbers ascend, so the first of equals stays
                        if constexpr (V > 1)
                            __stcs(reinterpret_cast<uint4*>(out + at), *reinterpret_cast<const uint4*>(x[j]));
                        else
                            out[at] = x[j][0];
                    } else {  // partly outside the row
#pragma unroll
                        for (uint32_t k = 0; k < V; ++k) {
                            if (i + k >= s1 || at + k < a) continue;
                            if (!((allowed >> k) & 1u)) from_f32(-INFINITY, x[j][k]);
                            if (const float v = to_f32(x[j][k]); v > best.v && v < INFINITY) best.v = v, best.at = at;
                            out[at + k] = x[j][k];
                        }
                    }
                }
            }
            w0 = w1;
        }
        if (c0 + chunk < v_end) __syncthreads();  // bits and list are set anew
    }
    if (p.best) {
        if (best.at != 0xffffffffu) {  // the first of its vector that has the value (the thread wrote it itself)
            uint32_t t = max(best.at, a);
            while (to_f32(out[t]) != best.v) ++t;
            best.at = t - a;
        }
        unsigned long long key = best.at == 0xffffffffu
                                     ? 0ull
                                     : ((unsigned long long)ordered(best.v) << 32) | (unsigned long long)(~best.at);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
            key = other > key ? other : key;
        }
        if (lane == 0) s_best[warp] = key;
        __syncthreads();
        if (tid == 0)
#pragma unroll
            for (uint32_t w = 1; w < kLogitsThreads / 32; ++w) key = s_best[w] > key ? s_best[w] : key;
        if (gridDim.x > 1u) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // CTA 0 is ready
        if (tid == 0 && blockIdx.x != 0)
            st_async_u64(shared_of(&s_keys[blockIdx.x], 0), key, shared_of(&keys_in, 0));
        if (tid == 0 && blockIdx.x == 0) {
            if (gridDim.x > 1u && mbar_wait_cluster(&keys_in, 0, err))
                for (uint32_t c = 1; c < gridDim.x; ++c) key = s_keys[c] > key ? s_keys[c] : key;
            p.best[row] = key ? (int32_t)~(uint32_t)(key & 0xffffffffull) : -1;
        }
    } else if (gridDim.x > 1u) {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

template <typename T, int V, bool Shift>
cudaError_t launch_logits(const LogitsProcess& p, uint32_t row0, uint32_t rows, cudaStream_t stream) {
    // CTAs per row: as many as give the least waves x (tokens of a CTA + what a CTA costs beside them).  Measured for
    // 152064 tokens with all constraints: 128 rows 61 / 46 / 52 / 69 / 108 us with 1 / 2 / 4 / 8 / 16, 64 rows 54 / 32 / 28
    // / 36 / 57, 20 rows 48 / 27 / 19 / 19 / 23, 1 row 46 / 26 / 19 / 15 / 13.
    constexpr uint64_t kSlots = 2u * 148u, kCtaCost = 7500u;
    uint32_t ctas = 1;
    uint64_t least = ~0ull;
    for (uint32_t c = 1; c <= 16u; c *= 2u) {
        const uint64_t t = ((uint64_t)p.n_rows * c + kSlots - 1u) / kSlots * (p.vocab / c + kCtaCost);
        if (t < least) least = t, ctas = c;
    }
    const uint32_t slice = ((p.vocab + V - 1u + ctas - 1u) / ctas + 31u) / 32u * 32u;
    const uint32_t chunk = std::min(slice, kChunk);
    const bool counts = p.history && (p.repetition || p.frequency || p.presence);
    const uint32_t smem = counts || p.bias_start
                              ? (chunk + 31u) / 32u * 8u + 4u + 4u * kList + 4u * kNamed * (p.bias_start ? 3u : 2u)
                              : 0u;
    cudaError_t e = allow_shared<logits_process_kernel<T, V, Shift>, true>(kChunk / 4 + 4 + 4 * kList + 12 * kNamed);
    if (e != cudaSuccess) return e;
    LogitsProcess q = p;
    q.n_rows = rows;
    q.logits = static_cast<const T*>(p.logits) + (uint64_t)row0 * p.stride;
    q.out = static_cast<T*>(p.out) + (uint64_t)row0 * p.out_stride;
    auto shift = [&](auto* ptr, uint64_t by) { return ptr ? ptr + by : ptr; };
    q.history = shift(p.history, (uint64_t)row0 * p.history_stride);
    q.prompt_len = shift(p.prompt_len, row0);
    q.total_len = shift(p.total_len, row0);
    q.repetition = shift(p.repetition, row0);
    q.frequency = shift(p.frequency, row0);
    q.presence = shift(p.presence, row0);
    q.bias_start = shift(p.bias_start, row0);
    q.mask = shift(p.mask, (uint64_t)row0 * p.mask_stride);
    q.best = shift(p.best, row0);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, rows);
    cfg.blockDim = dim3(kLogitsThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (pdl_enabled()) {
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    e = cudaLaunchKernelEx(&cfg, logits_process_kernel<T, V, Shift>, q, slice, chunk, dev_error_word());
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T>
cudaError_t launch_logits_type(const LogitsProcess& p, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    // 16-byte vectors when the rows of logits and out lie the same way to 16 bytes
    const uintptr_t in = reinterpret_cast<uintptr_t>(p.logits), out = reinterpret_cast<uintptr_t>(p.out);
    const bool vec = (in - out) % 16u == 0u && (p.stride - p.out_stride) % V == 0u;
    const bool aligned = vec && in % 16u == 0u && p.stride % V == 0u;
    const auto launch = aligned ? launch_logits<T, V, false> : vec ? launch_logits<T, V, true> : launch_logits<T, 1, false>;
    constexpr uint32_t kMaxGridY = 65535u;
    for (uint32_t r = 0; r < p.n_rows; r += kMaxGridY) {
        const uint32_t rows = std::min(kMaxGridY, p.n_rows - r);
        const cudaError_t e = launch(p, r, rows, stream);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace

int logits_process(int type, const LogitsProcess& p, cudaStream_t stream) {
    if (p.n_rows == 0) return ARC_OK;
    if (!p.logits || !p.out) return set_error(ARC_E_INVALID_ARGUMENT, "logits: null pointer");
    if (type != ARC_GGML_F32 && type != ARC_GGML_F16 && type != ARC_GGML_BF16)
        return set_error(ARC_E_INVALID_ARGUMENT, "logits: type must be F32, F16 or BF16");
    if (p.vocab == 0 || p.vocab > 0x7fffffffu - 512u || p.n_rows > 0x7fffffffu || p.stride < p.vocab ||
        p.out_stride < p.vocab)
        return set_error(ARC_E_INVALID_ARGUMENT, "logits: bad shape");
    if (p.history && (!p.total_len || p.history_stride > 0x1fffffffu))
        return set_error(ARC_E_INVALID_ARGUMENT, "logits: a history needs total_len and a stride below 2^29");
    if ((p.repetition || p.frequency || p.presence) && !p.history)
        return set_error(ARC_E_INVALID_ARGUMENT, "logits: penalties need a history");
    if (p.bias_start && (!p.bias_ids || !p.bias_values))
        return set_error(ARC_E_INVALID_ARGUMENT, "logits: bias_start needs bias_ids and bias_values");
    if (p.mask && p.mask_stride < (p.vocab + 31u) / 32u)
        return set_error(ARC_E_INVALID_ARGUMENT, "logits: mask rows shorter than the vocabulary");
    const uint64_t size = type == ARC_GGML_F32 ? 4u : 2u;
    const uintptr_t a = reinterpret_cast<uintptr_t>(p.logits), b = reinterpret_cast<uintptr_t>(p.out);
    if ((a | b) % size) return set_error(ARC_E_ALIGNMENT, "logits: pointers aligned to their type");
    if (any_off(4u, p.history, p.prompt_len, p.total_len, p.repetition, p.frequency, p.presence, p.bias_start, p.bias_ids,
                p.bias_values, p.mask, p.best))
        return set_error(ARC_E_ALIGNMENT, "logits: arrays of 32-bit words");
    // in place (the same rows) or apart
    const uint64_t na = ((uint64_t)(p.n_rows - 1u) * p.stride + p.vocab) * size;
    const uint64_t nb = ((uint64_t)(p.n_rows - 1u) * p.out_stride + p.vocab) * size;
    if (a < b + nb && b < a + na && !(a == b && p.stride == p.out_stride))
        return set_error(ARC_E_INVALID_ARGUMENT, "logits: out overlaps logits without being the same rows");
    cudaError_t e;
    if (type == ARC_GGML_F32)
        e = launch_logits_type<float>(p, stream);
    else if (type == ARC_GGML_F16)
        e = launch_logits_type<__half>(p, stream);
    else
        e = launch_logits_type<__nv_bfloat16>(p, stream);
    return launch_checked(e, "logits launch");
}

}  // namespace arc
