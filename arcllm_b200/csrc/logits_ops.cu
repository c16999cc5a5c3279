// Sampling constraints on a batch of logits (B200, sm_100a): penalties for
// tokens that already stand in a request, biases of single tokens, a grammar's
// mask of allowed tokens, and the greedy choice among what is left -- the step
// between the LM head and the next token when requests carry such settings
// (arcllm_cuda_argmax is the choice without them).
#include <algorithm>

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "arcllm_cuda_internal.h"
#include "common.cuh"
#include "decode_ops.h"
#include "paged_ops.h"

namespace arc {
namespace {

constexpr uint32_t kLogitsThreads = 512;
constexpr uint32_t kLogitsCluster = 8;      // CTAs per row
constexpr uint32_t kLogitsWords = 20480;    // per-token words of a chunk in shared memory (80 KB: two CTAs per SM)
constexpr uint32_t kPromptSeen = 0x80000000u;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

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

// A cluster of 8 CTAs per row, each over a contiguous eighth of the
// vocabulary.  Per chunk of its slice a CTA counts the row's history into
// shared memory (one word per token: generated count, top bit: in the prompt;
// with biases a second word: 1 + the index of the token's last entry), then
// streams the logits through once: read, constrain, round, write, and keep the
// best finite value with the lowest index.  The eight bests meet in CTA 0
// through distributed shared memory, so no workspace, no atomics on global
// memory and no order of arrival is involved.  Many rows: HBM traffic of the
// logits in and out; one row: 8 CTAs, latency.
template <typename T, int V>
__global__ void __launch_bounds__(kLogitsThreads, 2)
    logits_process_kernel(LogitsProcess p, uint32_t slice, uint32_t chunk) {
    pdl_trigger();
    pdl_wait();  // logits come from the preceding kernels
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    extern __shared__ uint32_t words[];
    __shared__ unsigned long long s_best[kLogitsThreads / 32];
    __shared__ unsigned long long s_key;
    const uint32_t tid = threadIdx.x, row = blockIdx.y;
    const uint32_t v_begin = min(blockIdx.x * slice, p.vocab), v_end = min(v_begin + slice, p.vocab);
    const T* in = static_cast<const T*>(p.logits) + (uint64_t)row * p.stride;
    T* out = static_cast<T*>(p.out) + (uint64_t)row * p.out_stride;
    RowParams rp;
    rp.has_rep = p.repetition != nullptr, rp.has_freq = p.frequency != nullptr, rp.has_pres = p.presence != nullptr;
    rp.rep = rp.has_rep ? p.repetition[row] : 1.f;
    rp.freq = rp.has_freq ? p.frequency[row] : 0.f;
    rp.pres = rp.has_pres ? p.presence[row] : 0.f;
    uint32_t n_hist = 0, n_prompt = 0, b0 = 0, b1 = 0;
    if (p.history && (rp.has_rep || rp.has_freq || rp.has_pres)) {
        n_hist = (uint32_t)min(max(p.total_len[row], 0), (int32_t)p.history_stride);
        n_prompt = p.prompt_len ? (uint32_t)max(p.prompt_len[row], 0) : 0u;
    }
    if (p.bias_start) {
        b0 = (uint32_t)max(p.bias_start[row], 0);
        b1 = (uint32_t)max(p.bias_start[row + 1], (int32_t)b0);
    }
    const int32_t* hist = p.history + (uint64_t)row * p.history_stride;
    const uint32_t* mask = p.mask ? p.mask + (uint64_t)row * p.mask_stride : nullptr;
    uint32_t* count = words;
    uint32_t* last = words + chunk;  // only with biases
    float best = -INFINITY;
    uint32_t best_at = 0xffffffffu;
    for (uint32_t c0 = v_begin; c0 < v_end; c0 += chunk) {
        const uint32_t n = min(chunk, v_end - c0);
        const bool counted = n_hist != 0u, biased = b1 != b0;
        if (counted || biased) {
            for (uint32_t i = tid; i < n; i += kLogitsThreads) {
                if (counted) count[i] = 0u;
                if (biased) last[i] = 0u;
            }
            __syncthreads();
            for (uint32_t i = tid; i < n_hist; i += kLogitsThreads) {
                const uint32_t id = (uint32_t)hist[i] - c0;  // outside the chunk, or no token: a large number
                if (id < n) {
                    if (i < n_prompt)
                        atomicOr(&count[id], kPromptSeen);
                    else
                        atomicAdd(&count[id], 1u);
                }
            }
            for (uint32_t e = b0 + tid; e < b1; e += kLogitsThreads) {
                const uint32_t id = (uint32_t)p.bias_ids[e] - c0;
                if (id < n) atomicMax(&last[id], e - b0 + 1u);
            }
            __syncthreads();
        }
        constexpr uint32_t U = 4;  // vectors in flight per thread
        for (uint32_t i0 = 0; i0 < n; i0 += kLogitsThreads * V * U) {
            T x[U][V];
#pragma unroll
            for (uint32_t j = 0; j < U; ++j) {
                const uint32_t i = i0 + (j * kLogitsThreads + tid) * V;
                if (i + V <= n) {
                    if constexpr (V > 1)
                        *reinterpret_cast<uint4*>(x[j]) = __ldcs(reinterpret_cast<const uint4*>(in + c0 + i));
                    else
                        x[j][0] = in[c0 + i];
                } else {
#pragma unroll
                    for (uint32_t k = 0; k < V; ++k)
                        if (i + k < n) x[j][k] = in[c0 + i + k];
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < U; ++j) {
                const uint32_t i = i0 + (j * kLogitsThreads + tid) * V;
                if (i >= n) continue;
                // V consecutive tokens start on a multiple of V, so their mask bits lie in one word
                const uint32_t allowed = mask ? mask[(c0 + i) >> 5] >> ((c0 + i) & 31u) : 0xffffffffu;
#pragma unroll
                for (uint32_t k = 0; k < V; ++k) {
                    if (i + k >= n) continue;
                    float v = constrained(to_f32(x[j][k]), counted ? count[i + k] : 0u, rp);
                    if (biased && last[i + k]) v = __fadd_rn(v, p.bias_values[b0 + last[i + k] - 1u]);
                    if (!((allowed >> k) & 1u)) v = -INFINITY;
                    from_f32(v, x[j][k]);
                    v = to_f32(x[j][k]);
                    if (isfinite(v) && (v > best || best_at == 0xffffffffu)) best = v, best_at = c0 + i + k;
                }
                if (i + V <= n) {
                    if constexpr (V > 1)
                        __stcs(reinterpret_cast<uint4*>(out + c0 + i), *reinterpret_cast<const uint4*>(x[j]));
                    else
                        out[c0 + i] = x[j][0];
                } else {
#pragma unroll
                    for (uint32_t k = 0; k < V; ++k)
                        if (i + k < n) out[c0 + i + k] = x[j][k];
                }
            }
        }
        if (c0 + chunk < v_end) __syncthreads();  // the words are filled anew
    }
    if (!p.best) return;
    unsigned long long key =
        best_at == 0xffffffffu ? 0ull : ((unsigned long long)ordered(best) << 32) | (unsigned long long)(~best_at);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
        key = other > key ? other : key;
    }
    if ((tid & 31u) == 0) s_best[tid >> 5] = key;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (uint32_t w = 1; w < kLogitsThreads / 32; ++w) key = s_best[w] > key ? s_best[w] : key;
        s_key = key;
    }
    cl.sync();
    if (cl.block_rank() == 0 && tid == 0) {
        for (uint32_t c = 1; c < kLogitsCluster; ++c) {
            const unsigned long long other = *cl.map_shared_rank(&s_key, c);
            key = other > key ? other : key;
        }
        p.best[row] = key ? (int32_t)~(uint32_t)(key & 0xffffffffull) : -1;
    }
    cl.sync();  // no CTA leaves while CTA 0 still reads its key
}

template <typename T, int V>
cudaError_t launch_logits(const LogitsProcess& p, uint32_t row0, uint32_t rows, cudaStream_t stream) {
    const bool counts = p.history && (p.repetition || p.frequency || p.presence);
    const uint32_t slice = ((p.vocab + kLogitsCluster - 1u) / kLogitsCluster + 31u) / 32u * 32u;  // whole mask words
    const uint32_t most = p.bias_start ? kLogitsWords / 2u : kLogitsWords;
    const uint32_t parts = (slice + most - 1u) / most;
    const uint32_t chunk = ((slice + parts - 1u) / parts + 31u) / 32u * 32u;
    const uint32_t smem = p.bias_start ? 8u * chunk : counts ? 4u * chunk : 0u;
    cudaError_t e = cudaFuncSetAttribute(logits_process_kernel<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         4 * kLogitsWords);
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
    cfg.gridDim = dim3(kLogitsCluster, rows);
    cfg.blockDim = dim3(kLogitsThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kLogitsCluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (pdl_enabled()) {
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    e = cudaLaunchKernelEx(&cfg, logits_process_kernel<T, V>, q, slice, chunk);
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T>
cudaError_t launch_logits_type(const LogitsProcess& p, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const uintptr_t all = reinterpret_cast<uintptr_t>(p.logits) | reinterpret_cast<uintptr_t>(p.out);
    // 16-byte vectors when every row starts on 16 bytes
    const bool vec = (all & 15u) == 0u && p.stride % V == 0u && p.out_stride % V == 0u;
    constexpr uint32_t kMaxGridY = 65535u;
    for (uint32_t r = 0; r < p.n_rows; r += kMaxGridY) {
        const uint32_t rows = std::min(kMaxGridY, p.n_rows - r);
        const cudaError_t e = vec ? launch_logits<T, V>(p, r, rows, stream) : launch_logits<T, 1>(p, r, rows, stream);
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
    if (p.history && (!p.total_len || p.history_stride > 0x3fffffffu))
        return set_error(ARC_E_INVALID_ARGUMENT, "logits: a history needs total_len and a stride below 2^30");
    if ((p.repetition || p.frequency || p.presence) && !p.history)
        return set_error(ARC_E_INVALID_ARGUMENT, "logits: penalties need a history");
    if (p.bias_start && (!p.bias_ids || !p.bias_values))
        return set_error(ARC_E_INVALID_ARGUMENT, "logits: bias_start needs bias_ids and bias_values");
    if (p.mask && p.mask_stride < (p.vocab + 31u) / 32u)
        return set_error(ARC_E_INVALID_ARGUMENT, "logits: mask rows shorter than the vocabulary");
    const uint64_t size = type == ARC_GGML_F32 ? 4u : 2u;
    const uintptr_t a = reinterpret_cast<uintptr_t>(p.logits), b = reinterpret_cast<uintptr_t>(p.out);
    if ((a | b) % size) return set_error(ARC_E_ALIGNMENT, "logits: pointers aligned to their type");
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
