// One warp waits on a barrier that another warp completes after a while, or
// never; its lanes come to the wait at different times.  Every loop here ends by
// itself.
#include "attention_paged.cuh"

namespace {

__device__ void pass_time(unsigned long long from, unsigned long long ns) {
    for (uint32_t i = 0; i < (1u << 24) && arc::globaltimer() - from < ns; ++i) {
    }
}

__global__ void wait_kernel(uint32_t lane_ns, uint32_t arrive_ns, uint32_t limit_ns, int32_t* result, unsigned int* err) {
    __shared__ uint64_t bar;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    if (threadIdx.x == 0) {
        arc::mbar_init(&bar, 1);
        arc::fence_mbar_init();
    }
    __syncthreads();
    const unsigned long long t0 = arc::globaltimer();
    if (warp == 0) {
        pass_time(t0, (unsigned long long)lane * lane_ns);
        result[lane] = arc::paged::warp_wait(&bar, 0, err, [] { return false; }, limit_ns);
    } else if (lane == 0 && arrive_ns != 0) {
        pass_time(t0, arrive_ns);
        arc::mbar_arrive(&bar);
    }
    __syncthreads();
}

}  // namespace

// result: 32 numbers, err: one word (device memory); waits for the kernel.
extern "C" __attribute__((visibility("default"))) int warp_wait_run(uint32_t lane_ns, uint32_t arrive_ns,
                                                                    uint32_t limit_ns, int32_t* result,
                                                                    unsigned int* err) {
    wait_kernel<<<1, 64>>>(lane_ns, arrive_ns, limit_ns, result, err);
    const cudaError_t e = cudaGetLastError();
    return (int)(e != cudaSuccess ? e : cudaDeviceSynchronize());
}
