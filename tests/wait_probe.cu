// A barrier that nobody completes: the waits of both warps have to end by their limit.
#include "common.cuh"

__global__ void wait_probe_kernel(int* ended, unsigned long long* took) {
    __shared__ uint64_t bar[2];  // the second one is complete
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) wzyb::mbar_init(&bar[i], 1);
        wzyb::fence_mbar_init();
        wzyb::mbar_arrive(&bar[1]);
    }
    __syncthreads();
    const unsigned long long t0 = wzyb::globaltimer_ns();
    int bits = 0;
    for (int i = 0; i < 2; ++i) bits |= (int)wzyb::mbar_wait_asleep(&bar[i], 0) << i;
    if (lane == 0) {
        ended[warp] = bits;
        took[warp] = wzyb::globaltimer_ns() - t0;
    }
}

extern "C" int wait_probe(int* ended, unsigned long long* took, unsigned int* faults) {
    int* e;
    unsigned long long* t;
    if (cudaMalloc(&e, 2 * sizeof(int)) != cudaSuccess || cudaMalloc(&t, 2 * sizeof(*t)) != cudaSuccess) return -1;
    wait_probe_kernel<<<1, 64>>>(e, t);
    cudaMemcpy(ended, e, 2 * sizeof(int), cudaMemcpyDeviceToHost);
    cudaMemcpy(took, t, 2 * sizeof(*t), cudaMemcpyDeviceToHost);
    cudaMemcpyFromSymbol(faults, wzyb::g_fault_word, sizeof(*faults));
    cudaFree(e);
    cudaFree(t);
    return (int)cudaGetLastError();
}
