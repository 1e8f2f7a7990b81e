// Waits of csrc/tc05.cuh with a short limit on a barrier that nothing completes: they end and say so.
#include "../../nesle_b200/csrc/tc05.cuh"

using namespace nesle;

__global__ void wait_probe(int* out, long long* took, long long limit) {
    __shared__ uint64_t bar;
    if (threadIdx.x == 0) {
        tc::mbar_init(&bar, 1);
        tc::mbar_init_fence();
    }
    __syncwarp();
    const long long t0 = clock64();
    const bool early = tc::mbar_wait_warp(&bar, 0, limit);
    const long long t1 = clock64();
    const bool lane = tc::mbar_wait(&bar, 0, threadIdx.x * 10);  // another limit in every lane
    __syncwarp();
    if (threadIdx.x == 0) tc::mbar_arrive(&bar);
    const bool over = tc::mbar_wait_warp(&bar, 0, limit);
    tc::mbar_see(&bar, 0);
    if (threadIdx.x == 0) tc::mbar_expect_tx(&bar, 16);  // bytes that never come
    const bool bytes = tc::mbar_wait_warp(&bar, 1, limit);
    out[threadIdx.x] = early | lane << 1 | over << 2 | bytes << 3;
    if (threadIdx.x == 0) *took = t1 - t0;
}

extern "C" int run_wait_probe(int* out, long long* took, long long limit) {
    int* d_out = nullptr;
    long long* d_took = nullptr;
    cudaError_t e = cudaMalloc(&d_out, 32 * sizeof(int));
    if (e == cudaSuccess) e = cudaMalloc(&d_took, sizeof(long long));
    if (e == cudaSuccess) {
        wait_probe<<<1, 32>>>(d_out, d_took, limit);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) e = cudaMemcpy(out, d_out, 32 * sizeof(int), cudaMemcpyDeviceToHost);
    if (e == cudaSuccess) e = cudaMemcpy(took, d_took, sizeof(long long), cudaMemcpyDeviceToHost);
    cudaFree(d_out);
    cudaFree(d_took);
    return static_cast<int>(e);
}
