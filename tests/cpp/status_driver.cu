// A bounded wait that runs out, and the status word that says so: the wait of csrc/ptx.cuh on a barrier that nothing arrives at, with a limit of
// a few polls, on a stream that does not wait for the default one, and the read of csrc/device_plan.hpp.
#include <cstdio>

#include "device_plan.hpp"
#include "ptx.cuh"

using namespace cutespmm;

__device__ uint32_t g_status;

// Sleeps a while first, so that a read that waits for nothing comes too early.
__global__ void gives_up(uint32_t arrive)
{
    __shared__ uint64_t bar;
    if (threadIdx.x == 0) {
        ptx::mbar_init(&bar, 1);
        ptx::fence_mbar_init();
        for (int i = 0; i < 5000; ++i) __nanosleep(1000);
        if (arrive) ptx::mbar_arrive(&bar);
        if (!ptx::mbar_wait(&bar, 0, 16)) atomicExch(&g_status, 1u);
    }
}

int main()
{
    cudaStream_t s;
    uint32_t word = 7, after = 7, fine = 7;
    if (cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking) != cudaSuccess) return 1;
    gives_up<<<1, 32, 0, s>>>(0);
    if (read_status(g_status, &word) != cudaSuccess || read_status(g_status, &after) != cudaSuccess) return 1;
    gives_up<<<1, 32, 0, s>>>(1);
    if (read_status(g_status, &fine) != cudaSuccess) return 1;
    std::printf("ran out %u, read again %u, arrived %u\n", word, after, fine);
    return 0;
}
