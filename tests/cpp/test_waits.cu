// A wait for a barrier that nobody arrives at ends by itself, with its flag set, and those behind it do not wait at all.
#include <cstdio>

#include "tensor.cuh"

using namespace mtxc;

struct Seen {
    int first, failed, second, third, fourth;
    long long first_cycles, second_cycles;
};

__global__ void wait_kernel(Seen* seen) {
    __shared__ alignas(8) uint64_t bars[2];
    __shared__ int failed;
    if (threadIdx.x) return;
    const uint32_t silent = shared_address(bars), other = silent + 8;
    barrier_init(silent, 1);
    barrier_init(other, 1);
    failed = 0;
    barrier_arrive(other);
    seen->third = barrier_wait(other, 0, &failed);  // its phase has ended
    long long t = clock64();
    seen->first = barrier_wait(silent, 0, &failed);
    seen->first_cycles = clock64() - t;
    seen->failed = failed;
    t = clock64();
    seen->second = barrier_wait(silent, 0, &failed);
    seen->second_cycles = clock64() - t;
    seen->fourth = barrier_wait(other, 0, &failed);
}

int main() {
    Seen* seen;
    if (cudaMallocManaged(&seen, sizeof *seen) != cudaSuccess) return 2;
    wait_kernel<<<1, 32>>>(seen);
    if (cudaDeviceSynchronize() != cudaSuccess) return 3;
    std::printf("%d %d %d %d %d %lld %lld\n", seen->first, seen->failed, seen->second, seen->third, seen->fourth, seen->first_cycles,
                seen->second_cycles);
    return 0;
}
