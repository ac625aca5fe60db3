// A warp whose lanes' limits differ waits for a barrier that is reached between them: mbar_wait_warp gives all
// lanes one answer. Nothing after the wait is the warp's together, and every loop has a limit.
#include <cstdio>

#include "q3_sm100.cuh"

using namespace q3::sm100;

__global__ void __launch_bounds__(64) wait_kernel(int* answers, long long few, long long many, long long pause) {
    __shared__ __align__(8) uint64_t bar;
    __shared__ int abort_flag;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        mbar_init(&bar, 1);
        abort_flag = 0;
        mbar_fence_init();
    }
    __syncthreads();
    if (warp == 0) {
        const bool ok = mbar_wait_warp(&bar, 0, lane < 16 ? few : many, &abort_flag);
        answers[lane] = ok ? 1 : 0;
    } else if (lane == 0) {
        const long long t0 = clock64();
        while (clock64() - t0 < pause) {}
        mbar_arrive(&bar);
    }
}

int main() {
    int* answers = nullptr;
    if (cudaMallocManaged(&answers, 32 * sizeof(int)) != cudaSuccess) return 1;
    const struct {
        long long few, many, pause;
    } cases[] = {{1000, 400000000, 20000000}, {400000000, 1000, 20000000}, {400000000, 400000000, 1000},
                 {1000, 1000, 20000000}};
    for (const auto& c : cases) {
        for (int i = 0; i < 32; ++i) answers[i] = -1;
        wait_kernel<<<1, 64>>>(answers, c.few, c.many, c.pause);
        if (cudaDeviceSynchronize() != cudaSuccess) return 1;
        for (int i = 0; i < 32; ++i) {
            if (answers[i] < 0 || answers[i] != answers[0]) {
                std::printf("lane %d: %d, lane 0: %d (limits %lld, %lld)\n", i, answers[i], answers[0], c.few, c.many);
                return 1;
            }
        }
        std::printf("limits %lld and %lld, reached after %lld: %d\n", c.few, c.many, c.pause, answers[0]);
    }
    std::printf("wait tests passed\n");
    return 0;
}
