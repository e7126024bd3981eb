// Kernels that the operators on rows and sequences share.
#include "sequence_util.cuh"

namespace gcb {

__global__ void __launch_bounds__(kSumWarps * 32) sum_rows_kernel(const __grid_constant__ SumParams P) {
    __shared__ float sm[kSumWarps][33];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long blocks = (P.cols + 31) / 32;
    const int plane = static_cast<int>(blockIdx.x / blocks);
    const long long col = (blockIdx.x - plane * blocks) * 32 + lane;
    double sum = 0.0;
    if (col < P.cols) {
        const float *src = P.part + (static_cast<long long>(warp) * P.planes + plane) * P.cols + col;
        const long long step = static_cast<long long>(kSumWarps) * P.planes * P.cols;
        for (long long left = (P.rows - warp + kSumWarps - 1) / kSumWarps; left > 0; left -= kSumRun) {
            const int run = static_cast<int>(min(left, static_cast<long long>(kSumRun)));
            float s = 0.0f;
#pragma unroll 8
            for (int u = 0; u < run; ++u, src += step) s += *src;
            sum += s;
        }
    }
    sm[warp][lane] = static_cast<float>(sum);
    __syncthreads();
    if (warp == 0 && col < P.cols) {
        float s = sm[0][lane];
#pragma unroll
        for (int w = 1; w < kSumWarps; ++w) s += sm[w][lane];
        if (P.out[plane] != nullptr) store_param(P.out[plane], P.type[plane], col * P.mul[plane] + P.add[plane], s);
    }
}

}  // namespace gcb
