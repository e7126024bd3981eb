// Kernels that the operators on rows and sequences share.
#include "sequence_util.cuh"

#include "host_util.h"

namespace gcb {

template <int COLS>
__global__ void __launch_bounds__(kSumThreads) sum_rows_kernel(const __grid_constant__ SumParams P) {
    constexpr int BATCH = 8, WORKERS = kSumThreads / COLS, SHARE = WORKERS / (32 / COLS);
    __shared__ float sm[WORKERS][COLS + 1];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x % COLS, worker = threadIdx.x / COLS;
    const long long blocks = (P.cols + COLS - 1) / COLS;
    const int plane = static_cast<int>(blockIdx.x / blocks);
    const long long col = (blockIdx.x - plane * blocks) * COLS + lane;
    double sum = 0.0;
    if (col < P.cols) {
        const float *src = P.part + (static_cast<long long>(worker) * P.planes + plane) * P.cols + col;
        const long long step = static_cast<long long>(WORKERS) * P.planes * P.cols;
        for (long long left = (P.rows - worker + WORKERS - 1) / WORKERS; left > 0; left -= kSumRun) {
            const int run = static_cast<int>(min(left, static_cast<long long>(kSumRun)));
            float s = 0.0f;
            for (int u = 0; u < run; u += BATCH, src += BATCH * step) {
                float v[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; ++k) v[k] = u + k < run ? src[k * step] : 0.0f;
#pragma unroll
                for (int k = 0; k < BATCH; ++k) s += v[k];
            }
            sum += s;
        }
    }
    sm[worker][lane] = static_cast<float>(sum);
    __syncthreads();
    if (threadIdx.x >= 32) return;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < SHARE; ++w) s += sm[worker * SHARE + w][lane];
#pragma unroll
    for (int o = COLS; o < 32; o *= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (worker == 0 && col < P.cols && P.out[plane] != nullptr)
        store_param(P.out[plane], P.type[plane], col * P.mul[plane] + P.add[plane], s);
}

cudaError_t launch_sum_rows(SumParams &P, cudaStream_t stream) {
    const bool narrow = P.rows > 256;
    const void *fn = narrow ? reinterpret_cast<const void *>(&sum_rows_kernel<8>) : reinterpret_cast<const void *>(&sum_rows_kernel<32>);
    void *args[] = {&P};
    return launch_pdl(fn, dim3(static_cast<unsigned>(P.planes * ceil_div(P.cols, narrow ? 8 : 32))), dim3(kSumThreads), args, 0, stream);
}

}  // namespace gcb
