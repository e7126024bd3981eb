// Dropout of a dense tensor from the counter-based generator, with an optional
// residual sum.  A thread takes eight elements at consecutive places, which is
// one generator block: 16 bytes of a 16-bit tensor or 32 of FP32.
#pragma once
#include "norm_util.cuh"

namespace gcb {

struct DropoutParams {
    const void *x, *residual;  // residual nullable
    void *y;
    uint64_t count;
    uint64_t groups;       // ceil(count / 8)
    uint64_t image, inner; // channel scope: elements of an image, and of a channel (1: channels last)
    uint64_t channels;
    DropParams drop;
};

// Decision index of the element at place i with one decision per channel.
__device__ __forceinline__ uint64_t channel_index(const DropoutParams &P, uint64_t i) {
    if (P.inner != 1) return i / P.inner;  // (n, c, pixels): n * C + c
    return i / P.image * P.channels + i % P.channels;
}

template <class T, bool VEC, bool CHANNEL>
__global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutParams P) {
    constexpr int V = kVec<T>;
    griddep_wait();
    griddep_launch_dependents();
    const DropState ds = drop_state(P.drop, blockIdx.x == 0 && threadIdx.x == 0);
    const T *x = static_cast<const T *>(P.x), *res = static_cast<const T *>(P.residual);
    T *y = static_cast<T *>(P.y);
    for (uint64_t g = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; g < P.groups;
         g += static_cast<uint64_t>(gridDim.x) * blockDim.x) {
        const uint64_t i0 = 8 * g;
        const int here = static_cast<int>(min(static_cast<uint64_t>(8), P.count - i0));
        uint32_t keep = 0;
        if (!CHANNEL) {
            keep = keep_bits<8>(P.drop, ds, i0);
        } else {
            uint64_t block = ~static_cast<uint64_t>(0);
            uint32_t bits = 0;
            for (int k = 0; k < here; ++k) {
                const uint64_t j = channel_index(P, i0 + k);
                if (j >> 3 != block) {
                    block = j >> 3;
                    bits = keep_bits<8>(P.drop, ds, block << 3);
                }
                keep |= (bits >> (j & 7) & 1u) << k;
            }
        }
        if (VEC && here == 8) {
#pragma unroll
            for (int h = 0; h < 8 / V; ++h) {
                float v[V];
                load_elems<T, V>(x + i0 + h * V, v);
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = keep >> (h * V + k) & 1u ? v[k] * P.drop.scale : 0.0f;
                if (res != nullptr) {
                    float r[V];
                    load_elems<T, V>(res + i0 + h * V, r);
#pragma unroll
                    for (int k = 0; k < V; ++k) v[k] += r[k];
                }
                store_elems<T, V>(y + i0 + h * V, v);
            }
        } else {
            for (int k = 0; k < here; ++k) {
                float v = keep >> k & 1u ? to_float(x[i0 + k]) * P.drop.scale : 0.0f;
                if (res != nullptr) v += to_float(res[i0 + k]);
                y[i0 + k] = from_float<T>(v);
            }
        }
    }
}

}  // namespace gcb
