// Dropout from the counter-based generator, with an optional residual sum.
//
// dropout_kernel          one decision per element, or (MAP) per channel of
//                         many small images in either order
// channel_dropout_kernel  one decision per channel of an image, channels last
// plane_dropout_kernel    the same in plain order
// A decision per channel is drawn once for all the pixels that a thread takes.
// All three stream 16-byte vectors through the per-thread rings, or single
// elements where a tensor is not aligned.
#pragma once
#include "norm_util.cuh"

namespace gcb {

struct DropoutParams {
    const void *x, *residual;  // residual nullable
    void *y;
    uint64_t count;            // elements
    // one decision per channel
    uint64_t decisions;        // images * channels
    uint64_t row;              // pixels of an image
    uint64_t chunk, chunks;    // pixels per block (channels last) or warp (plain), chunks of an image or plane
    uint64_t image;            // MAP: elements of an image, channels last; 0 in plain order
    int channels, vcols, vb, cblocks, lanes;  // channels last: columns as in the norm's split path
    DropParams drop;
};

// y = drop(x) [+ residual] for the vectors at k * step from x, y, residual;
// drop(k, vector).
template <class T, int V, class F>
__device__ __forceinline__ void drop_vectors(uint4 *ring, const T *x, const T *residual, T *y, long long step, int count,
                                             F drop) {
    if (residual != nullptr) {
        start_vector_pairs<V>(ring, x, step, residual, step, count);
        for_vector_pairs<T, V>(ring, x, step, residual, step, count, [&](int k, const Lanes<V> &v, const Lanes<V> &r) {
            Lanes<V> s = drop(k, v);
#pragma unroll
            for (int i = 0; i < Lanes<V>::kPairs; ++i) s.p[i] = s.p[i] + r.p[i];
            store_lanes<T, V>(y, s);
            y += step;
        });
    } else {
        start_vectors<V>(ring, x, step, count);
        for_vectors<T, V>(ring, x, step, count, [&](int k, const Lanes<V> &v) {
            store_lanes<T, V>(y, drop(k, v));
            y += step;
        });
    }
}

// The channel of an image that element i belongs to.
__device__ __forceinline__ uint64_t decision_of(const DropoutParams &P, uint64_t i) {
    if (P.count <= 0xffffffffu) {  // for the shorter division
        const uint32_t k = static_cast<uint32_t>(i), c = static_cast<uint32_t>(P.channels);
        if (P.image == 0) return k / static_cast<uint32_t>(P.row);
        return k / static_cast<uint32_t>(P.image) * c + k % c;
    }
    return P.image == 0 ? i / P.row : i / P.image * P.channels + i % P.channels;
}

// The decisions on the V elements from i, a multiple of V; channels last, V
// divides the channels.
template <int V>
__device__ __forceinline__ uint32_t mapped_bits(const DropoutParams &P, const Philox &gen, uint64_t i) {
    uint64_t j = decision_of(P, i);
    if (P.image != 0) return Draws<V>(gen, j).bits(P.drop.limit);
    uint64_t left = (j + 1) * P.row - i;  // of the plane that i lies in
    uint32_t bits = 0;
    for (int k = 0; k < V; left = P.row, ++j) {
        const int take = static_cast<int>(min(left, static_cast<uint64_t>(V - k)));
        if (Draws<1>(gen, j).keep(0, P.drop.limit)) bits |= ((1u << take) - 1u) << k;
        k += take;
    }
    return bits;
}

// Two neighbouring threads of an FP32 tensor compute the same generator block,
// which costs less than accesses of half a sector.  16-bit tensors are bound
// by the generator's products (19 of 32 x 32 -> 64 bits for eight elements).
template <class T, int V, bool MAP>
__global__ void __launch_bounds__(kStreamThreads, 3) dropout_kernel(const __grid_constant__ DropoutParams P) {
    extern __shared__ __align__(16) unsigned char nsm[];
    griddep_wait();
    griddep_launch_dependents();
    const Philox gen(P.drop, blockIdx.x == 0 && threadIdx.x == 0);
    const T *x = static_cast<const T *>(P.x), *res = static_cast<const T *>(P.residual);
    T *y = static_cast<T *>(P.y);
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * kStreamThreads;
    const uint64_t first = static_cast<uint64_t>(blockIdx.x) * kStreamThreads + threadIdx.x, whole = P.count / V;
    // every 2^31 - 1 vectors of a thread anew: the loops count in 32 bits
    constexpr uint64_t kMost = 0x7fffffff;
    for (uint64_t g = first; g < whole; g += kMost * step) {
        const int count = static_cast<int>(min(kMost, (whole - g + step - 1) / step));
        drop_vectors<T, V>(reinterpret_cast<uint4 *>(nsm), x + V * g, res == nullptr ? res : res + V * g, y + V * g,
                           static_cast<long long>(V * step), count, [&](int k, const Lanes<V> &v) {
                               if (P.drop.threshold == 0) return v;
                               const uint64_t i = V * (g + k * step);
                               if constexpr (MAP) return drop_lanes<V>(v, mapped_bits<V>(P, gen, i), P.drop);
                               else return drop_lanes<V>(v, Draws<V>(gen, i), P.drop);
                           });
    }
    const uint64_t i = whole * V + first;  // fewer than V elements are left
    if (i < P.count) {
        const bool keep = P.drop.threshold == 0 || Draws<1>(gen, MAP ? decision_of(P, i) : i).keep(0, P.drop.limit);
        float v = keep ? to_float(x[i]) * P.drop.scale : 0.0f;
        if (res != nullptr) v += to_float(res[i]);
        y[i] = from_float<T>(v);
    }
}

// A thread keeps one vector of channels (V = 1: one channel) for the pixels of
// its block's chunk.
template <class T, int V>
__global__ void __launch_bounds__(kStreamThreads, 3) channel_dropout_kernel(const __grid_constant__ DropoutParams P) {
    extern __shared__ __align__(16) unsigned char nsm[];
    griddep_wait();
    griddep_launch_dependents();
    const Philox gen(P.drop, blockIdx.x == 0 && threadIdx.x == 0);
    const unsigned cb = blockIdx.x % P.cblocks, t = blockIdx.x / P.cblocks;
    const uint64_t n = t / P.chunks, first = (t - n * P.chunks) * P.chunk;
    const int lane = threadIdx.x / P.vb, col = static_cast<int>(cb) * P.vb + threadIdx.x % P.vb;
    const uint64_t p0 = first + lane, last = min(P.row, first + P.chunk);
    if (lane >= P.lanes || col >= P.vcols || p0 >= last) return;
    const uint64_t c0 = static_cast<uint64_t>(col) * V;
    uint32_t keep = ~0u;
    if (P.drop.threshold) keep = Draws<V>(gen, n * P.channels + c0).bits(P.drop.limit);
    const uint64_t at = (n * P.row + p0) * P.channels + c0;
    const T *res = static_cast<const T *>(P.residual);
    drop_vectors<T, V>(reinterpret_cast<uint4 *>(nsm), static_cast<const T *>(P.x) + at, res == nullptr ? res : res + at,
                       static_cast<T *>(P.y) + at, static_cast<long long>(P.lanes) * P.channels,
                       static_cast<int>((last - p0 + P.lanes - 1) / P.lanes),
                       [&](int, const Lanes<V> &v) { return drop_lanes<V>(v, keep, P.drop); });
}

// A warp takes a chunk of one channel's pixels, with single elements up to the
// first 16-byte boundary and behind the last (V > 1: the bases of the three
// tensors are aligned).
template <class T, int V>
__global__ void __launch_bounds__(kStreamThreads, 3) plane_dropout_kernel(const __grid_constant__ DropoutParams P) {
    extern __shared__ __align__(16) unsigned char nsm[];
    griddep_wait();
    griddep_launch_dependents();
    const Philox gen(P.drop, blockIdx.x == 0 && threadIdx.x == 0);
    const T *x = static_cast<const T *>(P.x), *res = static_cast<const T *>(P.residual);
    T *y = static_cast<T *>(P.y);
    const int lane = threadIdx.x & 31;
    const uint64_t warps = static_cast<uint64_t>(gridDim.x) * (kStreamThreads / 32);
    for (uint64_t item = static_cast<uint64_t>(blockIdx.x) * (kStreamThreads / 32) + threadIdx.x / 32;
         item < P.decisions * P.chunks; item += warps) {
        const uint64_t j = item / P.chunks, p0 = (item - j * P.chunks) * P.chunk;
        const uint64_t begin = j * P.row + p0, end = j * P.row + min(P.row, p0 + P.chunk);
        const uint32_t keep = P.drop.threshold == 0 || Draws<1>(gen, j).keep(0, P.drop.limit) ? ~0u : 0u;
        const uint64_t low = min(end, (begin + V - 1) / V * V), high = max(low, end / V * V), i0 = low + lane * V;
        auto single = [&](uint64_t i) {  // fewer than a warp's lanes on either side
            float v = keep ? to_float(x[i]) * P.drop.scale : 0.0f;
            if (res != nullptr) v += to_float(res[i]);
            y[i] = from_float<T>(v);
        };
        if (begin + lane < low) single(begin + lane);
        if (high + lane < end) single(high + lane);
        const int count = i0 < high ? static_cast<int>((high - i0 + 32 * V - 1) / (32 * V)) : 0;
        drop_vectors<T, V>(reinterpret_cast<uint4 *>(nsm), x + i0, res == nullptr ? res : res + i0, y + i0, 32 * V, count,
                           [&](int, const Lanes<V> &v) { return drop_lanes<V>(v, keep, P.drop); });
        cp_async_wait<0>();  // the ring is used again
    }
}

}  // namespace gcb
