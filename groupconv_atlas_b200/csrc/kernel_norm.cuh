// Group normalisation of channels-last tensors with an activation and dropout
// in its epilogue, and its gradient.
//
//   mean, var over the pixels and channels of one group of one image
//   z = (x - mean) * a + beta[c],  a = gamma[c] / sqrt(var + eps)
//   y = keep ? act(z) / (1 - q) : 0
//   dz = keep ? dy / (1 - q) * act'(z) : 0
//   dbeta[c] = sum dz,  dgamma[c] = rstd * sum dz (x - mean)
//   dx = a dz - k1 - k2 (x - mean),  k1 = rstd S1 / M,  k2 = rstd^2 S2 / M,
//        S1 = sum gamma dz, S2 = rstd * sum gamma dz (x - mean) over the group,
//        M the elements of a group of one image
// z and x - mean come from the same two operations in both directions, so the
// gradient sees the activation's argument that the forward pass saw.
//
// The split path below runs for every supported tensor: partial results of
// chunks of pixels per channel, one reduction per group, and a second pass
// over the data.  A vector of V channels per thread (16 bytes, or one element
// where a pixel is not a multiple of 16 bytes); a block covers up to 256
// vector columns and walks down its chunk of pixels.
#pragma once
#include "norm_util.cuh"

namespace gcb {

constexpr int kNormThreads = 256;
constexpr int kNormRun = 64;  // pixels of a thread that share a pivot (below)

struct NormParams {
    const void *x, *dy;
    void *y;  // y or dx
    long long x_ldn, x_ldp, dy_ldn, dy_ldp, y_ldn, y_ldp;  // element strides of an image and a pixel
    const void *gamma, *beta;                              // nullable
    int gamma_type, beta_type;                             // ElemType
    void *dgamma, *dbeta;                                  // nullable
    int dgamma_type, dbeta_type;
    float2 *stats;  // [n][groups]: mean, 1 / sqrt(var + eps)
    float2 *part;   // [n][chunks][c]: (mean, sum of squares about it), or the gradient's two sums
    float2 *chan;   // [n][c]: the gradient's sums of a channel
    float2 *gsum;   // [n][groups]: k1, k2
    long long n, px;
    int c, groups, cpg;
    float eps;
    int act;
    // split path
    long long chunk_rows;  // pixels per chunk
    int chunks;            // per image
    int vcols;             // c / V
    int vb;                // vector columns per block (at most 256)
    int cblocks;           // ceil(vcols / vb)
    int lanes;             // 256 / vb pixels at a time
    long long items;       // n * chunks * cblocks
    DropParams drop;
};

struct NormItem {
    long long n, p0, p1;  // image, first and one-past-last pixel
    int chunk, vcol;
};

__device__ __forceinline__ NormItem norm_item(const NormParams &P, long long item, int col) {
    NormItem it;
    const int cb = static_cast<int>(item % P.cblocks);
    const long long t = item / P.cblocks;
    it.chunk = static_cast<int>(t % P.chunks);
    it.n = t / P.chunks;
    it.vcol = cb * P.vb + col;
    it.p0 = it.chunk * P.chunk_rows;
    it.p1 = min(P.px, it.p0 + P.chunk_rows);
    return it;
}

// (count, mean, sum of squares about the mean) of two disjoint sets joined.
__device__ __forceinline__ void join_moments(float &n, float &mean, float &m2, float nb, float mb, float m2b) {
    if (nb == 0.0f) return;
    const float total = n + nb, f = nb / total, d = mb - mean;
    mean = fmaf(d, f, mean);
    m2 += m2b + d * d * (n * f);
    n = total;
}

template <int ACT>
__device__ __forceinline__ float act_fwd(int act, float z) {
    if constexpr (ACT >= 0) return activate<ACT>(z);
    if (act == kActRelu) return activate<kActRelu>(z);
    if (act == kActRelu6) return activate<kActRelu6>(z);
    if (act == kActSilu) return activate<kActSilu>(z);
    return z;
}
template <int ACT>
__device__ __forceinline__ float act_bwd(int act, float z, float g) {
    if constexpr (ACT >= 0) return activate_grad<ACT>(z, g);
    if (act == kActRelu) return activate_grad<kActRelu>(z, g);
    if (act == kActRelu6) return activate_grad<kActRelu6>(z, g);
    if (act == kActSilu) return activate_grad<kActSilu>(z, g);
    return g;
}

// Sum of v over the block (every thread gets it).  red: 32 floats of shared memory.
__device__ __forceinline__ float block_sum(float v, float *red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();  // red is free
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = lane < warps ? red[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// ---- split path, forward ---------------------------------------------------------------
// Moments of one chunk per channel.  A thread sums x - pivot and its square
// over runs of at most 64 of its pixels, the pivot being the run's first
// value: it is one of the values, so the squares about it exceed the squares
// about the mean at most by the run's length, and the cancellation in
// sum d^2 - (sum d)^2 / n costs at most 64 rounding errors whatever the data's
// mean.  Runs, pixel lanes and chunks are joined as (count, mean, squares).
template <class T, int V>
__global__ void __launch_bounds__(kNormThreads) norm_moments_kernel(const __grid_constant__ NormParams P) {
    __shared__ float2 sm[kNormThreads * V];
    __shared__ float cnt[kNormThreads];
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x, lane = tid / P.vb, col = tid - lane * P.vb;
    int half = 1;
    while (half * 2 < P.lanes) half *= 2;
    for (long long item = blockIdx.x; item < P.items; item += gridDim.x) {
        const NormItem it = norm_item(P, item, col);
        const bool active = lane < P.lanes && it.vcol < P.vcols;
        float mean[V], m2[V], n = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) mean[j] = m2[j] = 0.0f;
        if (active) {
            const T *x = static_cast<const T *>(P.x) + it.n * P.x_ldn + static_cast<long long>(it.vcol) * V;
            const long long step = static_cast<long long>(P.lanes) * kNormRun;
            for (long long base = it.p0 + lane; base < it.p1; base += step) {
                const long long end = min(it.p1, base + step);
                float piv[V], s[V], q[V];
                load_elems<T, V>(x + base * P.x_ldp, piv);
#pragma unroll
                for (int j = 0; j < V; ++j) s[j] = q[j] = 0.0f;
                float k = 1.0f;
#pragma unroll 4
                for (long long p = base + P.lanes; p < end; p += P.lanes) {
                    float v[V];
                    load_elems<T, V>(x + p * P.x_ldp, v);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float d = v[j] - piv[j];
                        s[j] += d;
                        q[j] = fmaf(d, d, q[j]);
                    }
                    k += 1.0f;
                }
                const float inv = 1.0f / k;
                const float before = n;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float nj = before;
                    join_moments(nj, mean[j], m2[j], k, fmaf(s[j], inv, piv[j]), fmaxf(0.0f, fmaf(-s[j] * inv, s[j], q[j])));
                    if (j == V - 1) n = nj;
                }
            }
        }
        __syncthreads();  // the previous item's values are no longer read
        if (lane < P.lanes) {
            if (col == 0) cnt[lane] = n;
#pragma unroll
            for (int j = 0; j < V; ++j) sm[tid * V + j] = make_float2(mean[j], m2[j]);
        }
        for (int h = half; h > 0; h >>= 1) {
            __syncthreads();
            float nb = 0.0f;
            if (lane < h && lane + h < P.lanes) {
                n = cnt[lane];
                nb = cnt[lane + h];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float2 b = sm[(tid + h * P.vb) * V + j];
                    float nj = n;
                    join_moments(nj, mean[j], m2[j], nb, b.x, b.y);
                    sm[tid * V + j] = make_float2(mean[j], m2[j]);
                }
            }
            __syncthreads();
            if (lane < h && lane + h < P.lanes && col == 0) cnt[lane] = n + nb;
        }
        if (lane == 0 && it.vcol < P.vcols) {
            float2 *out = P.part + (it.n * P.chunks + it.chunk) * P.c + static_cast<long long>(it.vcol) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) out[j] = make_float2(mean[j], m2[j]);
        }
    }
}

// Joins a group's chunks and channels: one block per (image, group).
__global__ void __launch_bounds__(kNormThreads) norm_finalize_kernel(const __grid_constant__ NormParams P) {
    __shared__ float red[32];
    griddep_wait();
    griddep_launch_dependents();
    const float total = static_cast<float>(P.px) * static_cast<float>(P.cpg);
    const long long entries = static_cast<long long>(P.chunks) * P.cpg;
    for (long long ng = blockIdx.x; ng < P.n * P.groups; ng += gridDim.x) {
        const long long n = ng / P.groups;
        const float2 *part = P.part + n * P.chunks * P.c + (ng - n * P.groups) * P.cpg;
        float s = 0.0f;
        for (long long i = threadIdx.x; i < entries; i += kNormThreads) {
            const long long k = i / P.cpg;
            const float rows = static_cast<float>(min(P.chunk_rows, P.px - k * P.chunk_rows));
            s = fmaf(rows, part[k * P.c + (i - k * P.cpg)].x, s);
        }
        const float mean = block_sum(s, red) / total;
        float q = 0.0f;
        for (long long i = threadIdx.x; i < entries; i += kNormThreads) {
            const long long k = i / P.cpg;
            const float rows = static_cast<float>(min(P.chunk_rows, P.px - k * P.chunk_rows));
            const float2 v = part[k * P.c + (i - k * P.cpg)];
            const float d = v.x - mean;
            q += fmaf(rows * d, d, v.y);
        }
        const float var = block_sum(q, red) / total;
        if (threadIdx.x == 0) P.stats[ng] = make_float2(mean, 1.0f / sqrtf(var + P.eps));
    }
}

// Normalises, activates and drops out: the second pass over x.
template <class T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_apply_kernel(const __grid_constant__ NormParams P) {
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x, lane = tid / P.vb, col = tid - lane * P.vb;
    DropState ds{};
    if (P.drop.threshold) ds = drop_state(P.drop, blockIdx.x == 0 && tid == 0);
    for (long long item = blockIdx.x; item < P.items; item += gridDim.x) {
        const NormItem it = norm_item(P, item, col);
        if (lane >= P.lanes || it.vcol >= P.vcols) continue;
        const int c0 = it.vcol * V;
        float mean[V], a[V], b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 st = P.stats[it.n * P.groups + (c0 + j) / P.cpg];
            mean[j] = st.x;
            a[j] = st.y * (P.gamma ? load_param(P.gamma, P.gamma_type, c0 + j) : 1.0f);
            b[j] = P.beta ? load_param(P.beta, P.beta_type, c0 + j) : 0.0f;
        }
        uint32_t keep = ~0u;
        if (P.drop.threshold && P.drop.channel) keep = keep_bits<V>(P.drop, ds, static_cast<uint64_t>(it.n) * P.c + c0);
        const T *x = static_cast<const T *>(P.x) + it.n * P.x_ldn + c0;
        T *y = static_cast<T *>(P.y) + it.n * P.y_ldn + c0;
#pragma unroll 2
        for (long long p = it.p0 + lane; p < it.p1; p += P.lanes) {
            float v[V];
            load_elems<T, V>(x + p * P.x_ldp, v);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = act_fwd<ACT>(P.act, fmaf(v[j] - mean[j], a[j], b[j]));
            if (P.drop.threshold) {
                if (!P.drop.channel)
                    keep = keep_bits<V>(P.drop, ds, (static_cast<uint64_t>(it.n) * P.px + p) * P.c + c0);
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = keep >> j & 1u ? v[j] * P.drop.scale : 0.0f;
            }
            store_elems<T, V>(y + p * P.y_ldp, v);
        }
    }
}

// ---- split path, gradient ----------------------------------------------------------------
// Per chunk and channel: sum dz, sum dz (x - mean).
template <class T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_grad_sums_kernel(const __grid_constant__ NormParams P) {
    __shared__ float2 sm[kNormThreads * V];
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x, lane = tid / P.vb, col = tid - lane * P.vb;
    DropState ds{};
    if (P.drop.threshold) ds = drop_state(P.drop, false);
    int half = 1;
    while (half * 2 < P.lanes) half *= 2;
    for (long long item = blockIdx.x; item < P.items; item += gridDim.x) {
        const NormItem it = norm_item(P, item, col);
        float s[V], t[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = t[j] = 0.0f;
        if (lane < P.lanes && it.vcol < P.vcols) {
            const int c0 = it.vcol * V;
            float mean[V], a[V], b[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float2 st = P.stats[it.n * P.groups + (c0 + j) / P.cpg];
                mean[j] = st.x;
                a[j] = st.y * (P.gamma ? load_param(P.gamma, P.gamma_type, c0 + j) : 1.0f);
                b[j] = P.beta ? load_param(P.beta, P.beta_type, c0 + j) : 0.0f;
            }
            uint32_t keep = ~0u;
            if (P.drop.threshold && P.drop.channel)
                keep = keep_bits<V>(P.drop, ds, static_cast<uint64_t>(it.n) * P.c + c0);
            const T *x = static_cast<const T *>(P.x) + it.n * P.x_ldn + c0;
            const T *dy = static_cast<const T *>(P.dy) + it.n * P.dy_ldn + c0;
#pragma unroll 2
            for (long long p = it.p0 + lane; p < it.p1; p += P.lanes) {
                float v[V], g[V];
                load_elems<T, V>(x + p * P.x_ldp, v);
                load_elems<T, V>(dy + p * P.dy_ldp, g);
                if (P.drop.threshold) {
                    if (!P.drop.channel)
                        keep = keep_bits<V>(P.drop, ds, (static_cast<uint64_t>(it.n) * P.px + p) * P.c + c0);
#pragma unroll
                    for (int j = 0; j < V; ++j) g[j] = keep >> j & 1u ? g[j] * P.drop.scale : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = v[j] - mean[j];
                    const float dz = act_bwd<ACT>(P.act, fmaf(d, a[j], b[j]), g[j]);
                    s[j] += dz;
                    t[j] = fmaf(dz, d, t[j]);
                }
            }
        }
        __syncthreads();
        if (lane < P.lanes) {
#pragma unroll
            for (int j = 0; j < V; ++j) sm[tid * V + j] = make_float2(s[j], t[j]);
        }
        for (int h = half; h > 0; h >>= 1) {
            __syncthreads();
            if (lane < h && lane + h < P.lanes) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float2 o = sm[(tid + h * P.vb) * V + j];
                    s[j] += o.x;
                    t[j] += o.y;
                    sm[tid * V + j] = make_float2(s[j], t[j]);
                }
            }
        }
        if (lane == 0 && it.vcol < P.vcols) {
            float2 *out = P.part + (it.n * P.chunks + it.chunk) * P.c + static_cast<long long>(it.vcol) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) out[j] = make_float2(s[j], t[j]);
        }
    }
}

// Per (image, group): the channels' sums over all chunks, and the group's k1, k2.
__global__ void __launch_bounds__(kNormThreads) norm_grad_finalize_kernel(const __grid_constant__ NormParams P) {
    __shared__ float red[32];
    griddep_wait();
    griddep_launch_dependents();
    const float total = static_cast<float>(P.px) * static_cast<float>(P.cpg);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (long long ng = blockIdx.x; ng < P.n * P.groups; ng += gridDim.x) {
        const long long n = ng / P.groups;
        const int c0 = static_cast<int>(ng - n * P.groups) * P.cpg;
        const float2 st = P.stats[ng];
        float s1 = 0.0f, s2 = 0.0f;
        for (int k = warp; k < P.cpg; k += warps) {
            const float2 *part = P.part + n * P.chunks * P.c + c0 + k;
            float s = 0.0f, t = 0.0f;
            for (int i = lane; i < P.chunks; i += 32) {
                const float2 v = part[static_cast<long long>(i) * P.c];
                s += v.x;
                t += v.y;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                s += __shfl_xor_sync(0xffffffffu, s, o);
                t += __shfl_xor_sync(0xffffffffu, t, o);
            }
            t *= st.y;
            if (lane == 0) {
                const float gm = P.gamma ? load_param(P.gamma, P.gamma_type, c0 + k) : 1.0f;
                P.chan[n * P.c + c0 + k] = make_float2(s, t);
                s1 = fmaf(gm, s, s1);
                s2 = fmaf(gm, t, s2);
            }
        }
        s1 = block_sum(s1, red);
        s2 = block_sum(s2, red);
        if (threadIdx.x == 0) P.gsum[ng] = make_float2(st.y * s1 / total, st.y * st.y * s2 / total);
    }
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_grad_apply_kernel(const __grid_constant__ NormParams P) {
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x, lane = tid / P.vb, col = tid - lane * P.vb;
    DropState ds{};
    if (P.drop.threshold) ds = drop_state(P.drop, blockIdx.x == 0 && tid == 0);
    for (long long item = blockIdx.x; item < P.items; item += gridDim.x) {
        const NormItem it = norm_item(P, item, col);
        if (lane >= P.lanes || it.vcol >= P.vcols) continue;
        const int c0 = it.vcol * V;
        float mean[V], a[V], b[V], k1[V], k2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const long long ng = it.n * P.groups + (c0 + j) / P.cpg;
            const float2 st = P.stats[ng], k = P.gsum[ng];
            mean[j] = st.x;
            a[j] = st.y * (P.gamma ? load_param(P.gamma, P.gamma_type, c0 + j) : 1.0f);
            b[j] = P.beta ? load_param(P.beta, P.beta_type, c0 + j) : 0.0f;
            k1[j] = k.x;
            k2[j] = k.y;
        }
        uint32_t keep = ~0u;
        if (P.drop.threshold && P.drop.channel) keep = keep_bits<V>(P.drop, ds, static_cast<uint64_t>(it.n) * P.c + c0);
        const T *x = static_cast<const T *>(P.x) + it.n * P.x_ldn + c0;
        const T *dy = static_cast<const T *>(P.dy) + it.n * P.dy_ldn + c0;
        T *dx = static_cast<T *>(P.y) + it.n * P.y_ldn + c0;
#pragma unroll 2
        for (long long p = it.p0 + lane; p < it.p1; p += P.lanes) {
            float v[V], g[V];
            load_elems<T, V>(x + p * P.x_ldp, v);
            load_elems<T, V>(dy + p * P.dy_ldp, g);
            if (P.drop.threshold) {
                if (!P.drop.channel)
                    keep = keep_bits<V>(P.drop, ds, (static_cast<uint64_t>(it.n) * P.px + p) * P.c + c0);
#pragma unroll
                for (int j = 0; j < V; ++j) g[j] = keep >> j & 1u ? g[j] * P.drop.scale : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = v[j] - mean[j];
                const float dz = act_bwd<ACT>(P.act, fmaf(d, a[j], b[j]), g[j]);
                v[j] = fmaf(a[j], dz, -fmaf(d, k2[j], k1[j]));
            }
            store_elems<T, V>(dx + p * P.y_ldp, v);
        }
    }
}

// dgamma, dbeta: the channels' sums over the images.  A block takes 32
// channels, eight images at a time.
__global__ void __launch_bounds__(kNormThreads) norm_grad_params_kernel(const __grid_constant__ NormParams P) {
    __shared__ float2 sm[kNormThreads];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float s = 0.0f, t = 0.0f;
    if (c < P.c)
        for (long long n = row; n < P.n; n += kNormThreads / 32) {
            const float2 v = P.chan[n * P.c + c];
            s += v.x;
            t += v.y;
        }
    sm[threadIdx.x] = make_float2(s, t);
    __syncthreads();
    if (row == 0 && c < P.c) {
#pragma unroll
        for (int r = 1; r < kNormThreads / 32; ++r) {
            s += sm[r * 32 + lane].x;
            t += sm[r * 32 + lane].y;
        }
        if (P.dbeta) store_param(P.dbeta, P.dbeta_type, c, s);
        if (P.dgamma) store_param(P.dgamma, P.dgamma_type, c, t);
    }
}

}  // namespace gcb
