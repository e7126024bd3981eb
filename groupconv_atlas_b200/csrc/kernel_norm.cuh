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
// Two paths.  The resident path (end of this file) reads x, and dy, once: a
// cluster of CTAs holds all pixels of some whole groups of an image in shared
// memory.  It takes every tensor whose pixels are multiples of 16 bytes and
// whose groups fit.
//
// The split path runs for every supported tensor: partial results of chunks of
// pixels per channel, one reduction per group, and a second pass over the
// data.  A vector of V channels per thread (16 bytes, or one element where a
// pixel is not a multiple of 16 bytes); a block covers up to 256 vector columns
// and walks down its chunk of pixels.
#pragma once
#include <cooperative_groups.h>

#include "norm_util.cuh"

namespace gcb {

constexpr int kNormThreads = 256;      // split path
constexpr int kResidentThreads = 512;  // resident path, at most
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
    long long sum_rows;    // rows of chan that the parameters' gradients add up
    // resident path
    int cb;       // channels of a unit (whole groups, whole vectors)
    int vr;       // cb / V vector columns; a thread keeps one of them
    int sub;      // sums of a thread's V channels that stay apart (1: one group a vector)
    int gcols;    // such sums of one pixel lane that make up a group
    int gb;       // groups of a unit
    int bundles;  // c / cb
    int cluster;  // CTAs that share a unit's pixels
    int rows;     // pixels per CTA
    int iters;    // ceil(rows / lanes) vectors per thread
    long long stride;  // clusters per bundle: each takes every stride-th image
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

// The per-channel values of a thread, as pairs.
template <int V>
struct Coefs {
    Lanes<V> minus_mean, a, b;
};
// z = (x - mean) a + b; also d = x - mean.
template <int V>
__device__ __forceinline__ f2 normalise(const Coefs<V> &k, int i, f2 x, f2 &d) {
    d = x + k.minus_mean.p[i];
    return fma2(d, k.a.p[i], k.b.p[i]);
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

template <int V>
__device__ __forceinline__ Coefs<V> split_coefs(const NormParams &P, long long n, int c0) {
    float mean[V], a[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 st = P.stats[n * P.groups + (c0 + j) / P.cpg];
        mean[j] = -st.x;
        a[j] = st.y * (P.gamma ? load_param(P.gamma, P.gamma_type, c0 + j) : 1.0f);
        b[j] = P.beta ? load_param(P.beta, P.beta_type, c0 + j) : 0.0f;
    }
    return {lanes_of<V>(mean), lanes_of<V>(a), lanes_of<V>(b)};
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
        const Coefs<V> coefs = split_coefs<V>(P, it.n, c0);
        uint32_t keep = ~0u;
        if (P.drop.threshold && P.drop.channel) keep = keep_bits<V>(P.drop, ds, static_cast<uint64_t>(it.n) * P.c + c0);
        const T *x = static_cast<const T *>(P.x) + it.n * P.x_ldn + c0;
        T *y = static_cast<T *>(P.y) + it.n * P.y_ldn + c0;
#pragma unroll 2
        for (long long p = it.p0 + lane; p < it.p1; p += P.lanes) {
            Lanes<V> v = load_lanes<T, V>(x + p * P.x_ldp);
#pragma unroll
            for (int i = 0; i < Lanes<V>::kPairs; ++i) {
                f2 d;
                v.p[i] = activate<ACT>(P.act, normalise<V>(coefs, i, v.p[i], d));
            }
            if (P.drop.threshold) {
                if (!P.drop.channel)
                    keep = keep_bits<V>(P.drop, ds, (static_cast<uint64_t>(it.n) * P.px + p) * P.c + c0);
                v = keep_lanes<V>(v, keep, P.drop.scale);
            }
            store_lanes<T, V>(y + p * P.y_ldp, v);
        }
    }
}

// ---- split path, gradient ----------------------------------------------------------------
template <int V, int ACT>
__device__ __forceinline__ void grad_sums(int act, const Coefs<V> &k, const Lanes<V> &v, const Lanes<V> &g, Lanes<V> &s,
                                          Lanes<V> &t) {
#pragma unroll
    for (int i = 0; i < Lanes<V>::kPairs; ++i) {
        f2 d;
        const f2 z = normalise<V>(k, i, v.p[i], d);
        const f2 dz = activate_grad<ACT>(act, z, g.p[i]);
        s.p[i] = s.p[i] + dz;
        t.p[i] = fma2(dz, d, t.p[i]);
    }
}
// a dz - k1 - k2 (x - mean), with k1 and k2 given negated
template <int V, int ACT>
__device__ __forceinline__ Lanes<V> grad_result(int act, const Coefs<V> &k, const Lanes<V> &minus_k1,
                                                const Lanes<V> &minus_k2, const Lanes<V> &v, const Lanes<V> &g) {
    Lanes<V> r;
#pragma unroll
    for (int i = 0; i < Lanes<V>::kPairs; ++i) {
        f2 d;
        const f2 z = normalise<V>(k, i, v.p[i], d);
        const f2 dz = activate_grad<ACT>(act, z, g.p[i]);
        r.p[i] = fma2(k.a.p[i], dz, fma2(d, minus_k2.p[i], minus_k1.p[i]));
    }
    return r;
}

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
            const Coefs<V> coefs = split_coefs<V>(P, it.n, c0);
            Lanes<V> s2, t2;
#pragma unroll
            for (int i = 0; i < Lanes<V>::kPairs; ++i) s2.p[i] = t2.p[i] = pair(0.0f);
            uint32_t keep = ~0u;
            if (P.drop.threshold && P.drop.channel)
                keep = keep_bits<V>(P.drop, ds, static_cast<uint64_t>(it.n) * P.c + c0);
            const T *x = static_cast<const T *>(P.x) + it.n * P.x_ldn + c0;
            const T *dy = static_cast<const T *>(P.dy) + it.n * P.dy_ldn + c0;
#pragma unroll 2
            for (long long p = it.p0 + lane; p < it.p1; p += P.lanes) {
                const Lanes<V> v = load_lanes<T, V>(x + p * P.x_ldp);
                Lanes<V> g = load_lanes<T, V>(dy + p * P.dy_ldp);
                if (P.drop.threshold) {
                    if (!P.drop.channel)
                        keep = keep_bits<V>(P.drop, ds, (static_cast<uint64_t>(it.n) * P.px + p) * P.c + c0);
                    g = keep_lanes<V>(g, keep, P.drop.scale);
                }
                grad_sums<V, ACT>(P.act, coefs, v, g, s2, t2);
            }
            values_of<V>(s2, s);
            values_of<V>(t2, t);
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
        const Coefs<V> coefs = split_coefs<V>(P, it.n, c0);
        float k1[V], k2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 k = P.gsum[it.n * P.groups + (c0 + j) / P.cpg];
            k1[j] = -k.x;
            k2[j] = -k.y;
        }
        const Lanes<V> mk1 = lanes_of<V>(k1), mk2 = lanes_of<V>(k2);
        uint32_t keep = ~0u;
        if (P.drop.threshold && P.drop.channel) keep = keep_bits<V>(P.drop, ds, static_cast<uint64_t>(it.n) * P.c + c0);
        const T *x = static_cast<const T *>(P.x) + it.n * P.x_ldn + c0;
        const T *dy = static_cast<const T *>(P.dy) + it.n * P.dy_ldn + c0;
        T *dx = static_cast<T *>(P.y) + it.n * P.y_ldn + c0;
#pragma unroll 2
        for (long long p = it.p0 + lane; p < it.p1; p += P.lanes) {
            const Lanes<V> v = load_lanes<T, V>(x + p * P.x_ldp);
            Lanes<V> g = load_lanes<T, V>(dy + p * P.dy_ldp);
            if (P.drop.threshold) {
                if (!P.drop.channel)
                    keep = keep_bits<V>(P.drop, ds, (static_cast<uint64_t>(it.n) * P.px + p) * P.c + c0);
                g = keep_lanes<V>(g, keep, P.drop.scale);
            }
            store_lanes<T, V>(dx + p * P.y_ldp, grad_result<V, ACT>(P.act, coefs, mk1, mk2, v, g));
        }
    }
}

// dgamma, dbeta: the channels' sums over all rows (images, or CTAs of the
// resident path).  A block takes 32 channels, eight rows at a time.
__global__ void __launch_bounds__(kNormThreads) norm_grad_params_kernel(const __grid_constant__ NormParams P) {
    __shared__ float2 sm[kNormThreads];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float s = 0.0f, t = 0.0f;
    if (c < P.c)
        for (long long n = row; n < P.sum_rows; n += kNormThreads / 32) {
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

// ---- resident path -------------------------------------------------------------------------
// A unit is some whole groups (cb channels) of one image; a cluster of CTAs
// shares its pixels, and takes every stride-th image of its channels.  Thread
// (lane, col) takes vector column col of the pixels lane, lane + lanes, ...,
// and copies them to shared memory at [k][thread]: it reads back only what it
// copied itself, so the data needs no barrier, no bank conflicts arise
// whatever cb is, and as soon as the last pass has read a vector the next
// image's can be copied into its place: one buffer overlaps a unit's
// arithmetic and stores with the next unit's loads.  Only the sums cross
// threads (shared memory) and CTAs (distributed shared memory), in a fixed
// order.

namespace cg = cooperative_groups;

struct Resident {
    int lane, col, count;  // count: vectors of this thread
    int rows;              // pixels of this CTA
    int c0, local;         // first channel of the thread, in the tensor and in the unit
    long long p0;          // first pixel of the thread
};

__device__ __forceinline__ Resident resident_place(const NormParams &P, int rank, int bundle, int v) {
    Resident r;
    r.lane = threadIdx.x / P.vr;
    r.col = threadIdx.x - r.lane * P.vr;
    const long long first = static_cast<long long>(rank) * P.rows;
    r.rows = static_cast<int>(max(0LL, min(static_cast<long long>(P.rows), P.px - first)));
    r.count = r.lane < P.lanes && r.lane < r.rows ? (r.rows - r.lane + P.lanes - 1) / P.lanes : 0;
    r.local = r.lane < P.lanes ? r.col * v : 0;
    r.c0 = bundle * P.cb + r.local;
    r.p0 = first + r.lane;
    return r;
}

// The copies are committed in kParts groups so that the first pass over the
// data can start while the last ones are in flight.
constexpr int kParts = 4;
__device__ __forceinline__ int part_end(int iters, int count, int part) {
    return min(count, (iters * (part + 1) + kParts - 1) / kParts);
}
__device__ __forceinline__ void wait_part(int part) {
    if (part == 0) cp_async_wait<kParts - 1>();
    else if (part == 1) cp_async_wait<kParts - 2>();
    else if (part == 2) cp_async_wait<kParts - 3>();
    else cp_async_wait<0>();
}
__device__ __forceinline__ void copy_vector(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Calls f(j, group) for a thread's V channels, the group counted within the unit.
template <int V, class F>
__device__ __forceinline__ void for_channels(const NormParams &P, const Resident &r, F f) {
    int g = r.local / P.cpg, at = r.local - g * P.cpg;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        f(j, g);
        if (++at == P.cpg) at = 0, ++g;
    }
}

// Rows of the gradient's channel sums that meet in shared memory: one a warp
// where a warp holds whole pixel lanes (they are added by shuffles first),
// else one a lane.
__host__ __device__ inline int grad_rows(int threads, int vr, int lanes) { return 32 % vr == 0 ? threads / 32 : lanes; }

// Shared memory of the resident kernels behind the tiles.
__host__ __device__ inline size_t resident_extra(const NormParams &P, int threads, bool grad) {
    const size_t gb = P.gb, cb = P.cb;
    const size_t entries = grad ? grad_rows(threads, P.vr, P.lanes) * cb + threads + 2 * cb
                                : static_cast<size_t>(P.lanes) * P.vr * P.sub;
    return (entries + 4 * gb) * sizeof(float2);
}

template <class T, int ACT, bool DROP>
__global__ void __launch_bounds__(kResidentThreads, 1) norm_resident_kernel(const __grid_constant__ NormParams P) {
    constexpr int V = kVec<T>, kPairs = Lanes<V>::kPairs;
    extern __shared__ __align__(16) unsigned char nsm[];
    const int threads = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
    uint4 *tile = reinterpret_cast<uint4 *>(nsm);
    float2 *exch = reinterpret_cast<float2 *>(tile + static_cast<size_t>(P.iters) * threads);  // [2][gb]
    float2 *fin = exch + 2 * P.gb;
    float *pivot = reinterpret_cast<float *>(fin + P.gb);
    float2 *red = fin + 2 * P.gb;  // [lanes][vr][sub]
    const int rank = blockIdx.x % P.cluster;
    const unsigned unit = blockIdx.x / P.cluster;
    const int bundle = unit % P.bundles;
    const Resident r = resident_place(P, rank, bundle, V);
    const uint4 *tile_at = tile + tid;
    const uint32_t tile_addr = smem_addr(tile_at), pitch = 16 * threads;
    griddep_wait();
    griddep_launch_dependents();
    DropState ds{};
    if (DROP) ds = drop_state(P.drop, blockIdx.x == 0 && tid == 0);
    const long long xstep = static_cast<long long>(P.lanes) * P.x_ldp, ystep = static_cast<long long>(P.lanes) * P.y_ldp;
    const T *x = static_cast<const T *>(P.x) + (unit / P.bundles) * P.x_ldn + r.p0 * P.x_ldp + r.c0;
    {
        const T *src = x;
        int k = 0;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            const int to = part_end(P.iters, r.count, part);
#pragma unroll 4
            for (; k < to; ++k, src += xstep) copy_vector(tile_addr + k * pitch, src);
            cp_async_commit();
        }
    }
    float gm[V], bt[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        gm[j] = P.gamma ? load_param(P.gamma, P.gamma_type, r.c0 + j) : 1.0f;
        bt[j] = P.beta ? load_param(P.beta, P.beta_type, r.c0 + j) : 0.0f;
    }
    Coefs<V> coefs;
    coefs.b = lanes_of<V>(bt);
    const float total = static_cast<float>(P.px) * static_cast<float>(P.cpg);
    const float members = static_cast<float>(r.rows) * static_cast<float>(P.cpg);
    int turn = 0;
    for (long long n = unit / P.bundles; n < P.n; n += P.stride, turn ^= 1) {
        // First pass: sums about the thread's first vector.  It is one of the
        // summed values, so the squares about it exceed those about the mean at
        // most by the factor `count`, and so does the cancellation below.
        Lanes<V> minus, s2, q2;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) minus.p[i] = s2.p[i] = q2.p[i] = pair(0.0f);
        int k = 0;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            wait_part(part);
            if (part == 0 && r.count > 0) {
                const Lanes<V> v = unpack_lanes<T, V>(tile_at[0], x);
#pragma unroll
                for (int i = 0; i < kPairs; ++i) minus.p[i] = v.p[i] * pair(-1.0f);
            }
            const int to = part_end(P.iters, r.count, part);
#pragma unroll 4
            for (; k < to; ++k) {
                const Lanes<V> v = unpack_lanes<T, V>(tile_at[k * threads], x);
#pragma unroll
                for (int i = 0; i < kPairs; ++i) {
                    const f2 d = v.p[i] + minus.p[i];
                    s2.p[i] = s2.p[i] + d;
                    q2.p[i] = fma2(d, d, q2.p[i]);
                }
            }
        }
        // Per thread and channel: mean and squares about it; then both about
        // one value of the CTA per group, the mean of the first channel's
        // pixels of lane 0, so that the CTA's threads add up.
        float mean[V], m2[V];
        {
            float s[V], q[V], first[V];
            values_of<V>(s2, s);
            values_of<V>(q2, q);
            values_of<V>(minus, first);
            const float cnt = static_cast<float>(r.count), inv = r.count > 0 ? 1.0f / cnt : 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                mean[j] = fmaf(s[j], inv, -first[j]);
                m2[j] = fmaxf(0.0f, fmaf(-s[j] * inv, s[j], q[j]));
                if (q[j] != q[j]) m2[j] = q[j];  // NaN
            }
            if (r.lane == 0) for_channels<V>(P, r, [&](int j, int g) {
                if (r.local + j == g * P.cpg) pivot[g] = mean[j];
            });
            __syncthreads();
            for_channels<V>(P, r, [&](int j, int g) {
                const float e = mean[j] - pivot[g], ne = cnt * e;
                mean[j] = ne;
                m2[j] = r.count > 0 ? fmaf(ne, e, m2[j]) : 0.0f;
            });
        }
        if (r.lane < P.lanes) {
            if (r.count == 0) {
#pragma unroll
                for (int j = 0; j < V; ++j) mean[j] = m2[j] = 0.0f;
            }
            float2 *out = red + (r.lane * P.vr + r.col) * P.sub;
            if (P.sub == V) {
#pragma unroll
                for (int j = 0; j < V; ++j) out[j] = make_float2(mean[j], m2[j]);
            }
#pragma unroll
            for (int w = V / 2; w >= 1; w /= 2) {  // neighbours added until P.sub values remain
#pragma unroll
                for (int j = 0; j < w; ++j) {
                    mean[j] = mean[2 * j] + mean[2 * j + 1];
                    m2[j] = m2[2 * j] + m2[2 * j + 1];
                }
                if (w == P.sub) {
#pragma unroll
                    for (int j = 0; j < w; ++j) out[j] = make_float2(mean[j], m2[j]);
                }
            }
        }
        __syncthreads();
        float2 *mine = exch + turn * P.gb;
        for (int g = warp; g < P.gb; g += warps) {
            const int each = P.lanes * P.gcols, pitch_f = P.vr * P.sub;
            float a = 0.0f, b = 0.0f;
            for (int m = lane; m < each; m += 32) {
                const int row = m / P.gcols;
                const float2 v = red[row * pitch_f + g * P.gcols + (m - row * P.gcols)];
                a += v.x;
                b += v.y;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                a += __shfl_xor_sync(0xffffffffu, a, o);
                b += __shfl_xor_sync(0xffffffffu, b, o);
            }
            if (lane == 0) {
                const float d = r.rows > 0 ? a / members : 0.0f;
                mine[g] = make_float2(r.rows > 0 ? pivot[g] + d : 0.0f, b - d * a);
            }
        }
        // the cluster's moments joined: lane q reads CTA q's
        if (P.cluster > 1) cg::this_cluster().sync();
        else __syncwarp();
        for (int g = warp; g < P.gb; g += warps) {
            float2 m = make_float2(0.0f, 0.0f);
            if (P.cluster == 1) {
                m = mine[g];
            } else {
                const long long left = P.px - static_cast<long long>(lane) * P.rows;
                float rows = 0.0f;
                float2 o = make_float2(0.0f, 0.0f);
                if (lane < P.cluster && left > 0) {
                    rows = static_cast<float>(min(static_cast<long long>(P.rows), left));
                    o = cg::this_cluster().map_shared_rank(mine, lane)[g];
                }
                float sum = rows * o.x;
#pragma unroll
                for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
                sum = __shfl_sync(0xffffffffu, sum, 0) / static_cast<float>(P.px);
                const float d = o.x - sum;
                float squares = rows > 0.0f ? fmaf(rows * static_cast<float>(P.cpg) * d, d, o.y) : 0.0f;
#pragma unroll
                for (int w = 8; w > 0; w >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, w);
                m = make_float2(sum, squares);
            }
            if (lane == 0) {
                const float2 st = make_float2(m.x, 1.0f / sqrtf((m.y < 0.0f ? 0.0f : m.y) / total + P.eps));
                fin[g] = st;
                if (rank == 0 && P.stats != nullptr) P.stats[n * P.groups + bundle * P.gb + g] = st;
            }
        }
        __syncthreads();
        // Second pass: normalise, activate, drop out, store; the next image's
        // vector is copied into each place that has been read.
        {
            float a[V];
            for_channels<V>(P, r, [&](int j, int g) {
                const float2 st = fin[g];
                mean[j] = -st.x;
                a[j] = st.y * gm[j];
            });
            coefs.minus_mean = lanes_of<V>(mean);
            coefs.a = lanes_of<V>(a);
        }
        T *y = static_cast<T *>(P.y) + n * P.y_ldn + r.p0 * P.y_ldp + r.c0;
        uint32_t keep = ~0u;
        if (DROP && P.drop.channel) keep = keep_bits<V>(P.drop, ds, static_cast<uint64_t>(n) * P.c + r.c0);
        uint64_t at = (static_cast<uint64_t>(n) * P.px + r.p0) * P.c + r.c0;
        const bool more = n + P.stride < P.n;
        x += P.stride * P.x_ldn;
        const T *src = x;
        k = 0;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            const int to = part_end(P.iters, r.count, part);
#pragma unroll 2
            for (; k < to; ++k, y += ystep) {
                Lanes<V> v = unpack_lanes<T, V>(tile_at[k * threads], x);
                if (more) {
                    copy_vector(tile_addr + k * pitch, src);
                    src += xstep;
                }
#pragma unroll
                for (int i = 0; i < kPairs; ++i) {
                    f2 d;
                    v.p[i] = activate<ACT>(P.act, normalise<V>(coefs, i, v.p[i], d));
                }
                if (DROP) {
                    if (!P.drop.channel) keep = keep_bits<V>(P.drop, ds, at);
                    at += static_cast<uint64_t>(P.lanes) * P.c;
                    v = keep_lanes<V>(v, keep, P.drop.scale);
                }
                store_lanes<T, V>(y, v);
            }
            cp_async_commit();
        }
    }
    // no CTA leaves while another may read its exchange
    if (P.cluster > 1) cg::this_cluster().sync();
}

// The gradient: x and dy resident.  First pass: sum dz and sum dz (x - mean)
// per channel; second pass: dx.  Element decisions of the dropout are drawn in
// the first pass and kept as one byte a vector in shared memory.
template <class T, int ACT, bool DROP>
__global__ void __launch_bounds__(kResidentThreads, 1) norm_resident_grad_kernel(const __grid_constant__ NormParams P) {
    constexpr int V = kVec<T>;
    extern __shared__ __align__(16) unsigned char nsm[];
    const int threads = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
    const size_t tiles = static_cast<size_t>(P.iters) * threads;
    uint4 *tx = reinterpret_cast<uint4 *>(nsm);
    float2 *exch = reinterpret_cast<float2 *>(tx + 2 * tiles);  // [2][gb]
    float2 *fin = exch + 2 * P.gb;
    float2 *gst = fin + P.gb;           // mean, rstd of the unit's groups
    float2 *weighted = gst + P.gb;      // [cb]: gamma * the channel's sums
    float2 *acc = weighted + P.cb;      // [cb]: the channel's sums over this CTA's images
    float2 *segsum = acc + P.cb;        // [segs][cb]
    float2 *red = segsum + threads;     // [rows][cb]
    const int rows = grad_rows(threads, P.vr, P.lanes);
    const bool warp_rows = 32 % P.vr == 0;
    uint8_t *bits = reinterpret_cast<uint8_t *>(red + rows * P.cb);
    const int rank = blockIdx.x % P.cluster;
    const unsigned unit = blockIdx.x / P.cluster;
    const int bundle = unit % P.bundles;
    const Resident r = resident_place(P, rank, bundle, V);
    // threads that share a channel's summing (none where a unit has more channels than threads)
    const int segs = threads / P.cb;
    const uint4 *x_at = tx + tid, *g_at = x_at + tiles;
    const uint32_t x_addr = smem_addr(x_at), g_addr = smem_addr(g_at), pitch = 16 * threads;
    griddep_wait();
    griddep_launch_dependents();
    DropState ds{};
    if (DROP) ds = drop_state(P.drop, blockIdx.x == 0 && tid == 0);
    const long long xstep = static_cast<long long>(P.lanes) * P.x_ldp;
    const long long gstep = static_cast<long long>(P.lanes) * P.dy_ldp;
    const long long ystep = static_cast<long long>(P.lanes) * P.y_ldp;
    const T *x = static_cast<const T *>(P.x) + (unit / P.bundles) * P.x_ldn + r.p0 * P.x_ldp + r.c0;
    const T *dy = static_cast<const T *>(P.dy) + (unit / P.bundles) * P.dy_ldn + r.p0 * P.dy_ldp + r.c0;
    {
        const T *sx = x, *sg = dy;
        int k = 0;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            const int to = part_end(P.iters, r.count, part);
#pragma unroll 2
            for (; k < to; ++k, sx += xstep, sg += gstep) {
                copy_vector(x_addr + k * pitch, sx);
                copy_vector(g_addr + k * pitch, sg);
            }
            cp_async_commit();
        }
    }
    for (int c = tid; c < P.cb; c += threads) acc[c] = make_float2(0.0f, 0.0f);
    for (int g = tid; g < P.gb; g += threads) gst[g] = P.stats[(unit / P.bundles) * P.groups + bundle * P.gb + g];
    float gm[V], bt[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        gm[j] = P.gamma ? load_param(P.gamma, P.gamma_type, r.c0 + j) : 1.0f;
        bt[j] = P.beta ? load_param(P.beta, P.beta_type, r.c0 + j) : 0.0f;
    }
    Coefs<V> coefs;
    coefs.b = lanes_of<V>(bt);
    const float total = static_cast<float>(P.px) * static_cast<float>(P.cpg);
    int turn = 0;
    for (long long n = unit / P.bundles; n < P.n; n += P.stride, turn ^= 1) {
        __syncthreads();  // gst
        {
            float mean[V], a[V];
            for_channels<V>(P, r, [&](int j, int g) {
                const float2 st = gst[g];
                mean[j] = -st.x;
                a[j] = st.y * gm[j];
            });
            coefs.minus_mean = lanes_of<V>(mean);
            coefs.a = lanes_of<V>(a);
        }
        Lanes<V> s2, t2;
#pragma unroll
        for (int i = 0; i < Lanes<V>::kPairs; ++i) s2.p[i] = t2.p[i] = pair(0.0f);
        uint32_t keep = ~0u;
        if (DROP && P.drop.channel) keep = keep_bits<V>(P.drop, ds, static_cast<uint64_t>(n) * P.c + r.c0);
        uint64_t at = (static_cast<uint64_t>(n) * P.px + r.p0) * P.c + r.c0;
        int k = 0;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            wait_part(part);
            const int to = part_end(P.iters, r.count, part);
#pragma unroll 2
            for (; k < to; ++k) {
                const Lanes<V> v = unpack_lanes<T, V>(x_at[k * threads], x);
                Lanes<V> g = unpack_lanes<T, V>(g_at[k * threads], x);
                if (DROP) {
                    if (!P.drop.channel) {
                        keep = keep_bits<V>(P.drop, ds, at);
                        bits[k * threads + tid] = static_cast<uint8_t>(keep);
                    }
                    at += static_cast<uint64_t>(P.lanes) * P.c;
                    g = keep_lanes<V>(g, keep, P.drop.scale);
                }
                grad_sums<V, ACT>(P.act, coefs, v, g, s2, t2);
            }
        }
        // channel sums over the CTA's pixels: by shuffles, then in two steps
        if (r.lane < P.lanes) {
            float s[V], t[V];
            values_of<V>(s2, s);
            values_of<V>(t2, t);
            if (warp_rows)  // every lane of the block takes part: 32 is a multiple of vr
                for (int o = P.vr; o < 32; o <<= 1) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
                        t[j] += __shfl_xor_sync(0xffffffffu, t[j], o);
                    }
                }
            if (!warp_rows || lane < P.vr) {
                float2 *out = red + (warp_rows ? warp : r.lane) * P.cb + r.local;
#pragma unroll
                for (int j = 0; j < V; ++j) out[j] = make_float2(s[j], t[j]);
            }
        }
        __syncthreads();
        if (segs > 1) {
            const int seg = tid / P.cb, c = tid - seg * P.cb;
            float2 sum = make_float2(0.0f, 0.0f);
            if (seg < segs) {
                for (int l = seg; l < rows; l += segs) {
                    const float2 v = red[l * P.cb + c];
                    sum.x += v.x;
                    sum.y += v.y;
                }
                segsum[tid] = sum;
            }
            __syncthreads();
        }
        const float2 *parts = segs > 1 ? segsum : red;
        const int count = segs > 1 ? segs : rows;
        for (int c = tid; c < P.cb; c += threads) {
            float2 sum = make_float2(0.0f, 0.0f);
            for (int i = 0; i < count; ++i) {
                const float2 v = parts[i * P.cb + c];
                sum.x += v.x;
                sum.y += v.y;
            }
            sum.y *= gst[c / P.cpg].y;
            const float w = P.gamma ? load_param(P.gamma, P.gamma_type, bundle * P.cb + c) : 1.0f;
            weighted[c] = make_float2(w * sum.x, w * sum.y);
            acc[c] = make_float2(acc[c].x + sum.x, acc[c].y + sum.y);
        }
        __syncthreads();
        float2 *mine = exch + turn * P.gb;
        for (int g = warp; g < P.gb; g += warps) {
            float s1 = 0.0f, w2 = 0.0f;
            for (int c = lane; c < P.cpg; c += 32) {
                s1 += weighted[g * P.cpg + c].x;
                w2 += weighted[g * P.cpg + c].y;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                s1 += __shfl_xor_sync(0xffffffffu, s1, o);
                w2 += __shfl_xor_sync(0xffffffffu, w2, o);
            }
            if (lane == 0) mine[g] = make_float2(s1, w2);
        }
        if (P.cluster > 1) cg::this_cluster().sync();
        else __syncwarp();
        for (int g = warp; g < P.gb; g += warps) {
            float2 o = make_float2(0.0f, 0.0f);
            if (P.cluster == 1) {
                o = mine[g];
            } else {
                if (lane < P.cluster) o = cg::this_cluster().map_shared_rank(mine, lane)[g];
#pragma unroll
                for (int w = 8; w > 0; w >>= 1) {
                    o.x += __shfl_xor_sync(0xffffffffu, o.x, w);
                    o.y += __shfl_xor_sync(0xffffffffu, o.y, w);
                }
            }
            const float rstd = gst[g].y;
            if (lane == 0) fin[g] = make_float2(rstd * o.x / total, rstd * rstd * o.y / total);
        }
        __syncthreads();
        Lanes<V> mk1, mk2;
        {
            float k1[V], k2[V];
            for_channels<V>(P, r, [&](int j, int g) {
                k1[j] = -fin[g].x;
                k2[j] = -fin[g].y;
            });
            mk1 = lanes_of<V>(k1);
            mk2 = lanes_of<V>(k2);
        }
        T *dx = static_cast<T *>(P.y) + n * P.y_ldn + r.p0 * P.y_ldp + r.c0;
        const bool more = n + P.stride < P.n;
        // the next image's statistics: gst was last read before the barrier above
        if (more)
            for (int g = tid; g < P.gb; g += threads) gst[g] = P.stats[(n + P.stride) * P.groups + bundle * P.gb + g];
        x += P.stride * P.x_ldn;
        dy += P.stride * P.dy_ldn;
        const T *sx = x, *sg = dy;
        k = 0;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            const int to = part_end(P.iters, r.count, part);
#pragma unroll 2
            for (; k < to; ++k, dx += ystep) {
                const Lanes<V> v = unpack_lanes<T, V>(x_at[k * threads], x);
                Lanes<V> g = unpack_lanes<T, V>(g_at[k * threads], x);
                if (more) {
                    copy_vector(x_addr + k * pitch, sx);
                    copy_vector(g_addr + k * pitch, sg);
                    sx += xstep;
                    sg += gstep;
                }
                if (DROP) {
                    if (!P.drop.channel) keep = bits[k * threads + tid];
                    g = keep_lanes<V>(g, keep, P.drop.scale);
                }
                store_lanes<T, V>(dx, grad_result<V, ACT>(P.act, coefs, mk1, mk2, v, g));
            }
            cp_async_commit();
        }
    }
    if (P.part != nullptr)
        for (int c = tid; c < P.cb; c += threads)
            P.part[(static_cast<long long>(unit / P.bundles) * P.cluster + rank) * P.c + bundle * P.cb + c] = acc[c];
    if (P.cluster > 1) cg::this_cluster().sync();
}

}  // namespace gcb
