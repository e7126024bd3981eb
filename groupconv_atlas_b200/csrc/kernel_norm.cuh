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
// Three paths, of which the host takes the one that it estimates to be fastest.
// The resident path (end of this file) reads x, and dy, once: a cluster of CTAs
// holds all pixels of some whole groups of an image in shared memory.  One
// launch forward, two for the gradient.
//
// The split path takes what does not fit: partial results of chunks of pixels
// per channel, one reduction per group, and a second pass over the data.
//
// In both a thread works on vectors of V channels: 16 bytes, or one element
// where a pixel is not a multiple of 16 bytes.
//
// The small path takes many images of few pixels: a few threads hold a whole
// group of an image in registers.
//
// Sums.  An FP32 sum of n values of one sign, added one after the other, is off
// by up to n half steps, and by a third of that where the values are alike (a
// mean's gradient).  Here at most kNormRun values, on the resident path a
// thread's vectors (some 100), are added in a row before sums are joined: by
// trees, by as many runs again, or in 64 bits where there may be thousands of
// them (chunks, images).
#pragma once
#include <cooperative_groups.h>

#include <type_traits>

#include "norm_util.cuh"

namespace gcb {

constexpr int kNormThreads = kStreamThreads;  // split path
constexpr int kResidentThreads = 512;         // resident path, at most

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
    // small path (gb: groups of a block)
    int team;            // threads of a group, a power of two
    int gblocks;         // ceil(groups / gb)
    long long nblocks;   // blocks over the images
    DropParams drop;
};

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

// value(i) for i, i + step, .. below end, added in 32 bits over runs of kNormRun
// and in 64 bits over the runs.  (64-bit additions of each value cost 14 us where
// a group has 290 chunks of 255 channels.)
constexpr int kNormRun = 64;
template <int UNROLL, class I, class F>
__device__ __forceinline__ float long_sum(I i, I end, I step, F value) {
    double total = 0.0;
    while (i < end) {
        const I stop = (end - i) / kNormRun < step ? end : i + kNormRun * step;
        float run = 0.0f;
#pragma unroll UNROLL
        for (; i < stop; i += step) run += value(i);
        total += run;
    }
    return static_cast<float>(total);
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

// ---- sums of a block ---------------------------------------------------------------------
// Where a thread (lane, col) holds a value pair for each of its V channels:
// rows of channel pairs that meet in shared memory, one a warp where a warp
// holds whole pixel lanes (they are added by shuffles first), else one a lane.
__host__ __device__ inline int sum_rows_of(int threads, int vr, int lanes) { return 32 % vr == 0 ? threads / 32 : lanes; }
// Entries of shared memory that channel_sums needs for a block of cb channels.
__host__ __device__ inline size_t channel_sums_space(int threads, int vr, int lanes, int cb) {
    return static_cast<size_t>(sum_rows_of(threads, vr, lanes)) * cb + threads;
}

// Adds s and t over the block's pixel lanes and calls f(c, sums) once for each
// channel c of the block, from some thread.  `scratch` may be reused after the
// next barrier.
template <int V, class F>
__device__ __forceinline__ void channel_sums(int vr, int lanes, int cb, int at, int local, float (&s)[V], float (&t)[V],
                                             float2 *scratch, F f) {
    const int threads = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool warp_rows = 32 % vr == 0;
    const int rows = sum_rows_of(threads, vr, lanes), segs = threads / cb;
    float2 *segsum = scratch, *red = scratch + threads;
    if (at < lanes) {
        if (warp_rows)  // every lane of the block takes part: 32 is a multiple of vr
            for (int o = vr; o < 32; o <<= 1) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
                    t[j] += __shfl_xor_sync(0xffffffffu, t[j], o);
                }
            }
        if (!warp_rows || lane < vr) {
            float2 *out = red + (warp_rows ? warp : at) * cb + local;
#pragma unroll
            for (int j = 0; j < V; ++j) out[j] = make_float2(s[j], t[j]);
        }
    }
    __syncthreads();
    if (segs > 1) {
        const int seg = tid / cb, c = tid - seg * cb;
        float2 sum = make_float2(0.0f, 0.0f);
        if (seg < segs) {
            for (int l = seg; l < rows; l += segs) {
                const float2 v = red[l * cb + c];
                sum.x += v.x;
                sum.y += v.y;
            }
            segsum[tid] = sum;
        }
        __syncthreads();
    }
    const float2 *parts = segs > 1 ? segsum : red;
    const int count = segs > 1 ? min(segs, rows) : rows;
    for (int c = tid; c < cb; c += threads) {
        float2 sum = make_float2(0.0f, 0.0f);
        for (int i = 0; i < count; ++i) {
            const float2 v = parts[i * cb + c];
            sum.x += v.x;
            sum.y += v.y;
        }
        f(c, sum);
    }
}

// ---- split path ----------------------------------------------------------------------------
// A block streams a chunk of pixels of up to 256 vector columns.  Blocks per
// SM: what the rings of shared memory and the registers of the vector kernels
// allow; single elements need more threads to keep as many bytes in flight.
__host__ __device__ constexpr int split_blocks(int v, bool backward) { return v == 1 ? 4 : backward ? 2 : 3; }

struct SplitPlace {
    long long n, p0;  // image, first pixel of the thread
    int chunk, lane, col, count;  // count: vectors of this thread
    int c0;                       // first channel of the thread, 0 where it has none
    int width;                    // channels of this block
    int first;                    // first channel of this block
};
__device__ __forceinline__ SplitPlace split_place(const NormParams &P, int v) {
    SplitPlace s;
    const unsigned item = blockIdx.x;
    const unsigned cb = item % P.cblocks, t = item / P.cblocks;
    s.chunk = t % P.chunks;
    s.n = t / P.chunks;
    s.lane = threadIdx.x / P.vb;
    s.col = threadIdx.x - s.lane * P.vb;
    const int columns = min(P.vb, P.vcols - static_cast<int>(cb) * P.vb);
    s.first = static_cast<int>(cb) * P.vb * v;
    s.width = columns * v;
    const bool active = s.lane < P.lanes && s.col < columns;
    const long long p0 = s.chunk * P.chunk_rows, p1 = min(P.px, p0 + P.chunk_rows);
    s.p0 = p0 + s.lane;
    s.count = active && s.p0 < p1 ? static_cast<int>((p1 - s.p0 + P.lanes - 1) / P.lanes) : 0;
    s.c0 = active ? s.first + s.col * v : 0;
    return s;
}

// Moments of a thread's values of one channel each: sums about a pivot, which
// is the first of at most 64 values.  As one of the values it lies so near the
// mean that the squares about it exceed those about the mean at most by the
// factor 64; cancellation in q - s^2 / n costs no more than that many roundings
// whatever the data's mean.  Runs of 64 are joined as (mean, squares).
template <int V>
struct Moments {
    Lanes<V> minus, s, q;
    float mean[V], m2[V], n = 0.0f;
    __device__ __forceinline__ void start(const Lanes<V> &v) {
#pragma unroll
        for (int i = 0; i < Lanes<V>::kPairs; ++i) {
            minus.p[i] = v.p[i] * pair(-1.0f);
            s.p[i] = q.p[i] = pair(0.0f);
        }
    }
    __device__ __forceinline__ void add(const Lanes<V> &v) {
#pragma unroll
        for (int i = 0; i < Lanes<V>::kPairs; ++i) {
            const f2 d = v.p[i] + minus.p[i];
            s.p[i] = s.p[i] + d;
            q.p[i] = fma2(d, d, q.p[i]);
        }
    }
    // The run's count values become part of (n, mean, m2).
    __device__ __forceinline__ void finish(int count) {
        float first[V], sv[V], qv[V];
        values_of<V>(minus, first);
        values_of<V>(s, sv);
        values_of<V>(q, qv);
        const float k = static_cast<float>(count), inv = 1.0f / k, total = n + k, f = k / total;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float run = fmaf(sv[j], inv, -first[j]);
            float squares = fmaf(-sv[j] * inv, sv[j], qv[j]);
            squares = squares < 0.0f ? 0.0f : squares;  // a NaN stays
            if (n == 0.0f) {
                mean[j] = run;
                m2[j] = squares;
            } else {
                const float d = run - mean[j];
                mean[j] = fmaf(d, f, mean[j]);
                m2[j] += squares + d * d * (n * f);
            }
        }
        n = total;
    }
};

// Per chunk and channel: mean and squares about it.  The threads' moments are
// moved to one pivot per channel, the mean of pixel lane 0, and then add up.
// Bound by the memory once a launch's fixed 7 us are behind (first copies,
// sums across the block, SMs that finish late): N8 C128 256x256 bf16, 134 MB,
// 29 us.
template <class T, int V>
__global__ void __launch_bounds__(kNormThreads, split_blocks(V, false)) norm_moments_kernel(const __grid_constant__ NormParams P) {
    extern __shared__ __align__(16) unsigned char nsm[];
    uint4 *ring = reinterpret_cast<uint4 *>(nsm);
    // the sums' space is the ring's, which is read no more by then
    float *pivot = reinterpret_cast<float *>(nsm);  // [width]
    float2 *scratch = reinterpret_cast<float2 *>(pivot + (P.vb * V + 1) / 2 * 2);
    griddep_wait();
    griddep_launch_dependents();
    const SplitPlace at = split_place(P, V);
    Moments<V> m;
#pragma unroll
    for (int j = 0; j < V; ++j) m.mean[j] = m.m2[j] = 0.0f;
    const T *x = static_cast<const T *>(P.x) + at.n * P.x_ldn + at.p0 * P.x_ldp + at.c0;
    const long long step = static_cast<long long>(P.lanes) * P.x_ldp;
    start_vectors<V>(ring, x, step, at.count);
    for_vectors<T, V>(ring, x, step, at.count, [&](int i, const Lanes<V> &v) {
        if (i % kNormRun == 0) {
            if (i > 0) m.finish(kNormRun);
            m.start(v);
        }
        m.add(v);
    });
    if (at.count > 0) m.finish((at.count - 1) % kNormRun + 1);
    const int local = at.c0 - at.first;
    __syncthreads();
    if (at.lane == 0 && at.count > 0) {
#pragma unroll
        for (int j = 0; j < V; ++j) pivot[local + j] = m.mean[j];
    }
    __syncthreads();
    const bool any = at.count > 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float e = any ? m.mean[j] - pivot[local + j] : 0.0f, ne = m.n * e;
        m.mean[j] = ne;
        m.m2[j] = any ? fmaf(ne, e, m.m2[j]) : 0.0f;
    }
    float2 *out = P.part + (at.n * P.chunks + at.chunk) * P.c + at.first;
    const float rows = static_cast<float>(min(P.chunk_rows, P.px - at.chunk * P.chunk_rows));
    channel_sums<V>(P.vb, P.lanes, P.vb * V, at.lane, at.lane < P.lanes ? at.col * V : 0, m.mean, m.m2, scratch, [&](int c, float2 sum) {
        const float d = sum.x / rows;
        if (c < at.width) out[c] = make_float2(pivot[c] + d, fmaf(-d, sum.x, sum.y));
    });
}

// Joins a group's chunks and channels: a team of TEAM threads (a warp, or the
// block) per (image, group).
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float *red) {
    if constexpr (TEAM == 32) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    } else {
        return block_sum(v, red);
    }
}

template <int TEAM>
__global__ void __launch_bounds__(kNormThreads) norm_finalize_kernel(const __grid_constant__ NormParams P) {
    constexpr int kHeld = 8;  // entries a thread holds on to for the second pass
    __shared__ float red[32];
    griddep_wait();
    griddep_launch_dependents();
    const float total = static_cast<float>(P.px) * static_cast<float>(P.cpg);
    const unsigned entries = static_cast<unsigned>(P.chunks) * P.cpg;
    const int me = threadIdx.x % TEAM;
    const long long teams = static_cast<long long>(gridDim.x) * (kNormThreads / TEAM);
    for (long long ng = (static_cast<long long>(blockIdx.x) * kNormThreads + threadIdx.x) / TEAM; ng < P.n * P.groups;
         ng += teams) {
        const long long n = ng / P.groups;
        const float2 *part = P.part + n * P.chunks * P.c + (ng - n * P.groups) * P.cpg;
        auto entry = [&](unsigned i, float &rows) {
            const unsigned chunk = i / P.cpg;
            rows = static_cast<float>(min(P.chunk_rows, P.px - chunk * P.chunk_rows));
            return part[static_cast<long long>(chunk) * P.c + (i - chunk * P.cpg)];
        };
        float2 held[kHeld];
        float held_rows[kHeld], s = 0.0f, q = 0.0f;
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            const unsigned i = me + u * TEAM;
            held[u] = make_float2(0.0f, 0.0f);
            held_rows[u] = 0.0f;
            if (i < entries) held[u] = entry(i, held_rows[u]);
        }
#pragma unroll
        for (int u = 0; u < kHeld; ++u) s = fmaf(held_rows[u], held[u].x, s);
        const unsigned rest = me + kHeld * TEAM;
        s += long_sum<4, unsigned>(rest, entries, TEAM, [&](unsigned i) {
            float rows;
            const float2 v = entry(i, rows);
            return rows * v.x;
        });
        const float mean = team_sum<TEAM>(s, red) / total;
#pragma unroll
        for (int u = 0; u < kHeld; ++u) {
            const float d = held[u].x - mean;
            if (held_rows[u] > 0.0f) q += fmaf(held_rows[u] * d, d, held[u].y);
        }
        q += long_sum<4, unsigned>(rest, entries, TEAM, [&](unsigned i) {
            float rows;
            const float2 v = entry(i, rows);
            const float d = v.x - mean;
            return fmaf(rows * d, d, v.y);
        });
        const float var = team_sum<TEAM>(q, red) / total;
        if (me == 0) P.stats[ng] = make_float2(mean, 1.0f / sqrtf(var + P.eps));
    }
}

// gamma and beta of a thread's channels.
template <int V>
struct Affine {
    float gamma[V], beta[V];
    __device__ __forceinline__ Affine(const NormParams &P, int c0) {
        load_params<V>(P.gamma, P.gamma_type, c0, 1.0f, gamma);
        load_params<V>(P.beta, P.beta_type, c0, 0.0f, beta);
    }
};
template <int V>
__device__ __forceinline__ Coefs<V> split_coefs(const NormParams &P, const Affine<V> &affine, long long n, int c0) {
    float mean[V], a[V];
    const float2 *stats = P.stats + n * P.groups;
    int g = c0 / P.cpg, at = c0 - g * P.cpg;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 st = stats[g];
        mean[j] = -st.x;
        a[j] = st.y * affine.gamma[j];
        if (++at == P.cpg) at = 0, g = min(g + 1, P.groups - 1);
    }
    return {lanes_of<V>(mean), lanes_of<V>(a), lanes_of<V>(affine.beta)};
}

// Dropout of a thread's vectors, pixel by pixel.
template <int V, bool DROP>
struct Keeper {
    Philox gen;
    Draws<V> draws;
    uint64_t at, step;
    __device__ __forceinline__ Keeper(const NormParams &P, bool writer, long long n, long long p0, int c0, int lanes) {
        if (!DROP) return;
        gen = Philox(P.drop, writer);
        at = (static_cast<uint64_t>(n) * P.px + p0) * P.c + c0;
        step = static_cast<uint64_t>(static_cast<long long>(lanes) * P.c);  // modulo 2^64 where it goes down
        if (P.drop.channel) draws = Draws<V>(gen, static_cast<uint64_t>(n) * P.c + c0);
    }
    __device__ __forceinline__ Lanes<V> apply(const NormParams &P, const Lanes<V> &v) {
        if (!DROP) return v;
        if (!P.drop.channel) draws = Draws<V>(gen, at);
        at += step;
        return drop_lanes<V>(v, draws, P.drop);
    }
};

// Normalises, activates and drops out: the second pass over x, from a chunk's
// end to its start, because the first pass left the ends in the L2 cache.  x
// is not written by the launches that this one follows, so its first copies
// are issued before the wait for their results.  N8 C128 256x256 bf16 with
// SiLU: 268 MB read and written in 42 us (6.4 TB/s).
template <class T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(kNormThreads, split_blocks(V, false)) norm_apply_kernel(const __grid_constant__ NormParams P) {
    extern __shared__ __align__(16) unsigned char nsm[];
    uint4 *ring = reinterpret_cast<uint4 *>(nsm);
    const SplitPlace at = split_place(P, V);
    const long long last = at.p0 + static_cast<long long>(max(0, at.count - 1)) * P.lanes;
    const T *x = static_cast<const T *>(P.x) + at.n * P.x_ldn + last * P.x_ldp + at.c0;
    const long long xstep = -static_cast<long long>(P.lanes) * P.x_ldp, ystep = -static_cast<long long>(P.lanes) * P.y_ldp;
    start_vectors<V>(ring, x, xstep, at.count);
    const Affine<V> affine(P, at.c0);
    griddep_wait();
    griddep_launch_dependents();
    Keeper<V, DROP> drop(P, blockIdx.x == 0 && threadIdx.x == 0, at.n, last, at.c0, -P.lanes);
    if (at.count == 0) return;
    const Coefs<V> coefs = split_coefs<V>(P, affine, at.n, at.c0);
    T *y = static_cast<T *>(P.y) + at.n * P.y_ldn + last * P.y_ldp + at.c0;
    for_vectors<T, V>(ring, x, xstep, at.count, [&](int, Lanes<V> v) {
#pragma unroll
        for (int i = 0; i < Lanes<V>::kPairs; ++i) {
            f2 d;
            v.p[i] = activate<ACT>(P.act, normalise<V>(coefs, i, v.p[i], d));
        }
        store_lanes<T, V>(y, drop.apply(P, v));
        y += ystep;
    });
}

// ---- split path, gradient ----------------------------------------------------------------
// dz = drop(g act'(z)), and x - mean.  The slope comes before the mask, so that
// a dropped place is 0 whatever it is (NaN where z is infinite).
template <int V, int ACT, class F>
__device__ __forceinline__ Lanes<V> grad_inner(int act, const Coefs<V> &k, const Lanes<V> &v, const Lanes<V> &g, Lanes<V> &d,
                                               F drop) {
    Lanes<V> dz;
#pragma unroll
    for (int i = 0; i < Lanes<V>::kPairs; ++i) {
        const f2 z = normalise<V>(k, i, v.p[i], d.p[i]);
        dz.p[i] = activate_grad<ACT>(act, z, g.p[i]);
    }
    return drop(dz);
}
template <int V, int ACT, class F>
__device__ __forceinline__ void grad_sums(int act, const Coefs<V> &k, const Lanes<V> &v, const Lanes<V> &g, Lanes<V> &s,
                                          Lanes<V> &t, F drop) {
    Lanes<V> d;
    const Lanes<V> dz = grad_inner<V, ACT>(act, k, v, g, d, drop);
#pragma unroll
    for (int i = 0; i < Lanes<V>::kPairs; ++i) {
        s.p[i] = s.p[i] + dz.p[i];
        t.p[i] = fma2(dz.p[i], d.p[i], t.p[i]);
    }
}
// a dz - k1 - k2 (x - mean), with k1 and k2 given negated
template <int V, int ACT, class F>
__device__ __forceinline__ Lanes<V> grad_result(int act, const Coefs<V> &k, const Lanes<V> &minus_k1,
                                                const Lanes<V> &minus_k2, const Lanes<V> &v, const Lanes<V> &g, F drop) {
    Lanes<V> d, r = grad_inner<V, ACT>(act, k, v, g, d, drop);
#pragma unroll
    for (int i = 0; i < Lanes<V>::kPairs; ++i)
        r.p[i] = fma2(k.a.p[i], r.p[i], fma2(d.p[i], minus_k2.p[i], minus_k1.p[i]));
    return r;
}

// Per chunk and channel: sum dz, sum dz (x - mean).  N8 C128 256x256 bf16 with
// SiLU: 268 MB in 47 us (5.7 TB/s).
template <class T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(kNormThreads, DROP ? 2 : split_blocks(V, true)) norm_grad_sums_kernel(const __grid_constant__ NormParams P) {
    extern __shared__ __align__(16) unsigned char nsm[];
    griddep_wait();
    griddep_launch_dependents();
    const SplitPlace at = split_place(P, V);
    uint4 *ring = reinterpret_cast<uint4 *>(nsm);
    const T *x = static_cast<const T *>(P.x) + at.n * P.x_ldn + at.p0 * P.x_ldp + at.c0;
    const T *dy = static_cast<const T *>(P.dy) + at.n * P.dy_ldn + at.p0 * P.dy_ldp + at.c0;
    const long long xstep = static_cast<long long>(P.lanes) * P.x_ldp, gstep = static_cast<long long>(P.lanes) * P.dy_ldp;
    start_vector_pairs<V>(ring, x, xstep, dy, gstep, at.count);
    const Affine<V> affine(P, at.c0);
    Keeper<V, DROP> drop(P, false, at.n, at.p0, at.c0, P.lanes);
    const Coefs<V> coefs = split_coefs<V>(P, affine, at.n, at.c0);
    Lanes<V> s2, t2, all_s, all_t;  // of a run, of the runs
#pragma unroll
    for (int i = 0; i < Lanes<V>::kPairs; ++i) s2.p[i] = t2.p[i] = all_s.p[i] = all_t.p[i] = pair(0.0f);
    auto join = [&] {
#pragma unroll
        for (int i = 0; i < Lanes<V>::kPairs; ++i) {
            all_s.p[i] = all_s.p[i] + s2.p[i];
            all_t.p[i] = all_t.p[i] + t2.p[i];
            s2.p[i] = t2.p[i] = pair(0.0f);
        }
    };
    for_vector_pairs<T, V, kNormRun>(
        ring, x, xstep, dy, gstep, at.count,
        [&](int, const Lanes<V> &v, const Lanes<V> &g) {
            grad_sums<V, ACT>(P.act, coefs, v, g, s2, t2, [&](const Lanes<V> &dz) { return drop.apply(P, dz); });
        },
        join);
    float s[V], t[V];
    values_of<V>(all_s, s);
    values_of<V>(all_t, t);
    float2 *out = P.part + (at.n * P.chunks + at.chunk) * P.c + at.first;
    __syncthreads();  // the sums' space is the ring's
    channel_sums<V>(P.vb, P.lanes, P.vb * V, at.lane, at.lane < P.lanes ? at.col * V : 0, s, t,
                    reinterpret_cast<float2 *>(nsm), [&](int c, float2 sum) {
                        if (c < at.width) out[c] = sum;
                    });
}

// Per (image, channel): the sums over all chunks; then per group k1 and k2.  A
// team per group: channel by channel, its lanes over the chunks.
template <int TEAM>
__global__ void __launch_bounds__(kNormThreads) norm_grad_finalize_kernel(const __grid_constant__ NormParams P) {
    __shared__ float red[32];
    griddep_wait();
    griddep_launch_dependents();
    const float total = static_cast<float>(P.px) * static_cast<float>(P.cpg);
    const int lane = threadIdx.x & 31, warp = threadIdx.x % TEAM / 32;
    const long long teams = static_cast<long long>(gridDim.x) * (kNormThreads / TEAM);
    for (long long ng = (static_cast<long long>(blockIdx.x) * kNormThreads + threadIdx.x) / TEAM; ng < P.n * P.groups;
         ng += teams) {
        const long long n = ng / P.groups;
        const int c0 = static_cast<int>(ng - n * P.groups) * P.cpg;
        const float2 st = P.stats[ng];
        float s1 = 0.0f, s2 = 0.0f, run1 = 0.0f, run2 = 0.0f;
        int in_run = 0;
        // four channels at a time, so that their loads are in flight together
        for (int k = 4 * warp; k < P.cpg; k += 4 * (TEAM / 32)) {
            const float2 *part = P.part + n * P.chunks * P.c + c0 + k;
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f}, t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
            for (int i = lane; i < P.chunks; i += 32) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (k + j < P.cpg) {
                        const float2 v = part[static_cast<long long>(i) * P.c + j];
                        s[j] += v.x;
                        t[j] += v.y;
                    }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
                    t[j] += __shfl_xor_sync(0xffffffffu, t[j], o);
                }
                if (lane == j && k + j < P.cpg) {
                    const float w = t[j] * st.y;
                    const float gm = P.gamma ? load_param(P.gamma, P.gamma_type, c0 + k + j) : 1.0f;
                    P.chan[n * P.c + c0 + k + j] = make_float2(s[j], w);
                    run1 = fmaf(gm, s[j], run1);
                    run2 = fmaf(gm, w, run2);
                }
            }
            if (++in_run == kNormRun) {
                s1 += run1;
                s2 += run2;
                run1 = run2 = 0.0f;
                in_run = 0;
            }
        }
        s1 = team_sum<TEAM>(s1 + run1, red);
        s2 = team_sum<TEAM>(s2 + run2, red);
        if (threadIdx.x % TEAM == 0) P.gsum[ng] = make_float2(st.y * s1 / total, st.y * st.y * s2 / total);
    }
}

// The second pass over x and dy, like norm_apply_kernel.  The same shape: 403 MB
// in 63 us (6.4 TB/s); with dropout the generator's products bound both.
template <class T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(kNormThreads, DROP ? 2 : split_blocks(V, true)) norm_grad_apply_kernel(const __grid_constant__ NormParams P) {
    extern __shared__ __align__(16) unsigned char nsm[];
    uint4 *ring = reinterpret_cast<uint4 *>(nsm);
    const SplitPlace at = split_place(P, V);
    const long long last = at.p0 + static_cast<long long>(max(0, at.count - 1)) * P.lanes;
    const T *x = static_cast<const T *>(P.x) + at.n * P.x_ldn + last * P.x_ldp + at.c0;
    const T *dy = static_cast<const T *>(P.dy) + at.n * P.dy_ldn + last * P.dy_ldp + at.c0;
    const long long down = -static_cast<long long>(P.lanes), xstep = down * P.x_ldp, gstep = down * P.dy_ldp;
    start_vector_pairs<V>(ring, x, xstep, dy, gstep, at.count);
    const Affine<V> affine(P, at.c0);
    griddep_wait();
    griddep_launch_dependents();
    Keeper<V, DROP> drop(P, blockIdx.x == 0 && threadIdx.x == 0, at.n, last, at.c0, -P.lanes);
    if (at.count == 0) return;
    const Coefs<V> coefs = split_coefs<V>(P, affine, at.n, at.c0);
    Lanes<V> mk1, mk2;
    {
        float k1[V], k2[V];
        const float2 *sums = P.gsum + at.n * P.groups;
        int g = at.c0 / P.cpg, in = at.c0 - g * P.cpg;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 k = sums[g];
            k1[j] = -k.x;
            k2[j] = -k.y;
            if (++in == P.cpg) in = 0, g = min(g + 1, P.groups - 1);
        }
        mk1 = lanes_of<V>(k1);
        mk2 = lanes_of<V>(k2);
    }
    T *dx = static_cast<T *>(P.y) + at.n * P.y_ldn + last * P.y_ldp + at.c0;
    const long long ystep = down * P.y_ldp;
    for_vector_pairs<T, V>(ring, x, xstep, dy, gstep, at.count, [&](int, const Lanes<V> &v, const Lanes<V> &g) {
        store_lanes<T, V>(dx, grad_result<V, ACT>(P.act, coefs, mk1, mk2, v, g,
                                                  [&](const Lanes<V> &dz) { return drop.apply(P, dz); }));
        dx += ystep;
    });
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
    if (c < P.c && row < P.sum_rows) {
        double sum_s = 0.0, sum_t = 0.0;
        const float2 *src = P.chan + static_cast<long long>(row) * P.c + c;
        const long long step = static_cast<long long>(kNormThreads / 32) * P.c;
        for (long long left = (P.sum_rows - row + kNormThreads / 32 - 1) / (kNormThreads / 32); left > 0; left -= kNormRun) {
            const int run = static_cast<int>(min(left, static_cast<long long>(kNormRun)));
            s = t = 0.0f;
#pragma unroll 8
            for (int u = 0; u < run; ++u, src += step) {
                const float2 v = *src;
                s += v.x;
                t += v.y;
            }
            sum_s += s;
            sum_t += t;
        }
        s = static_cast<float>(sum_s);
        t = static_cast<float>(sum_t);
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
//
// Measured (forward, SiLU): N32 C256 56x56 bf16 27 us, of which 4.4 us are the
// first load at the memory's rate, 2 x 4 us first pass and sums, 7 us a second
// pass that stores and loads (memory) and 6.6 us one that only stores (issue
// slots and special functions); the tensor is 1.7 times what the SMs hold.
// N16 C256 14x14 FP32 4.8 us, N1 C32 56x56 FP32 4.5 us (latencies: a load, two
// block barriers, one cluster barrier, a store).  Gradient of N32 C256 28x28
// bf16 19 us: load 4.7, first pass 3.4, sums 2.2, second pass 4.1, the launch
// that adds up the parameters' gradients 3.

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

// Bytes of iters slots per thread, rounded up for what follows.
__host__ __device__ inline size_t tile_bytes(int iters, int threads, int slot) {
    return (static_cast<size_t>(iters) * threads * slot + 15) / 16 * 16;
}
// Shared memory of the resident kernels behind the tiles.
__host__ __device__ inline size_t resident_extra(const NormParams &P, int threads, bool grad) {
    const size_t gb = P.gb, cb = P.cb;
    const size_t entries = grad ? channel_sums_space(threads, P.vr, P.lanes, P.cb) + 3 * cb
                                : static_cast<size_t>(P.lanes) * P.vr * P.sub;
    return (entries + 4 * gb) * sizeof(float2);
}

// A thread's place in a tile: a 16-byte vector, or one element (V = 1, for
// tensors whose pixels are not multiples of 16 bytes; 16-bit elements have no
// asynchronous copy and pass through a register).
template <class T, int V>
using Slot = typename std::conditional<V == 1, T, uint4>::type;
template <class T, int V>
__device__ __forceinline__ void copy_slot(Slot<T, V> *dst, uint32_t addr, const T *src) {
    if constexpr (V > 1) copy_vector(addr, src);
    else if constexpr (sizeof(T) == 4) cp_async_4(dst, src, true);
    else *dst = *src;
}
template <class T, int V>
__device__ __forceinline__ Lanes<V> read_slot(const Slot<T, V> &s) {
    if constexpr (V > 1) {
        return unpack_lanes<T, V>(s, static_cast<const T *>(nullptr));
    } else {
        const float v[1] = {to_float(s)};
        return lanes_of<1>(v);
    }
}

template <class T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(kResidentThreads, 1) norm_resident_kernel(const __grid_constant__ NormParams P) {
    constexpr int kPairs = Lanes<V>::kPairs;
    extern __shared__ __align__(16) unsigned char nsm[];
    const int threads = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
    Slot<T, V> *tile = reinterpret_cast<Slot<T, V> *>(nsm);
    float2 *exch = reinterpret_cast<float2 *>(nsm + tile_bytes(P.iters, threads, sizeof(Slot<T, V>)));  // [2][gb]
    float2 *fin = exch + 2 * P.gb;
    float *pivot = reinterpret_cast<float *>(fin + P.gb);
    float2 *red = fin + 2 * P.gb;  // [lanes][vr][sub]
    const int rank = blockIdx.x % P.cluster;
    const unsigned unit = blockIdx.x / P.cluster;
    const int bundle = unit % P.bundles;
    const Resident r = resident_place(P, rank, bundle, V);
    Slot<T, V> *tile_at = tile + tid;
    const uint32_t tile_addr = smem_addr(tile_at), pitch = sizeof(Slot<T, V>) * threads;
    griddep_wait();
    griddep_launch_dependents();
    Philox gen;
    if (DROP) gen = Philox(P.drop, blockIdx.x == 0 && tid == 0);
    const long long xstep = static_cast<long long>(P.lanes) * P.x_ldp, ystep = static_cast<long long>(P.lanes) * P.y_ldp;
    const T *x = static_cast<const T *>(P.x) + (unit / P.bundles) * P.x_ldn + r.p0 * P.x_ldp + r.c0;
    {
        const T *src = x;
        int k = 0;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            const int to = part_end(P.iters, r.count, part);
#pragma unroll 4
            for (; k < to; ++k, src += xstep) copy_slot<T, V>(tile_at + k * threads, tile_addr + k * pitch, src);
            cp_async_commit();
        }
    }
    const Affine<V> affine(P, r.c0);
    Coefs<V> coefs;
    coefs.b = lanes_of<V>(affine.beta);
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
                const Lanes<V> v = read_slot<T, V>(tile_at[0]);
#pragma unroll
                for (int i = 0; i < kPairs; ++i) minus.p[i] = v.p[i] * pair(-1.0f);
            }
            const int to = part_end(P.iters, r.count, part);
#pragma unroll 4
            for (; k < to; ++k) {
                const Lanes<V> v = read_slot<T, V>(tile_at[k * threads]);
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
                a[j] = st.y * affine.gamma[j];
            });
            coefs.minus_mean = lanes_of<V>(mean);
            coefs.a = lanes_of<V>(a);
        }
        T *y = static_cast<T *>(P.y) + n * P.y_ldn + r.p0 * P.y_ldp + r.c0;
        Draws<V> draws;
        if (DROP && P.drop.channel) draws = Draws<V>(gen, static_cast<uint64_t>(n) * P.c + r.c0);
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
                Lanes<V> v = read_slot<T, V>(tile_at[k * threads]);
                if (more) {
                    copy_slot<T, V>(tile_at + k * threads, tile_addr + k * pitch, src);
                    src += xstep;
                }
#pragma unroll
                for (int i = 0; i < kPairs; ++i) {
                    f2 d;
                    v.p[i] = activate<ACT>(P.act, normalise<V>(coefs, i, v.p[i], d));
                }
                if (DROP) {
                    if (!P.drop.channel) draws = Draws<V>(gen, at);
                    at += static_cast<uint64_t>(P.lanes) * P.c;
                    v = drop_lanes<V>(v, draws, P.drop);
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
template <class T, int V, int ACT, bool DROP>
__global__ void __launch_bounds__(kResidentThreads, 1) norm_resident_grad_kernel(const __grid_constant__ NormParams P) {
    extern __shared__ __align__(16) unsigned char nsm[];
    const int threads = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
    const size_t tiles = static_cast<size_t>(P.iters) * threads;
    Slot<T, V> *tx = reinterpret_cast<Slot<T, V> *>(nsm);
    float2 *exch = reinterpret_cast<float2 *>(nsm + tile_bytes(2 * P.iters, threads, sizeof(Slot<T, V>)));  // [2][gb]
    float2 *fin = exch + 2 * P.gb;
    float2 *gst = fin + P.gb;           // mean, rstd of the unit's groups
    float2 *weighted = gst + P.gb;      // [cb]: gamma * the channel's sums
    double *acc = reinterpret_cast<double *>(weighted + P.cb);  // [2][cb]: the channel's sums over this CTA's images
    float2 *scratch = weighted + 3 * P.cb;                      // channel_sums
    uint8_t *bits = reinterpret_cast<uint8_t *>(scratch + channel_sums_space(threads, P.vr, P.lanes, P.cb));
    const int rank = blockIdx.x % P.cluster;
    const unsigned unit = blockIdx.x / P.cluster;
    const int bundle = unit % P.bundles;
    const Resident r = resident_place(P, rank, bundle, V);
    Slot<T, V> *x_at = tx + tid, *g_at = x_at + tiles;
    const uint32_t x_addr = smem_addr(x_at), g_addr = smem_addr(g_at), pitch = sizeof(Slot<T, V>) * threads;
    griddep_wait();
    griddep_launch_dependents();
    Philox gen;
    if (DROP) gen = Philox(P.drop, blockIdx.x == 0 && tid == 0);
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
                copy_slot<T, V>(x_at + k * threads, x_addr + k * pitch, sx);
                copy_slot<T, V>(g_at + k * threads, g_addr + k * pitch, sg);
            }
            cp_async_commit();
        }
    }
    for (int c = tid; c < P.cb; c += threads) acc[c] = acc[P.cb + c] = 0.0;
    for (int g = tid; g < P.gb; g += threads) gst[g] = P.stats[(unit / P.bundles) * P.groups + bundle * P.gb + g];
    const Affine<V> affine(P, r.c0);
    Coefs<V> coefs;
    coefs.b = lanes_of<V>(affine.beta);
    const float total = static_cast<float>(P.px) * static_cast<float>(P.cpg);
    int turn = 0;
    for (long long n = unit / P.bundles; n < P.n; n += P.stride, turn ^= 1) {
        __syncthreads();  // gst
        {
            float mean[V], a[V];
            for_channels<V>(P, r, [&](int j, int g) {
                const float2 st = gst[g];
                mean[j] = -st.x;
                a[j] = st.y * affine.gamma[j];
            });
            coefs.minus_mean = lanes_of<V>(mean);
            coefs.a = lanes_of<V>(a);
        }
        Lanes<V> s2, t2;
#pragma unroll
        for (int i = 0; i < Lanes<V>::kPairs; ++i) s2.p[i] = t2.p[i] = pair(0.0f);
        uint32_t keep = ~0u;
        auto drop = [&](const Lanes<V> &dz) { return DROP ? drop_lanes<V>(dz, keep, P.drop) : dz; };
        if (DROP && P.drop.channel) keep = Draws<V>(gen, static_cast<uint64_t>(n) * P.c + r.c0).bits(P.drop.limit);
        uint64_t at = (static_cast<uint64_t>(n) * P.px + r.p0) * P.c + r.c0;
        int k = 0;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            wait_part(part);
            const int to = part_end(P.iters, r.count, part);
#pragma unroll 2
            for (; k < to; ++k) {
                const Lanes<V> v = read_slot<T, V>(x_at[k * threads]), g = read_slot<T, V>(g_at[k * threads]);
                if (DROP) {
                    if (!P.drop.channel) {
                        keep = Draws<V>(gen, at).bits(P.drop.limit);
                        bits[k * threads + tid] = static_cast<uint8_t>(keep);
                    }
                    at += static_cast<uint64_t>(P.lanes) * P.c;
                }
                grad_sums<V, ACT>(P.act, coefs, v, g, s2, t2, drop);
            }
        }
        // channel sums over the CTA's pixels
        {
            float s[V], t[V];
            values_of<V>(s2, s);
            values_of<V>(t2, t);
            channel_sums<V>(P.vr, P.lanes, P.cb, r.lane, r.local, s, t, scratch, [&](int c, float2 sum) {
                sum.y *= gst[c / P.cpg].y;
                const float w = P.gamma ? load_param(P.gamma, P.gamma_type, bundle * P.cb + c) : 1.0f;
                weighted[c] = make_float2(w * sum.x, w * sum.y);
                acc[c] += sum.x;
                acc[P.cb + c] += sum.y;
            });
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
                const Lanes<V> v = read_slot<T, V>(x_at[k * threads]), g = read_slot<T, V>(g_at[k * threads]);
                if (more) {
                    copy_slot<T, V>(x_at + k * threads, x_addr + k * pitch, sx);
                    copy_slot<T, V>(g_at + k * threads, g_addr + k * pitch, sg);
                    sx += xstep;
                    sg += gstep;
                }
                if (DROP && !P.drop.channel) keep = bits[k * threads + tid];
                store_lanes<T, V>(dx, grad_result<V, ACT>(P.act, coefs, mk1, mk2, v, g, drop));
            }
            cp_async_commit();
        }
    }
    if (P.part != nullptr)
        for (int c = tid; c < P.cb; c += threads)
            P.part[(static_cast<long long>(unit / P.bundles) * P.cluster + rank) * P.c + bundle * P.cb + c] =
                make_float2(static_cast<float>(acc[c]), static_cast<float>(acc[P.cb + c]));
    if (P.cluster > 1) cg::this_cluster().sync();
}

// ---- small path -----------------------------------------------------------------------------
// Groups of at most 32 E elements: a team of P.team threads of a warp holds a
// group of one image in registers, E elements a thread, and exchanges sums by
// shuffles.  A block takes gb neighbouring groups of as many images as it has
// teams for, and goes on to other images with the same channels, so that the
// parameters' gradients add up in registers.  Neighbouring threads take
// neighbouring channels, one element an access, which keeps few bytes in flight
// and bounds the kernel.  65536 rows of 64 channels in 8 groups, FP32 with SiLU:
// 21 us, gradient 50 us (by the call 18 us forward against 770 on the resident
// path, where a cluster needs a round of barriers for each few rows); 1000000
// rows of 16: 71 us (128 MB, 1.8 TB/s), gradient 132 us.
template <class T, int E, bool GRAD>
__global__ void __launch_bounds__(kNormThreads) norm_small_kernel(const __grid_constant__ NormParams P) {
    __shared__ float2 sm[GRAD ? kNormThreads * E : 1];
    griddep_wait();
    griddep_launch_dependents();
    const bool drop = P.drop.threshold != 0;
    Philox gen;
    if (drop) gen = Philox(P.drop, blockIdx.x == 0 && threadIdx.x == 0);
    const int team = threadIdx.x / P.team, t = threadIdx.x % P.team, images = kNormThreads / P.team / P.gb;
    const int gl = team % P.gb, il = team / P.gb;
    const unsigned gblock = blockIdx.x % P.gblocks, nblock = blockIdx.x / P.gblocks;
    const int g = static_cast<int>(gblock) * P.gb + gl, elements = static_cast<int>(P.px) * P.cpg;
    const bool active = il < images && g < P.groups;
    const float total = static_cast<float>(elements);
    int p[E], c[E];  // pixel and channel of an element; channel -1: none
    float gm[E], bt[E], sum_s[E], sum_t[E];
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int i = t + k * P.team;
        p[k] = i / P.cpg;
        c[k] = active && i < elements ? g * P.cpg + (i - p[k] * P.cpg) : -1;
        gm[k] = P.gamma != nullptr && c[k] >= 0 ? load_param(P.gamma, P.gamma_type, c[k]) : 1.0f;
        bt[k] = P.beta != nullptr && c[k] >= 0 ? load_param(P.beta, P.beta_type, c[k]) : 0.0f;
        sum_s[k] = sum_t[k] = 0.0f;
    }
    auto team_total = [&](float v) {
        for (int o = P.team / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    auto one = [](f2 v) {
        float a, b;
        split(v, a, b);
        return a;
    };
    // every thread of the block makes the same turns: the shuffles need whole warps
    for (long long base = nblock * static_cast<long long>(images); base < P.n; base += P.nblocks * images) {
        const long long n = base + il;
        const bool here = n < P.n;
        const T *x = static_cast<const T *>(P.x) + n * P.x_ldn;
        float v[E], f[E];  // f: dropout's factor
#pragma unroll
        for (int k = 0; k < E; ++k) v[k] = here && c[k] >= 0 ? to_float(x[p[k] * P.x_ldp + c[k]]) : 0.0f;
        bool keep[E];
#pragma unroll
        for (int k = 0; k < E; ++k) {
            keep[k] = true;
            f[k] = 1.0f;
            if (drop && c[k] >= 0) {
                const uint64_t row = static_cast<uint64_t>(n) * (P.drop.channel ? 1 : P.px) + (P.drop.channel ? 0 : p[k]);
                keep[k] = Draws<1>(gen, row * P.c + c[k]).keep(0, P.drop.limit);
                f[k] = P.drop.scale;
            }
        }
        T *y = static_cast<T *>(P.y) + n * P.y_ldn;
        if constexpr (!GRAD) {
            float s = 0.0f, q = 0.0f;
#pragma unroll
            for (int k = 0; k < E; ++k) s += v[k];
            const float mean = team_total(s) / total;
#pragma unroll
            for (int k = 0; k < E; ++k)
                if (c[k] >= 0) q = fmaf(v[k] - mean, v[k] - mean, q);
            const float rstd = 1.0f / sqrtf(team_total(q) / total + P.eps);
            if (here && active && t == 0 && P.stats != nullptr) P.stats[n * P.groups + g] = make_float2(mean, rstd);
#pragma unroll
            for (int k = 0; k < E; ++k)
                if (here && c[k] >= 0) {
                    const float z = fmaf(v[k] - mean, rstd * gm[k], bt[k]);
                    const float a = one(activate<-1>(P.act, pair(z, 0.0f)));
                    y[p[k] * P.y_ldp + c[k]] = from_float<T>(keep[k] ? a * f[k] : 0.0f);
                }
        } else {
            const T *dy = static_cast<const T *>(P.dy) + n * P.dy_ldn;
            const float2 st = here && active ? P.stats[n * P.groups + g] : make_float2(0.0f, 0.0f);
            float dz[E], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
            for (int k = 0; k < E; ++k) {
                dz[k] = 0.0f;
                if (here && c[k] >= 0) {
                    const float d = v[k] - st.x, up = to_float(dy[p[k] * P.dy_ldp + c[k]]);
                    const float z = fmaf(d, st.y * gm[k], bt[k]);
                    dz[k] = one(activate_grad<-1>(P.act, pair(z, 0.0f), pair(up * f[k], 0.0f)));
                    if (!keep[k]) dz[k] = 0.0f;
                    s1 = fmaf(gm[k], dz[k], s1);
                    s2 = fmaf(gm[k] * dz[k], d, s2);
                    sum_s[k] += dz[k];
                    sum_t[k] = fmaf(dz[k], d * st.y, sum_t[k]);
                }
            }
            const float k1 = st.y * team_total(s1) / total, k2 = st.y * st.y * (st.y * team_total(s2)) / total;
#pragma unroll
            for (int k = 0; k < E; ++k)
                if (here && c[k] >= 0) {
                    const float d = v[k] - st.x;
                    y[p[k] * P.y_ldp + c[k]] = from_float<T>(fmaf(st.y * gm[k], dz[k], -fmaf(d, k2, k1)));
                }
        }
    }
    if constexpr (GRAD) {
        if (P.part == nullptr) return;
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (c[k] >= 0) sm[team * elements + t + k * P.team] = make_float2(sum_s[k], sum_t[k]);
        __syncthreads();
        // images, then pixels, folded by halves
        const int block = P.gb * elements;
        for (int left = images; left > 1;) {
            const int half = (left + 1) / 2;
            for (int i = threadIdx.x; i < (left - half) * block; i += kNormThreads) {
                sm[i].x += sm[i + half * block].x;
                sm[i].y += sm[i + half * block].y;
            }
            left = half;
            __syncthreads();
        }
        for (int left = static_cast<int>(P.px); left > 1;) {
            const int half = (left + 1) / 2, each = (left - half) * P.cpg;
            for (int i = threadIdx.x; i < P.gb * each; i += kNormThreads) {
                const int at = i / each * elements + i % each;
                sm[at].x += sm[at + half * P.cpg].x;
                sm[at].y += sm[at + half * P.cpg].y;
            }
            left = half;
            __syncthreads();
        }
        for (int i = threadIdx.x; i < P.gb * P.cpg; i += kNormThreads) {
            const int gi = i / P.cpg, ci = i - gi * P.cpg, group = static_cast<int>(gblock) * P.gb + gi;
            if (group >= P.groups) break;
            P.part[static_cast<long long>(nblock) * P.c + group * P.cpg + ci] = sm[gi * elements + ci];
        }
    }
}

}  // namespace gcb
