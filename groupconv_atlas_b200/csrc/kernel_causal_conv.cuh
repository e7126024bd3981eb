// Causal depthwise convolution along sequences of tokens (channels innermost),
// its gradient, and its form for one new token of every sequence.
//
//   v[t] = bias + sum_k w[k] u[t + k],  u = the K - 1 inputs before the sequence, then x
//   y[t] = act(v[t]);  g[t] = dy[t] act'(v[t])
//   dx[s] = sum_k w[k] g[s + K - 1 - k],  dw[k] = sum_t g[t] u[t + k],  dbias = sum_t g[t]
//
// Bound by memory: a thread walks along some tokens of a few channels with the
// window of its last inputs in registers, so each input is read once (but for
// the window in front of each thread's stretch, which its neighbour's reads have
// brought into the caches).  The kernels hold KT taps, K or more; what a missing
// tap would multiply is left out, not multiplied by 0.
#pragma once
#include <type_traits>

#include "norm_util.cuh"

namespace gcb {

struct ConvSeqParams {
    const void *x, *dy;
    void *y;  // or dx
    long long x_ldn, x_ldt, dy_ldn, dy_ldt, y_ldn, y_ldt;
    long long n, l;
    int c, vcols, taps;
    const void *w, *bias;  // w: [c][taps]
    int w_type, bias_type;
    int act;
    const int *lengths;    // nullable
    const void *state;     // nullable, [n][taps - 1][c]
    void *state_out;       // nullable; in the gradient: of the first state
    const void *dstate;    // gradient, nullable: of the last state
    long long s_ldn, s_ldt, so_ldn, so_ldt, ds_ldn, ds_ldt;
    int stretch;           // tokens of a thread
    long long segs;        // stretches of a sequence
    // gradient
    int cols, workers;     // vector columns and workers of a block
    long long blocks_y;    // blocks that share a tile of columns
    float *part;           // [block][taps + 1][c] or NULL
};

constexpr int kConvThreads = 256;

// V elements as they lie in memory: 16 or 8 bytes, or one element.
template <class T, int V>
struct Group {
    static constexpr int kBytes = V * static_cast<int>(sizeof(T));
    typename std::conditional<kBytes == 16, uint4, typename std::conditional<V == 1, T, uint2>::type>::type u;
};
template <class T, int V>
__device__ __forceinline__ Group<T, V> load_group(const T *p) {
    Group<T, V> g;
    if constexpr (V == 1) g.u = *p;
    else g.u = *reinterpret_cast<const decltype(g.u) *>(p);
    return g;
}
template <class T, int V>
__device__ __forceinline__ Lanes<V> lanes_of_group(const Group<T, V> &g) {
    Lanes<V> r;
    if constexpr (V == 1) {
        r.p[0] = pair(to_float(g.u), 0.0f);
    } else if constexpr (Group<T, V>::kBytes == 16) {
        r = unpack_lanes<T, V>(g.u, static_cast<const T *>(nullptr));
    } else {
        float v[8];
        unpack(make_uint4(g.u.x, g.u.y, 0u, 0u), v, static_cast<const T *>(nullptr));
        r.p[0] = pair(v[0], v[1]);
        r.p[1] = pair(v[2], v[3]);
    }
    return r;
}
template <class T, int V>
__device__ __forceinline__ void store_group(T *p, const Lanes<V> &l) {
    if constexpr (V == 1 || Group<T, V>::kBytes == 16) {
        store_lanes<T, V>(p, l);
    } else {
        float v[8] = {};
        split(l.p[0], v[0], v[1]);
        split(l.p[1], v[2], v[3]);
        const uint4 u = pack(v, p);
        __stcs(reinterpret_cast<uint2 *>(p), make_uint2(u.x, u.y));
    }
}
template <int V>
__device__ __forceinline__ Lanes<V> no_lanes() {
    Lanes<V> r;
#pragma unroll
    for (int i = 0; i < Lanes<V>::kPairs; ++i) r.p[i] = pair(0.0f);
    return r;
}

// The weights of V channels, tap by tap, right-aligned in KT.
template <int V, int KT>
__device__ __forceinline__ void load_taps(const ConvSeqParams &P, int c0, Lanes<V> (&w)[KT]) {
    const int pad = KT - P.taps;
#pragma unroll
    for (int k = 0; k < KT; ++k) {
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j)
            v[j] = k >= pad ? load_param(P.w, P.w_type, static_cast<long long>(c0 + j) * P.taps + k - pad) : 0.0f;
        w[k] = lanes_of<V>(v);
    }
}
template <int V>
__device__ __forceinline__ Lanes<V> load_bias(const ConvSeqParams &P, int c0) {
    float v[V];
    load_params<V>(P.bias, P.bias_type, c0, 0.0f, v);
    return lanes_of<V>(v);
}

// u at token t of sequence n, where t < 0 lies in the state.
template <class T, int V>
__device__ __forceinline__ Lanes<V> input_at(const ConvSeqParams &P, long long n, long long t, int c0) {
    if (t >= 0) return lanes_of_group<T, V>(load_group<T, V>(static_cast<const T *>(P.x) + n * P.x_ldn + t * P.x_ldt + c0));
    const long long j = t + P.taps - 1;
    if (P.state == nullptr || j < 0) return no_lanes<V>();
    return lanes_of_group<T, V>(load_group<T, V>(static_cast<const T *>(P.state) + n * P.s_ldn + j * P.s_ldt + c0));
}

__device__ __forceinline__ long long length_of(const int *lengths, long long n, long long l) {
    if (lengths == nullptr) return l;
    const int v = lengths[n];
    return v < 0 ? 0 : min(static_cast<long long>(v), l);
}

template <int V, int KT, int ACT>
__device__ __forceinline__ Lanes<V> conv_at(const ConvSeqParams &P, const Lanes<V> (&w)[KT], const Lanes<V> (&window)[KT - 1],
                                            const Lanes<V> &cur, const Lanes<V> &bias) {
    const int pad = KT - P.taps;
    Lanes<V> v = bias;
#pragma unroll
    for (int k = 0; k < KT; ++k)
        if (k >= pad) {
#pragma unroll
            for (int i = 0; i < Lanes<V>::kPairs; ++i)
                v.p[i] = fma2(w[k].p[i], k < KT - 1 ? window[k < KT - 1 ? k : 0].p[i] : cur.p[i], v.p[i]);
        }
    return v;
}

// A thread's groups at p, p + step, .. copied ahead through a ring in shared memory
// that is its own: D copies under way, no barrier, no registers.  The ring holds
// kConvRing groups of every thread.
constexpr int kConvRing = 16;
template <class T, int V>
struct ConvRing {
    static constexpr bool kCopies = Group<T, V>::kBytes >= 4;
    Group<T, V> *mine;
    __device__ __forceinline__ explicit ConvRing(char *space) : mine(reinterpret_cast<Group<T, V> *>(space) + threadIdx.x) {}
    __device__ __forceinline__ void copy(int slot, const T *p) const {
        const uint32_t dst = smem_addr(mine + slot * kConvThreads);
        if constexpr (Group<T, V>::kBytes == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(p) : "memory");
        else if constexpr (Group<T, V>::kBytes == 8)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(p) : "memory");
        else if constexpr (kCopies)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(p) : "memory");
    }
    // What cannot be copied asynchronously (two bytes): `count` groups at once, for
    // slots first, first + every, ..
    template <int MOST>
    __device__ __forceinline__ void fill(int first, int every, const T *p, long long step, int count) const {
        if constexpr (!kCopies) {
            Group<T, V> g[MOST];
#pragma unroll
            for (int k = 0; k < MOST; ++k)
                if (k < count) g[k] = load_group<T, V>(p + k * step);
#pragma unroll
            for (int k = 0; k < MOST; ++k)
                if (k < count) mine[(first + k * every) * kConvThreads] = g[k];
        }
    }
    __device__ __forceinline__ Lanes<V> at(int slot) const { return lanes_of_group<T, V>(mine[slot * kConvThreads]); }
};

template <class T, int V, int KT, int ACT>
__global__ void __launch_bounds__(kConvThreads) causal_conv_kernel(const __grid_constant__ ConvSeqParams P) {
    extern __shared__ __align__(16) char space[];
    griddep_wait();
    griddep_launch_dependents();
    const long long id = static_cast<long long>(blockIdx.x) * kConvThreads + threadIdx.x;
    const int c0 = static_cast<int>(id % P.vcols) * V;
    const long long rest = id / P.vcols, seg = rest % P.segs, n = rest / P.segs;
    if (n >= P.n) return;
    const long long len = length_of(P.lengths, n, P.l), t0 = seg * P.stretch, t1 = min(P.l, t0 + P.stretch);
    const long long end = min(len, t1);
    Lanes<V> w[KT], window[KT - 1];
    T *y = static_cast<T *>(P.y) + n * P.y_ldn + c0;
    if (t0 < end) {
        const ConvRing<T, V> ring(space);
        const int count = static_cast<int>(end - t0);
        const T *x = static_cast<const T *>(P.x) + n * P.x_ldn + t0 * P.x_ldt + c0;
#pragma unroll
        for (int k = 0; k < kConvRing; ++k, x += P.x_ldt) {
            if (k < count) ring.copy(k, x);
            cp_async_commit();
        }
        load_taps<V, KT>(P, c0, w);
        const Lanes<V> bias = load_bias<V>(P, c0);
#pragma unroll
        for (int k = 0; k < KT - 1; ++k) window[k] = k >= KT - P.taps ? input_at<T, V>(P, n, t0 - (KT - 1) + k, c0) : no_lanes<V>();
        T *out = y + t0 * P.y_ldt;
#pragma unroll 4
        for (int k = 0; k < count; ++k, x += P.x_ldt, out += P.y_ldt) {
            cp_async_wait<kConvRing - 1>();
            const int slot = k % kConvRing;
            if (slot == 0) ring.template fill<kConvRing>(0, 1, x - kConvRing * P.x_ldt, P.x_ldt, count - k);
            const Lanes<V> cur = ring.at(slot);
            if (k + kConvRing < count) ring.copy(slot, x);
            cp_async_commit();
            Lanes<V> v = conv_at<V, KT, ACT>(P, w, window, cur, bias);
#pragma unroll
            for (int i = 0; i < Lanes<V>::kPairs; ++i) v.p[i] = activate<ACT>(P.act, v.p[i]);
            store_group<T, V>(out, v);
#pragma unroll
            for (int i = 0; i + 1 < KT - 1; ++i) window[i] = window[i + 1];
            window[KT - 2] = cur;
        }
    }
    for (long long t = max(end, t0); t < t1; ++t) store_group<T, V>(y + t * P.y_ldt, no_lanes<V>());
    if (P.state_out != nullptr && seg == 0) {
        T *out = static_cast<T *>(P.state_out) + n * P.so_ldn + c0;
        for (int j = 0; j < P.taps - 1; ++j)
            store_group<T, V>(out + j * P.so_ldt, input_at<T, V>(P, n, len + j - (P.taps - 1), c0));
    }
}

// One token: x and y are [n][c].  A thread has read all of its channels' state
// before it writes, so state_out may be the state itself.
template <class T, int V, int KT, int ACT>
__global__ void __launch_bounds__(kConvThreads) causal_conv_step_kernel(const __grid_constant__ ConvSeqParams P) {
    griddep_wait();
    griddep_launch_dependents();
    const long long id = static_cast<long long>(blockIdx.x) * kConvThreads + threadIdx.x;
    const int c0 = static_cast<int>(id % P.vcols) * V;
    const long long n = id / P.vcols;
    if (n >= P.n) return;
    Lanes<V> w[KT], window[KT - 1];
#pragma unroll
    for (int k = 0; k < KT - 1; ++k) window[k] = k >= KT - P.taps ? input_at<T, V>(P, n, k - (KT - 1), c0) : no_lanes<V>();
    const Lanes<V> cur = input_at<T, V>(P, n, 0, c0);
    load_taps<V, KT>(P, c0, w);
    Lanes<V> v = conv_at<V, KT, ACT>(P, w, window, cur, load_bias<V>(P, c0));
#pragma unroll
    for (int i = 0; i < Lanes<V>::kPairs; ++i) v.p[i] = activate<ACT>(P.act, v.p[i]);
    store_group<T, V>(static_cast<T *>(P.y) + n * P.y_ldn + c0, v);
    if (P.taps == 1) return;
    T *out = static_cast<T *>(P.state_out) + n * P.so_ldn + c0;
    const int pad = KT - P.taps;
#pragma unroll
    for (int k = 1; k < KT - 1; ++k)
        if (k > pad) store_group<T, V>(out + (k - 1 - pad) * P.so_ldt, window[k]);
    store_group<T, V>(out + (P.taps - 2) * P.so_ldt, cur);
}

// The gradient.  A block takes a tile of `cols` vector columns; its workers take
// stretches of sequences in turn.  Walking forward, a worker forms g[t] and
// finishes dx[t - (KT - 1)]; the KT - 1 tokens behind its stretch are formed once
// more.  dw and dbias add up over a stretch, then over stretches, then over the
// workers of the block in a fixed order.
template <class T, int V, int KT, int ACT>
__global__ void __launch_bounds__(kConvThreads, KT <= 4 ? 2 : 1) causal_conv_grad_kernel(const __grid_constant__ ConvSeqParams P) {
    constexpr int NP = Lanes<V>::kPairs, D = kConvRing / 2;  // D: tokens under way, of x and of dy
    extern __shared__ __align__(16) char space[];
    __shared__ float sm[kConvThreads * V];
    griddep_wait();
    griddep_launch_dependents();
    const long long tile = blockIdx.x / P.blocks_y, by = blockIdx.x - tile * P.blocks_y;
    const int worker = threadIdx.x / P.cols, col = threadIdx.x - worker * P.cols;
    const long long vcol = tile * P.cols + col;
    const bool live = worker < P.workers && vcol < P.vcols;
    const int c0 = static_cast<int>(vcol) * V, pad = KT - P.taps;
    Lanes<V> dw[KT], db = no_lanes<V>();
#pragma unroll
    for (int k = 0; k < KT; ++k) dw[k] = no_lanes<V>();
    if (live) {
        Lanes<V> w[KT];
        load_taps<V, KT>(P, c0, w);
        const Lanes<V> bias = load_bias<V>(P, c0);
        for (long long item = by * P.workers + worker; item < P.n * P.segs; item += P.blocks_y * P.workers) {
            const long long n = item / P.segs, seg = item - n * P.segs;
            const long long len = length_of(P.lengths, n, P.l), t0 = seg * P.stretch, t1 = min(P.l, t0 + P.stretch);
            const T *x = static_cast<const T *>(P.x) + n * P.x_ldn + c0, *dy = static_cast<const T *>(P.dy) + n * P.dy_ldn + c0;
            T *dx = static_cast<T *>(P.y) + n * P.y_ldn + c0;
            const ConvRing<T, V> ring(space);
            const int count = static_cast<int>(t1 + KT - 1 - t0);                                 // tokens to walk over
            const int inside = static_cast<int>(max(0LL, min(len, t1 + KT - 1) - t0));  // of those, in the sequence
            const T *px = x + t0 * P.x_ldt, *pg = dy + t0 * P.dy_ldt;
#pragma unroll
            for (int k = 0; k < D; ++k, px += P.x_ldt, pg += P.dy_ldt) {
                if (k < inside) {
                    ring.copy(2 * k, px);
                    ring.copy(2 * k + 1, pg);
                }
                cp_async_commit();
            }
            Lanes<V> xw[KT - 1], gw[KT - 1], dw1[KT], db1 = no_lanes<V>();
#pragma unroll
            for (int k = 0; k < KT; ++k) dw1[k] = no_lanes<V>();
#pragma unroll
            for (int k = 0; k < KT - 1; ++k) {
                xw[k] = k >= pad && inside > 0 ? input_at<T, V>(P, n, t0 - (KT - 1) + k, c0) : no_lanes<V>();
                gw[k] = no_lanes<V>();
            }
            const int first = seg == 0 ? KT - P.taps : KT - 1;  // from here on a finished place is the stretch's, or the state's
            T *out = dx + (t0 - (KT - 1)) * P.y_ldt;
            for (int k = 0; k < count; ++k, px += P.x_ldt, pg += P.dy_ldt, out += P.y_ldt) {
                cp_async_wait<D - 1>();
                const int slot = k % D * 2;
                if (slot == 0) {
                    ring.template fill<D>(0, 2, px - D * P.x_ldt, P.x_ldt, inside - k);
                    ring.template fill<D>(1, 2, pg - D * P.dy_ldt, P.dy_ldt, inside - k);
                }
                Lanes<V> cur = no_lanes<V>(), g = no_lanes<V>();
                if (k < inside) {
                    cur = ring.at(slot);
                    g = ring.at(slot + 1);
                }
                if (k + D < inside) {
                    ring.copy(slot, px);
                    ring.copy(slot + 1, pg);
                }
                cp_async_commit();
                if (k < inside) {
                    if (ACT != kActNone) {
                        const Lanes<V> v = conv_at<V, KT, ACT>(P, w, xw, cur, bias);
#pragma unroll
                        for (int i = 0; i < NP; ++i) g.p[i] = activate_grad<ACT>(P.act, v.p[i], g.p[i]);
                    }
                    if (k < t1 - t0) {
#pragma unroll
                        for (int i = 0; i < NP; ++i) {
                            db1.p[i] = db1.p[i] + g.p[i];
#pragma unroll
                            for (int j = 0; j < KT; ++j)
                                if (j >= pad)
                                    dw1[j].p[i] = fma2(g.p[i], j < KT - 1 ? xw[j < KT - 1 ? j : 0].p[i] : cur.p[i], dw1[j].p[i]);
                        }
                    }
                }
                if (k >= first) {
                    const long long s = t0 + k - (KT - 1);
                    Lanes<V> d = no_lanes<V>();
                    if (s < len) {
#pragma unroll
                        for (int j = 0; j < KT; ++j)
                            if (j >= pad) {
#pragma unroll
                                for (int i = 0; i < NP; ++i)
                                    d.p[i] = fma2(w[j].p[i], j == 0 ? g.p[i] : gw[j == 0 ? 0 : KT - 1 - j].p[i], d.p[i]);
                            }
                        const long long j = s + P.taps - 1 - len;  // its place in the last state
                        if (P.dstate != nullptr && j >= 0) {
                            const Lanes<V> e = lanes_of_group<T, V>(load_group<T, V>(
                                static_cast<const T *>(P.dstate) + n * P.ds_ldn + j * P.ds_ldt + c0));
#pragma unroll
                            for (int i = 0; i < NP; ++i) d.p[i] = d.p[i] + e.p[i];
                        }
                    }
                    if (s >= 0) store_group<T, V>(out, d);
                    else if (P.state_out != nullptr)
                        store_group<T, V>(static_cast<T *>(P.state_out) + n * P.so_ldn + (s + P.taps - 1) * P.so_ldt + c0, d);
                }
#pragma unroll
                for (int i = 0; i + 1 < KT - 1; ++i) {
                    xw[i] = xw[i + 1];
                    gw[i] = gw[i + 1];
                }
                xw[KT - 2] = cur;
                gw[KT - 2] = g;
            }
            cp_async_wait<0>();
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                db.p[i] = db.p[i] + db1.p[i];
#pragma unroll
                for (int k = 0; k < KT; ++k) dw[k].p[i] = dw[k].p[i] + dw1[k].p[i];
            }
        }
    }
    if (P.part == nullptr) return;
#pragma unroll
    for (int q = 0; q <= KT; ++q) {
        if (q < pad) continue;
        float v[V];
        values_of<V>(q < KT ? dw[q < KT ? q : 0] : db, v);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (worker < P.workers) sm[(j * P.workers + worker) * P.cols + col] = v[j];
        __syncthreads();
        if (worker == 0 && vcol < P.vcols) {
            float *out = P.part + (by * (P.taps + 1) + (q < KT ? q - pad : P.taps)) * P.c + c0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float s = sm[j * P.workers * P.cols + col];
                for (int i = 1; i < P.workers; ++i) s += sm[(j * P.workers + i) * P.cols + col];
                out[j] = s;
            }
        }
    }
}

}  // namespace gcb
