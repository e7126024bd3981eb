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
// tap would multiply is left out, not multiplied by 0.  N8 L2048 C2048 bf16, K 4,
// SiLU: forward 29 us (4.6 TB/s), gradient 59 (3.4 TB/s).  Both run 256 blocks, two to a
// multiprocessor, on 148: one uneven round.  Backwards 13 warps a multiprocessor issue in
// 50 % of the slots and wait for one another's results more than for memory; 128
// registers hold the four-channel kernels but for 32 to 176 bytes a thread.  K 3, whose
// taps are counted at run time: 40 and 77 us, K 8 in its kernel of 243 registers 68 and 142.
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
    int w_four;            // four taps, aligned
    int act;
    const int *lengths;    // nullable
    const void *state;     // nullable, [n][taps - 1][c]
    void *state_out;       // nullable; in the gradient: of the first state
    const void *dstate;    // gradient, nullable: of the last state
    long long s_ldn, s_ldt, so_ldn, so_ldt, ds_ldn, ds_ldt;
    int stretch;           // tokens of a thread
    long long segs;        // stretches of a sequence
    int small;             // fewer than 2^32 threads
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

// The weights of V channels, tap by tap, right-aligned in KT.  Four taps of four
// channels lie side by side: two or four 16-byte accesses.
template <int V, int KT>
__device__ __forceinline__ void load_taps(const ConvSeqParams &P, int c0, Lanes<V> (&w)[KT]) {
    if constexpr (V > 1 && KT == 4) {
        if (P.w_four) {
            float f[V][4];  // [channel][tap]
            if (P.w_type == kElemF32) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    unpack(__ldg(reinterpret_cast<const uint4 *>(static_cast<const float *>(P.w) + c0 * 4) + j), f[j],
                           static_cast<const float *>(nullptr));
            } else {
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const uint4 u = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(P.w) + c0 * 4) + j);
                    float v[8];
                    if (P.w_type == kElemBF16) unpack(u, v, static_cast<const __nv_bfloat16 *>(nullptr));
                    else unpack(u, v, static_cast<const __half *>(nullptr));
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[2 * j + i / 4][i % 4] = v[i];
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float v[V];
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = f[j][k];
                w[k] = lanes_of<V>(v);
            }
            return;
        }
    }
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

// FULL: as many taps as the kernel holds.
// The window of a thread is a ring of KT inputs, the newest at place `u`; loops over
// tokens are unrolled by KT, so that places are known at compile time and nothing
// is moved.
template <int V, int KT, bool FULL>
__device__ __forceinline__ Lanes<V> conv_at(const ConvSeqParams &P, const Lanes<V> (&w)[KT], const Lanes<V> (&window)[KT], int u,
                                            const Lanes<V> &bias) {
    const int pad = FULL ? 0 : KT - P.taps;
    Lanes<V> v = bias;
#pragma unroll
    for (int k = 0; k < KT; ++k)
        if (k >= pad) {
#pragma unroll
            for (int i = 0; i < Lanes<V>::kPairs; ++i) v.p[i] = fma2(w[k].p[i], window[(u + 1 + k) % KT].p[i], v.p[i]);
        }
    return v;
}
// The window in front of token t.
template <class T, int V, int KT>
__device__ __forceinline__ void load_window(const ConvSeqParams &P, long long n, long long t, int c0, bool any, Lanes<V> (&window)[KT]) {
    window[0] = no_lanes<V>();
#pragma unroll
    for (int k = 1; k < KT; ++k)
        window[k] = any && k > KT - P.taps ? input_at<T, V>(P, n, t - KT + k, c0) : no_lanes<V>();
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

template <class T, int V, int KT, bool FULL, int ACT>
__global__ void __launch_bounds__(kConvThreads) causal_conv_kernel(const __grid_constant__ ConvSeqParams P) {
    extern __shared__ __align__(16) char space[];
    griddep_wait();
    griddep_launch_dependents();
    long long n, seg;
    int c0;
    if (P.small) {  // 32-bit divisions
        const unsigned id = blockIdx.x * kConvThreads + threadIdx.x, vcols = P.vcols, segs = static_cast<unsigned>(P.segs);
        const unsigned rest = id / vcols;
        c0 = static_cast<int>(id - rest * vcols) * V;
        n = rest / segs;
        seg = rest % segs;
    } else {
        const long long id = static_cast<long long>(blockIdx.x) * kConvThreads + threadIdx.x, rest = id / P.vcols;
        c0 = static_cast<int>(id % P.vcols) * V;
        seg = rest % P.segs;
        n = rest / P.segs;
    }
    if (n >= P.n) return;
    const long long len = length_of(P.lengths, n, P.l), t0 = seg * P.stretch, t1 = min(P.l, t0 + P.stretch);
    const long long end = min(len, t1);
    Lanes<V> w[KT], window[KT];
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
        load_window<T, V, KT>(P, n, t0, c0, true, window);
        T *out = y + t0 * P.y_ldt;
        for (int k0 = 0; k0 < count; k0 += KT) {
            if (k0 % kConvRing == 0) ring.template fill<kConvRing>(0, 1, x - kConvRing * P.x_ldt, P.x_ldt, count - k0);
            const int slot = k0 % kConvRing;
#pragma unroll
            for (int u = 0; u < KT; ++u, x += P.x_ldt, out += P.y_ldt) {
                cp_async_wait<kConvRing - 1>();
                window[u] = ring.at(slot + u);
                if (k0 + u + kConvRing < count) ring.copy(slot + u, x);
                cp_async_commit();
                Lanes<V> v = conv_at<V, KT, FULL>(P, w, window, u, bias);
#pragma unroll
                for (int i = 0; i < Lanes<V>::kPairs; ++i) v.p[i] = activate<ACT>(P.act, v.p[i]);
                if (k0 + u < count) store_group<T, V>(out, v);
            }
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
template <class T, int V, int KT, bool FULL, int ACT>
__global__ void __launch_bounds__(kConvThreads) causal_conv_step_kernel(const __grid_constant__ ConvSeqParams P) {
    griddep_wait();
    griddep_launch_dependents();
    long long n;
    int c0;
    if (P.small) {
        const unsigned id = blockIdx.x * kConvThreads + threadIdx.x, vcols = P.vcols;
        n = id / vcols;
        c0 = static_cast<int>(id % vcols) * V;
    } else {
        const long long id = static_cast<long long>(blockIdx.x) * kConvThreads + threadIdx.x;
        n = id / P.vcols;
        c0 = static_cast<int>(id % P.vcols) * V;
    }
    if (n >= P.n) return;
    Lanes<V> w[KT], window[KT];
    load_window<T, V, KT>(P, n, 0, c0, true, window);
    window[0] = input_at<T, V>(P, n, 0, c0);
    load_taps<V, KT>(P, c0, w);
    Lanes<V> v = conv_at<V, KT, FULL>(P, w, window, 0, load_bias<V>(P, c0));
#pragma unroll
    for (int i = 0; i < Lanes<V>::kPairs; ++i) v.p[i] = activate<ACT>(P.act, v.p[i]);
    store_group<T, V>(static_cast<T *>(P.y) + n * P.y_ldn + c0, v);
    if (P.taps == 1) return;
    T *out = static_cast<T *>(P.state_out) + n * P.so_ldn + c0;
    const int pad = KT - P.taps;
#pragma unroll
    for (int k = 2; k < KT; ++k)
        if (k > pad + 1) store_group<T, V>(out + (k - 2 - pad) * P.so_ldt, window[k]);
    store_group<T, V>(out + (P.taps - 2) * P.so_ldt, window[0]);
}

// The gradient.  A block takes a tile of `cols` vector columns; its workers take
// stretches of sequences in turn.  Walking forward, a worker forms g[t] and
// finishes dx[t - (KT - 1)]; the KT - 1 tokens behind its stretch are formed once
// more.  dw and dbias add up over a stretch (128 tokens at most), then over 64
// stretches at most (the plan sees to that), then over the workers of the block, in a
// fixed order.
template <class T, int V, int KT, bool FULL, int ACT>
__global__ void __launch_bounds__(kConvThreads, KT <= 4 ? 2 : 1) causal_conv_grad_kernel(const __grid_constant__ ConvSeqParams P) {
    constexpr int NP = Lanes<V>::kPairs, D = kConvRing / 2;  // D: tokens under way, of x and of dy
    extern __shared__ __align__(16) char space[];
    griddep_wait();
    griddep_launch_dependents();
    const long long tile = blockIdx.x / P.blocks_y, by = blockIdx.x - tile * P.blocks_y;
    const int worker = threadIdx.x / P.cols, col = threadIdx.x - worker * P.cols;
    const long long vcol = tile * P.cols + col;
    const bool live = worker < P.workers && vcol < P.vcols;
    const int c0 = static_cast<int>(vcol) * V, pad = FULL ? 0 : KT - P.taps;
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
            Lanes<V> xw[KT], gw[KT], dw1[KT], db1 = no_lanes<V>();
#pragma unroll
            for (int k = 0; k < KT; ++k) dw1[k] = gw[k] = no_lanes<V>();
            load_window<T, V, KT>(P, n, t0, c0, inside > 0, xw);
            const int first = seg == 0 ? KT - P.taps : KT - 1;  // from here on a finished place is the stretch's, or the state's
            const int own = static_cast<int>(t1 - t0);
            // tokens between which nothing has to be asked: all places finished are tokens of the
            // sequence away from its last state, all tokens are the stretch's
            const int plain_from = KT - 1, plain_to = P.dstate != nullptr ? 0 : min(inside, own);
            T *out = dx + (t0 - (KT - 1)) * P.y_ldt;
            const auto token = [&](int k, int u, auto ask) {
                constexpr bool ASK = decltype(ask)::value;
                cp_async_wait<D - 1>();
                const int slot = k % D * 2;
                const bool live = !ASK || k < inside;
                xw[u] = gw[u] = no_lanes<V>();
                if (live) {
                    xw[u] = ring.at(slot);
                    gw[u] = ring.at(slot + 1);
                }
                if (k + D < inside) {
                    ring.copy(slot, px);
                    ring.copy(slot + 1, pg);
                }
                cp_async_commit();
                if (live) {
                    if (ACT != kActNone) {
                        const Lanes<V> v = conv_at<V, KT, FULL>(P, w, xw, u, bias);
#pragma unroll
                        for (int i = 0; i < NP; ++i) gw[u].p[i] = activate_grad<ACT>(P.act, v.p[i], gw[u].p[i]);
                    }
                    if (!ASK || k < own) {
#pragma unroll
                        for (int i = 0; i < NP; ++i) {
                            db1.p[i] = db1.p[i] + gw[u].p[i];
#pragma unroll
                            for (int j = 0; j < KT; ++j)
                                if (j >= pad) dw1[j].p[i] = fma2(gw[u].p[i], xw[(u + 1 + j) % KT].p[i], dw1[j].p[i]);
                        }
                    }
                }
                if (!ASK || k >= first) {
                    const long long s = t0 + k - (KT - 1);
                    Lanes<V> d = no_lanes<V>();
                    if (!ASK || s < len) {
#pragma unroll
                        for (int j = 0; j < KT; ++j)
                            if (j >= pad) {
#pragma unroll
                                for (int i = 0; i < NP; ++i) d.p[i] = fma2(w[j].p[i], gw[(u - j + KT) % KT].p[i], d.p[i]);
                            }
                        const long long j = s + P.taps - 1 - len;  // its place in the last state
                        if (ASK && P.dstate != nullptr && j >= 0) {
                            const Lanes<V> e = lanes_of_group<T, V>(load_group<T, V>(
                                static_cast<const T *>(P.dstate) + n * P.ds_ldn + j * P.ds_ldt + c0));
#pragma unroll
                            for (int i = 0; i < NP; ++i) d.p[i] = d.p[i] + e.p[i];
                        }
                    }
                    if (!ASK || s >= 0) store_group<T, V>(out, d);
                    else if (P.state_out != nullptr)
                        store_group<T, V>(static_cast<T *>(P.state_out) + n * P.so_ldn + (s + P.taps - 1) * P.so_ldt + c0, d);
                }
                px += P.x_ldt;
                pg += P.dy_ldt;
                out += P.y_ldt;
            };
            for (int k0 = 0; k0 < count; k0 += KT) {
                if (k0 % D == 0) {
                    ring.template fill<D>(0, 2, px - D * P.x_ldt, P.x_ldt, inside - k0);
                    ring.template fill<D>(1, 2, pg - D * P.dy_ldt, P.dy_ldt, inside - k0);
                }
                if (k0 >= plain_from && k0 + KT <= plain_to) {
#pragma unroll
                    for (int u = 0; u < KT; ++u) token(k0 + u, u, std::false_type());
                } else {
#pragma unroll
                    for (int u = 0; u < KT; ++u)
                        if (k0 + u < count) token(k0 + u, u, std::true_type());
                }
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
    // all sums side by side in the ring's place, each then joined by one thread
    float *sm = reinterpret_cast<float *>(space);
    const int pitch = P.workers * P.cols;
    __syncthreads();
#pragma unroll
    for (int q = 0; q <= KT; ++q) {
        float v[V];
        values_of<V>(q < KT ? dw[q < KT ? q : 0] : db, v);
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (worker < P.workers && q >= pad) sm[((q - pad) * V + j) * pitch + worker * P.cols + col] = v[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (P.taps + 1) * V * P.cols; i += kConvThreads) {
        const int k = i % P.cols, j = i / P.cols % V, q = i / P.cols / V;  // column, element, tap (the last: bias)
        if (tile * P.cols + k >= P.vcols) continue;
        const float *src = sm + (q * V + j) * pitch + k;
        float s = src[0];
        for (int w = 1; w < P.workers; ++w) s += src[w * P.cols];
        P.part[(by * (P.taps + 1) + q) * P.c + (tile * P.cols + k) * V + j] = s;
    }
}

}  // namespace gcb
