// Selective state space scan over sequences, its gradient, and its form for one
// new token of every sequence.
//
//   delta = softplus(dt + dt_bias);  h[t] = a[t] h[t-1] + delta[t] x[t] B[t],  a[t] = exp(delta[t] A)
//   v[t] = C[t] . h[t] + D x[t];  y[t] = v[t] z[t] / (1 + exp(-z[t]))
//
// with a state h of S numbers for each channel of each sequence; B and C are
// shared by the channels of a group.  Backwards, with f = dy times the gate and
// q[t] = f[t] C[t] + a[t+1] q[t+1]:
//   dB[t] += q[t] delta x,  dC[t] += f h[t],  dA += q[t] a[t] h[t-1] delta,
//   dx = delta (q . B) + D f,  ddelta = (q a h[t-1]) . A + x (q . B)
//
// What bounds these kernels is the exponential of every (token, channel, state):
// the special-function unit does 16 a clock and multiprocessor.  A channel's
// states are spread over P lanes of R = 4 each, held as pairs of floats; a block
// takes 2 THREADS / P channels and walks along the tokens in tiles.  A tile's
// inputs are copied to shared memory while the tile before is worked on; softplus,
// gate and products of a token and channel are then formed once for its P lanes.
// Where sequences and channels alone are too few to fill the GPU, each
// sequence is cut into segments: a first launch gives each segment's effect on
// the state (what it adds, and the sum of its deltas, whose product with A is its
// decay's logarithm), from which every block forms the state that it starts with.
//
// N4 L2048 C2048 S16 bf16, kernel after kernel: segments' effects 88 us, scan 173;
// backwards 102 and 370, sums 22.  The exponentials alone would take 58 us in each.
// There are 10 to 15 warps a multiprocessor at a time, which keep the shared memory's
// pipe (every lane reads each product, B and C of its states) 44 to 57 % busy and issue in
// 48 to 62 % of the slots: dependent instructions wait for one another.
#pragma once
#include <cstring>
#include <type_traits>

#include "norm_util.cuh"

namespace gcb {

// Tokens between the states that the scan keeps for its gradient; the gradient
// takes so many at a time.  (With 16 the states of two channels take the registers
// of half of the warps: 570 us against 432 at N4 L2048 C2048 bf16, for half of the
// memory.)
constexpr int kScanChunk = 8;
// Tiles of the gradient whose sums for A, D and dt_bias are added up in 32 bits one
// after the other; such runs are joined by sum_rows_kernel.
constexpr int kScanRun = 64;

// A tensor of tokens: strides of a sequence, a token and (B, C) a group.
struct TokenView {
    const void *p;
    long long ldn, ldt, ldg;
};
struct ScanParams {
    TokenView x, dt, z, b, c, dy;      // z.p nullable
    TokenView y, dx, ddt, dz;          // outputs
    const void *a, *d, *bias;          // a: [channels][states]; d, bias nullable
    int a_type, d_type, bias_type;
    const float *state, *dlast;        // nullable: first state; gradient of the last
    float *state_out;                  // nullable: last state, or the first one's gradient
    long long s_ldn, s_ldc, so_ldn, so_ldc, dl_ldn, dl_ldc;
    const int *lengths;                // nullable
    long long n, l;
    int channels, states, groups, cpg; // cpg: channels of a group
    int vec, bvec, softplus;           // vec, bvec: four channels, four states of B and C in one access
    int tiles;                         // blocks that share a group's channels
    long long seg_len;
    int segs;
    float *carry, *sums;               // [n][segs][channels][states], [n][segs][channels]
    float *kept;                       // [n][chunks][channels][states] or NULL
    float *part_bc;                    // gradient: [tile][n][l][groups][2][states]
    float *part_a, *part_d;            // [n * segs * runs][channels][states], [n * segs * runs][2][channels] (D, dt_bias)
    int runs;                          // of kScanRun tiles, in a segment
};

// ---- four elements ---------------------------------------------------------------------------
template <class T>
struct Four {
    typename std::conditional<sizeof(T) == 4, uint4, uint2>::type u;
};
// `valid` elements from p; in one access where `vec` (valid is then 4 or none).
template <class T>
__device__ __forceinline__ Four<T> load_four(const T *p, bool vec, int valid) {
    Four<T> r;
    if (vec && valid > 0) {
        r.u = *reinterpret_cast<const decltype(r.u) *>(p);
    } else {
        T e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = i < valid ? p[i] : from_float<T>(0.0f);
        memcpy(&r.u, e, sizeof(r.u));
    }
    return r;
}
template <class T>
__device__ __forceinline__ void floats_of(const Four<T> &r, f2 (&v)[2]) {
    if constexpr (sizeof(T) == 4) {
        v[0] = pair(__uint_as_float(r.u.x), __uint_as_float(r.u.y));
        v[1] = pair(__uint_as_float(r.u.z), __uint_as_float(r.u.w));
    } else {
        float w[8];
        unpack(make_uint4(r.u.x, r.u.y, 0u, 0u), w, static_cast<const T *>(nullptr));
        v[0] = pair(w[0], w[1]);
        v[1] = pair(w[2], w[3]);
    }
}
template <class T>
__device__ __forceinline__ void store_zeros(T *p, bool vec, int valid) {
    if (vec && valid > 0) {
        Four<T> r;
        memset(&r.u, 0, sizeof(r.u));
        *reinterpret_cast<decltype(r.u) *>(p) = r.u;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < valid) p[i] = from_float<T>(0.0f);
    }
}
// Four elements to a thread's own place in shared memory.
template <class T>
__device__ __forceinline__ void copy_four(const void *dst, const T *p) {
    if constexpr (sizeof(T) == 4)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(p) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_addr(dst)), "l"(p) : "memory");
}

// ---- functions of a token and channel -----------------------------------------------------
__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ f2 exp2_fast(f2 v) {
    float a, b;
    split(v, a, b);
    return pair(exp2_fast(a), exp2_fast(b));
}
__device__ __forceinline__ float rcp_fast(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// The larger, or NaN where one of them is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float sum_of(f2 v) {
    float a, b;
    split(v, a, b);
    return a + b;
}
constexpr float kLog2E = 1.4426950408889634f;

// softplus(v) = max(v, 0) + log(1 + e), e = exp(-|v|), and (SLOPE) its slope, the
// sigmoid.  log(1 + e) = 2 artanh(e / (2 + e)) by the series of the inverse
// hyperbolic tangent, whose argument is at most 1/3: the first term left out is
// below 2e-8 of the sum.  Step sizes far below 1 come from small e, where a
// logarithm of the rounded 1 + e would lose what matters.  Two denominators share
// a reciprocal; they are between 1 and 3 whatever the arguments are, since a NaN, which
// would reach the other value through it, takes no part: |v| is held below 128, where
// e is 0 already (the smaller of a NaN and a number is the number), and a NaN comes
// back with max(v, 0).
template <bool SLOPE>
__device__ __forceinline__ void softplus2(f2 v, f2 &value, f2 &slope) {
    float v0, v1, p0, p1;
    split(v, v0, v1);
    const f2 e = exp2_fast(pair(fminf(fabsf(v0), 128.0f), fminf(fabsf(v1), 128.0f)) * pair(-kLog2E));
    split(e + pair(2.0f), p0, p1);
    const f2 u = e * (pair(p1, p0) * pair(rcp_fast(p0 * p1))), w = u * u;
    f2 s = fma2(w, pair(1.0f / 13.0f), pair(1.0f / 11.0f));
    s = fma2(w, s, pair(1.0f / 9.0f));
    s = fma2(w, s, pair(1.0f / 7.0f));
    s = fma2(w, s, pair(1.0f / 5.0f));
    s = fma2(w, s, pair(1.0f / 3.0f));
    s = fma2(w, s, pair(1.0f));
    value = fma2(u + u, s, pair(max_nan(v0, 0.0f), max_nan(v1, 0.0f)));
    if constexpr (SLOPE) {
        float e0, e1;
        split(e, e0, e1);
        split(e + pair(1.0f), p0, p1);
        const f2 r = pair(p1, p0) * pair(rcp_fast(p0 * p1));  // 1 / (1 + e)
        slope = pair(v0 >= 0.0f ? 1.0f : e0, v1 >= 0.0f ? 1.0f : e1) * r;
    }
}
// delta of four channels, and its slope against dt.
template <bool SLOPE>
__device__ __forceinline__ void scan_deltas(bool softplus, const f2 (&raw)[2], const f2 (&bias)[2], f2 (&delta)[2],
                                            f2 (&slope)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f2 v = raw[i] + bias[i];
        if (softplus) {
            softplus2<SLOPE>(v, delta[i], slope[i]);
        } else {
            delta[i] = v;
            slope[i] = pair(1.0f);
        }
    }
}
// z / (1 + exp(-z)) and (SLOPE) its slope, of two values.
template <bool SLOPE>
__device__ __forceinline__ void gate2(f2 z, f2 &gate, f2 &slope) {
    f2 s, rest;
    sigmoid2(z, s, rest);
    gate = z * s;
    if constexpr (SLOPE) slope = s * fma2(z, rest, pair(1.0f));
}

// ---- shapes and places ---------------------------------------------------------------------
// A thread takes a part of the states of two neighbouring channels, so that what
// it reads of B and C serves both.
template <int SP_, int MOST, int THREADS_, int T_>
struct ScanShape {
    static constexpr int SP = SP_, THREADS = THREADS_, T = T_;           // T: tokens of a tile
    static constexpr int R = SP < MOST ? SP : MOST, NP = (R + 1) / 2;    // states of a lane and channel, as pairs
    static constexpr int P = SP / R, CB = 2 * THREADS / P;       // lanes of a channel, channels of a block
    static constexpr int GROUPS = CB / 4, NG = T * GROUPS > THREADS ? T * GROUPS / THREADS : 1;
    static constexpr int QUADS = SP >= 4 ? SP / 4 : 1;           // of a token's B or C
    // Values of pairs of channels, 16 bytes each: even pairs, then odd ones, a place
    // apart in the banks, and tokens two.  Threads that store the pairs of their four
    // channels, lanes that read one token's pairs and lanes that read pairs of four
    // tokens all meet different banks.
    static constexpr int ODD = GROUPS + 1, PAIRS = 2 * ODD;
    __device__ __forceinline__ static int place(int chan) { return (chan >> 1 & 1) * ODD + (chan >> 2); }
};

// A warp's lanes: pair of channels * P + part; a part has the states part * R ...
template <class S>
struct ScanPlace {
    long long n, len, begin, stop, end;  // the segment's tokens; end: of those in the sequence
    int seg, group, tile, first, count;  // first channel of the block, its channels
    int chan, part, channel;             // the thread's first channel, in the block and in all
    bool live[2];
    __device__ __forceinline__ explicit ScanPlace(const ScanParams &Q) {
        // 32-bit divisions: those of 64 bits would be most of a step's instructions
        const unsigned tiles = Q.tiles, per = Q.groups * tiles, segs = Q.segs, b = blockIdx.x / per, gt = blockIdx.x - b * per;
        n = b / segs;
        seg = static_cast<int>(b % segs);
        group = static_cast<int>(gt / tiles);
        tile = static_cast<int>(gt % tiles);
        first = group * Q.cpg + tile * S::CB;
        count = min(S::CB, Q.cpg - tile * S::CB);
        chan = threadIdx.x / S::P * 2;
        part = threadIdx.x % S::P;
        channel = first + chan;
        live[0] = chan < count;
        live[1] = chan + 1 < count;
        len = Q.l;
        if (Q.lengths != nullptr) {
            const int v = Q.lengths[n];
            len = v < 0 ? 0 : min(static_cast<long long>(v), Q.l);
        }
        begin = seg * Q.seg_len;
        stop = min(Q.l, begin + Q.seg_len);
        end = min(len, stop);
    }
};

// A lane's states of a [..][states] tensor, as pairs; zeros where there are none.
// `swap` reorders them: place r holds state r ^ swap.
// Four floats in the order that `swap` asks for.
__device__ __forceinline__ float4 reorder(float4 v, int swap) {
    if (swap & 2) v = make_float4(v.z, v.w, v.x, v.y);
    if (swap & 1) v = make_float4(v.y, v.x, v.w, v.z);
    return v;
}
__device__ __forceinline__ bool whole_states(const void *p, int states) {
    return states % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}
template <class S>
__device__ __forceinline__ void load_states(const float *p, int part, int states, bool live, int swap, f2 (&v)[S::NP]) {
    const bool whole = whole_states(p, states);
#pragma unroll
    for (int r = 0; r < S::R; r += 4) {
        float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float *q = p + part * S::R + r;
        const int left = live ? min(states - part * S::R - r, S::R - r) : 0;
        if (S::R >= 4 && whole) {
            if (left > 0) f = *reinterpret_cast<const float4 *>(q);
        } else {
            if (left > 0) f.x = q[0];
            if (left > 1) f.y = q[1];
            if (left > 2) f.z = q[2];
            if (left > 3) f.w = q[3];
        }
        f = reorder(f, swap);
        v[r / 2] = pair(f.x, f.y);
        if constexpr (S::NP > 1) v[r / 2 + 1] = pair(f.z, f.w);
    }
}
template <class S>
__device__ __forceinline__ void store_states(float *p, int part, int states, bool live, int swap, const f2 (&v)[S::NP]) {
    const bool whole = whole_states(p, states);
#pragma unroll
    for (int r = 0; r < S::R; r += 4) {
        float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        split(v[r / 2], f.x, f.y);
        if constexpr (S::NP > 1) split(v[r / 2 + 1], f.z, f.w);
        f = reorder(f, swap);  // its own inverse
        float *q = p + part * S::R + r;
        const int left = live ? min(states - part * S::R - r, S::R - r) : 0;
        if (S::R >= 4 && whole) {
            if (left > 0) *reinterpret_cast<float4 *>(q) = f;
        } else {
            if (left > 0) q[0] = f.x;
            if (left > 1) q[1] = f.y;
            if (left > 2) q[2] = f.z;
            if (left > 3) q[3] = f.w;
        }
    }
}
// A log2(e): the exponentials are powers of 2.  Infinities become the largest
// numbers, whose exponentials are the same, so that a step size of 0 leaves a
// state as it is; tiles are filled up with such steps.  A NaN stays one.
__device__ __forceinline__ f2 decay_exponent(f2 v) {
    float a, b;
    split(v * pair(kLog2E), a, b);
    a = a > 3e38f ? 3e38f : a < -3e38f ? -3e38f : a;
    b = b > 3e38f ? 3e38f : b < -3e38f ? -3e38f : b;
    return pair(a, b);
}
template <class S>
__device__ __forceinline__ void load_decay(const ScanParams &Q, const ScanPlace<S> &at, int k, int swap, f2 (&v)[S::NP]) {
    if (Q.a_type == kElemF32) {
        load_states<S>(static_cast<const float *>(Q.a) + static_cast<long long>(at.channel + k) * Q.states, at.part, Q.states,
                       at.live[k], swap, v);
    } else {
#pragma unroll
        for (int r = 0; r < S::R; r += 4) {
            float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const int first = at.part * S::R + r, left = at.live[k] ? min(Q.states - first, S::R - r) : 0;
            const long long i = static_cast<long long>(at.channel + k) * Q.states + first;
            if (left > 0) f.x = load_param(Q.a, Q.a_type, i);
            if (left > 1) f.y = load_param(Q.a, Q.a_type, i + 1);
            if (left > 2) f.z = load_param(Q.a, Q.a_type, i + 2);
            if (left > 3) f.w = load_param(Q.a, Q.a_type, i + 3);
            f = reorder(f, swap);
            v[r / 2] = pair(f.x, f.y);
            if constexpr (S::NP > 1) v[r / 2 + 1] = pair(f.z, f.w);
        }
    }
#pragma unroll
    for (int i = 0; i < S::NP; ++i) v[i] = decay_exponent(v[i]);
}
// The states of a thread's own place, in its order.
template <class S>
__device__ __forceinline__ void own_states(float4 f, int swap, f2 (&v)[S::NP]) {
    f = reorder(f, swap);
    v[0] = pair(f.x, f.y);
    if constexpr (S::NP > 1) v[1] = pair(f.z, f.w);
}
// Element (or, where `vec`, both at once) of the two channels from p.
template <class T>
__device__ __forceinline__ void store_two(T *p, bool vec, const bool (&live)[2], float a, float b) {
    if (vec && live[1]) {  // pairs lie on pairs
        struct alignas(2 * sizeof(T)) Two {
            T a, b;
        };
        *reinterpret_cast<Two *>(p) = Two{from_float<T>(a), from_float<T>(b)};
    } else {
        if (live[0]) p[0] = from_float<T>(a);
        if (live[1]) p[1] = from_float<T>(b);
    }
}
// A lane's states of a token from shared memory.
template <class S>
__device__ __forceinline__ void tile_states(const float *p, f2 (&v)[S::NP]) {
    if constexpr (S::R >= 4) {
#pragma unroll
        for (int i = 0; i < S::NP; i += 2) {
            const float4 f = *reinterpret_cast<const float4 *>(p + 2 * i);
            v[i] = pair(f.x, f.y);
            v[i + 1] = pair(f.z, f.w);
        }
    } else {
        v[0] = pair(*p, 0.0f);
    }
}

// The copies of a tile: fours of channels of NT tensors, and quads of the states
// of B (PB) and C (PC).  A thread reads only what it copied itself, so that no
// barrier is needed, and the copies take no registers while they are under way;
// tensors that cannot be copied in groups are read directly.
template <class T, class S, int NT, int NP>
struct ScanRaw {
    static constexpr int NQ = (NP * S::T * S::QUADS + S::THREADS - 1) / S::THREADS;
    Four<T> four[NT][S::NG][S::THREADS];
    Four<T> quad[NQ][S::THREADS];
};
template <class T, class S, int NT, bool PB, bool PC>
struct ScanFetch {
    static constexpr int NP = PB + PC, ROWS = S::THREADS / S::GROUPS;  // ROWS: tokens that the threads take at once
    using Raw = ScanRaw<T, S, NT, NP>;
    TokenView in[NT], b, c;
    const ScanPlace<S> &at;
    int gc, valid, row;   // the thread's first channel in the block, how many of its four there are, its first token
    int states;
    bool vec, bvec;
    __device__ __forceinline__ ScanFetch(const ScanParams &Q, const ScanPlace<S> &place) : b(Q.b), c(Q.c), at(place) {
        gc = (threadIdx.x % S::GROUPS) * 4;
        valid = at.count - gc;
        row = threadIdx.x / S::GROUPS;
        states = Q.states;
        vec = Q.vec;
        bvec = Q.bvec;
    }
    __device__ __forceinline__ const T *four_at(int k, int g, long long t0) const {
        return static_cast<const T *>(in[k].p) + at.n * in[k].ldn + (t0 + row + g * ROWS) * in[k].ldt + at.first + gc;
    }
    __device__ __forceinline__ static bool is_b(int id) { return PB && (!PC || id < S::T * S::QUADS); }
    __device__ __forceinline__ const T *quad_at(int id, long long t0, int t, int s) const {
        return is_b(id) ? static_cast<const T *>(b.p) + at.n * b.ldn + (t0 + t) * b.ldt + at.group * b.ldg + s
                        : static_cast<const T *>(c.p) + at.n * c.ldn + (t0 + t) * c.ldt + at.group * c.ldg + s;
    }
    // tokens: from t0 on, of which a tile is copied at most
    __device__ __forceinline__ void start(Raw &raw, long long t0, int tokens) const {
        if (vec && valid > 0) {
#pragma unroll
            for (int g = 0; g < S::NG; ++g) {
                const int t = row + g * ROWS;
                if (t < tokens && (S::NG * ROWS <= S::T || t < S::T)) {  // threads may be more than a tile's tokens need
#pragma unroll
                    for (int k = 0; k < NT; ++k)
                        if (in[k].p != nullptr) copy_four<T>(&raw.four[k][g][threadIdx.x], four_at(k, g, t0));
                }
            }
        }
        if (bvec) {
#pragma unroll
            for (int i = 0; i < Raw::NQ; ++i) {
                const int id = threadIdx.x + i * S::THREADS, t = id / S::QUADS % S::T, s = id % S::QUADS * 4;
                if (id < NP * S::T * S::QUADS && t < tokens && s < states)
                    copy_four<T>(&raw.quad[i][threadIdx.x], quad_at(id, t0, t, s));
            }
        }
        cp_async_commit();
    }
    // four channels of tensor k at the thread's g-th token, which is one of the tile's
    __device__ __forceinline__ void four(const Raw &raw, int k, int g, long long t0, f2 (&v)[2]) const {
        Four<T> f;
        if (vec && valid > 0) f = raw.four[k][g][threadIdx.x];
        else f = load_four<T>(four_at(k, g, t0), false, valid);
        floats_of<T>(f, v);
    }
    // put(is B, token, first state, four states) for every quad of the tile; zeros where there are none
    template <class F>
    __device__ __forceinline__ void quads(const Raw &raw, long long t0, int tokens, F put) const {
#pragma unroll
        for (int i = 0; i < Raw::NQ; ++i) {
            const int id = threadIdx.x + i * S::THREADS, t = id / S::QUADS % S::T, s = id % S::QUADS * 4;
            if (id >= NP * S::T * S::QUADS) continue;
            f2 v[2] = {pair(0.0f), pair(0.0f)};
            if (t < tokens && s < states) {
                Four<T> f;
                if (bvec) f = raw.quad[i][threadIdx.x];
                else f = load_four<T>(quad_at(id, t0, t, s), false, states - s);
                floats_of<T>(f, v);
            }
            float4 w;
            split(v[0], w.x, w.y);
            split(v[1], w.z, w.w);
            put(is_b(id), t, s, w);
        }
    }
};

// Sums of four values over the P lanes of a channel.  The lanes share the work:
// afterwards lane p < 4 of a channel has the sums first .. first + N - 1 in v.
template <int P>
struct FourSums {
    static constexpr int N = P == 1 ? 4 : P == 2 ? 2 : 1;
    __device__ __forceinline__ static int first(int part) { return P == 1 ? 0 : P == 2 ? 2 * part : 2 * (part & 1) + (part >> 1 & 1); }
    __device__ __forceinline__ static void sum(float (&v)[4], int part) {
        if constexpr (P >= 2) {
            const bool up = part & 1;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float send = up ? v[i] : v[i + 2], keep = up ? v[i + 2] : v[i];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, send, 1);
            }
        }
        if constexpr (P >= 4) {
            const bool up = part & 2;
            const float send = up ? v[0] : v[1], keep = up ? v[1] : v[0];
            v[0] = keep + __shfl_xor_sync(0xffffffffu, send, 2);
        }
#pragma unroll
        for (int o = 4; o < P; o *= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
};

// The exponent of what v has grown by over many tokens: 0 where v is, which an infinite
// growth (A > 0) would make no number.
__device__ __forceinline__ f2 growth(f2 exponent, f2 v) {
    float a, b, x, y;
    split(exponent, a, b);
    split(v, x, y);
    return pair(x == 0.0f ? 0.0f : a, y == 0.0f ? 0.0f : b);
}
template <class T>
__device__ __forceinline__ T *token_at(const TokenView &v, long long n, long long t) {
    return static_cast<T *>(const_cast<void *>(v.p)) + n * v.ldn + t * v.ldt;
}

// The state (or, backwards, its gradient) after the segments first, first + step, ..
// before `stop`: each adds what it adds to what its decay leaves.  Four segments'
// effects are loaded at once.
template <class S>
__device__ __forceinline__ void pass_segments(const ScanParams &Q, const ScanPlace<S> &at, int k, int swap, int first, int count,
                                              int step, const f2 (&a2)[S::NP], f2 (&h)[S::NP]) {
    for (int j0 = 0; j0 < count; j0 += 4) {
        f2 e[4][S::NP];
        float sum[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool any = at.live[k] && j0 + j < count;
            const long long row = (at.n * Q.segs + first + (j0 + j) * step) * Q.channels + at.channel + k;
            load_states<S>(Q.carry + row * Q.states, at.part, Q.states, any, swap, e[j]);
            sum[j] = any ? Q.sums[row] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j0 + j >= count) continue;
#pragma unroll
            for (int i = 0; i < S::NP; ++i) h[i] = fma2(exp2_fast(growth(pair(sum[j]) * a2[i], h[i])), h[i], e[j][i]);
        }
    }
}

enum ScanMode { kScanMain, kScanCarry, kScanCarryBack };

// ---- forward ------------------------------------------------------------------------------
template <class T, class S, int MODE>
struct ScanTile {
    static constexpr bool kMain = MODE == kScanMain, kB = MODE != kScanCarryBack, kC = MODE != kScanCarry;
    using Fetch = ScanFetch<T, S, MODE == kScanCarry ? 2 : 3, kB, kC>;
    typename Fetch::Raw raw;
    float4 du[2][S::T][S::PAIRS];                           // delta, delta x (backwards f) of two channels
    float4 ep[kMain ? 2 : 1][kMain ? S::T : 1][S::PAIRS];   // D x, gate
    float bc[2][kMain ? 2 : 1][S::T][S::SP];
};

// kScanMain       y and the last state, the states for the gradient where wanted
// kScanCarry      a segment's effect on the state: what it adds, sum of deltas
// kScanCarryBack  a segment's effect on the gradient of the state behind it
// Two buffers and one barrier a tile: a tile's values are formed after the one
// before has been worked on, from copies that were under way meanwhile.  Tiles are
// filled up with steps of size 0.
// The bounds hold registers down; what fits a multiprocessor is up to shared memory as
// well.  At 16 states in 16 bits that is eight blocks of the main kernel, whose bound is
// ten: N4 L2048 C2048 bf16, whole call, 244 us with 96 registers, 252 with 80 (twelve), 250
// with 96 otherwise arranged (nine), 231 with 128 (eight).  The other modes would take 240
// and get 168, six blocks (N1 L8192 C2048 S16 bf16, whole call: 257 us left to itself, 245
// so, 261 with 128, 272 with 72; the training step of N4 L2048 C2048 771, 738, 745, 737).
template <class E, class S, int MODE>
__global__ void __launch_bounds__(S::THREADS, S::P < 4 ? 8 : MODE == kScanMain ? 10 : 6) scan_kernel(const __grid_constant__ ScanParams Q) {
    constexpr int P = S::P, R = S::R, NP = S::NP, T = S::T, N = FourSums<P>::N;
    using Tile = ScanTile<E, S, MODE>;
    extern __shared__ __align__(16) char space[];
    Tile &sm = *reinterpret_cast<Tile *>(space);
    griddep_wait();
    griddep_launch_dependents();
    const ScanPlace<S> at(Q);
    // the effect of the last segment, backwards the first, reaches no other one
    if (MODE != kScanMain && at.seg == (MODE == kScanCarry ? Q.segs - 1 : 0)) return;
    typename Tile::Fetch fetch(Q, at);
    fetch.in[0] = Q.dt;
    if constexpr (MODE == kScanCarryBack) fetch.in[1] = Q.dy;
    else fetch.in[1] = Q.x;
    if constexpr (MODE != kScanCarry) fetch.in[2] = Q.z;
    const int gc = fetch.gc, valid = fetch.valid;
    long long t0 = at.begin;
    int left = static_cast<int>(max(0LL, at.end - t0));  // tokens from the tile on
    fetch.start(sm.raw, t0, left);

    f2 a2[2][NP], h[2][NP];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        load_decay<S>(Q, at, k, 0, a2[k]);
#pragma unroll
        for (int i = 0; i < NP; ++i) h[k][i] = pair(0.0f);
        if (MODE != kScanMain) continue;
        if (Q.state != nullptr)
            load_states<S>(Q.state + at.n * Q.s_ldn + (at.channel + k) * Q.s_ldc, at.part, Q.states, at.live[k], 0, h[k]);
        pass_segments<S>(Q, at, k, 0, 0, at.seg, 1, a2[k], h[k]);
    }
    f2 bias[2], skip[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float b[2] = {}, d[2] = {};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (Q.bias != nullptr && 2 * i + k < valid) b[k] = load_param(Q.bias, Q.bias_type, at.first + gc + 2 * i + k);
            if (MODE == kScanMain && Q.d != nullptr && 2 * i + k < valid) d[k] = load_param(Q.d, Q.d_type, at.first + gc + 2 * i + k);
        }
        bias[i] = pair(b[0], b[1]);
        skip[i] = pair(d[0], d[1]);
    }
    const bool gated = MODE != kScanCarry && Q.z.p != nullptr, softplus = Q.softplus;
    // the values of a tile whose copies have arrived
    const auto form = [&](long long t0, int tokens, int buf) {
        cp_async_wait<0>();
#pragma unroll
        for (int g = 0; g < S::NG; ++g) {
            const int t = fetch.row + g * Tile::Fetch::ROWS;
            if (t >= T) continue;
            f2 delta[2] = {pair(0.0f), pair(0.0f)}, u[2] = {pair(0.0f), pair(0.0f)};
            f2 gate[2] = {pair(1.0f), pair(1.0f)}, dx[2] = {pair(0.0f), pair(0.0f)};
            if (t < tokens) {
                f2 raw[2], x[2], slope[2];
                fetch.four(sm.raw, 0, g, t0, raw);
                fetch.four(sm.raw, 1, g, t0, x);
                scan_deltas<false>(softplus, raw, bias, delta, slope);
                if constexpr (MODE != kScanCarry) {
                    if (gated) {
                        f2 z[2];
                        fetch.four(sm.raw, 2, g, t0, z);
#pragma unroll
                        for (int i = 0; i < 2; ++i) gate2<false>(z[i], gate[i], slope[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    u[i] = x[i] * (MODE == kScanCarryBack ? gate[i] : delta[i]);
                    dx[i] = x[i] * skip[i];
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float4 w;
                split(delta[i], w.x, w.z);
                split(u[i], w.y, w.w);
                sm.du[buf][t][i * S::ODD + gc / 4] = w;
                if constexpr (MODE == kScanMain) {
                    split(dx[i], w.x, w.z);
                    split(gate[i], w.y, w.w);
                    sm.ep[buf][t][i * S::ODD + gc / 4] = w;
                }
            }
        }
        fetch.quads(sm.raw, t0, tokens, [&](bool is_b, int t, int s, const float4 &v) {
            float *p = &sm.bc[buf][MODE == kScanMain && !is_b ? 1 : 0][t][s];
            if constexpr (R >= 4) *reinterpret_cast<float4 *>(p) = v;
            else *p = v.x;
        });
    };
    form(t0, left, 0);
    fetch.start(sm.raw, t0 + T, left - T);
    float sum[2] = {0.0f, 0.0f};  // of the deltas
    const long long chunks = (Q.l + kScanChunk - 1) / kScanChunk;
    float *kept = Q.kept + ((at.n * chunks + at.begin / kScanChunk) * Q.channels + at.channel) * Q.states;
    const bool writes = at.part < 4, vec = Q.vec;
    const int place = S::place(at.chan);
    for (int buf = 0; left > 0; left -= T, t0 += T, buf ^= 1) {
        __syncthreads();
        E *y_at = token_at<E>(Q.y, at.n, t0 + FourSums<P>::first(at.part)) + at.channel;  // the lane's token of each four
        const float4 *du = &sm.du[buf][0][place];
        const float *b = &sm.bc[buf][0][0][at.part * R], *c = &sm.bc[buf][MODE == kScanMain ? 1 : 0][0][at.part * R];
#pragma unroll
        for (int t4 = 0; t4 < T; t4 += 4) {
            if (MODE == kScanMain && t4 % kScanChunk == 0 && Q.kept != nullptr && t4 < left) {
#pragma unroll
                for (int k = 0; k < 2; ++k) store_states<S>(kept + k * Q.states, at.part, Q.states, at.live[k], 0, h[k]);
                kept += static_cast<long long>(Q.channels) * Q.states;
            }
            float y[2][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = t4 + j;
                const float4 v = du[t * S::PAIRS];
                const float delta[2] = {v.x, v.z}, u[2] = {v.y, v.w};
                float since[2];  // the segment's deltas so far, where f is not 0 (an infinite growth of nothing is nothing)
                f2 wb[NP], wc[NP];
                tile_states<S>(b + t * S::SP, wb);
                if constexpr (MODE == kScanMain) tile_states<S>(c + t * S::SP, wc);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if constexpr (MODE != kScanMain) sum[k] += delta[k];
                    since[k] = MODE != kScanCarryBack || u[k] == 0.0f ? 0.0f : sum[k];
                    if constexpr (MODE == kScanCarryBack) {
#pragma unroll
                        for (int i = 0; i < NP; ++i) h[k][i] = fma2(exp2_fast(pair(since[k]) * a2[k][i]), pair(u[k]) * wb[i], h[k][i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < NP; ++i) h[k][i] = fma2(exp2_fast(pair(delta[k]) * a2[k][i]), h[k][i], pair(u[k]) * wb[i]);
                    }
                    if constexpr (MODE == kScanMain) {
                        f2 p = wc[0] * h[k][0];
#pragma unroll
                        for (int i = 1; i < NP; ++i) p = fma2(wc[i], h[k][i], p);
                        y[k][j] = sum_of(p);
                    }
                }
            }
            if constexpr (MODE == kScanMain) {
                FourSums<P>::sum(y[0], at.part);
                FourSums<P>::sum(y[1], at.part);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int t = t4 + FourSums<P>::first(at.part) + i;
                    if (writes && t < left) {
                        const float4 e = sm.ep[buf][t][place];
                        store_two<E>(y_at + i * Q.y.ldt, vec, at.live, (y[0][i] + e.x) * e.y, (y[1][i] + e.z) * e.w);
                    }
                }
                y_at += 4 * Q.y.ldt;
            }
            asm volatile("" ::: "memory");  // loads of later tokens stay behind: their registers are the states'
        }
        if (left > T) {
            form(t0 + T, left - T, buf ^ 1);
            fetch.start(sm.raw, t0 + 2 * T, left - 2 * T);
        }
    }
    cp_async_wait<0>();
    if (MODE == kScanMain) {
        if (Q.state_out != nullptr && at.seg == Q.segs - 1)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                store_states<S>(Q.state_out + at.n * Q.so_ldn + (at.channel + k) * Q.so_ldc, at.part, Q.states, at.live[k], 0, h[k]);
        for (long long i = max(at.end, at.begin) * S::GROUPS + threadIdx.x; i < at.stop * S::GROUPS; i += S::THREADS) {
            const int c0 = static_cast<int>(i % S::GROUPS) * 4;
            store_zeros<E>(token_at<E>(Q.y, at.n, i / S::GROUPS) + at.first + c0, Q.vec, at.count - c0);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const long long row = (at.n * Q.segs + at.seg) * Q.channels + at.channel + k;
            store_states<S>(Q.carry + row * Q.states, at.part, Q.states, at.live[k], 0, h[k]);
            if (at.part == 0 && at.live[k]) Q.sums[row] = sum[k];
        }
    }
}

// ---- gradient -------------------------------------------------------------------------------
// Sums over the channels of a warp of what a lane has for B and for C, R values
// each.  Each step halves what a lane holds.  Lanes keep their states in an order
// of their own (place r holds state r ^ swap), so that in the first steps every
// lane sends the same places and nothing is selected.
template <class S>
struct ChannelSums {
    static constexpr int P = S::P, R = S::R;
    static constexpr bool kTwo = R == 4 && P <= 16, kOne = R == 4 && P <= 8, kSides = P <= 4;
    static constexpr int LEFT = !kTwo ? R : !kOne ? 2 : 1;  // of B and of C, before the sides are shared
    __device__ __forceinline__ static int swap(int lane) { return (kTwo && (lane & 16) ? 2 : 0) | (kOne && (lane & 8) ? 1 : 0); }
    // b, c: what the lane has; store(place in [2][SP], value)
    template <class F>
    __device__ __forceinline__ static void sum(float (&b)[4], float (&c)[4], int lane, int part, F store) {
        if constexpr (kTwo) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                b[r] += __shfl_xor_sync(0xffffffffu, b[r + 2], 16);
                c[r] += __shfl_xor_sync(0xffffffffu, c[r + 2], 16);
            }
        }
        if constexpr (kOne) {
            b[0] += __shfl_xor_sync(0xffffffffu, b[1], 8);
            c[0] += __shfl_xor_sync(0xffffffffu, c[1], 8);
        }
        // place 0 of a lane now holds state 0 ^ swap
        const int s = part * R;
        if constexpr (kSides) {  // one lane takes B, its neighbour C
            constexpr int O = R == 4 ? 4 : 16;
            const bool up = (lane & O) != 0;
            float v = (up ? c[0] : b[0]) + __shfl_xor_sync(0xffffffffu, up ? b[0] : c[0], O);
            bool writes = true;
#pragma unroll
            for (int o = R == 4 ? 2 : 8; o >= P; o /= 2) {
                v += __shfl_xor_sync(0xffffffffu, v, o);
                writes = writes && (lane & o) == 0;
            }
            if (writes) store((up ? S::SP : 0) + s + swap(lane), v);
        } else {
#pragma unroll
            for (int r = 0; r < LEFT; ++r) {
                store(s + (r ^ swap(lane)), b[r]);
                store(S::SP + s + (r ^ swap(lane)), c[r]);
            }
        }
    }
};

template <class T, class S>
struct ScanGradTile {
    static constexpr int PITCH = S::T * S::SP + 16;  // of a copy in another order: apart in the banks
    using Fetch = ScanFetch<T, S, 4, true, true>;
    typename Fetch::Raw raw;
    float4 du[S::T][S::PAIRS];         // delta, delta x of two channels
    float4 e[S::T][S::PAIRS];          // slope of delta, dy times the gate's slope
    alignas(16) float f[S::T][S::CB + 8], x[S::T][S::CB + 8];
    alignas(16) float bc[2][S::R][PITCH];  // B and C in the orders that lanes keep
    alignas(16) float red[S::THREADS / 32][S::T][2 * S::SP];
    // a thread's own: the states in front of this tile and the next, bias of its four
    // channels, sums for D and dt_bias of its two
    float4 kept[2][2][S::THREADS], bias[S::THREADS], sums[S::THREADS];
};

// Tiles of 8 tokens, from a segment's last to its first.  A tile's states are
// formed once more from the state kept in front of it and stay in registers for
// the way back; the decays are formed twice (kept too they would take the
// registers of half of the warps).
template <class E, class S>
__global__ void __launch_bounds__(S::THREADS, 512 / S::THREADS) scan_grad_kernel(const __grid_constant__ ScanParams Q) {
    constexpr int P = S::P, R = S::R, NP = S::NP, T = S::T, WARPS = S::THREADS / 32, N = FourSums<P>::N;
    using Tile = ScanGradTile<E, S>;
    using Sums = ChannelSums<S>;
    extern __shared__ __align__(16) char space[];
    Tile &sm = *reinterpret_cast<Tile *>(space);
    griddep_wait();
    griddep_launch_dependents();
    const ScanPlace<S> at(Q);
    const bool gated = Q.z.p != nullptr, softplus = Q.softplus;
    const long long chunks = (Q.l + T - 1) / T;
    const int place = S::place(at.chan);
    // the states in front of a tile to the thread's own place
    const auto keep = [&](long long t0, int buf) {
        const bool whole = whole_states(Q.kept, Q.states);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int left = at.live[k] ? min(Q.states - at.part * R, R) : 0;
            const float *p = Q.kept + ((at.n * chunks + t0 / T) * Q.channels + at.channel + k) * Q.states + at.part * R;
            float4 &own = sm.kept[buf][k][threadIdx.x];
            if (R == 4 && whole && left > 0)
                cp_async_16(&own, p);
            else
                own = make_float4(left > 0 ? p[0] : 0.0f, left > 1 ? p[1] : 0.0f, left > 2 ? p[2] : 0.0f, left > 3 ? p[3] : 0.0f);
        }
    };
    // the last tile with tokens of the sequence, and how many tiles there are
    int tiles = at.end > at.begin ? static_cast<int>((at.end - at.begin + T - 1) / T) : 0;
    long long t0 = at.begin + (tiles - 1) * static_cast<long long>(T);
    int tokens = static_cast<int>(at.end - t0);
    typename Tile::Fetch fetch(Q, at);
    fetch.in[0] = Q.dt;
    fetch.in[1] = Q.x;
    fetch.in[2] = Q.dy;
    fetch.in[3] = Q.z;
    const int gc = fetch.gc, valid = fetch.valid, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int swap = Sums::swap(lane);
    if (tiles > 0) {
        keep(t0, 0);
        fetch.start(sm.raw, t0, tokens);
    }

    f2 a2[2][NP], q[2][NP], da[2][NP];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        load_decay<S>(Q, at, k, swap, a2[k]);
#pragma unroll
        for (int i = 0; i < NP; ++i) q[k][i] = da[k][i] = pair(0.0f);
        if (Q.dlast != nullptr)
            load_states<S>(Q.dlast + at.n * Q.dl_ldn + (at.channel + k) * Q.dl_ldc, at.part, Q.states, at.live[k], swap, q[k]);
        pass_segments<S>(Q, at, k, swap, Q.segs - 1, Q.segs - 1 - at.seg, -1, a2[k], q[k]);
    }
    {
        float b[4] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (Q.bias != nullptr && i < valid) b[i] = load_param(Q.bias, Q.bias_type, at.first + gc + i);
        sm.bias[threadIdx.x] = make_float4(b[0], b[1], b[2], b[3]);
        sm.sums[threadIdx.x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    float skip[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) skip[k] = Q.d != nullptr && at.live[k] ? load_param(Q.d, Q.d_type, at.channel + k) : 0.0f;
    const bool writes = at.part < 4, vec = Q.vec;
    // A run's sums to its row of the partial results, and the next run's from 0.
    const auto end_run = [&](int run) {
        const long long row = (at.n * Q.segs + at.seg) * Q.runs + run;
        const float4 own = sm.sums[threadIdx.x];
        float dskip[2] = {own.x, own.y}, dbias[2] = {own.z, own.w};
        sm.sums[threadIdx.x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (Q.part_a != nullptr)
                store_states<S>(Q.part_a + (row * Q.channels + at.channel + k) * Q.states, at.part, Q.states, at.live[k], swap, da[k]);
#pragma unroll
            for (int i = 0; i < NP; ++i) da[k][i] = pair(0.0f);
            if (Q.part_d == nullptr) continue;
#pragma unroll
            for (int o = 1; o < P; o *= 2) {
                dskip[k] += __shfl_xor_sync(0xffffffffu, dskip[k], o);
                dbias[k] += __shfl_xor_sync(0xffffffffu, dbias[k], o);
            }
            if (at.part == 0 && at.live[k]) {
                Q.part_d[row * 2 * Q.channels + at.channel + k] = dskip[k];
                Q.part_d[(row * 2 + 1) * Q.channels + at.channel + k] = dbias[k];
            }
        }
    };
    for (int run = (tiles + kScanRun - 1) / kScanRun; run < Q.runs; ++run) end_run(run);  // behind the sequence's end

    for (int buf = 0; tiles > 0; --tiles, t0 -= T, tokens = T, buf ^= 1) {
        f2 h[T][2][NP];
        cp_async_wait<0>();
#pragma unroll
        for (int g = 0; g < S::NG; ++g) {
            const int t = fetch.row + g * Tile::Fetch::ROWS;
            if (t >= T) continue;
            f2 delta[2], slope[2], x[2], f[2], w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) delta[i] = slope[i] = x[i] = f[i] = w[i] = pair(0.0f);
            if (t < tokens) {
                const float4 b4 = sm.bias[threadIdx.x];
                const f2 bias[2] = {pair(b4.x, b4.y), pair(b4.z, b4.w)};
                f2 raw[2];
                fetch.four(sm.raw, 0, g, t0, raw);
                fetch.four(sm.raw, 1, g, t0, x);
                fetch.four(sm.raw, 2, g, t0, f);
                scan_deltas<true>(softplus, raw, bias, delta, slope);
                if (gated) {
                    f2 z[2], gate, gslope;
                    fetch.four(sm.raw, 3, g, t0, z);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        gate2<true>(z[i], gate, gslope);
                        w[i] = f[i] * gslope;
                        f[i] = f[i] * gate;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float4 d, e;
                split(delta[i], d.x, d.z);
                split(delta[i] * x[i], d.y, d.w);
                split(slope[i], e.x, e.z);
                split(w[i], e.y, e.w);
                sm.du[t][i * S::ODD + gc / 4] = d;
                sm.e[t][i * S::ODD + gc / 4] = e;
            }
            float4 f4, x4;
            split(f[0], f4.x, f4.y);
            split(f[1], f4.z, f4.w);
            split(x[0], x4.x, x4.y);
            split(x[1], x4.z, x4.w);
            *reinterpret_cast<float4 *>(&sm.f[t][gc]) = f4;
            *reinterpret_cast<float4 *>(&sm.x[t][gc]) = x4;
        }
        fetch.quads(sm.raw, t0, tokens, [&](bool is_b, int t, int s, const float4 &v) {
            float *p = &sm.bc[is_b ? 0 : 1][0][t * S::SP + s];
            if constexpr (R == 4) {
                *reinterpret_cast<float4 *>(p) = v;
                if constexpr (Sums::kOne) *reinterpret_cast<float4 *>(p + Tile::PITCH) = make_float4(v.y, v.x, v.w, v.z);
                if constexpr (Sums::kTwo) *reinterpret_cast<float4 *>(p + 2 * Tile::PITCH) = make_float4(v.z, v.w, v.x, v.y);
                if constexpr (Sums::kOne) *reinterpret_cast<float4 *>(p + 3 * Tile::PITCH) = make_float4(v.w, v.z, v.y, v.x);
            } else {
                *p = v.x;
            }
        });
        __syncthreads();
        if (tiles > 1) {
            keep(t0 - T, buf ^ 1);
            fetch.start(sm.raw, t0 - T, T);
        }
        const auto before = [&](int k, f2 (&v)[NP]) { own_states<S>(sm.kept[buf][k][threadIdx.x], swap, v); };
        const float *b = &sm.bc[0][R == 4 ? swap : 0][at.part * R], *c = &sm.bc[1][R == 4 ? swap : 0][at.part * R];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const float4 v = sm.du[t][place];
            const float delta[2] = {v.x, v.z}, u[2] = {v.y, v.w};
            f2 w[NP];
            tile_states<S>(b + t * S::SP, w);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                f2 last[NP];
                if (t == 0) before(k, last);
#pragma unroll
                for (int i = 0; i < NP; ++i)
                    h[t][k][i] = fma2(exp2_fast(pair(delta[k]) * a2[k][i]), t == 0 ? last[i] : h[t == 0 ? 0 : t - 1][k][i],
                                      pair(u[k]) * w[i]);
            }
            // loads of later tokens stay behind: their registers are the states'
            if (t % 4 == 3) asm volatile("" ::: "memory");
        }
        f2 da1[2][NP];  // sums of this tile
        float dskip1[2] = {0.0f, 0.0f}, dbias1[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NP; ++i) da1[0][i] = da1[1][i] = pair(0.0f);
#pragma unroll
        for (int t4 = T - 4; t4 >= 0; t4 -= 4) {
            float qb[2][4], qa[2][4], y[2][4];  // q . B, (q a h) . A, C . h
#pragma unroll
            for (int j = 3; j >= 0; --j) {
                const int t = t4 + j;
                const float4 v = sm.du[t][place];
                const float2 f2v = *reinterpret_cast<const float2 *>(&sm.f[t][at.chan]);
                const float delta[2] = {v.x, v.z}, u[2] = {v.y, v.w}, f[2] = {f2v.x, f2v.y};
                f2 wb[NP], wc[NP], gb[NP], gc2[NP];
                tile_states<S>(c + t * S::SP, wc);
                tile_states<S>(b + t * S::SP, wb);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    f2 sb, sa, sy, last[NP];
                    if (t == 0) before(k, last);
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        q[k][i] = fma2(pair(f[k]), wc[i], q[k][i]);
                        gb[i] = k == 0 ? q[k][i] * pair(u[k]) : fma2(q[k][i], pair(u[k]), gb[i]);
                        gc2[i] = k == 0 ? h[t][k][i] * pair(f[k]) : fma2(h[t][k][i], pair(f[k]), gc2[i]);
                        sb = i == 0 ? q[k][0] * wb[0] : fma2(q[k][i], wb[i], sb);
                        sy = i == 0 ? h[t][k][0] * wc[0] : fma2(h[t][k][i], wc[i], sy);
                        q[k][i] = q[k][i] * exp2_fast(pair(delta[k]) * a2[k][i]);
                        const f2 m = q[k][i] * (t == 0 ? last[i] : h[t == 0 ? 0 : t - 1][k][i]);
                        sa = i == 0 ? m * a2[k][0] : fma2(m, a2[k][i], sa);
                        da1[k][i] = fma2(m, pair(delta[k]), da1[k][i]);
                    }
                    qb[k][j] = sum_of(sb);
                    qa[k][j] = sum_of(sa);
                    y[k][j] = sum_of(sy);
                }
                float gbv[4], gcv[4];
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    split(gb[i], gbv[2 * i], gbv[2 * i + 1]);
                    split(gc2[i], gcv[2 * i], gcv[2 * i + 1]);
                }
                Sums::sum(gbv, gcv, lane, at.part, [&](int p, float s) { sm.red[warp][t][p] = s; });
                asm volatile("" ::: "memory");
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                FourSums<P>::sum(qb[k], at.part);
                FourSums<P>::sum(qa[k], at.part);
                if (gated) FourSums<P>::sum(y[k], at.part);
            }
            const long long row = t0 + t4 + FourSums<P>::first(at.part);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int t = t4 + FourSums<P>::first(at.part) + i;
                if (writes && t < tokens) {
                    const float4 e = sm.e[t][place], d = sm.du[t][place];
                    const float2 ff = *reinterpret_cast<const float2 *>(&sm.f[t][at.chan]);
                    const float2 xx = *reinterpret_cast<const float2 *>(&sm.x[t][at.chan]);
                    const float delta[2] = {d.x, d.z}, f[2] = {ff.x, ff.y}, x[2] = {xx.x, xx.y};
                    const float slope[2] = {e.x, e.z}, w[2] = {e.y, e.w};
                    float dx[2], ddt[2], dz[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        dx[k] = fmaf(delta[k], qb[k][i], skip[k] * f[k]);
                        // qa holds A log2(e), not A
                        ddt[k] = fmaf(x[k], qb[k][i], qa[k][i] * (1.0f / kLog2E)) * slope[k];
                        dz[k] = w[k] * fmaf(skip[k], x[k], y[k][i]);
                        dskip1[k] = fmaf(f[k], x[k], dskip1[k]);
                        dbias1[k] += ddt[k];
                    }
                    store_two<E>(token_at<E>(Q.dx, at.n, row + i) + at.channel, vec, at.live, dx[0], dx[1]);
                    store_two<E>(token_at<E>(Q.ddt, at.n, row + i) + at.channel, vec, at.live, ddt[0], ddt[1]);
                    if (gated) store_two<E>(token_at<E>(Q.dz, at.n, row + i) + at.channel, vec, at.live, dz[0], dz[1]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int i = 0; i < NP; ++i) da[k][i] = da[k][i] + da1[k][i];
        }
        {
            const float4 v = sm.sums[threadIdx.x];
            sm.sums[threadIdx.x] = make_float4(v.x + dskip1[0], v.y + dskip1[1], v.z + dbias1[0], v.w + dbias1[1]);
        }
        if ((tiles - 1) % kScanRun == 0) end_run((tiles - 1) / kScanRun);
        __syncthreads();
        float *part = Q.part_bc + (((at.tile * Q.n + at.n) * Q.l + t0) * Q.groups + at.group) * 2 * Q.states;
        const long long next = static_cast<long long>(Q.groups) * 2 * Q.states;  // a token further
        if (R == 4 && Q.states % 4 == 0) {
            for (int i = threadIdx.x; i < tokens * 2 * S::QUADS; i += S::THREADS) {
                const int t = i / (2 * S::QUADS), j = i % (2 * S::QUADS) * 4, s = j % S::SP;
                if (s >= Q.states) continue;
                float4 sum = *reinterpret_cast<const float4 *>(&sm.red[0][t][j]);
#pragma unroll
                for (int w = 1; w < WARPS; ++w) {
                    const float4 v = *reinterpret_cast<const float4 *>(&sm.red[w][t][j]);
                    sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
                }
                *reinterpret_cast<float4 *>(part + t * next + (j / S::SP) * Q.states + s) = sum;
            }
        } else {
            for (int i = threadIdx.x; i < tokens * 2 * S::SP; i += S::THREADS) {
                const int t = i / (2 * S::SP), j = i % (2 * S::SP), s = j % S::SP;
                if (s >= Q.states) continue;
                float sum = sm.red[0][t][j];
#pragma unroll
                for (int w = 1; w < WARPS; ++w) sum += sm.red[w][t][j];
                part[t * next + (j / S::SP) * Q.states + s] = sum;
            }
        }
    }
    const auto zeros = [&](const TokenView &w) {
        if (w.p == nullptr) return;
        for (long long i = max(at.end, at.begin) * S::GROUPS + threadIdx.x; i < at.stop * S::GROUPS; i += S::THREADS) {
            const int c0 = static_cast<int>(i % S::GROUPS) * 4;
            store_zeros<E>(token_at<E>(w, at.n, i / S::GROUPS) + at.first + c0, Q.vec, at.count - c0);
        }
    };
    zeros(Q.dx);
    zeros(Q.ddt);
    zeros(Q.dz);
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (Q.state_out != nullptr && at.seg == 0)
            store_states<S>(Q.state_out + at.n * Q.so_ldn + (at.channel + k) * Q.so_ldc, at.part, Q.states, at.live[k], swap, q[k]);
}

// dB and dC: the sums over the blocks that share a group's channels.
struct ScanJoinParams {
    const float *part;      // [tiles][rows][2][states], rows = n * l * groups
    long long rows, l;
    int tiles, states, groups, type;
    TokenView db, dc;       // p nullable
    const int *lengths;
};
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) scan_join_kernel(const __grid_constant__ ScanJoinParams Q);

// One token of every sequence: x, dt, z, y are [n][channels].  A thread has read its
// part of a state before it writes it, so state_out may be the state itself.
//
// WHOLE: every access of a thread is one access of 16, 8 or 4 bytes and nothing has
// to be asked: as many states as lanes have, blocks full of channels, parameters in
// 32 bits, a gate.  A step moves 76 bytes for each channel and part, and the
// general kernel's questions are five times its arithmetic (N64 C4096 bf16: 16 us
// there).
template <class E, class S, bool WHOLE>
__global__ void __launch_bounds__(S::THREADS) scan_step_kernel(const __grid_constant__ ScanParams Q) {
    constexpr int P = S::P, R = S::R, NP = S::NP;
    griddep_wait();
    griddep_launch_dependents();
    f2 a2[2][NP], h[2][NP], b[2], c[2];
    float x[2], dt[2], z[2], bias[2] = {}, skip[2] = {};
    long long n;
    int channel, part;
    bool live[2] = {true, true};
    if constexpr (WHOLE) {
        n = blockIdx.y;
        const int group = Q.groups == 1 ? 0 : static_cast<int>(blockIdx.x / static_cast<unsigned>(Q.tiles));
        channel = static_cast<int>(blockIdx.x * S::CB + threadIdx.x / P * 2);
        part = threadIdx.x % P;
        const int at = channel * S::SP + part * R;
        const auto two = [&](const TokenView &v, float (&e)[2]) {
            const E *p = static_cast<const E *>(v.p) + n * v.ldn + channel;
            E r[2];
            memcpy(r, __builtin_assume_aligned(p, 2 * sizeof(E)), 2 * sizeof(E));
            e[0] = to_float(r[0]);
            e[1] = to_float(r[1]);
        };
        const auto quad = [&](const float *p, f2 (&v)[NP]) {
            const float4 f = *reinterpret_cast<const float4 *>(p);
            v[0] = pair(f.x, f.y);
            v[NP - 1] = pair(f.z, f.w);
        };
        const float *state = Q.state + n * Q.s_ldn + at, *decay = static_cast<const float *>(Q.a) + at;
#pragma unroll
        for (int k = 0; k < 2; ++k) quad(state + k * S::SP, h[k]);
        two(Q.x, x);
        two(Q.dt, dt);
        two(Q.z, z);
        const E *pb = static_cast<const E *>(Q.b.p) + n * Q.b.ldn + group * Q.b.ldg + part * R;
        const E *pc = static_cast<const E *>(Q.c.p) + n * Q.c.ldn + group * Q.c.ldg + part * R;
        const Four<E> fb = load_four<E>(pb, true, 4), fc = load_four<E>(pc, true, 4);
        const float2 vb = *reinterpret_cast<const float2 *>(static_cast<const float *>(Q.bias) + channel);
        const float2 vd = *reinterpret_cast<const float2 *>(static_cast<const float *>(Q.d) + channel);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            quad(decay + k * S::SP, a2[k]);
#pragma unroll
            for (int i = 0; i < NP; ++i) a2[k][i] = decay_exponent(a2[k][i]);
        }
        floats_of<E>(fb, b);
        floats_of<E>(fc, c);
        bias[0] = vb.x, bias[1] = vb.y;
        skip[0] = vd.x, skip[1] = vd.y;
    } else {
        const ScanPlace<S> at(Q);
        n = at.n;
        channel = at.channel;
        part = at.part;
        const auto two = [&](const TokenView &v, float (&e)[2]) {
            const E *p = static_cast<const E *>(v.p) + n * v.ldn + channel;
#pragma unroll
            for (int k = 0; k < 2; ++k) e[k] = at.live[k] ? to_float(p[k]) : 0.0f;
        };
        const auto pairs = [&](const TokenView &v, f2 (&e)[2]) {
            const int s = part * R;
            floats_of<E>(load_four<E>(static_cast<const E *>(v.p) + n * v.ldn + at.group * v.ldg + s, false, min(Q.states - s, R)), e);
        };
        two(Q.x, x);
        two(Q.dt, dt);
        if (Q.z.p != nullptr) two(Q.z, z);
        pairs(Q.b, b);
        pairs(Q.c, c);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            live[k] = at.live[k];
            load_states<S>(Q.state + n * Q.s_ldn + (channel + k) * Q.s_ldc, part, Q.states, live[k], 0, h[k]);
            load_decay<S>(Q, at, k, 0, a2[k]);
            if (Q.bias != nullptr && live[k]) bias[k] = load_param(Q.bias, Q.bias_type, channel + k);
            if (Q.d != nullptr && live[k]) skip[k] = load_param(Q.d, Q.d_type, channel + k);
        }
    }
    f2 delta = pair(dt[0], dt[1]) + pair(bias[0], bias[1]), slope;
    if (Q.softplus) softplus2<false>(delta, delta, slope);
    float d[2], y[2], gate[2] = {1.0f, 1.0f};
    split(delta, d[0], d[1]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        f2 s = pair(0.0f);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            h[k][i] = fma2(exp2_fast(pair(d[k]) * a2[k][i]), h[k][i], pair(d[k] * x[k]) * b[i]);
            s = fma2(c[i], h[k][i], s);
        }
        y[k] = sum_of(s);
        float *out = Q.state_out + n * Q.so_ldn;
        if constexpr (WHOLE) {
            float4 f;
            split(h[k][0], f.x, f.y);
            split(h[k][NP - 1], f.z, f.w);
            *reinterpret_cast<float4 *>(out + channel * S::SP + part * R + k * S::SP) = f;
        } else {
            store_states<S>(out + (channel + k) * Q.so_ldc, part, Q.states, live[k], 0, h[k]);
        }
#pragma unroll
        for (int o = 1; o < P; o *= 2) y[k] += __shfl_xor_sync(0xffffffffu, y[k], o);
        y[k] = fmaf(skip[k], x[k], y[k]);
    }
    if (part != 0) return;
    if (WHOLE || Q.z.p != nullptr) {
        f2 g;
        gate2<false>(pair(z[0], z[1]), g, slope);
        split(g, gate[0], gate[1]);
    }
    store_two<E>(token_at<E>(Q.y, n, 0) + channel, WHOLE, live, y[0] * gate[0], y[1] * gate[1]);
}

// ---- instances, one translation unit for each element type -----------------------------------
enum ScanKernel { kMain, kCarry, kCarryBack, kGrad, kStep, kStepWhole };
struct ScanLaunch {
    const void *fn;
    int threads;
    size_t smem;
};
// Threads of a block of the gradient: what the tiles of few lanes take of shared
// memory grows with the channels of a block.
constexpr int kScanThreads = 64, kScanStates = 4;  // states of a lane: with 8 the scan was slower by a third
constexpr int grad_threads(int sp) { return sp >= 16 ? 128 : kScanThreads; }

template <class E, int SP>
ScanLaunch scan_instance(ScanKernel k) {
    // few lanes mean many channels a block, whose tiles take the shared memory of blocks
    using S = ScanShape<SP, kScanStates, kScanThreads, SP >= 16 ? 16 : 8>;
    using G = ScanShape<SP, kScanStates, grad_threads(SP), kScanChunk>;
    switch (k) {
    case kMain:
        return {reinterpret_cast<const void *>(&scan_kernel<E, S, kScanMain>), S::THREADS, sizeof(ScanTile<E, S, kScanMain>)};
    case kCarry:
        return {reinterpret_cast<const void *>(&scan_kernel<E, S, kScanCarry>), S::THREADS, sizeof(ScanTile<E, S, kScanCarry>)};
    case kCarryBack:
        return {reinterpret_cast<const void *>(&scan_kernel<E, S, kScanCarryBack>), S::THREADS,
                sizeof(ScanTile<E, S, kScanCarryBack>)};
    case kGrad: return {reinterpret_cast<const void *>(&scan_grad_kernel<E, G>), G::THREADS, sizeof(ScanGradTile<E, G>)};
    case kStepWhole:
        if constexpr (SP >= 4) return {reinterpret_cast<const void *>(&scan_step_kernel<E, S, true>), S::THREADS, 0};
        else return {nullptr, 0, 0};  // not planned
    default: return {reinterpret_cast<const void *>(&scan_step_kernel<E, S, false>), S::THREADS, 0};
    }
}
template <class E>
ScanLaunch scan_launch(ScanKernel k, int sp) {
    switch (sp) {
    case 1: return scan_instance<E, 1>(k);
    case 4: return scan_instance<E, 4>(k);
    case 8: return scan_instance<E, 8>(k);
    case 16: return scan_instance<E, 16>(k);
    case 32: return scan_instance<E, 32>(k);
    default: return scan_instance<E, 64>(k);
    }
}
extern template ScanLaunch scan_launch<float>(ScanKernel, int);
extern template ScanLaunch scan_launch<__half>(ScanKernel, int);
extern template ScanLaunch scan_launch<__nv_bfloat16>(ScanKernel, int);

}  // namespace gcb
