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
// states are spread over P lanes of R each; a block takes THREADS / P channels
// and walks along the tokens in tiles that are staged in shared memory, where
// softplus, gate and products of a token and channel are formed once for its P
// lanes.  Where sequences and channels alone are too few to fill the GPU, each
// sequence is cut into segments: a first launch gives each segment's effect on
// the state (what it adds, and the sum of its deltas, whose product with A is its
// decay's logarithm), from which every block forms the state that it starts with.
#pragma once
#include "norm_util.cuh"

namespace gcb {

// Tokens between the states that the forward pass keeps for the gradient, and
// that the gradient's kernel takes at a time.
constexpr int kScanChunk = 16;

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
    int type, vec, softplus;           // vec: four channels in one access
    int tiles;                         // blocks that share a group's channels
    long long seg_len;
    int segs;
    float *carry, *sums;               // [n][segs][channels][states], [n][segs][channels]
    float *kept;                       // [n][chunks][channels][states] or NULL
    float *part_bc;                    // gradient: [tile][n][l][groups][2][states]
    float *part_a, *part_d;            // [n * segs][channels][states], [n * segs][2][channels] (D, dt_bias)
};

// ---- four channels of a token -----------------------------------------------------------
struct Four {
    uint4 u;
};
__device__ __forceinline__ Four load_four(const void *p, int type, bool vec, long long at, int valid) {
    Four r;
    r.u = make_uint4(0u, 0u, 0u, 0u);
    if (valid <= 0) return r;
    if (type == kElemF32) {
        const float *q = static_cast<const float *>(p) + at;
        if (vec) {
            r.u = __ldg(reinterpret_cast<const uint4 *>(q));
        } else {
            r.u.x = __float_as_uint(q[0]);
            if (valid > 1) r.u.y = __float_as_uint(q[1]);
            if (valid > 2) r.u.z = __float_as_uint(q[2]);
            if (valid > 3) r.u.w = __float_as_uint(q[3]);
        }
    } else {
        const unsigned short *q = static_cast<const unsigned short *>(p) + at;
        if (vec) {
            const uint2 t = __ldg(reinterpret_cast<const uint2 *>(q));
            r.u.x = t.x;
            r.u.y = t.y;
        } else {
            r.u.x = q[0];
            if (valid > 1) r.u.x |= static_cast<uint32_t>(q[1]) << 16;
            if (valid > 2) r.u.y = q[2];
            if (valid > 3) r.u.y |= static_cast<uint32_t>(q[3]) << 16;
        }
    }
    return r;
}
__device__ __forceinline__ void floats_of(const Four &r, int type, float (&v)[4]) {
    if (type == kElemF32) {
        unpack(r.u, v, static_cast<const float *>(nullptr));
    } else {
        float w[8];
        if (type == kElemBF16) unpack(r.u, w, static_cast<const __nv_bfloat16 *>(nullptr));
        else unpack(r.u, w, static_cast<const __half *>(nullptr));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = w[i];
    }
}
__device__ __forceinline__ void store_four(const void *p, int type, bool vec, long long at, int valid, const float (&v)[4]) {
    if (valid <= 0) return;
    void *out = const_cast<void *>(p);
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < valid) store_param(out, type, at + i, v[i]);
    } else if (type == kElemF32) {
        float *q = static_cast<float *>(out) + at;
        __stcs(reinterpret_cast<uint4 *>(q), pack(v, q));
    } else {
        const float w[8] = {v[0], v[1], v[2], v[3], 0.0f, 0.0f, 0.0f, 0.0f};
        const uint4 u = type == kElemBF16 ? pack(w, static_cast<const __nv_bfloat16 *>(nullptr))
                                          : pack(w, static_cast<const __half *>(nullptr));
        __stcs(reinterpret_cast<uint2 *>(static_cast<unsigned short *>(out) + at), make_uint2(u.x, u.y));
    }
}

// ---- scalars ------------------------------------------------------------------------------
__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp_fast(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
constexpr float kLog2E = 1.4426950408889634f;

// softplus(v) = max(v, 0) + log(1 + e), e = exp(-|v|), and its slope, the sigmoid.
// log(1 + e) = 2 artanh(e / (2 + e)) by the series of the inverse hyperbolic
// tangent, whose argument is at most 1/3: the first term left out is below 2e-8
// of the sum.  Step sizes far below 1 come from small e, where a logarithm of the
// rounded 1 + e would lose what matters.
__device__ __forceinline__ void softplus(float v, float &value, float &slope) {
    const float e = exp2_fast(-fabsf(v) * kLog2E);
    const float u = e * rcp_fast(2.0f + e), w = u * u;
    float s = fmaf(w, 1.0f / 13.0f, 1.0f / 11.0f);
    s = fmaf(w, s, 1.0f / 9.0f);
    s = fmaf(w, s, 1.0f / 7.0f);
    s = fmaf(w, s, 1.0f / 5.0f);
    s = fmaf(w, s, 1.0f / 3.0f);
    s = fmaf(w, s, 1.0f);
    value = fmaxf(v, 0.0f) + 2.0f * u * s;
    const float r = rcp_fast(1.0f + e);
    slope = v >= 0.0f ? r : e * r;
}
__device__ __forceinline__ float scan_delta(const ScanParams &P, float raw, float &slope) {
    if (!P.softplus) {
        slope = 1.0f;
        return raw;
    }
    float v;
    softplus(raw, v, slope);
    return v;
}
// z / (1 + exp(-z)) and its slope for four values.
__device__ __forceinline__ void gates(const float (&z)[4], float (&gate)[4], float (&slope)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        f2 s, rest;
        const f2 zz = pair(z[i], z[i + 1]);
        sigmoid2(zz, s, rest);
        split(zz * s, gate[i], gate[i + 1]);
        split(s * fma2(zz, rest, pair(1.0f)), slope[i], slope[i + 1]);
    }
}

// ---- a thread's place ---------------------------------------------------------------------
// A warp's lanes: channel * P + part; a part has the states part * R ...
template <int SP, int R, int THREADS>
struct ScanPlace {
    static constexpr int P = SP / R, CB = THREADS / P;
    long long n, len;
    int seg, group, tile, first, count;  // first channel of the block, its channels
    int chan, part;                      // the thread's, from `first`
    __device__ __forceinline__ explicit ScanPlace(const ScanParams &Q) {
        const int per = Q.groups * Q.tiles;
        long long b = blockIdx.x;
        const int gt = static_cast<int>(b % per);
        b /= per;
        seg = static_cast<int>(b % Q.segs);
        n = b / Q.segs;
        group = gt / Q.tiles;
        tile = gt - group * Q.tiles;
        first = group * Q.cpg + tile * CB;
        count = min(CB, Q.cpg - tile * CB);
        chan = threadIdx.x / P;
        part = threadIdx.x % P;
        len = Q.l;
        if (Q.lengths != nullptr) {
            const int v = Q.lengths[n];
            len = v < 0 ? 0 : min(static_cast<long long>(v), Q.l);
        }
    }
    __device__ __forceinline__ bool live() const { return chan < count; }
    __device__ __forceinline__ int channel() const { return first + chan; }
};

// R states of a [..][states] tensor at `p`, zeros where there are none.
template <int R>
__device__ __forceinline__ void load_states(const float *p, int part, int states, bool live, float (&v)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = live && part * R + r < states ? p[part * R + r] : 0.0f;
}
template <int R>
__device__ __forceinline__ void store_states(float *p, int part, int states, bool live, const float (&v)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (live && part * R + r < states) p[part * R + r] = v[r];
}
// A log2(e): the exponentials are powers of 2.
template <int R>
__device__ __forceinline__ void load_decay(const ScanParams &Q, long long channel, int part, bool live, float (&v)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
        v[r] = live && part * R + r < Q.states ? load_param(Q.a, Q.a_type, channel * Q.states + part * R + r) * kLog2E : 0.0f;
}

// B or C of `count` tokens from t0 into sm[token][SP], zeros beyond.
template <int SP>
__device__ __forceinline__ void stage_states(const ScanParams &Q, const TokenView &v, long long n, long long t0, int group,
                                             int count, int tokens, float *sm) {
    for (int i = threadIdx.x; i < tokens * SP; i += blockDim.x) {
        const int t = i / SP, s = i - t * SP;
        sm[i] = t < count && s < Q.states ? load_param(v.p, Q.type, n * v.ldn + (t0 + t) * v.ldt + group * v.ldg + s) : 0.0f;
    }
}

// Sums of four values over the P lanes of a channel.  The lanes share the work:
// afterwards lane p of a channel has the sums first .. first + N - 1 in v.
template <int P>
struct FourSums {
    static constexpr int N = P == 1 ? 4 : P == 2 ? 2 : 1;
    int first = 0;
    __device__ __forceinline__ void operator()(float (&v)[4], int part) {
        if constexpr (P >= 2) {
            const bool up = part & 1;
            first = up ? 2 : 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float send = up ? v[i] : v[i + 2], keep = up ? v[i + 2] : v[i];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, send, 1);
            }
        }
        if constexpr (P >= 4) {
            const bool up = part & 2;
            first += up ? 1 : 0;
            const float send = up ? v[0] : v[1], keep = up ? v[1] : v[0];
            v[0] = keep + __shfl_xor_sync(0xffffffffu, send, 2);
        }
#pragma unroll
        for (int o = 4; o < P; o *= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
};

enum ScanMode { kScanMain, kScanCarry, kScanCarryBack };

// kScanMain       y and the last state, the states for the gradient where wanted
// kScanCarry      a segment's effect on the state: what it adds, sum of deltas
// kScanCarryBack  a segment's effect on the gradient of the state behind it
template <int SP, int R, int TT, int THREADS, int MODE>
__global__ void __launch_bounds__(THREADS) scan_kernel(const __grid_constant__ ScanParams Q) {
    using Place = ScanPlace<SP, R, THREADS>;
    constexpr int P = Place::P, CB = Place::CB, GROUPS = CB / 4;
    constexpr int NG = (TT * GROUPS + THREADS - 1) / THREADS;  // groups of four channels of a thread and tile
    __shared__ float2 du[TT][CB];
    __shared__ __align__(16) float bs[TT][SP], cs[MODE == kScanMain ? TT : 1][SP];
    griddep_wait();
    griddep_launch_dependents();
    const Place at(Q);
    // the effect of the last segment, backwards the first, reaches no other one
    if (MODE != kScanMain && at.seg == (MODE == kScanCarry ? Q.segs - 1 : 0)) return;
    const long long begin = at.seg * Q.seg_len, stop = min(Q.l, begin + Q.seg_len), end = min(at.len, stop);
    const int channel = at.channel();
    const bool live = at.live();
    float a2[R], h[R];
    load_decay<R>(Q, channel, at.part, live, a2);
#pragma unroll
    for (int r = 0; r < R; ++r) h[r] = 0.0f;
    if (MODE == kScanMain) {
        if (Q.state != nullptr && live)
            load_states<R>(Q.state + at.n * Q.s_ldn + channel * Q.s_ldc, at.part, Q.states, live, h);
        for (int j = 0; j < at.seg; ++j) {
            const long long row = (at.n * Q.segs + j) * Q.channels + channel;
            float e[R];
            load_states<R>(Q.carry + row * Q.states, at.part, Q.states, live, e);
            const float sum = live ? Q.sums[row] : 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r) h[r] = fmaf(exp2_fast(sum * a2[r]), h[r], e[r]);
        }
    }
    // the thread's groups of four channels: the same channels in every tile
    const int gc = (threadIdx.x % GROUPS) * 4, valid = at.count - gc;
    float bias[4], skip[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bias[i] = Q.bias != nullptr && i < valid ? load_param(Q.bias, Q.bias_type, at.first + gc + i) : 0.0f;
        skip[i] = MODE == kScanMain && Q.d != nullptr && i < valid ? load_param(Q.d, Q.d_type, at.first + gc + i) : 0.0f;
    }
    float sum = 0.0f;  // of the deltas
    for (long long t0 = begin; t0 < stop; t0 += TT) {
        const int tokens = static_cast<int>(max(0LL, min(static_cast<long long>(TT), end - t0)));
        if (MODE != kScanMain && tokens == 0) break;
        Four x[NG], z[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int t = (threadIdx.x + g * THREADS) / GROUPS;
            if (t >= tokens) continue;
            const long long c = at.first + gc, tt = t0 + t;
            const TokenView &in = MODE == kScanCarryBack ? Q.dy : Q.x;
            x[g] = load_four(in.p, Q.type, Q.vec, at.n * in.ldn + tt * in.ldt + c, valid);
            if (MODE != kScanCarry && Q.z.p != nullptr)
                z[g] = load_four(Q.z.p, Q.type, Q.vec, at.n * Q.z.ldn + tt * Q.z.ldt + c, valid);
            float d[4], v[4];
            floats_of(load_four(Q.dt.p, Q.type, Q.vec, at.n * Q.dt.ldn + tt * Q.dt.ldt + c, valid), Q.type, d);
            floats_of(x[g], Q.type, v);
            if (MODE == kScanCarryBack && Q.z.p != nullptr) {
                float zz[4], gate[4], slope[4];
                floats_of(z[g], Q.type, zz);
                gates(zz, gate, slope);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] *= gate[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float slope;
                const float delta = scan_delta(Q, d[i] + bias[i], slope);
                du[t][gc + i] = make_float2(delta, MODE == kScanCarryBack ? v[i] : delta * v[i]);
            }
        }
        stage_states<SP>(Q, MODE == kScanCarryBack ? Q.c : Q.b, at.n, t0, at.group, tokens, tokens, &bs[0][0]);
        if (MODE == kScanMain) stage_states<SP>(Q, Q.c, at.n, t0, at.group, tokens, tokens, &cs[0][0]);
        __syncthreads();
        for (int t = 0; t < tokens; t += 4) {
            if (MODE == kScanMain && Q.kept != nullptr && (t0 + t) % kScanChunk == 0) {
                const long long chunks = (Q.l + kScanChunk - 1) / kScanChunk, chunk = (t0 + t) / kScanChunk;
                store_states<R>(Q.kept + ((at.n * chunks + chunk) * Q.channels + channel) * Q.states, at.part, Q.states, live, h);
            }
            float y[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                y[q] = 0.0f;
                if (t + q >= tokens) continue;
                const float2 v = du[t + q][at.chan];
                const float *b = &bs[t + q][at.part * R];
                if (MODE == kScanCarryBack) {
                    sum += v.x;
#pragma unroll
                    for (int r = 0; r < R; ++r) h[r] = fmaf(exp2_fast(sum * a2[r]), v.y * b[r], h[r]);
                } else {
                    if (MODE == kScanCarry) sum += v.x;
#pragma unroll
                    for (int r = 0; r < R; ++r) h[r] = fmaf(exp2_fast(v.x * a2[r]), h[r], v.y * b[r]);
                    if (MODE == kScanMain) {
                        const float *c = &cs[t + q][at.part * R];
#pragma unroll
                        for (int r = 0; r < R; ++r) y[q] = fmaf(c[r], h[r], y[q]);
                    }
                }
            }
            if (MODE == kScanMain) {
                FourSums<P> sums;
                sums(y, at.part);
                __syncwarp();  // every lane of the channel has read these tokens
                if (at.part < 4) {
#pragma unroll
                    for (int i = 0; i < FourSums<P>::N; ++i)
                        if (t + sums.first + i < tokens) du[t + sums.first + i][at.chan].x = y[i];
                }
            }
        }
        __syncthreads();
        if (MODE == kScanMain) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const int t = (threadIdx.x + g * THREADS) / GROUPS;
                if (t >= TT || t0 + t >= stop) continue;
                float out[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (t < tokens) {
                    float v[4];
                    floats_of(x[g], Q.type, v);
#pragma unroll
                    for (int i = 0; i < 4; ++i) out[i] = fmaf(skip[i], v[i], du[t][gc + i].x);
                    if (Q.z.p != nullptr) {
                        float zz[4], gate[4], slope[4];
                        floats_of(z[g], Q.type, zz);
                        gates(zz, gate, slope);
#pragma unroll
                        for (int i = 0; i < 4; ++i) out[i] *= gate[i];
                    }
                }
                store_four(Q.y.p, Q.type, Q.vec, at.n * Q.y.ldn + (t0 + t) * Q.y.ldt + at.first + gc, valid, out);
            }
            __syncthreads();
        }
    }
    if (MODE == kScanMain) {
        if (Q.state_out != nullptr && at.seg == Q.segs - 1 && live)
            store_states<R>(Q.state_out + at.n * Q.so_ldn + channel * Q.so_ldc, at.part, Q.states, live, h);
    } else if (live) {
        const long long row = (at.n * Q.segs + at.seg) * Q.channels + channel;
        store_states<R>(Q.carry + row * Q.states, at.part, Q.states, live, h);
        if (at.part == 0) Q.sums[row] = sum;
    }
}

// Sums of 2 R values over the channels of a warp.  Lanes share the work: each
// step halves what a lane holds, until one value is left.
template <int N, int O, int P>
__device__ __forceinline__ void channel_sums(float (&v)[N], int lane, int &first, bool &writes) {
    if constexpr (O >= P) {
        const bool up = (lane & O) != 0;
        if constexpr (N > 1) {
            float half[N / 2];
            if (up) first += N / 2;
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const float send = up ? v[i] : v[i + N / 2], keep = up ? v[i + N / 2] : v[i];
                half[i] = keep + __shfl_xor_sync(0xffffffffu, send, O);
            }
            channel_sums<N / 2, O / 2, P>(half, lane, first, writes);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) v[i] = half[i];
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], O);
            if (up) writes = false;
            channel_sums<1, O / 2, P>(v, lane, first, writes);
        }
    }
}
// Values left to a lane: 2 R over 32 / P channels, one at least.
template <int R, int P>
constexpr int kSumsLeft = 2 * R * P > 32 ? 2 * R * P / 32 : 1;

// The gradient: tiles of kScanChunk tokens, from a segment's last to its first.
// A tile's states and decays are formed once more from the state kept in front of
// it and stay in registers for the way back.
template <int SP, int R, int THREADS>
__global__ void __launch_bounds__(THREADS) scan_grad_kernel(const __grid_constant__ ScanParams Q) {
    using Place = ScanPlace<SP, R, THREADS>;
    constexpr int P = Place::P, CB = Place::CB, GROUPS = CB / 4, T = kScanChunk, WARPS = THREADS / 32;
    constexpr int NG = (T * GROUPS + THREADS - 1) / THREADS;
    __shared__ float4 sm[T][CB];  // delta, delta x, f; then q . B, (q a h) . A, ., and C . h last
    __shared__ __align__(16) float bs[T][SP], cs[T][SP];
    __shared__ float red[WARPS][T][2 * SP];
    griddep_wait();
    griddep_launch_dependents();
    const Place at(Q);
    const long long begin = at.seg * Q.seg_len, stop = min(Q.l, begin + Q.seg_len), end = min(at.len, stop);
    const long long chunks = (Q.l + T - 1) / T;
    const int channel = at.channel(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool live = at.live();
    float a2[R], q[R], da[R];
    load_decay<R>(Q, channel, at.part, live, a2);
#pragma unroll
    for (int r = 0; r < R; ++r) q[r] = da[r] = 0.0f;
    if (Q.dlast != nullptr && live)
        load_states<R>(Q.dlast + at.n * Q.dl_ldn + channel * Q.dl_ldc, at.part, Q.states, live, q);
    for (int j = Q.segs - 1; j > at.seg; --j) {
        const long long row = (at.n * Q.segs + j) * Q.channels + channel;
        float e[R];
        load_states<R>(Q.carry + row * Q.states, at.part, Q.states, live, e);
        const float sum = live ? Q.sums[row] : 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) q[r] = fmaf(exp2_fast(sum * a2[r]), q[r], e[r]);
    }
    const int gc = (threadIdx.x % GROUPS) * 4, valid = at.count - gc;
    float bias[4], skip[4], dskip[4], dbias[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bias[i] = Q.bias != nullptr && i < valid ? load_param(Q.bias, Q.bias_type, at.first + gc + i) : 0.0f;
        skip[i] = Q.d != nullptr && i < valid ? load_param(Q.d, Q.d_type, at.first + gc + i) : 0.0f;
        dskip[i] = dbias[i] = 0.0f;
    }
    for (long long t0 = begin + (stop - 1 - begin) / T * T; t0 >= begin; t0 -= T) {
        const int tokens = static_cast<int>(max(0LL, min(static_cast<long long>(T), end - t0)));
        Four rx[NG], rd[NG], rz[NG], rg[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int t = (threadIdx.x + g * THREADS) / GROUPS;
            if (t >= tokens) continue;
            const long long c = at.first + gc, tt = t0 + t;
            rx[g] = load_four(Q.x.p, Q.type, Q.vec, at.n * Q.x.ldn + tt * Q.x.ldt + c, valid);
            rd[g] = load_four(Q.dt.p, Q.type, Q.vec, at.n * Q.dt.ldn + tt * Q.dt.ldt + c, valid);
            rg[g] = load_four(Q.dy.p, Q.type, Q.vec, at.n * Q.dy.ldn + tt * Q.dy.ldt + c, valid);
            float x[4], d[4], f[4];
            floats_of(rx[g], Q.type, x);
            floats_of(rd[g], Q.type, d);
            floats_of(rg[g], Q.type, f);
            if (Q.z.p != nullptr) {
                rz[g] = load_four(Q.z.p, Q.type, Q.vec, at.n * Q.z.ldn + tt * Q.z.ldt + c, valid);
                float z[4], gate[4], slope[4];
                floats_of(rz[g], Q.type, z);
                gates(z, gate, slope);
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] *= gate[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float slope;
                const float delta = scan_delta(Q, d[i] + bias[i], slope);
                sm[t][gc + i] = make_float4(delta, delta * x[i], f[i], 0.0f);
            }
        }
        stage_states<SP>(Q, Q.b, at.n, t0, at.group, tokens, T, &bs[0][0]);
        stage_states<SP>(Q, Q.c, at.n, t0, at.group, tokens, T, &cs[0][0]);
        __syncthreads();
        if (tokens > 0) {
            float before[R], h[T][R], a[T][R];
            load_states<R>(Q.kept + ((at.n * chunks + t0 / T) * Q.channels + channel) * Q.states, at.part, Q.states, live, before);
#pragma unroll
            for (int t4 = 0; t4 < T; t4 += 4) {
                float y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int t = t4 + k;
                    y[k] = 0.0f;
                    if (t >= tokens) continue;
                    const float4 v = sm[t][at.chan];
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        a[t][r] = exp2_fast(v.x * a2[r]);
                        h[t][r] = fmaf(a[t][r], t == 0 ? before[r] : h[t == 0 ? 0 : t - 1][r], v.y * bs[t][at.part * R + r]);
                        y[k] = fmaf(cs[t][at.part * R + r], h[t][r], y[k]);
                    }
                }
                if (Q.z.p != nullptr) {
                    FourSums<P> sums;
                    sums(y, at.part);
                    if (at.part < 4) {
#pragma unroll
                        for (int i = 0; i < FourSums<P>::N; ++i)
                            if (t4 + sums.first + i < tokens) sm[t4 + sums.first + i][at.chan].w = y[i];
                    }
                }
            }
            float da1[R];
#pragma unroll
            for (int r = 0; r < R; ++r) da1[r] = 0.0f;
#pragma unroll
            for (int t4 = T - 4; t4 >= 0; t4 -= 4) {
                float db[4], dd[4];
#pragma unroll
                for (int k = 3; k >= 0; --k) {
                    const int t = t4 + k;
                    db[k] = dd[k] = 0.0f;
                    if (t >= tokens) continue;
                    const float4 v = sm[t][at.chan];
                    float g[2 * R];
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        q[r] = fmaf(v.z, cs[t][at.part * R + r], q[r]);
                        g[r] = live ? q[r] * v.y : 0.0f;
                        g[R + r] = live ? v.z * h[t][r] : 0.0f;
                        db[k] = fmaf(q[r], bs[t][at.part * R + r], db[k]);
                        q[r] *= a[t][r];
                        const float m = q[r] * (t == 0 ? before[r] : h[t == 0 ? 0 : t - 1][r]);
                        dd[k] = fmaf(m, a2[r], dd[k]);
                        da1[r] = fmaf(m, v.x, da1[r]);
                    }
                    int first = 0;
                    bool writes = true;
                    channel_sums<2 * R, 16, P>(g, lane, first, writes);
                    if (writes) {
#pragma unroll
                        for (int i = 0; i < (kSumsLeft<R, P>); ++i) {
                            const int j = first + i;
                            red[warp][t][j < R ? at.part * R + j : SP + at.part * R + j - R] = g[i];
                        }
                    }
                }
                FourSums<P> sums, other;
                sums(db, at.part);
                other(dd, at.part);
                __syncwarp();  // every lane of the channel has read these tokens
                if (at.part < 4) {
#pragma unroll
                    for (int i = 0; i < FourSums<P>::N; ++i)
                        if (t4 + sums.first + i < tokens) {
                            float4 &v = sm[t4 + sums.first + i][at.chan];
                            v.x = db[i];
                            v.y = dd[i] * (1.0f / kLog2E);  // A, not A log2(e)
                        }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) da[r] += da1[r];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < tokens * 2 * SP; i += THREADS) {
            const int t = i / (2 * SP), j = i - t * 2 * SP, s = j % SP;
            if (s >= Q.states) continue;
            float v = red[0][t][j];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) v += red[w][t][j];
            const long long row = ((at.tile * Q.n + at.n) * Q.l + t0 + t) * Q.groups + at.group;
            Q.part_bc[(row * 2 + j / SP) * Q.states + s] = v;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int t = (threadIdx.x + g * THREADS) / GROUPS;
            if (t >= T || t0 + t >= stop) continue;
            float dx[4] = {}, ddt[4] = {}, dz[4] = {};
            if (t < tokens) {
                float x[4], d[4], f[4], z[4], gate[4], gslope[4];
                floats_of(rx[g], Q.type, x);
                floats_of(rd[g], Q.type, d);
                floats_of(rg[g], Q.type, f);
                if (Q.z.p != nullptr) {
                    floats_of(rz[g], Q.type, z);
                    gates(z, gate, gslope);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 v = sm[t][gc + i];
                    float slope;
                    const float delta = scan_delta(Q, d[i] + bias[i], slope);
                    if (Q.z.p != nullptr) {
                        dz[i] = f[i] * fmaf(skip[i], x[i], v.w) * gslope[i];
                        f[i] *= gate[i];
                    }
                    dx[i] = fmaf(delta, v.x, skip[i] * f[i]);
                    ddt[i] = fmaf(x[i], v.x, v.y) * slope;
                    if (i < valid) {
                        dskip[i] = fmaf(f[i], x[i], dskip[i]);
                        dbias[i] += ddt[i];
                    }
                }
            }
            const long long c = at.first + gc, tt = t0 + t;
            store_four(Q.dx.p, Q.type, Q.vec, at.n * Q.dx.ldn + tt * Q.dx.ldt + c, valid, dx);
            store_four(Q.ddt.p, Q.type, Q.vec, at.n * Q.ddt.ldn + tt * Q.ddt.ldt + c, valid, ddt);
            if (Q.z.p != nullptr) store_four(Q.dz.p, Q.type, Q.vec, at.n * Q.dz.ldn + tt * Q.dz.ldt + c, valid, dz);
        }
        __syncthreads();
    }
    if (Q.state_out != nullptr && at.seg == 0 && live)
        store_states<R>(Q.state_out + at.n * Q.so_ldn + channel * Q.so_ldc, at.part, Q.states, live, q);
    const long long row = at.n * Q.segs + at.seg;
    if (Q.part_a != nullptr && live)
        store_states<R>(Q.part_a + (row * Q.channels + channel) * Q.states, at.part, Q.states, live, da);
    if (Q.part_d == nullptr) return;
    // D and dt_bias: over the threads that take the same four channels
    float *join = reinterpret_cast<float *>(&sm[0][0]);
    constexpr int ROWS = THREADS / GROUPS;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        for (int base = 0; base < ROWS; base += T) {  // T rows at a time
            __syncthreads();
            const int r = static_cast<int>(threadIdx.x) / GROUPS - base;
            if (r >= 0 && r < T) {
#pragma unroll
                for (int i = 0; i < 4; ++i) join[r * CB + gc + i] = half == 0 ? dskip[i] : dbias[i];
            }
            __syncthreads();
            for (int c = threadIdx.x; c < at.count; c += THREADS) {
                float *out = Q.part_d + (row * 2 + half) * Q.channels + at.first + c;
                float s = base == 0 ? 0.0f : *out;
                for (int k = 0; k < min(T, ROWS - base); ++k) s += join[k * CB + c];
                *out = s;
            }
        }
    }
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

// One token of every sequence: x, dt, z, y are [n][channels].  A thread has read
// its part of the state before it writes it, so state_out may be the state itself.
template <int SP, int R, int THREADS>
__global__ void __launch_bounds__(THREADS) scan_step_kernel(const __grid_constant__ ScanParams Q) {
    using Place = ScanPlace<SP, R, THREADS>;
    constexpr int P = Place::P;
    griddep_wait();
    griddep_launch_dependents();
    const Place at(Q);
    const int channel = at.channel();
    const bool live = at.live();
    float y = 0.0f, x = 0.0f;
    if (live) {
        float a2[R], h[R];
        load_states<R>(Q.state + at.n * Q.s_ldn + channel * Q.s_ldc, at.part, Q.states, live, h);
        load_decay<R>(Q, channel, at.part, live, a2);
        x = load_param(Q.x.p, Q.type, at.n * Q.x.ldn + channel);
        float raw = load_param(Q.dt.p, Q.type, at.n * Q.dt.ldn + channel), slope;
        if (Q.bias != nullptr) raw += load_param(Q.bias, Q.bias_type, channel);
        const float delta = scan_delta(Q, raw, slope), u = delta * x;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int s = at.part * R + r;
            if (s >= Q.states) continue;
            const float b = load_param(Q.b.p, Q.type, at.n * Q.b.ldn + at.group * Q.b.ldg + s);
            const float c = load_param(Q.c.p, Q.type, at.n * Q.c.ldn + at.group * Q.c.ldg + s);
            h[r] = fmaf(exp2_fast(delta * a2[r]), h[r], u * b);
            y = fmaf(c, h[r], y);
        }
        store_states<R>(Q.state_out + at.n * Q.so_ldn + channel * Q.so_ldc, at.part, Q.states, live, h);
    }
#pragma unroll
    for (int o = 1; o < P; o *= 2) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (live && at.part == 0) {
        if (Q.d != nullptr) y = fmaf(load_param(Q.d, Q.d_type, channel), x, y);
        if (Q.z.p != nullptr) {
            const float z = load_param(Q.z.p, Q.type, at.n * Q.z.ldn + channel);
            const float zz[4] = {z, 0.0f, 0.0f, 0.0f};
            float gate[4], slope[4];
            gates(zz, gate, slope);
            y *= gate[0];
        }
        store_param(const_cast<void *>(Q.y.p), Q.type, at.n * Q.y.ldn + channel, y);
    }
}

}  // namespace gcb
