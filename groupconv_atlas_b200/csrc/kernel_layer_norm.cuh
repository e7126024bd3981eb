// Layer normalisation of rows, and its gradient.
//
//   y  = (x - mean) rstd gamma + beta,  rstd = 1 / sqrt(var + eps)
//   dx = rstd (g - mean(g) - xhat mean(g xhat)),  g = dy gamma, xhat = (x - mean) rstd
//   dgamma = sum over rows of dy xhat,  dbeta = sum over rows of dy
//
// All of it is bound by memory: x (and dy) is read once, held in registers
// through the sums, and the result written.  A team of threads takes a row: a
// power of two of at most 32, several to a warp, or a whole block.  The variance
// is the mean of squares about the mean, from the values in registers.  Forward
// 16384 x 2048 bf16 takes 32 us (4.2 TB/s), 100352 x 96 FP32 16 us (4.8 TB/s) and
// its gradient 22 us (5.3 TB/s).  Where whole blocks are teams the gradient takes 68 us
// at 16384 x 2048 bf16 and 140 at 8192 x 8192 (2.9 TB/s): three blocks of 256
// threads, or one of 512, are all that their registers let a multiprocessor hold, and a block has no loads under way while it
// sums.
#pragma once
#include <cstring>

#include "norm_util.cuh"

namespace gcb {

struct LayerNormParams {
    const void *x, *dy;  // dy: gradient only
    void *y;             // or dx
    long long rows, x_ld, dy_ld, y_ld;
    int c, vcols;        // elements and vectors of a row
    int team;            // threads that take a row
    const void *gamma, *beta;
    int gamma_type, beta_type;
    int aligned;         // whether both can be read 16 bytes at a time
    float eps;
    float2 *stats;       // mean and rstd of each row; nullable in the forward pass
    float *part;         // gradient: dgamma and dbeta of each block, [block][2][c]; NULL where neither is wanted
};

constexpr int kRowThreads = 256, kRowMost = 512;  // threads of a block of small teams; of a block that is a team

// Sums over a team, the same in every thread.  buf: two turns of [warps][N].
template <int N>
__device__ __forceinline__ void team_sums(float (&v)[N], int team, float *buf, int &turn) {
    for (int o = min(team, 32) / 2; o > 0; o /= 2) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
    if (team <= 32) return;
    // A turn's buffer is written again two sums later, behind a barrier that
    // every thread reaches after reading it.
    float *mine = buf + turn * (kRowMost / 32) * N;
    turn ^= 1;
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) mine[warp * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = mine[i];
    for (int w = 1; w < warps; ++w) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += mine[w * N + i];
    }
}

// A parameter's values at a vector's columns; 16-byte accesses where they are aligned.
template <int V>
__device__ __forceinline__ Lanes<V> row_params(const void *p, int type, bool aligned, int i, float none) {
    float v[V];
    if constexpr (V == 8) {
        if (p != nullptr && aligned) {
            if (type == kElemF32) {
                const float4 a = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i));
                const float4 b = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i) + 1);
                Lanes<V> r;
                r.p[0] = pair(a.x, a.y);
                r.p[1] = pair(a.z, a.w);
                r.p[2] = pair(b.x, b.y);
                r.p[3] = pair(b.z, b.w);
                return r;
            }
            const uint4 u = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i));
            return type == kElemBF16 ? unpack_lanes<__nv_bfloat16, V>(u, static_cast<const __nv_bfloat16 *>(nullptr))
                                     : unpack_lanes<__half, V>(u, static_cast<const __half *>(nullptr));
        }
    } else if constexpr (V == 4) {
        if (p != nullptr && aligned)
            return unpack_lanes<float, V>(__ldg(reinterpret_cast<const uint4 *>(static_cast<const float *>(p) + i)),
                                          static_cast<const float *>(nullptr));
    }
    load_params<V>(p, type, i, none, v);
    return lanes_of<V>(v);
}
template <int V>
__device__ __forceinline__ Lanes<V> float_params(const float *p) {
    float v[V];
    if constexpr (V == 1) {
        v[0] = *p;
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 f = __ldg(reinterpret_cast<const float4 *>(p + i));
            v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
        }
    }
    return lanes_of<V>(v);
}
// g = dy gamma, rounded by itself in its sum and in dx alike, so that what is g's mean
// leaves 0 (rows of one column, rows whose g is one value).  Of pairs a product and a
// sum behind it become one fma, .rn or not; of single values they do not.
__device__ __forceinline__ f2 rounded_product(f2 a, f2 b) {
    float a0, a1, b0, b1;
    split(a, a0, a1);
    split(b, b0, b1);
    return pair(__fmul_rn(a0, b0), __fmul_rn(a1, b1));
}
template <int V>
__device__ __forceinline__ float lanes_sum(const Lanes<V> &l) {
    f2 s = l.p[0];
#pragma unroll
    for (int i = 1; i < Lanes<V>::kPairs; ++i) s = s + l.p[i];
    float a, b;
    split(s, a, b);
    return a + b;
}

// NV vectors a thread and row, ROWS rows at a time.
template <class T, int V, int NV, int ROWS>
__global__ void __launch_bounds__(kRowMost) layer_norm_kernel(const __grid_constant__ LayerNormParams P) {
    constexpr int NP = Lanes<V>::kPairs;
    __shared__ float buf[2 * (kRowMost / 32) * ROWS];
    griddep_wait();
    griddep_launch_dependents();
    const int teams = blockDim.x / P.team, team = threadIdx.x / P.team, lane = threadIdx.x - team * P.team;
    const long long all = static_cast<long long>(gridDim.x) * teams;
    const float inv = 1.0f / static_cast<float>(P.c);
    const bool plain = P.aligned && P.gamma != nullptr && P.beta != nullptr && P.gamma_type == kElemF32 && P.beta_type == kElemF32;
    int turn = 0;
    for (long long first = static_cast<long long>(blockIdx.x) * teams; first < P.rows; first += all * ROWS) {
        Raw<T, V> raw[ROWS][NV];
        float s[ROWS], q[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = first + team + r * all;
            const T *src = static_cast<const T *>(P.x) + row * P.x_ld;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int v = lane + j * P.team;
                if (row < P.rows && v < P.vcols) raw[r][j] = load_raw<T, V>(src + static_cast<long long>(v) * V);
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            s[r] = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (first + team + r * all < P.rows && lane + j * P.team < P.vcols) s[r] += lanes_sum<V>(lanes_of_raw<T, V>(raw[r][j]));
        }
        team_sums<ROWS>(s, P.team, buf, turn);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            s[r] *= inv;
            f2 sum = pair(0.0f);
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (first + team + r * all < P.rows && lane + j * P.team < P.vcols) {
                    const Lanes<V> e = lanes_of_raw<T, V>(raw[r][j]);
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        const f2 d = e.p[i] + (V == 1 ? pair(-s[r], 0.0f) : pair(-s[r]));
                        sum = fma2(d, d, sum);
                    }
                }
            float a, b;
            split(sum, a, b);
            q[r] = a + b;
        }
        team_sums<ROWS>(q, P.team, buf, turn);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) q[r] = 1.0f / sqrtf(fmaf(q[r], inv, P.eps));
        const auto finish = [&](int j, int v, const Lanes<V> &gamma, const Lanes<V> &beta) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const long long row = first + team + r * all;
                if (row >= P.rows) continue;
                Lanes<V> e = lanes_of_raw<T, V>(raw[r][j]);
#pragma unroll
                for (int i = 0; i < NP; ++i)
                    e.p[i] = fma2((e.p[i] + pair(-s[r])) * pair(q[r]), gamma.p[i], beta.p[i]);
                store_lanes<T, V>(static_cast<T *>(P.y) + row * P.y_ld + static_cast<long long>(v) * V, e);
            }
        };
        if (V > 1 && plain) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int v = lane + j * P.team;
                if (v < P.vcols)
                    finish(j, v, float_params<V>(static_cast<const float *>(P.gamma) + v * V),
                           float_params<V>(static_cast<const float *>(P.beta) + v * V));
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int v = lane + j * P.team;
                if (v < P.vcols)
                    finish(j, v, row_params<V>(P.gamma, P.gamma_type, P.aligned, v * V, 1.0f),
                           row_params<V>(P.beta, P.beta_type, P.aligned, v * V, 0.0f));
            }
        }
        if (P.stats != nullptr && lane == 0) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const long long row = first + team + r * all;
                if (row < P.rows) P.stats[row] = make_float2(s[r], q[r]);
            }
        }
    }
}

// The gradient.  A block's teams take rows in turn and add up dgamma and dbeta of
// their columns in registers, over at most 64 rows (the launch sees to that); at
// the end the block joins its teams in a fixed order.  Dynamic shared memory:
// [warps][2][c] values where a row takes at most a warp.
template <class T, int V, int NV, int ROWS>
__global__ void __launch_bounds__(kRowMost) layer_norm_grad_kernel(const __grid_constant__ LayerNormParams P) {
    constexpr int NP = Lanes<V>::kPairs;
    extern __shared__ float joined[];
    __shared__ float buf[2 * (kRowMost / 32) * 2 * ROWS];
    griddep_wait();
    griddep_launch_dependents();
    const int teams = blockDim.x / P.team, team = threadIdx.x / P.team, lane = threadIdx.x - team * P.team;
    const long long all = static_cast<long long>(gridDim.x) * teams;
    const float inv = 1.0f / static_cast<float>(P.c);
    Lanes<V> gamma[NV], sum_g[NV], sum_b[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int v = lane + j * P.team;
        if (v < P.vcols) gamma[j] = row_params<V>(P.gamma, P.gamma_type, P.aligned, v * V, 1.0f);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            sum_g[j].p[i] = sum_b[j].p[i] = pair(0.0f);
            if (v >= P.vcols) gamma[j].p[i] = pair(0.0f);
        }
    }
    int turn = 0;
    for (long long first = static_cast<long long>(blockIdx.x) * teams; first < P.rows; first += all * ROWS) {
        Raw<T, V> rx[ROWS][NV], rg[ROWS][NV];
        float2 st[ROWS];
        float sums[2 * ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = first + team + r * all;
            st[r] = row < P.rows ? P.stats[row] : make_float2(0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const long long v = lane + j * P.team;
                if (row < P.rows && v < P.vcols) {
                    rx[r][j] = load_raw<T, V>(static_cast<const T *>(P.x) + row * P.x_ld + v * V);
                    rg[r][j] = load_raw<T, V>(static_cast<const T *>(P.dy) + row * P.dy_ld + v * V);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            f2 s1 = pair(0.0f), s2 = pair(0.0f);
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (first + team + r * all < P.rows && lane + j * P.team < P.vcols) {
                    const Lanes<V> e = lanes_of_raw<T, V>(rx[r][j]), d = lanes_of_raw<T, V>(rg[r][j]);
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        const f2 xhat = (e.p[i] + pair(-st[r].x)) * pair(st[r].y), g = rounded_product(d.p[i], gamma[j].p[i]);
                        s1 = s1 + g;
                        s2 = fma2(g, xhat, s2);
                        sum_g[j].p[i] = fma2(d.p[i], xhat, sum_g[j].p[i]);
                        sum_b[j].p[i] = sum_b[j].p[i] + d.p[i];
                    }
                }
            float a, b;
            split(s1, a, b);
            sums[2 * r] = V == 1 ? a : a + b;
            split(s2, a, b);
            sums[2 * r + 1] = V == 1 ? a : a + b;
        }
        team_sums<2 * ROWS>(sums, P.team, buf, turn);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const long long row = first + team + r * all;
            const f2 m1 = pair(-sums[2 * r] * inv), m2 = pair(-sums[2 * r + 1] * inv);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const long long v = lane + j * P.team;
                if (row < P.rows && v < P.vcols) {
                    const Lanes<V> e = lanes_of_raw<T, V>(rx[r][j]), d = lanes_of_raw<T, V>(rg[r][j]);
                    Lanes<V> o;
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        const f2 xhat = (e.p[i] + pair(-st[r].x)) * pair(st[r].y);
                        o.p[i] = pair(st[r].y) * fma2(xhat, m2, rounded_product(d.p[i], gamma[j].p[i]) + m1);
                    }
                    store_lanes<T, V>(static_cast<T *>(P.y) + row * P.y_ld + v * V, o);
                }
            }
        }
    }
    float dgamma[NV][V], dbeta[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        values_of<V>(sum_g[j], dgamma[j]);
        values_of<V>(sum_b[j], dbeta[j]);
    }
    if (P.part == nullptr) return;
    float *out = P.part + static_cast<long long>(blockIdx.x) * 2 * P.c;
    if (P.team > 32) {  // one team: the columns are the thread's own
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int v = lane + j * P.team;
            if (v >= P.vcols) continue;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                out[v * V + k] = dgamma[j][k];
                out[P.c + v * V + k] = dbeta[j][k];
            }
        }
        return;
    }
    for (int o = P.team; o < 32; o *= 2) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                dgamma[j][k] += __shfl_xor_sync(0xffffffffu, dgamma[j][k], o);
                dbeta[j][k] += __shfl_xor_sync(0xffffffffu, dbeta[j][k], o);
            }
    }
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) < P.team) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int v = lane + j * P.team;
            if (v >= P.vcols) continue;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                joined[(2 * warp) * P.c + v * V + k] = dgamma[j][k];
                joined[(2 * warp + 1) * P.c + v * V + k] = dbeta[j][k];
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * P.c; i += blockDim.x) {
        float s = joined[i];
        for (int w = 1; w < warps; ++w) s += joined[2 * w * P.c + i];
        out[i] = s;
    }
}

// ---- rows that do not start on 16 bytes -----------------------------------------------
// Rows of odd length lie one after the other, so each starts at a place of its own
// within 16 bytes.  A thread takes the aligned vectors that cover a row; its first
// and last ones hold columns of the neighbouring rows too, and are read and written
// element by element.  (Eight times fewer accesses than single elements: 8191 rows of
// 1001 bf16 37 us there, see the launch.)  x, dy and the result start alike.
template <class T>
struct EdgeVector {
    static constexpr int V = kVec<T>;
    int low, c;  // the vector's first column (negative in a row's first vector), columns of a row
    __device__ __forceinline__ bool any() const { return low < c; }
    __device__ __forceinline__ bool full() const { return low >= 0 && low + V <= c; }
    __device__ __forceinline__ bool has(int k) const { return low + k >= 0 && low + k < c; }
    // NEAREST: where a place is no column of the row, the value of the nearest that is;
    // else 0 there.
    template <bool NEAREST = false>
    __device__ __forceinline__ Raw<T, V> load(const T *row) const {
        Raw<T, V> r;
        if (full()) {
            r = load_raw<T, V>(row + low);
        } else {
            T e[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                if constexpr (NEAREST) e[k] = row[max(0, min(low + k, c - 1))];
                else e[k] = has(k) ? row[low + k] : from_float<T>(0.0f);
            }
            memcpy(&r.u, e, sizeof(r.u));
        }
        return r;
    }
    __device__ __forceinline__ void store(T *row, const Lanes<V> &l) const {
        if (full()) {
            store_lanes<T, V>(row + low, l);
        } else {
            float v[V];
            values_of<V>(l, v);
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (has(k)) row[low + k] = from_float<T>(v[k]);
        }
    }
};
// Values without those that are none of the row's.
template <class T>
__device__ __forceinline__ void mask_edges(const EdgeVector<T> &at, Lanes<kVec<T>> &l) {
    if (at.full()) return;
    float v[kVec<T>];
    values_of<kVec<T>>(l, v);
#pragma unroll
    for (int k = 0; k < kVec<T>; ++k)
        if (!at.has(k)) v[k] = 0.0f;
    l = lanes_of<kVec<T>>(v);
}
// Columns in shared memory: a gap after every vector, so that threads, which read a
// vector apart whatever the row's place is, meet different banks.
template <int V>
__device__ __forceinline__ int gapped(int c) { return c + c / V; }
template <class T>
__device__ __forceinline__ Lanes<kVec<T>> edge_params(const EdgeVector<T> &at, const float *p) {
    float v[kVec<T>];
#pragma unroll
    for (int k = 0; k < kVec<T>; ++k) v[k] = at.has(k) ? p[gapped<kVec<T>>(at.low + k)] : 0.0f;
    return lanes_of<kVec<T>>(v);
}
// A row's place within 16 bytes, in elements.
template <class T>
__device__ __forceinline__ int row_phase(const T *row) {
    return static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
}

// Dynamic shared memory: gamma and beta, gapped.  vcols: vectors that may touch a row.
template <class T, int NV>
__global__ void __launch_bounds__(kRowMost) layer_norm_edges_kernel(const __grid_constant__ LayerNormParams P) {
    constexpr int V = kVec<T>, NP = Lanes<V>::kPairs;
    extern __shared__ float params[];
    __shared__ float buf[2 * (kRowMost / 32)];
    griddep_wait();
    griddep_launch_dependents();
    float *gamma = params, *beta = params + gapped<V>(P.c - 1) + 1;
    for (int i = threadIdx.x; i < P.c; i += blockDim.x) {
        gamma[gapped<V>(i)] = P.gamma != nullptr ? load_param(P.gamma, P.gamma_type, i) : 1.0f;
        beta[gapped<V>(i)] = P.beta != nullptr ? load_param(P.beta, P.beta_type, i) : 0.0f;
    }
    __syncthreads();
    const int teams = blockDim.x / P.team, team = threadIdx.x / P.team, lane = threadIdx.x - team * P.team;
    const long long all = static_cast<long long>(gridDim.x) * teams;
    const float inv = 1.0f / static_cast<float>(P.c);
    int turn = 0;
    for (long long first = static_cast<long long>(blockIdx.x) * teams; first < P.rows; first += all) {
        const long long row = first + team;
        const T *x = static_cast<const T *>(P.x) + row * P.x_ld;
        const int phase = row_phase(x), count = row < P.rows ? P.c : -V;  // no columns in a row that is none
        Lanes<V> e[NV];
        float s[1] = {0.0f}, q[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const EdgeVector<T> at{(lane + j * P.team) * V - phase, count};
            if (at.any()) e[j] = lanes_of_raw<T, V>(at.load(x));
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (EdgeVector<T>{(lane + j * P.team) * V - phase, count}.any()) s[0] += lanes_sum<V>(e[j]);
        team_sums<1>(s, P.team, buf, turn);
        const float mean = s[0] * inv;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const EdgeVector<T> at{(lane + j * P.team) * V - phase, count};
            if (!at.any()) continue;
            f2 sum = pair(0.0f);
#pragma unroll
            for (int i = 0; i < NP; ++i) e[j].p[i] = e[j].p[i] + pair(-mean);
            mask_edges<T>(at, e[j]);
#pragma unroll
            for (int i = 0; i < NP; ++i) sum = fma2(e[j].p[i], e[j].p[i], sum);
            float a, b;
            split(sum, a, b);
            q[0] += a + b;
        }
        team_sums<1>(q, P.team, buf, turn);
        const float rstd = 1.0f / sqrtf(fmaf(q[0], inv, P.eps));
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const EdgeVector<T> at{(lane + j * P.team) * V - phase, count};
            if (!at.any()) continue;
            const Lanes<V> g = edge_params<T>(at, gamma), b = edge_params<T>(at, beta);
#pragma unroll
            for (int i = 0; i < NP; ++i) e[j].p[i] = fma2(e[j].p[i] * pair(rstd), g.p[i], b.p[i]);
            at.store(static_cast<T *>(P.y) + row * P.y_ld, e[j]);
        }
        if (P.stats != nullptr && lane == 0 && row < P.rows) P.stats[row] = make_float2(mean, rstd);
    }
}

// A team's rows all start at the same place (the launch sees to the step), so that
// its columns, their sums and gamma stay in its threads.  Dynamic shared memory:
// [teams][2][c] values where a row takes a warp.
template <class T, int NV>
__global__ void __launch_bounds__(kRowMost) layer_norm_edges_grad_kernel(const __grid_constant__ LayerNormParams P) {
    constexpr int V = kVec<T>, NP = Lanes<V>::kPairs;
    extern __shared__ float joined[];
    __shared__ float buf[2 * (kRowMost / 32) * 2];
    griddep_wait();
    griddep_launch_dependents();
    const int teams = blockDim.x / P.team, team = threadIdx.x / P.team, lane = threadIdx.x - team * P.team;
    const long long all = static_cast<long long>(gridDim.x) * teams;
    const float inv = 1.0f / static_cast<float>(P.c);
    const long long mine = static_cast<long long>(blockIdx.x) * teams + team;
    const int phase = row_phase(static_cast<const T *>(P.x) + mine * P.x_ld);
    Lanes<V> gamma[NV], sum_g[NV], sum_b[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const EdgeVector<T> at{(lane + j * P.team) * V - phase, P.c};
        float v[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            v[k] = 0.0f;
            if (at.has(k)) v[k] = P.gamma != nullptr ? load_param(P.gamma, P.gamma_type, at.low + k) : 1.0f;
        }
        gamma[j] = lanes_of<V>(v);
#pragma unroll
        for (int i = 0; i < NP; ++i) sum_g[j].p[i] = sum_b[j].p[i] = pair(0.0f);
    }
    int turn = 0;
    for (long long first = static_cast<long long>(blockIdx.x) * teams; first < P.rows; first += all) {
        const long long row = first + team;
        const int count = row < P.rows ? P.c : -V;
        const T *x = static_cast<const T *>(P.x) + row * P.x_ld, *dy = static_cast<const T *>(P.dy) + row * P.dy_ld;
        Raw<T, V> rx[NV], rg[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const EdgeVector<T> at{(lane + j * P.team) * V - phase, count};
            if (at.any()) {
                rx[j] = at.template load<true>(x);
                rg[j] = at.load(dy);
            }
        }
        const float2 st = row < P.rows ? P.stats[row] : make_float2(0.0f, 0.0f);
        float sums[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const EdgeVector<T> at{(lane + j * P.team) * V - phase, count};
            if (!at.any()) continue;
            // where a place is no column of the row dy and gamma are 0, and xhat is a
            // column's (with x = 0 there, (0 - mean) rstd could be infinite)
            const Lanes<V> e = lanes_of_raw<T, V>(rx[j]), d = lanes_of_raw<T, V>(rg[j]);
            f2 s1 = pair(0.0f), s2 = pair(0.0f);
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const f2 xhat = (e.p[i] + pair(-st.x)) * pair(st.y), g = rounded_product(d.p[i], gamma[j].p[i]);
                s1 = s1 + g;
                s2 = fma2(g, xhat, s2);
                sum_g[j].p[i] = fma2(d.p[i], xhat, sum_g[j].p[i]);
                sum_b[j].p[i] = sum_b[j].p[i] + d.p[i];
            }
            float a, b;
            split(s1, a, b);
            sums[0] += a + b;
            split(s2, a, b);
            sums[1] += a + b;
        }
        team_sums<2>(sums, P.team, buf, turn);
        const f2 m1 = pair(-sums[0] * inv), m2 = pair(-sums[1] * inv);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const EdgeVector<T> at{(lane + j * P.team) * V - phase, count};
            if (!at.any()) continue;
            const Lanes<V> e = lanes_of_raw<T, V>(rx[j]), d = lanes_of_raw<T, V>(rg[j]);
            Lanes<V> o;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const f2 xhat = (e.p[i] + pair(-st.x)) * pair(st.y);
                o.p[i] = pair(st.y) * fma2(xhat, m2, rounded_product(d.p[i], gamma[j].p[i]) + m1);
            }
            at.store(static_cast<T *>(P.y) + row * P.y_ld, o);
        }
    }
    if (P.part == nullptr) return;
    float *out = P.part + static_cast<long long>(blockIdx.x) * 2 * P.c;
    float *own = P.team > 32 ? out : joined + team * 2 * P.c;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const EdgeVector<T> at{(lane + j * P.team) * V - phase, P.c};
        float g[V], b[V];
        values_of<V>(sum_g[j], g);
        values_of<V>(sum_b[j], b);
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (at.has(k)) {
                own[at.low + k] = g[k];
                own[P.c + at.low + k] = b[k];
            }
    }
    if (P.team > 32) return;
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * P.c; i += blockDim.x) {
        float s = joined[i];
        for (int w = 1; w < teams; ++w) s += joined[2 * w * P.c + i];
        out[i] = s;
    }
}

// Rows too long for a block's registers: read three times (the second and third
// time from the caches), one row to a block.  Columns in 64 bits: a row may have up
// to 2^31 - 1, a step beyond which 32 do not hold, nor do they twice as many.
//
// A thread's share of such a row's sums, which has no bound: runs of 64 values in 32
// bits joined in 64.  add(column, the run's sums).
template <int N, class F>
__device__ __forceinline__ void long_sums(long long c, float (&v)[N], F add) {
    constexpr long long kRun = 64LL * kRowMost;
    double all[N] = {};
    for (long long start = threadIdx.x; start < c; start += kRun) {
        const long long stop = min(c, start + kRun);
        float run[N] = {};
        for (long long i = start; i < stop; i += kRowMost) add(i, run);
#pragma unroll
        for (int k = 0; k < N; ++k) all[k] += run[k];
    }
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = static_cast<float>(all[k]);
}
template <class T>
__global__ void __launch_bounds__(kRowMost) layer_norm_long_kernel(const __grid_constant__ LayerNormParams P) {
    __shared__ float buf[2 * (kRowMost / 32)];
    griddep_wait();
    griddep_launch_dependents();
    const float inv = 1.0f / static_cast<float>(P.c);
    int turn = 0;
    for (long long row = blockIdx.x; row < P.rows; row += gridDim.x) {
        const T *src = static_cast<const T *>(P.x) + row * P.x_ld;
        T *dst = static_cast<T *>(P.y) + row * P.y_ld;
        float s[1], q[1];
        long_sums<1>(P.c, s, [&](long long i, float (&run)[1]) { run[0] += to_float(src[i]); });
        team_sums<1>(s, kRowMost, buf, turn);
        const float mean = s[0] * inv;
        long_sums<1>(P.c, q, [&](long long i, float (&run)[1]) {
            const float d = to_float(src[i]) - mean;
            run[0] = fmaf(d, d, run[0]);
        });
        team_sums<1>(q, kRowMost, buf, turn);
        const float rstd = 1.0f / sqrtf(fmaf(q[0], inv, P.eps));
        for (long long i = threadIdx.x; i < P.c; i += kRowMost) {
            const float gamma = P.gamma != nullptr ? load_param(P.gamma, P.gamma_type, i) : 1.0f;
            const float beta = P.beta != nullptr ? load_param(P.beta, P.beta_type, i) : 0.0f;
            dst[i] = from_float<T>(fmaf((to_float(src[i]) - mean) * rstd, gamma, beta));
        }
        if (P.stats != nullptr && threadIdx.x == 0) P.stats[row] = make_float2(mean, rstd);
    }
}

// A thread's columns of the block's sums are its own, so they add up in the
// workspace.  Single elements, everything read twice and the sums read and written for
// every row: 4096 x 12288 bf16 400 us, where 46 would move x, dy and dx once.
template <class T>
__global__ void __launch_bounds__(kRowMost) layer_norm_long_grad_kernel(const __grid_constant__ LayerNormParams P) {
    __shared__ float buf[2 * (kRowMost / 32) * 2];
    griddep_wait();
    griddep_launch_dependents();
    const float inv = 1.0f / static_cast<float>(P.c);
    float *out = P.part == nullptr ? nullptr : P.part + static_cast<long long>(blockIdx.x) * 2 * P.c;
    int turn = 0;
    for (long long row = blockIdx.x; row < P.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(P.x) + row * P.x_ld, *dy = static_cast<const T *>(P.dy) + row * P.dy_ld;
        T *dst = static_cast<T *>(P.y) + row * P.y_ld;
        const float2 st = P.stats[row];
        float sums[2];
        long_sums<2>(P.c, sums, [&](long long i, float (&run)[2]) {
            const float gamma = P.gamma != nullptr ? load_param(P.gamma, P.gamma_type, i) : 1.0f;
            const float d = to_float(dy[i]), xhat = (to_float(x[i]) - st.x) * st.y, g = __fmul_rn(d, gamma);
            run[0] += g;
            run[1] = fmaf(g, xhat, run[1]);
            if (out != nullptr) {
                const bool fresh = row == blockIdx.x;
                out[i] = fmaf(d, xhat, fresh ? 0.0f : out[i]);
                out[P.c + i] = d + (fresh ? 0.0f : out[P.c + i]);
            }
        });
        team_sums<2>(sums, kRowMost, buf, turn);
        const float m1 = sums[0] * inv, m2 = sums[1] * inv;
        for (long long i = threadIdx.x; i < P.c; i += kRowMost) {
            const float gamma = P.gamma != nullptr ? load_param(P.gamma, P.gamma_type, i) : 1.0f;
            const float xhat = (to_float(x[i]) - st.x) * st.y;
            dst[i] = from_float<T>(st.y * (__fmul_rn(to_float(dy[i]), gamma) - m1 - xhat * m2));
        }
    }
}

}  // namespace gcb
