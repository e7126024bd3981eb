// Device-side building blocks of the normalisation and dropout kernels:
// element types, 16-byte vectors, the activations with their derivatives, and
// the counter-based generator.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "device_util.cuh"

namespace gcb {

constexpr int kActSilu = 3;  // beside kActNone, kActRelu, kActRelu6

// Element types of a tensor (dtype codes of groupconv.h in parentheses).
enum ElemType { kElemF32 = 0, kElemF16 = 1, kElemBF16 = 2 };  // GC_F32, GC_B200_F16, GC_B200_BF16

// ---- 16-byte vectors of elements, in 32-bit arithmetic --------------------------------
template <class T>
constexpr int kVec = 16 / sizeof(T);

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ void unpack(const uint4 &u, float (&v)[4], const float *) {
    v[0] = __uint_as_float(u.x);
    v[1] = __uint_as_float(u.y);
    v[2] = __uint_as_float(u.z);
    v[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4 &u, float (&v)[8], const __nv_bfloat16 *) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // a bf16 is the upper half of the float of the same value
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack(const uint4 &u, float (&v)[8], const __half *) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ uint4 pack(const float (&v)[4], const float *) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], const __nv_bfloat16 *) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], const __half *) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 b = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// V = kVec<T>: one 16-byte access (the address is 16-byte aligned); V = 1: one element.
template <class T, int V>
__device__ __forceinline__ void load_elems(const T *p, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = to_float(*p);
    } else {
        unpack(__ldg(reinterpret_cast<const uint4 *>(p)), v, p);
    }
}
// The results are not read again by the kernel that stores them: streaming stores.
template <class T, int V>
__device__ __forceinline__ void store_elems(T *p, const float (&v)[V]) {
    if constexpr (V == 1) {
        *p = from_float<T>(v[0]);
    } else {
        __stcs(reinterpret_cast<uint4 *>(p), pack(v, p));
    }
}

// Elements [i, i + V) of a parameter vector whose type is known at run time, or
// `none` where there is no vector.  One branch for all of them, so that their
// loads are in flight together.
template <int V>
__device__ __forceinline__ void load_params(const void *p, int type, long long i, float none, float (&v)[V]) {
    if (p == nullptr) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = none;
    } else if (type == kElemF32) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = __ldg(static_cast<const float *>(p) + i + j);
    } else {
        uint16_t u[V];
#pragma unroll
        for (int j = 0; j < V; ++j) u[j] = __ldg(static_cast<const unsigned short *>(p) + i + j);
#pragma unroll
        for (int j = 0; j < V; ++j)
            v[j] = type == kElemBF16 ? __uint_as_float(static_cast<uint32_t>(u[j]) << 16)
                                     : __half2float(__ushort_as_half(u[j]));
    }
}
// Element i of such a vector.
__device__ __forceinline__ float load_param(const void *p, int type, long long i) {
    if (type == kElemF32) return __ldg(static_cast<const float *>(p) + i);
    if (type == kElemF16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_param(void *p, int type, long long i, float v) {
    if (type == kElemF32) static_cast<float *>(p)[i] = v;
    else if (type == kElemF16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// ---- pairs of floats ------------------------------------------------------------------
// sm_100 adds and multiplies two floats in one instruction; the kernels are
// bound by issue slots at 16-bit types, so their arithmetic runs on pairs.
struct f2 {
    uint64_t v;
};
__device__ __forceinline__ f2 pair(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ f2 pair(float a) { return pair(a, a); }
__device__ __forceinline__ void split(f2 p, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v));
}
__device__ __forceinline__ f2 operator+(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f2 operator*(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// A thread's V values as pairs; V = 1 leaves the second half unused (0).
template <int V>
struct Lanes {
    static constexpr int kPairs = (V + 1) / 2;
    f2 p[kPairs];
};
template <int V>
__device__ __forceinline__ Lanes<V> lanes_of(const float (&v)[V]) {
    Lanes<V> r;
    if constexpr (V == 1) {
        r.p[0] = pair(v[0], 0.0f);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) r.p[i] = pair(v[2 * i], v[2 * i + 1]);
    }
    return r;
}
template <int V>
__device__ __forceinline__ void values_of(const Lanes<V> &l, float (&v)[V]) {
    if constexpr (V == 1) {
        float unused;
        split(l.p[0], v[0], unused);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) split(l.p[i], v[2 * i], v[2 * i + 1]);
    }
}
template <class T, int V>
__device__ __forceinline__ Lanes<V> load_lanes(const T *p) {
    float v[V];
    load_elems<T, V>(p, v);
    return lanes_of<V>(v);
}
template <class T, int V>
__device__ __forceinline__ Lanes<V> unpack_lanes(const uint4 &u, const T *tag) {
    float v[V];
    unpack(u, v, tag);
    return lanes_of<V>(v);
}
template <class T, int V>
__device__ __forceinline__ void store_lanes(T *p, const Lanes<V> &l) {
    float v[V];
    values_of<V>(l, v);
    store_elems<T, V>(p, v);
}
// ---- streaming ------------------------------------------------------------------------
// A thread of a 256-thread block walks over vectors that lie a fixed step
// apart.  16-byte vectors go through a ring in shared memory that is private
// to the thread (kRing copies in flight, no barrier: a read-only stream at
// 6.4 TB/s, where batches of eight register loads reached 5.5); single
// elements are loaded kAhead at a time.
constexpr int kStreamThreads = 256, kRing = 16, kAhead = 16;
__device__ __forceinline__ void copy_vector(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Raw elements as loaded: 16 bytes, or one element.
template <class T, int V>
struct Raw {
    uint4 u;
};
template <class T>
struct Raw<T, 1> {
    T u;
};
template <class T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T *p) {
    Raw<T, V> r;
    if constexpr (V == 1) r.u = *p;
    else r.u = __ldg(reinterpret_cast<const uint4 *>(p));
    return r;
}
template <class T, int V>
__device__ __forceinline__ Lanes<V> lanes_of_raw(const Raw<T, V> &r) {
    float v[V];
    if constexpr (V == 1) v[0] = to_float(r.u);
    else unpack(r.u, v, static_cast<const T *>(nullptr));
    return lanes_of<V>(v);
}

// Calls f(k, vector) for a thread's vectors.  ring: kRing * kStreamThreads
// vectors of shared memory (V > 1).  start_vectors issues the first copies and
// may run before the wait for an earlier launch that does not write the data.
template <int V, class T>
__device__ __forceinline__ void start_vectors(uint4 *ring, const T *p, long long step, int count) {
    if constexpr (V > 1) {
        const uint32_t addr = smem_addr(ring + threadIdx.x);
#pragma unroll
        for (int u = 0; u < kRing; ++u, p += step) {
            if (u < count) copy_vector(addr + u * kStreamThreads * sizeof(uint4), p);
            cp_async_commit();
        }
    }
}
template <class T, int V, class F>
__device__ __forceinline__ void for_vectors(uint4 *ring, const T *p, long long step, int count, F f) {
    if constexpr (V == 1) {
        for (int k = 0; k < count; k += kAhead) {
            Raw<T, V> raw[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u, p += step)
                if (k + u < count) raw[u] = load_raw<T, V>(p);
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (k + u < count) f(k + u, lanes_of_raw<T, V>(raw[u]));
        }
    } else {
        const uint4 *mine = ring + threadIdx.x;
        const uint32_t addr = smem_addr(mine);
        constexpr uint32_t kPitch = kStreamThreads * sizeof(uint4);
        p += kRing * step;
#pragma unroll 4
        for (int k = 0; k < count; ++k, p += step) {
            const int slot = k % kRing;
            cp_async_wait<kRing - 1>();
            const Lanes<V> v = unpack_lanes<T, V>(mine[slot * kStreamThreads], p);
            if (k + kRing < count) copy_vector(addr + slot * kPitch, p);
            cp_async_commit();
            f(k, v);
        }
    }
}
// The same for two tensors: f(k, vector of p, vector of q).
template <int V, class T>
__device__ __forceinline__ void start_vector_pairs(uint4 *ring, const T *p, long long pstep, const T *q, long long qstep,
                                                   int count) {
    if constexpr (V > 1) {
        const uint32_t addr = smem_addr(ring + threadIdx.x);
        constexpr uint32_t kPitch = kStreamThreads * sizeof(uint4);
#pragma unroll
        for (int u = 0; u < kRing / 2; ++u, p += pstep, q += qstep) {
            if (u < count) {
                copy_vector(addr + 2 * u * kPitch, p);
                copy_vector(addr + (2 * u + 1) * kPitch, q);
            }
            cp_async_commit();
        }
    }
}
// RUN > 0 (a multiple of kRing): end_run() after each RUN vectors and the last.
struct Nothing {
    __device__ __forceinline__ void operator()() const {}
};
template <class T, int V, int RUN = 0, class F, class E = Nothing>
__device__ __forceinline__ void for_vector_pairs(uint4 *ring, const T *p, long long pstep, const T *q, long long qstep,
                                                 int count, F f, E end_run = {}) {
    static_assert(RUN % kRing == 0 && RUN % kAhead == 0, "whole turns of the ring");
    if constexpr (V == 1) {
        constexpr int kPair = kAhead / 2;
        for (int start = 0; start < count;) {
            const int stop = RUN > 0 ? min(count, start + RUN) : count;
            for (int k = start; k < stop; k += kPair) {
                Raw<T, V> a[kPair], b[kPair];
#pragma unroll
                for (int u = 0; u < kPair; ++u, p += pstep, q += qstep)
                    if (k + u < stop) {
                        a[u] = load_raw<T, V>(p);
                        b[u] = load_raw<T, V>(q);
                    }
#pragma unroll
                for (int u = 0; u < kPair; ++u)
                    if (k + u < stop) f(k + u, lanes_of_raw<T, V>(a[u]), lanes_of_raw<T, V>(b[u]));
            }
            start = stop;
            end_run();
        }
    } else {
        constexpr int kHalf = kRing / 2;
        const uint4 *mine = ring + threadIdx.x;
        const uint32_t addr = smem_addr(mine);
        constexpr uint32_t kPitch = kStreamThreads * sizeof(uint4);
        p += kHalf * pstep;
        q += kHalf * qstep;
        for (int k = 0; k < count;) {
            const int stop = RUN > 0 ? min(count, k + RUN) : count;
#pragma unroll 2
            for (; k < stop; ++k, p += pstep, q += qstep) {
                const int slot = 2 * (k % kHalf);
                cp_async_wait<kHalf - 1>();
                const Lanes<V> v = unpack_lanes<T, V>(mine[slot * kStreamThreads], p);
                const Lanes<V> g = unpack_lanes<T, V>(mine[(slot + 1) * kStreamThreads], p);
                if (k + kHalf < count) {
                    copy_vector(addr + slot * kPitch, p);
                    copy_vector(addr + (slot + 1) * kPitch, q);
                }
                cp_async_commit();
                f(k, v, g);
            }
            end_run();
        }
    }
}
// Bytes of the ring.
__host__ __device__ inline size_t ring_space(int v) { return v == 1 ? 0 : kRing * kStreamThreads * sizeof(uint4); }

// ---- activations --------------------------------------------------------------------
// s = 1 / p, p = 1 + e, e = 2^(-z log2 e), and rest = 1 - s = e s of two values,
// with three of the special-function unit's instructions instead of four (that
// unit, a sixteenth of an SM's issue width, bounds the 16-bit kernels): one
// reciprocal serves both, r = 1 / (p q 2^-126), 1 / p = (q 2^-126) r.  The scale
// lets e go up to 2^127 in both: p q 2^-126 then is infinite and r 0.  e is held
// there, and s, below the normal numbers, becomes 0: z s is 0 for every finite z
// below -88, and NaN at -inf like v / (1 + exp(-v)).  (Branches for what leaves
// the range kept the pairs from overlapping and cost up to 16 %.)  1 - s is e s
// and not a difference because the slope multiplies it by z: the reciprocal's
// error would grow with z.  The approximate instructions are good to about 2^-22
// relative each, and the rounding of z log2 e moves the power by at most |z| 2^-24.
__device__ __forceinline__ void sigmoid2(f2 z, f2 &s, f2 &rest) {
    float a, b, p, q, r;
    split(z * pair(-1.4426950408889634f), a, b);
    a = fminf(a, 127.0f);
    b = fminf(b, 127.0f);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    split(fma2(pair(a, b), pair(0x1p-126f), pair(0x1p-126f)), p, q);  // p 2^-126, q 2^-126
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(p, b, p)));
    asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(s.v) : "l"(pair(q, p).v), "l"(pair(r).v));
    rest = pair(a, b) * s;
}

// Comparisons are written so that a NaN passes through.
__device__ __forceinline__ float relu(float z) { return z < 0.0f ? 0.0f : z; }
__device__ __forceinline__ float relu6(float z) { return z < 0.0f ? 0.0f : z > 6.0f ? 6.0f : z; }

// ACT -1: the activation is `act`, known at run time.
template <int ACT>
__device__ __forceinline__ f2 activate(int act, f2 z) {
    if constexpr (ACT >= 0) act = ACT;
    if (act == kActSilu) {
        f2 s, rest;
        sigmoid2(z, s, rest);
        return z * s;
    }
    if (act == kActNone) return z;
    float a, b;
    split(z, a, b);
    return act == kActRelu ? pair(relu(a), relu(b)) : pair(relu6(a), relu6(b));
}

// g * act'(z)
template <int ACT>
__device__ __forceinline__ f2 activate_grad(int act, f2 z, f2 g) {
    if constexpr (ACT >= 0) act = ACT;
    if (act == kActSilu) {
        f2 s, rest;
        sigmoid2(z, s, rest);
        return g * (s * fma2(z, rest, pair(1.0f)));
    }
    if (act == kActNone) return g;
    float a, b, ga, gb;
    split(z, a, b);
    split(g, ga, gb);
    const float top = act == kActRelu6 ? 6.0f : __int_as_float(0x7f800000);
    const bool open = act == kActRelu6;
    return pair(a <= 0.0f || (open && a >= top) ? 0.0f : ga, b <= 0.0f || (open && b >= top) ? 0.0f : gb);
}

// ---- dropout ------------------------------------------------------------------------
struct DropParams {
    uint32_t threshold;  // t: keep when the 16-bit draw is at least this; 0 = no dropout, 65536 = drop all
    uint32_t limit;      // 65536 t - 1: the draw in a word's upper half is kept when the word is above it
    float scale;         // 1 / (1 - t / 65536), 0 when everything is dropped
    int channel;         // one decision per channel of an image
    uint64_t seed, offset;
    const uint64_t *seed_ptr, *offset_ptr;  // nullable, added to seed and offset
    uint64_t *used;                         // nullable, receives what is in effect
};

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", 2011): ten rounds of two 32 x 32 -> 64 bit products.  Sixteen
// bits a decision make one block of four words serve eight elements: with 32
// bits the generator, not the memory, would bound 16-bit tensors.  The first
// product of the offset and the round keys are the same for every block of a
// launch and are computed once; the keys are kept from being recomputed (an
// integer addition takes as many issue slots as two of FP32).
struct Philox {
    uint32_t key[20], first, c3;  // first: high word of the first round's second product, keyed
    uint32_t low;                 // its low word
    __device__ __forceinline__ Philox() {}
    // To be called after the wait for earlier launches (the words may be theirs).
    __device__ __forceinline__ Philox(const DropParams &p, bool writer) {
        uint64_t seed = p.seed, offset = p.offset;
        if (p.seed_ptr != nullptr) seed += *p.seed_ptr;
        if (p.offset_ptr != nullptr) offset += *p.offset_ptr;
        if (writer && p.used != nullptr) {
            p.used[0] = seed;
            p.used[1] = offset;
        }
        uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
        for (int r = 0; r < 10; ++r) {
            key[2 * r] = k0;
            key[2 * r + 1] = k1;
            asm("" : "+r"(key[2 * r]), "+r"(key[2 * r + 1]));
            k0 += 0x9E3779B9u;
            k1 += 0xBB67AE85u;
        }
        const uint64_t b = static_cast<uint64_t>(static_cast<uint32_t>(offset)) * 0xCD9E8D57u;
        first = static_cast<uint32_t>(b >> 32) ^ key[0];
        low = static_cast<uint32_t>(b);
        c3 = static_cast<uint32_t>(offset >> 32) ^ key[1];
    }
    __device__ __forceinline__ uint4 operator()(uint64_t block) const {
        const uint64_t a = static_cast<uint64_t>(static_cast<uint32_t>(block)) * 0xD2511F53u;
        uint32_t x0 = first ^ static_cast<uint32_t>(block >> 32), x1 = low;
        uint32_t x2 = static_cast<uint32_t>(a >> 32) ^ c3, x3 = static_cast<uint32_t>(a);
#pragma unroll
        for (int r = 1; r < 10; ++r) {
            const uint64_t u = static_cast<uint64_t>(x0) * 0xD2511F53u;
            const uint64_t v = static_cast<uint64_t>(x2) * 0xCD9E8D57u;
            x0 = static_cast<uint32_t>(v >> 32) ^ x1 ^ key[2 * r];
            x1 = static_cast<uint32_t>(v);
            x2 = static_cast<uint32_t>(u >> 32) ^ x3 ^ key[2 * r + 1];
            x3 = static_cast<uint32_t>(u);
        }
        return make_uint4(x0, x1, x2, x3);
    }
};

// The draws of V consecutive decisions, two a word (V = 1: in the upper half).
template <int V>
struct Draws {
    uint32_t w[(V + 1) / 2];
    // j0 is a multiple of V and V divides 8, so that one block holds them all.
    __device__ __forceinline__ Draws(const Philox &gen, uint64_t j0) {
        const uint4 b = gen(j0 >> 3);
        const int at = static_cast<int>(j0 & 7);
        if constexpr (V == 8) {
            w[0] = b.x, w[1] = b.y, w[2] = b.z, w[3] = b.w;
        } else if constexpr (V == 4) {
            w[0] = at ? b.z : b.x, w[1] = at ? b.w : b.y;
        } else {
            static_assert(V == 1, "vectors of 8, 4 or 1");
            const uint32_t d = at < 4 ? (at < 2 ? b.x : b.y) : (at < 6 ? b.z : b.w);
            w[0] = at & 1 ? d : d << 16;
        }
    }
    __device__ __forceinline__ Draws() {}
    __device__ __forceinline__ bool keep(int j, uint32_t limit) const {
        return (V == 1 || (j & 1) ? w[j / 2] : w[j / 2] << 16) > limit;
    }
    __device__ __forceinline__ uint32_t bits(uint32_t limit) const {
        uint32_t r = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) r |= keep(j, limit) ? 1u << j : 0u;
        return r;
    }
};

// Kept values scaled, the others 0 whatever they hold.
template <int V>
__device__ __forceinline__ Lanes<V> drop_lanes(const Lanes<V> &l, const Draws<V> &d, const DropParams &p) {
    float v[V];
    values_of<V>(l, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = d.keep(j, p.limit) ? v[j] * p.scale : 0.0f;
    return lanes_of<V>(v);
}
template <int V>
__device__ __forceinline__ Lanes<V> drop_lanes(const Lanes<V> &l, uint32_t bits, const DropParams &p) {
    float v[V];
    values_of<V>(l, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = bits >> j & 1u ? v[j] * p.scale : 0.0f;
    return lanes_of<V>(v);
}

}  // namespace gcb
