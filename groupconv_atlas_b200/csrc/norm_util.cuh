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

// Element i of a parameter vector whose type is known at run time.
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

// ---- activations --------------------------------------------------------------------
// Comparisons are written so that a NaN passes through.
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if (ACT == kActRelu) return z < 0.0f ? 0.0f : z;
    if (ACT == kActRelu6) return z < 0.0f ? 0.0f : z > 6.0f ? 6.0f : z;
    if (ACT == kActSilu) return z * sigmoid(z);
    return z;
}

// g * act'(z)
template <int ACT>
__device__ __forceinline__ float activate_grad(float z, float g) {
    if (ACT == kActRelu) return z <= 0.0f ? 0.0f : g;
    if (ACT == kActRelu6) return z <= 0.0f || z >= 6.0f ? 0.0f : g;
    if (ACT == kActSilu) {
        const float s = sigmoid(z);
        return g * (s * fmaf(z, 1.0f - s, 1.0f));
    }
    return g;
}

// ---- dropout ------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", 2011): ten rounds of two 32 x 32 -> 64 bit products.  Sixteen
// bits a decision make one call serve eight elements: the ten rounds are about
// 50 instructions, and with 32 bits a decision the generator, not the memory,
// would bound 16-bit tensors.
__device__ __forceinline__ uint4 philox(uint64_t block, uint64_t offset, uint64_t seed) {
    uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32);
    uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u;
        const uint64_t b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
        c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
        c1 = static_cast<uint32_t>(b);
        c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
        c3 = static_cast<uint32_t>(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

struct DropParams {
    uint32_t threshold;  // keep when the 16-bit draw is at least this; 0 = keep all, 65536 = drop all
    float scale;         // 1 / (1 - threshold / 65536), 0 when everything is dropped
    int channel;         // one decision per channel of an image
    uint64_t seed, offset;
    const uint64_t *seed_ptr, *offset_ptr;  // nullable, added to seed and offset
    uint64_t *used;                         // nullable, receives what is in effect
};

struct DropState {
    uint64_t seed, offset;
};

// To be called after the wait for earlier launches (the words may be theirs).
__device__ __forceinline__ DropState drop_state(const DropParams &p, bool writer) {
    DropState s{p.seed, p.offset};
    if (p.seed_ptr != nullptr) s.seed += *p.seed_ptr;
    if (p.offset_ptr != nullptr) s.offset += *p.offset_ptr;
    if (writer && p.used != nullptr) {
        p.used[0] = s.seed;
        p.used[1] = s.offset;
    }
    return s;
}

// Keep bits (bit k: draw j0 + k) of V consecutive decisions; j0 is a multiple
// of V and V divides 8, so that one block holds them all.
template <int V>
__device__ __forceinline__ uint32_t keep_bits(const DropParams &p, const DropState &s, uint64_t j0) {
    const uint4 w = philox(j0 >> 3, s.offset, s.seed);
    const int first = static_cast<int>(j0 & 7);
    uint32_t bits = 0;
    if constexpr (V == 8) {
        const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            bits |= ((d[k] & 0xffffu) >= p.threshold ? 1u : 0u) << (2 * k);
            bits |= ((d[k] >> 16) >= p.threshold ? 2u : 0u) << (2 * k);
        }
    } else if constexpr (V == 4) {
        const uint32_t d[2] = {first ? w.z : w.x, first ? w.w : w.y};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            bits |= ((d[k] & 0xffffu) >= p.threshold ? 1u : 0u) << (2 * k);
            bits |= ((d[k] >> 16) >= p.threshold ? 2u : 0u) << (2 * k);
        }
    } else {
        static_assert(V == 1, "vectors of 8, 4 or 1");
        const uint32_t d = first < 4 ? (first < 2 ? w.x : w.y) : (first < 6 ? w.z : w.w);
        bits = ((first & 1 ? d >> 16 : d & 0xffffu) >= p.threshold) ? 1u : 0u;
    }
    return bits;
}

}  // namespace gcb
