// Checks of descriptors and calls that the entry points for strided tensors of
// several types share (group norm, dropout and the operators on sequences).
#pragma once
#include "groupconv.h"

#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "host_util.h"
#include "norm_util.cuh"

namespace gcb {

typedef __int128 wide;  // products of descriptor fields, before they are known to fit

inline int elem_type(int dtype) {
    return dtype == GC_F32 ? kElemF32 : dtype == GC_B200_F16 ? kElemF16
         : dtype == GC_B200_BF16 ? kElemBF16 : -1;
}
inline int elem_size(int type) { return type == kElemF32 ? 4 : 2; }

// What every descriptor of these entry points has to satisfy (GC_INVALID
// conditions, then FP64 as a valid type outside this set).
inline int check_fields(const gc_tensor *t, int rank_low, int rank_high, int64_t &count) {
    if (t == nullptr) return gc_error(GC_INVALID, "null tensor descriptor");
    if (t->rank < rank_low || t->rank > rank_high) return gc_error(GC_INVALID, "tensor rank out of range");
    if (t->device != GC_CUDA || t->device_index < 0) return gc_error(GC_INVALID, "tensor must be CUDA memory");
    if (t->dtype != GC_F64 && elem_type(t->dtype) < 0) return gc_error(GC_INVALID, "unknown tensor dtype");
    wide n = 1;
    for (int i = 0; i < t->rank; ++i) {
        if (t->dims[i] < 0) return gc_error(GC_INVALID, "tensor dimensions must not be negative");
        n *= t->dims[i];
        if (n > PTRDIFF_MAX / 8) return gc_error(GC_INVALID, "tensor element count overflow");
    }
    count = static_cast<int64_t>(n);
    if (count == 0) return GC_OK;
    if (t->data == nullptr) return gc_error(GC_INVALID, "null tensor buffer");
    const uintptr_t base = reinterpret_cast<uintptr_t>(t->data);
    const unsigned item = t->dtype == GC_F64 ? 8 : elem_size(elem_type(t->dtype));
    if (base % item != 0) return gc_error(GC_INVALID, "tensor data is not element aligned");
    if (t->bytes > UINTPTR_MAX - base) return gc_error(GC_INVALID, "tensor pointer range overflow");
    if (t->bytes / item < static_cast<uint64_t>(count)) return gc_error(GC_INVALID, "tensor buffer is too small");
    return GC_OK;
}

inline bool same_dims(const gc_tensor *a, const gc_tensor *b) {
    if (a->rank != b->rank) return false;
    for (int i = 0; i < a->rank; ++i)
        if (a->dims[i] != b->dims[i]) return false;
    return true;
}

inline bool ranges_meet(const void *a, uint64_t an, const void *b, uint64_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return an != 0 && bn != 0 && x < y + bn && y < x + an;
}
struct Range {
    const void *p;
    uint64_t bytes;
};
// Outputs against inputs and against one another.
inline bool outputs_meet(std::initializer_list<Range> outs, std::initializer_list<Range> ins) {
    for (const Range *o = outs.begin(); o != outs.end(); ++o) {
        for (const Range &i : ins)
            if (ranges_meet(o->p, o->bytes, i.p, i.bytes)) return true;
        for (const Range *q = outs.begin(); q != o; ++q)
            if (ranges_meet(o->p, o->bytes, q->p, q->bytes)) return true;
    }
    return false;
}

inline Range range_of(const gc_tensor *t) {
    if (t == nullptr) return {nullptr, 0};
    uint64_t n = t->dtype == GC_F64 ? 8 : elem_size(elem_type(t->dtype));
    for (int i = 0; i < t->rank; ++i) n *= static_cast<uint64_t>(t->dims[i]);
    return {t->data, n};
}

// The current device, the pointers' device and the stream (reference
// groupconv.cu:130-139, :185-191).
inline int check_call(std::initializer_list<const gc_tensor *> tensors, std::initializer_list<const void *> words,
                      int device_index, void *stream, int &dev) {
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return gc_error(GC_DEVICE_ERROR, cudaGetErrorString(e));
    for (const gc_tensor *t : tensors)
        if (t != nullptr && range_of(t).bytes != 0) {
            const int st = check_pointer(t, dev);
            if (st != GC_OK) return st;
        }
    for (const void *p : words)
        if (p != nullptr) {
            const int st = check_device_memory(p, device_index, dev);
            if (st != GC_OK) return st;
        }
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    e = cudaStreamIsCapturing(reinterpret_cast<cudaStream_t>(stream), &cs);
    return e == cudaSuccess ? GC_OK : gc_error(GC_DEVICE_ERROR, cudaGetErrorString(e));
}

inline int launched(cudaError_t e) {
    if (e == cudaSuccess) e = cudaGetLastError();
    else cudaGetLastError();
    return e == cudaSuccess ? gc_error(GC_OK, "") : gc_error(GC_DEVICE_ERROR, cudaGetErrorString(e));
}
// The same, with the plan of a call that succeeded.
template <class... T>
int launched(cudaError_t e, PlanRecord::Kind kind, const char *name, T... values) {
    const int st = launched(e);
    if (st == GC_OK) record_plan(kind, name, false, values...);
    return st;
}

inline uint64_t up16(uint64_t v) { return (v + 15) / 16 * 16; }

inline int check_workspace(const void *p, uint64_t bytes, uint64_t need) {
    if (need == 0) return GC_OK;
    if (p == nullptr || bytes < need) return gc_error(GC_INVALID, "workspace is missing or too small");
    if (!aligned16(p)) return gc_error(GC_INVALID, "workspace must be 16-byte aligned");
    return GC_OK;
}

// No exception leaves a C entry point; those that can arise here come from host
// memory that ran out.
inline int internal_error() { return gc_error(GC_DEVICE_ERROR, "host resources exhausted"); }

}  // namespace gcb
