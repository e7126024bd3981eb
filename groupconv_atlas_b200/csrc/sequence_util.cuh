// Building blocks of the operators on rows and sequences (layer norm, causal
// convolution, selective scan): views of strided tensors, and the sums of
// partial results over rows.
#pragma once
#include "tensor_checks.cuh"

namespace gcb {

// A strided tensor whose last axis is dense and whose elements do not share
// memory: strides in elements, the bytes from its first to its last element.
struct Strided {
    char *data = nullptr;
    int type = 0, rank = 0;
    long long d[4] = {}, s[4] = {};
    uint64_t span = 0;
    bool empty = false;
};

inline int strided_of(const gc_tensor *t, Strided &v) {
    if (t->dtype == GC_F64) return gc_error(GC_UNSUPPORTED, "FP64 tensors are not supported here");
    v = Strided{};
    v.data = static_cast<char *>(t->data);
    v.type = elem_type(t->dtype);
    v.rank = t->rank;
    int order[4] = {};
    int axes = 0;
    for (int i = 0; i < t->rank; ++i) {
        v.d[i] = t->dims[i];
        v.s[i] = t->dims[i] > 1 ? t->strides[i] : 0;
        v.empty = v.empty || t->dims[i] == 0;
        if (t->dims[i] <= 1) continue;
        int k = axes++;  // by ascending stride
        for (; k > 0 && t->strides[order[k - 1]] > t->strides[i]; --k) order[k] = order[k - 1];
        order[k] = i;
    }
    if (v.empty) return GC_OK;
    if (t->dims[t->rank - 1] > 1 && t->strides[t->rank - 1] != 1)
        return gc_error(GC_UNSUPPORTED, "the last axis must be dense");
    wide reach = 1;  // elements from the first to the last of the axes so far
    for (int k = 0; k < axes; ++k) {
        const int i = order[k];
        if (t->strides[i] < reach) return gc_error(GC_UNSUPPORTED, "tensor overlaps itself or has a negative stride");
        reach += static_cast<wide>(t->dims[i] - 1) * t->strides[i];
        if (reach > PTRDIFF_MAX / 8) return gc_error(GC_INVALID, "tensor extent overflow");
    }
    if (reach * elem_size(v.type) > static_cast<wide>(t->bytes)) return gc_error(GC_INVALID, "tensor buffer is too small");
    v.span = static_cast<uint64_t>(reach) * elem_size(v.type);
    return GC_OK;
}
inline Range range_of(const Strided &v) { return {v.data, v.span}; }

// Whether groups of `e` elements along the last axis start on their own size.
inline bool group_aligned(const Strided &v, int e) {
    if (reinterpret_cast<uintptr_t>(v.data) % (static_cast<size_t>(e) * elem_size(v.type)) != 0) return false;
    for (int i = 0; i + 1 < v.rank; ++i)
        if (v.s[i] % e != 0) return false;
    return v.d[v.rank - 1] % e == 0;
}

// A nullable dense parameter tensor, F32 or of `like`'s type, of the given dims.
inline int check_param(const gc_tensor *t, const gc_tensor *like, std::initializer_list<int64_t> dims) {
    if (t == nullptr) return GC_OK;
    int64_t count = 0;
    const int rank = static_cast<int>(dims.size());
    const int st = check_fields(t, rank, rank, count);
    if (st != GC_OK) return st;
    int i = 0;
    for (const int64_t d : dims)
        if (t->dims[i++] != d) return gc_error(GC_INVALID, "parameter dimensions do not fit the data");
    if (t->dtype != GC_F32 && t->dtype != like->dtype)
        return gc_error(GC_INVALID, "parameters must be F32 or of the data's type");
    if (t->device_index != like->device_index) return gc_error(GC_INVALID, "tensor device indices differ");
    return GC_OK;
}
inline int check_dense(const gc_tensor *t, const char *message) {
    if (t == nullptr) return GC_OK;
    wide expect = 1;
    for (int i = t->rank - 1; i >= 0; --i) {
        if (t->dims[i] > 1 && t->strides[i] != expect) return gc_error(GC_UNSUPPORTED, message);
        expect *= t->dims[i];
    }
    return GC_OK;
}

// ---- sums over rows of partial results ------------------------------------------------
// part holds `rows` rows of `planes` planes of `cols` 32-bit values; plane q's
// sum over the rows goes to element col * mul[q] + add[q] of out[q] (skipped
// where that is NULL).  A block takes 32 columns of a plane (a line of a row), or,
// of more than 256 rows, 8 (a sector): how many loads follow one another is then what
// counts.  With 32 columns 1184 rows of 2 x 1001 take 14 us, with 8 columns 9; 52 rows
// of 32768 take 7 and 15, 37 rows of 5 x 2048 4 and 6.  Its workers take the rows in
// turn, eight loads under way, in runs of 64 values in 32 bits joined in 64, and are
// joined in a fixed order.
constexpr int kSumPlanes = 9, kSumThreads = 512, kSumRun = 64;
struct SumParams {
    const float *part;
    long long rows, cols;
    int planes;
    void *out[kSumPlanes];
    int type[kSumPlanes];
    long long mul[kSumPlanes], add[kSumPlanes];
};
cudaError_t launch_sum_rows(SumParams &P, cudaStream_t stream);

}  // namespace gcb
