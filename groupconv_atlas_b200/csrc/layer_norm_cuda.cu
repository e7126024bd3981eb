// gc_b200_layer_norm and its gradient: descriptor checks, plans and launches.
// Nothing here allocates device memory, synchronizes or keeps anything of a call.
#include "groupconv.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "host_util.h"
#include "kernel_layer_norm.cuh"
#include "sequence_util.cuh"

namespace {

using namespace gcb;

// x as rows of its last axis, evenly spaced.
struct Rows {
    Strided t;
    long long rows = 1, ld = 0;
};
int rows_of(const gc_tensor *t, Rows &v) {
    const int st = strided_of(t, v.t);
    if (st != GC_OK) return st;
    const int last = t->rank - 1;
    v.rows = 1;
    v.ld = v.t.d[last];
    bool even = true;
    for (int i = last - 1; i >= 0; --i) {
        if (v.t.d[i] > 1) {
            if (v.rows == 1) v.ld = v.t.s[i];
            else even = even && static_cast<wide>(v.ld) * v.rows == v.t.s[i];
        }
        v.rows *= v.t.d[i];
    }
    return even || v.t.empty ? GC_OK : gc_error(GC_UNSUPPORTED, "rows are not evenly spaced");
}

// Data tensors of the same dims and type; views[0] is x's.
int check_rows(std::initializer_list<const gc_tensor *> tensors, Rows *views) {
    const gc_tensor *first = *tensors.begin();
    int64_t count = 0;
    for (const gc_tensor *t : tensors) {
        const int st = check_fields(t, 1, 4, count);
        if (st != GC_OK) return st;
        if (!same_dims(t, first)) return gc_error(GC_INVALID, "tensor dimensions differ");
        if (t->dtype != first->dtype) return gc_error(GC_INVALID, "tensor dtypes differ");
        if (t->device_index != first->device_index) return gc_error(GC_INVALID, "tensor device indices differ");
    }
    const int64_t c = first->dims[first->rank - 1];
    if (c < 1 || c > INT32_MAX) return gc_error(GC_INVALID, "row length out of range");
    for (const gc_tensor *t : tensors) {
        const int st = rows_of(t, *views++);
        if (st != GC_OK) return st;
    }
    return GC_OK;
}

int check_row_stats(const gc_tensor *t, const gc_tensor *x, long long rows) {
    int64_t count = 0;
    const int st = check_fields(t, 2, 2, count);
    if (st != GC_OK) return st;
    if (t->dtype != GC_F32 || t->dims[0] != rows || t->dims[1] != 2)
        return gc_error(GC_INVALID, "stats must be an F32 tensor of dims (rows, 2)");
    if (t->device_index != x->device_index) return gc_error(GC_INVALID, "tensor device indices differ");
    if (reinterpret_cast<uintptr_t>(t->data) % 8 != 0) return gc_error(GC_INVALID, "stats must be 8-byte aligned");
    return GC_OK;
}

struct RowPlan {
    bool vec = false, whole = false;  // whole: rows too long for registers
    bool edges = false;               // rows that start anywhere within 16 bytes, in vectors all the same
    int type = 0, v = 1, nv = 1, team = 1, threads = kRowThreads;
    size_t smem = 0;
    long long blocks = 0;
};

const char *const kDenseParams = "parameters must be dense";

// Vectors of a row for each thread, by how many of the threads' places stay empty,
// then by the longest run of a thread: sums between threads cost more than those in
// one (100352 rows of 96 FP32: 18 us in teams of 4 with six vectors each, 24 in teams
// of 8 with three), unless the rows are few, when each thread's own work is what
// takes the time (196 rows of 384 bf16: 6.0 us with six, 4.0 with three).  A team of
// up to 32 threads has no barriers; the gradient, which holds its columns' sums in
// registers, goes over to whole blocks earlier.  Single elements are taken four or
// sixteen (backwards eight) a thread.
void plan_rows(int c, int type, bool vec, bool backward, bool few, RowPlan &p) {
    p.type = type;
    p.vec = vec;
    p.v = !vec ? 1 : type == kElemF32 ? 4 : 8;
    const long long vcols = c / p.v;
    p.threads = kRowThreads;
    if (vec) {
        const int most = backward ? (p.v == 8 ? 3 : 4) : 8;
        long long best = 0;
        static const int longest[] = {8, 6, 4, 3, 2, 1}, shortest[] = {4, 3, 6, 8, 2, 1};
        for (int i = 0; i < 6; ++i) {
            const int nv = few ? shortest[i] : longest[i];
            if (nv > most) continue;
            int team = 1;
            while (static_cast<long long>(team) * nv < vcols) team *= 2;
            if (team > 32) continue;
            if (best == 0 || static_cast<long long>(team) * nv < best) {
                best = static_cast<long long>(team) * nv;
                p.nv = nv;
                p.team = team;
            }
        }
        if (best != 0) {
            if (backward) p.smem = static_cast<size_t>(p.threads / 32) * 2 * c * sizeof(float);
            return;
        }
        p.nv = backward ? 1 : 4;
        while (p.nv < (backward ? (p.v == 8 ? 2 : 4) : 8) && ceil_div(vcols, p.nv) > kRowMost) p.nv *= 2;
    } else {
        p.nv = ceil_div(vcols, 4) <= kRowMost ? 4 : backward ? 8 : 16;
    }
    const long long lanes = ceil_div(vcols, p.nv);
    p.whole = lanes > kRowMost;
    if (p.whole) {
        p.team = p.threads = kRowMost;
    } else if (lanes > 32) {
        p.team = p.threads = static_cast<int>(round_up(lanes, 32));
    } else {
        for (p.team = 1; p.team < lanes;) p.team *= 2;
        if (backward) p.smem = static_cast<size_t>(p.threads / 32) * 2 * c * sizeof(float);
    }
}

template <class T, int V>
const void *forward_typed(int nv) {
    if constexpr (V == 1) {
        return nv == 4 ? reinterpret_cast<const void *>(&layer_norm_kernel<T, 1, 4, 2>)
                       : reinterpret_cast<const void *>(&layer_norm_kernel<T, 1, 16, 1>);
    } else {
        switch (nv) {
        case 1: return reinterpret_cast<const void *>(&layer_norm_kernel<T, V, 1, 4>);
        case 2: return reinterpret_cast<const void *>(&layer_norm_kernel<T, V, 2, 2>);
        case 3: return reinterpret_cast<const void *>(&layer_norm_kernel<T, V, 3, 2>);
        case 4: return reinterpret_cast<const void *>(&layer_norm_kernel<T, V, 4, 1>);
        case 6: return reinterpret_cast<const void *>(&layer_norm_kernel<T, V, 6, 1>);
        default: return reinterpret_cast<const void *>(&layer_norm_kernel<T, V, 8, 1>);
        }
    }
}
template <class T, int V>
const void *backward_typed(int nv) {
    if constexpr (V == 1) {
        return nv == 4 ? reinterpret_cast<const void *>(&layer_norm_grad_kernel<T, 1, 4, 2>)
                       : reinterpret_cast<const void *>(&layer_norm_grad_kernel<T, 1, 8, 1>);
    } else {
        switch (nv) {
        case 1: return reinterpret_cast<const void *>(&layer_norm_grad_kernel<T, V, 1, 2>);
        case 2: return reinterpret_cast<const void *>(&layer_norm_grad_kernel<T, V, 2, 1>);
        case 3: return reinterpret_cast<const void *>(&layer_norm_grad_kernel<T, V, 3, 1>);
        default:
            if constexpr (V == 4) return reinterpret_cast<const void *>(&layer_norm_grad_kernel<T, V, 4, 1>);
            else return nullptr;  // not planned
        }
    }
}
// Rows that start anywhere: aligned vectors cover a row, one more than it would need,
// in teams of a warp at least.  False where that does not apply.
bool plan_edges(int c, int type, bool backward, RowPlan &p) {
    p = RowPlan{};
    p.type = type;
    p.v = type == kElemF32 ? 4 : 8;
    const int vcols = (c + p.v - 2) / p.v + 1, most = backward ? (p.v == 8 ? 2 : 4) : 4;
    if (vcols <= 32 || c > 4096) return false;
    p.edges = true;
    for (p.nv = 1; p.nv < most && vcols > 32 * p.nv;) p.nv *= 2;
    if (vcols <= 32 * p.nv) {
        p.team = 32;
        p.threads = kRowThreads;
        if (backward) p.smem = static_cast<size_t>(p.threads / 32) * 2 * c * sizeof(float);
    } else {
        for (p.nv = backward ? 1 : 2; p.nv < most && ceil_div(vcols, p.nv) > kRowMost;) p.nv *= 2;
        if (ceil_div(vcols, p.nv) > kRowMost) return false;
        p.team = p.threads = static_cast<int>(round_up(ceil_div(vcols, p.nv), 32));
    }
    if (!backward) p.smem = 2 * static_cast<size_t>((c - 1) + (c - 1) / p.v + 1) * sizeof(float);
    return true;
}
// Whether x, dy and the result start at the same place within 16 bytes in every row.
bool start_alike(std::initializer_list<const Rows *> views) {
    const Rows *first = *views.begin();
    const int size = elem_size(first->t.type);
    for (const Rows *v : views)
        if ((reinterpret_cast<uintptr_t>(v->t.data) - reinterpret_cast<uintptr_t>(first->t.data)) % 16 != 0 ||
            (v->rows > 1 && (v->ld - first->ld) * size % 16 != 0))
            return false;
    return true;
}
template <class T>
const void *edges_kernel(int nv, bool backward) {
    if (backward)
        return nv == 1   ? reinterpret_cast<const void *>(&layer_norm_edges_grad_kernel<T, 1>)
               : nv == 2 ? reinterpret_cast<const void *>(&layer_norm_edges_grad_kernel<T, 2>)
                         : reinterpret_cast<const void *>(&layer_norm_edges_grad_kernel<T, sizeof(T) == 4 ? 4 : 2>);
    return nv == 1   ? reinterpret_cast<const void *>(&layer_norm_edges_kernel<T, 1>)
           : nv == 2 ? reinterpret_cast<const void *>(&layer_norm_edges_kernel<T, 2>)
                     : reinterpret_cast<const void *>(&layer_norm_edges_kernel<T, 4>);
}

template <class T>
const void *row_kernel(const RowPlan &p, bool backward) {
    if (p.edges) return edges_kernel<T>(p.nv, backward);
    if (p.whole)
        return backward ? reinterpret_cast<const void *>(&layer_norm_long_grad_kernel<T>)
                        : reinterpret_cast<const void *>(&layer_norm_long_kernel<T>);
    if (p.vec) return backward ? backward_typed<T, kVec<T>>(p.nv) : forward_typed<T, kVec<T>>(p.nv);
    return backward ? backward_typed<T, 1>(p.nv) : forward_typed<T, 1>(p.nv);
}
const void *row_kernel(const RowPlan &p, bool backward) {
    return p.type == kElemF16    ? row_kernel<__half>(p, backward)
           : p.type == kElemBF16 ? row_kernel<__nv_bfloat16>(p, backward)
                                 : row_kernel<float>(p, backward);
}

// Blocks of the gradient: 1024 threads a multiprocessor, more where a team would add up
// more than 64 rows.  By their registers fewer fit at once: of 592 blocks at 16384 x 2048
// bf16 444 (70 registers, 1.33 rounds), of 1184 at 8191 x 1001 bf16 740 (83, 1.6 rounds).
long long grad_blocks(const RowPlan &p, long long rows, int sms) {
    const int teams = p.threads / p.team;
    const long long blocks = std::max(std::min(ceil_div(rows, teams), 2LL * sms * (kRowMost / p.threads)),
                                      ceil_div(rows, static_cast<long long>(kSumRun) * teams));
    // every eighth row at most starts at the same place: a team's rows lie so far apart
    return p.edges ? round_up(blocks, 8) : blocks;
}

// Whether the parameters can be read 16 bytes at a time (4 or 8 columns; their
// type may be wider than the data's).
bool aligned_params(std::initializer_list<const gc_tensor *> params, int v) {
    for (const gc_tensor *t : params)
        if (t != nullptr && (!aligned16(t->data) || (v == 4 && t->dtype != GC_F32))) return false;
    return true;
}

bool vectors(std::initializer_list<const Rows *> views);
RowPlan plan_backward(int c, const Rows (&v)[3]) {
    RowPlan plan;
    const bool vec = vectors({&v[0], &v[1], &v[2]});
    if (vec || !start_alike({&v[0], &v[1], &v[2]}) || !plan_edges(c, v[0].t.type, true, plan))
        plan_rows(c, v[0].t.type, vec, true, false, plan);
    return plan;
}

bool vectors(std::initializer_list<const Rows *> views) {
    for (const Rows *v : views) {
        const int e = v->t.type == kElemF32 ? 4 : 8;
        if (!group_aligned(v->t, e) || v->ld % e != 0) return false;
    }
    return true;
}

void set_param(const gc_tensor *t, const void *&p, int &type) {
    p = t != nullptr ? t->data : nullptr;
    type = t != nullptr ? elem_type(t->dtype) : kElemF32;
}

// Dynamic shared memory that a kernel may have beside its own buffer.
int dynamic_limit(const DeviceFacts &facts) { return facts.smem_optin - 2048; }

int current_facts(DeviceFacts &facts) {
    int dev = -1;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return gc_error(GC_DEVICE_ERROR, cudaGetErrorString(e));
    return device_facts(dev, facts);
}

}  // namespace

extern "C" {

int gc_b200_layer_norm(const gc_tensor *x, const gc_tensor *gamma, const gc_tensor *beta, gc_tensor *y,
                       gc_tensor *stats, double eps, void *stream) try {
    Rows v[2];
    int st = check_rows({x, y}, v);
    if (st != GC_OK) return st;
    if (!(eps >= 0.0) || !std::isfinite(eps)) return gc_error(GC_INVALID, "eps must be finite and not negative");
    const int64_t c = x->dims[x->rank - 1];
    for (const gc_tensor *t : {gamma, beta})
        if ((st = check_param(t, x, {c})) != GC_OK) return st;
    if (stats != nullptr && (st = check_row_stats(stats, x, v[0].rows)) != GC_OK) return st;
    if (outputs_meet({range_of(v[1].t), range_of(stats)}, {range_of(v[0].t), range_of(gamma), range_of(beta)}))
        return gc_error(GC_INVALID, "outputs must not overlap inputs or one another");
    for (const gc_tensor *t : {gamma, beta})
        if ((st = check_dense(t, kDenseParams)) != GC_OK) return st;
    if ((st = check_dense(stats, "stats must be dense")) != GC_OK) return st;
    if (v[0].t.empty) return gc_error(GC_OK, "");
    int dev = -1;
    if ((st = check_call({x, y, gamma, beta, stats}, {}, x->device_index, stream, dev)) != GC_OK) return st;
    DeviceFacts facts;
    if ((st = device_facts(dev, facts)) != GC_OK) return st;
    RowPlan plan;
    const bool vec = vectors({&v[0], &v[1]});
    if (vec || !start_alike({&v[0], &v[1]}) || !plan_edges(static_cast<int>(c), v[0].t.type, false, plan))
        plan_rows(static_cast<int>(c), v[0].t.type, vec, false, v[0].rows <= 4096LL * facts.sms / std::max<int64_t>(c, 1), plan);
    LayerNormParams P{};
    P.x = v[0].t.data;
    P.x_ld = v[0].ld;
    P.y = v[1].t.data;
    P.y_ld = v[1].ld;
    P.rows = v[0].rows;
    P.c = static_cast<int>(c);
    P.vcols = P.c / plan.v;
    P.team = plan.team;
    P.eps = static_cast<float>(eps);
    set_param(gamma, P.gamma, P.gamma_type);
    set_param(beta, P.beta, P.beta_type);
    P.aligned = aligned_params({gamma, beta}, plan.v) ? 1 : 0;
    P.stats = stats != nullptr ? static_cast<float2 *>(stats->data) : nullptr;
    const void *fn = row_kernel(plan, false);
    // Four times the blocks that a multiprocessor has threads for, which take rows in
    // turn where there are more: the multiprocessors are not served alike (16384 rows of
    // 2048 bf16, a row for each team then: 32 us, 35 with a quarter of the blocks).
    const long long grid = std::min(ceil_div(P.rows, plan.threads / plan.team), (plan.edges ? 2048LL : 8192LL) / plan.threads * facts.sms);
    void *args[] = {&P};
    const cudaError_t e = launch_pdl(fn, dim3(static_cast<unsigned>(grid)), dim3(plan.threads), args, plan.smem,
                                     reinterpret_cast<cudaStream_t>(stream));
    return launched(e, PlanRecord::kSequence, plan.whole ? "layer_norm_long" : plan.edges ? "layer_norm_edges" : "layer_norm", grid, plan.threads,
                    plan.vec ? 1 : 0, plan.team, plan.nv, 1, 1);
} catch (...) {
    return internal_error();
}

int gc_b200_layer_norm_backward_workspace(const gc_tensor *dy, const gc_tensor *x, const gc_tensor *dx,
                                          uint64_t *bytes) try {
    if (bytes == nullptr) return gc_error(GC_INVALID, "null size pointer");
    Rows v[3];
    int st = check_rows({x, dy, dx}, v);
    if (st != GC_OK) return st;
    *bytes = 0;
    if (v[0].t.empty) return gc_error(GC_OK, "");
    DeviceFacts facts;
    if ((st = current_facts(facts)) != GC_OK) return st;
    const int c = static_cast<int>(x->dims[x->rank - 1]);
    const RowPlan plan = plan_backward(c, v);
    *bytes = up16(static_cast<uint64_t>(grad_blocks(plan, v[0].rows, facts.sms)) * 2 * c * sizeof(float));
    return gc_error(GC_OK, "");
} catch (...) {
    return internal_error();
}

int gc_b200_layer_norm_backward(const gc_tensor *dy, const gc_tensor *x, const gc_tensor *gamma,
                                const gc_tensor *stats, gc_tensor *dx, gc_tensor *dgamma, gc_tensor *dbeta,
                                void *workspace, uint64_t workspace_bytes, void *stream) try {
    Rows v[3];
    int st = check_rows({x, dy, dx}, v);
    if (st != GC_OK) return st;
    const int64_t c = x->dims[x->rank - 1];
    const gc_tensor *const params[] = {gamma, dgamma, dbeta};
    for (const gc_tensor *t : params)
        if ((st = check_param(t, x, {c})) != GC_OK) return st;
    if ((st = check_row_stats(stats, x, v[0].rows)) != GC_OK) return st;
    if (outputs_meet({range_of(v[2].t), range_of(dgamma), range_of(dbeta), {workspace, workspace_bytes}},
                     {range_of(v[0].t), range_of(v[1].t), range_of(gamma), range_of(stats)}))
        return gc_error(GC_INVALID, "outputs and workspace must not overlap inputs or one another");
    for (const gc_tensor *t : params)
        if ((st = check_dense(t, kDenseParams)) != GC_OK) return st;
    if ((st = check_dense(stats, "stats must be dense")) != GC_OK) return st;
    int dev = -1;
    if ((st = check_call({x, dy, dx, gamma, stats, dgamma, dbeta}, {}, x->device_index, stream, dev)) != GC_OK) return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const bool sums = dgamma != nullptr || dbeta != nullptr;
    cudaError_t e = cudaSuccess;
    if (v[0].t.empty) {  // sums over nothing
        for (const gc_tensor *t : {dgamma, dbeta})
            if (t != nullptr && e == cudaSuccess) e = cudaMemsetAsync(t->data, 0, range_of(t).bytes, s);
        return launched(e);
    }
    DeviceFacts facts;
    if ((st = device_facts(dev, facts)) != GC_OK) return st;
    const RowPlan plan = plan_backward(static_cast<int>(c), v);
    const long long grid = grad_blocks(plan, v[0].rows, facts.sms);
    if (sums) {
        const uint64_t need = up16(static_cast<uint64_t>(grid) * 2 * c * sizeof(float));
        if ((st = check_workspace(workspace, workspace_bytes, need)) != GC_OK) return st;
        if ((st = check_device_memory(workspace, x->device_index, dev)) != GC_OK) return st;
    }
    if (grid > INT32_MAX) return gc_error(GC_UNSUPPORTED, "more rows than a grid has blocks");
    LayerNormParams P{};
    P.x = v[0].t.data;
    P.x_ld = v[0].ld;
    P.dy = v[1].t.data;
    P.dy_ld = v[1].ld;
    P.y = v[2].t.data;
    P.y_ld = v[2].ld;
    P.rows = v[0].rows;
    P.c = static_cast<int>(c);
    P.vcols = P.c / plan.v;
    P.team = plan.team;
    set_param(gamma, P.gamma, P.gamma_type);
    P.aligned = aligned_params({gamma}, plan.v) ? 1 : 0;
    P.stats = static_cast<float2 *>(stats->data);
    P.part = sums ? static_cast<float *>(workspace) : nullptr;
    const void *fn = row_kernel(plan, true);
    if (plan.smem > 40 * 1024 && (st = opt_in_smem(dev, fn, dynamic_limit(facts))) != GC_OK) return st;
    void *args[] = {&P};
    e = launch_pdl(fn, dim3(static_cast<unsigned>(grid)), dim3(plan.threads), args, plan.smem, s);
    if (e == cudaSuccess && sums) {
        SumParams S{};
        S.part = P.part;
        S.rows = grid;
        S.cols = c;
        S.planes = 2;
        int i = 0;
        for (const gc_tensor *t : {dgamma, dbeta}) {
            S.out[i] = t != nullptr ? t->data : nullptr;
            S.type[i] = t != nullptr ? elem_type(t->dtype) : kElemF32;
            S.mul[i++] = 1;
        }
        e = launch_sum_rows(S, s);
    }
    return launched(e, PlanRecord::kSequence, plan.whole ? "layer_norm_long_backward" : plan.edges ? "layer_norm_edges_backward" : "layer_norm_backward", grid,
                    plan.threads, plan.vec ? 1 : 0, plan.team, plan.nv, 1, sums ? 2 : 1);
} catch (...) {
    return internal_error();
}

}  // extern "C"
