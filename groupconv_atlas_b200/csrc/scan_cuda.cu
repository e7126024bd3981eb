// gc_b200_selective_scan, its gradient and its form for one token: descriptor
// checks, plans and launches.  Nothing here allocates device memory,
// synchronizes or keeps anything of a call.
#include "groupconv.h"

#include <cuda_runtime.h>

#include <algorithm>

#include "host_util.h"
#include "kernel_scan.cuh"
#include "sequence_util.cuh"

namespace gcb {

__global__ void __launch_bounds__(kJoinThreads) scan_join_kernel(const __grid_constant__ ScanJoinParams Q) {
    griddep_wait();
    griddep_launch_dependents();
    const long long width = 2LL * Q.states, id = static_cast<long long>(blockIdx.x) * kJoinThreads + threadIdx.x;
    const long long row = id / width;
    if (row >= Q.rows) return;
    const int j = static_cast<int>(id - row * width), which = j / Q.states, s = j - which * Q.states;
    const long long group = row % Q.groups, token = row / Q.groups, t = token % Q.l, n = token / Q.l;
    const TokenView &out = which == 0 ? Q.db : Q.dc;
    if (out.p == nullptr) return;
    double all = 0.0;
    if (Q.lengths == nullptr || t < Q.lengths[n]) {
        const float *src = Q.part + id;
        const long long step = Q.rows * width;
        for (int k0 = 0; k0 < Q.tiles; k0 += kSumRun) {  // runs in 32 bits, joined in 64
            const int stop = min(Q.tiles, k0 + kSumRun);
            float v = 0.0f;
#pragma unroll 4
            for (int k = k0; k < stop; ++k) v += src[k * step];
            all += v;
        }
    }
    store_param(const_cast<void *>(out.p), Q.type, n * out.ldn + t * out.ldt + group * out.ldg + s, static_cast<float>(all));
}

}  // namespace gcb

namespace {

using namespace gcb;

constexpr int kMostStates = 64;

// A call's tensors: the descriptors with the same index as their views.
struct ScanCall {
    int64_t n = 0, l = 1, c = 0, groups = 0, states = 0;
    Strided x, dt, z, b, bc, y;  // bc: C
    Strided state;
};

int check_like(const gc_tensor *t, const gc_tensor *like, int dtype, std::initializer_list<int64_t> dims) {
    const int rank = static_cast<int>(dims.size());
    int64_t count = 0;
    const int st = check_fields(t, rank, rank, count);
    if (st != GC_OK) return st;
    int i = 0;
    for (const int64_t d : dims)
        if (t->dims[i++] != d) return gc_error(GC_INVALID, "tensor dimensions differ");
    if (t->dtype != dtype) return gc_error(GC_INVALID, "tensor dtypes differ");
    if (t->device_index != like->device_index) return gc_error(GC_INVALID, "tensor device indices differ");
    return GC_OK;
}
int check_tokens(const gc_tensor *t, const gc_tensor *like, const ScanCall &c, bool step) {
    return step ? check_like(t, like, like->dtype, {c.n, c.c}) : check_like(t, like, like->dtype, {c.n, c.l, c.c});
}
int check_pairs(const gc_tensor *t, const gc_tensor *like, const ScanCall &c, bool step) {
    return step ? check_like(t, like, like->dtype, {c.n, c.groups, c.states})
                : check_like(t, like, like->dtype, {c.n, c.l, c.groups, c.states});
}
int check_state(const gc_tensor *t, const gc_tensor *like, const ScanCall &c) {
    return check_like(t, like, GC_F32, {c.n, c.c, c.states});
}

// The inputs' descriptors: every GC_INVALID condition of theirs.
int check_scan(const gc_b200_scan_args *q, ScanCall &c, bool step) {
    if (q == nullptr) return gc_error(GC_INVALID, "null arguments");
    int64_t count = 0;
    int st = check_fields(q->x, step ? 2 : 3, step ? 2 : 3, count);
    if (st != GC_OK) return st;
    c.n = q->x->dims[0];
    c.l = step ? 1 : q->x->dims[1];
    c.c = q->x->dims[step ? 1 : 2];
    if (c.c < 1 || c.c > INT32_MAX / 128) return gc_error(GC_INVALID, "channel count out of range");
    if ((st = check_fields(q->b, step ? 3 : 4, step ? 3 : 4, count)) != GC_OK) return st;
    c.groups = q->b->dims[step ? 1 : 2];
    c.states = q->b->dims[step ? 2 : 3];
    if (c.states < 1) return gc_error(GC_INVALID, "a channel has no states");
    if (c.groups < 1 || c.c % c.groups != 0) return gc_error(GC_INVALID, "channels must be divisible by groups");
    if ((st = check_tokens(q->dt, q->x, c, step)) != GC_OK) return st;
    if (q->z != nullptr && (st = check_tokens(q->z, q->x, c, step)) != GC_OK) return st;
    for (const gc_tensor *t : {q->b, q->c})
        if ((st = check_pairs(t, q->x, c, step)) != GC_OK) return st;
    if (q->a == nullptr) return gc_error(GC_INVALID, "null tensor descriptor");
    if ((st = check_param(q->a, q->x, {c.c, c.states})) != GC_OK) return st;
    for (const gc_tensor *t : {q->d, q->dt_bias})
        if ((st = check_param(t, q->x, {c.c})) != GC_OK) return st;
    if (q->state != nullptr && (st = check_state(q->state, q->x, c)) != GC_OK) return st;
    if (reinterpret_cast<uintptr_t>(q->lengths) % 4 != 0) return gc_error(GC_INVALID, "lengths are not aligned");
    return GC_OK;
}
// Their layouts.
int view_scan(const gc_b200_scan_args *q, ScanCall &c) {
    int st = GC_OK;
    const std::pair<const gc_tensor *, Strided *> views[] = {{q->x, &c.x}, {q->dt, &c.dt}, {q->z, &c.z},
                                                            {q->b, &c.b}, {q->c, &c.bc}, {q->state, &c.state}};
    for (const auto &v : views)
        if (v.first != nullptr && (st = strided_of(v.first, *v.second)) != GC_OK) return st;
    if (c.states > kMostStates) return gc_error(GC_UNSUPPORTED, "more than 64 states");
    if (c.l > INT32_MAX / 2) return gc_error(GC_UNSUPPORTED, "more than 2^30 tokens");
    for (const gc_tensor *t : {q->a, q->d, q->dt_bias})
        if ((st = check_dense(t, "parameters must be dense")) != GC_OK) return st;
    return GC_OK;
}
Range lengths_range(const gc_b200_scan_args *q, const ScanCall &c) {
    return {q->lengths, q->lengths != nullptr ? 4ull * c.n : 0};
}

// ---- plans ------------------------------------------------------------------------------------
// Lanes of four states; a state count is rounded up to a power of two.
struct ScanPlan {
    int type = 0, sp = 16, lanes = 4, per_lane = 4;
    int tiles = 1, grad_tiles = 1, segs = 1;  // blocks that share a group's channels
    int runs = 1;                             // of the gradient's sums, in a segment
    long long seg_len = 0, blocks = 0;
    bool vec = false, bvec = false;
};
int padded_states(int64_t s) {
    int sp = 1;
    while (sp < s) sp *= 2;
    return sp == 2 ? 4 : sp;
}
// Segments: as many as give each multiprocessor 16 blocks (24 in the gradient,
// whose own kernel has half as many), of at least 32 tokens.  Eight blocks fit at once at
// 16 states in 16 bits, so that 16 are two rounds there; FP32 has room for seven, 64 states
// for six, up to four states for four or five, and rounding up gives N4 L2048 C2048 2.16
// rounds.  N1 L8192 C2048 bf16 takes 8 % longer with ten blocks (1.3 rounds) and 5 % with 20
// (2.6), N5 L777 C330 FP32 20 % with 64 tokens.
ScanPlan plan_scan(const ScanCall &c, int sms, bool backward) {
    ScanPlan p;
    p.type = c.x.type;
    p.sp = padded_states(c.states);
    p.per_lane = std::min(p.sp, kScanStates);
    p.lanes = p.sp / p.per_lane;
    const int64_t cpg = c.c / c.groups;
    p.tiles = static_cast<int>(ceil_div(cpg, 2 * kScanThreads / p.lanes));
    p.grad_tiles = static_cast<int>(ceil_div(cpg, 2 * grad_threads(p.sp) / p.lanes));
    const long long blocks = std::max(1LL, static_cast<long long>(c.n) * c.groups * p.tiles);
    const long long wanted = std::min(ceil_div((backward ? 24LL : 16LL) * sms, blocks), static_cast<long long>(c.l / 32));
    p.seg_len = std::max(1LL, gcb::round_up(ceil_div(c.l, std::max(1LL, wanted)), 16));
    p.segs = static_cast<int>(std::max(1LL, ceil_div(c.l, p.seg_len)));
    p.runs = static_cast<int>(ceil_div(p.seg_len, kScanChunk * kScanRun));
    p.blocks = blocks * p.segs;
    return p;
}
bool fours(std::initializer_list<const Strided *> views, const ScanCall &c) {
    if (c.c / c.groups % 4 != 0) return false;
    for (const Strided *v : views)
        if (v->data != nullptr && !v->empty && !group_aligned(*v, 4)) return false;
    return true;
}

struct ScanSpace {  // parts of a workspace, in this order
    uint64_t carry = 0, sums = 0, bc = 0, a = 0, d = 0;
    uint64_t total() const { return carry + sums + bc + a + d; }
};
ScanSpace space_of(const ScanCall &c, const ScanPlan &p, bool backward) {
    ScanSpace s;
    const uint64_t rows = static_cast<uint64_t>(c.n) * p.segs;
    if (p.segs > 1) {
        s.carry = up16(rows * c.c * c.states * sizeof(float));
        s.sums = up16(rows * c.c * sizeof(float));
    }
    if (backward) {
        s.bc = up16(static_cast<uint64_t>(p.grad_tiles) * c.n * c.l * c.groups * 2 * c.states * sizeof(float));
        s.a = up16(rows * p.runs * c.c * c.states * sizeof(float));
        s.d = up16(rows * p.runs * 2 * c.c * sizeof(float));
    }
    return s;
}
uint64_t kept_bytes_of(const ScanCall &c) {
    return static_cast<uint64_t>(c.n) * ceil_div(c.l, kScanChunk) * c.c * c.states * sizeof(float);
}

TokenView tokens_of(const Strided &v, bool step) {
    return {v.empty ? nullptr : v.data, v.s[0], step ? 0 : v.s[1], 0};
}
TokenView pairs_of(const Strided &v, bool step) {
    return {v.empty ? nullptr : v.data, v.s[0], step ? 0 : v.s[1], v.s[step ? 1 : 2]};
}

void fill(ScanParams &P, const gc_b200_scan_args *q, const ScanCall &c, const ScanPlan &plan, bool step) {
    P.x = tokens_of(c.x, step);
    P.dt = tokens_of(c.dt, step);
    if (q->z != nullptr) P.z = tokens_of(c.z, step);
    P.b = pairs_of(c.b, step);
    P.c = pairs_of(c.bc, step);
    P.a = q->a->data;
    P.a_type = elem_type(q->a->dtype);
    P.d = q->d != nullptr ? q->d->data : nullptr;
    P.d_type = q->d != nullptr ? elem_type(q->d->dtype) : kElemF32;
    P.bias = q->dt_bias != nullptr ? q->dt_bias->data : nullptr;
    P.bias_type = q->dt_bias != nullptr ? elem_type(q->dt_bias->dtype) : kElemF32;
    P.state = q->state != nullptr && !c.state.empty ? reinterpret_cast<const float *>(c.state.data) : nullptr;
    P.s_ldn = c.state.s[0];
    P.s_ldc = c.state.s[1];
    P.lengths = q->lengths;
    P.n = c.n;
    P.l = c.l;
    P.channels = static_cast<int>(c.c);
    P.states = static_cast<int>(c.states);
    P.groups = static_cast<int>(c.groups);
    P.cpg = static_cast<int>(c.c / c.groups);
    P.vec = plan.vec ? 1 : 0;
    P.bvec = plan.bvec ? 1 : 0;
    P.softplus = q->softplus != 0;
    P.tiles = plan.tiles;
    P.seg_len = plan.seg_len;
    P.segs = plan.segs;
    P.runs = plan.runs;
}
void set_state_out(ScanParams &P, const Strided &v) {
    if (v.data == nullptr || v.empty) return;
    P.state_out = reinterpret_cast<float *>(v.data);
    P.so_ldn = v.s[0];
    P.so_ldc = v.s[1];
}

// ---- launches -----------------------------------------------------------------------------------
ScanLaunch launch_of(ScanKernel k, int type, int sp) {
    return type == kElemF16    ? scan_launch<__half>(k, sp)
           : type == kElemBF16 ? scan_launch<__nv_bfloat16>(k, sp)
                               : scan_launch<float>(k, sp);
}
int launch(ScanKernel k, const ScanPlan &p, ScanParams &P, int dev, const DeviceFacts &facts, cudaStream_t s, cudaError_t &e) {
    const ScanLaunch l = launch_of(k, p.type, p.sp);
    if (l.smem > 48 * 1024) {
        const int st = opt_in_smem(dev, l.fn, facts.smem_optin);
        if (st != GC_OK) return st;
    }
    P.tiles = k == kGrad ? p.grad_tiles : p.tiles;
    const long long blocks = P.n * P.groups * P.tiles * P.segs;
    if (blocks > INT32_MAX) return gc_error(GC_UNSUPPORTED, "more work than a grid has blocks");
    void *args[] = {&P};
    e = launch_pdl(l.fn, dim3(static_cast<unsigned>(blocks)), dim3(l.threads), args, l.smem, s);
    return GC_OK;
}

int current_facts(DeviceFacts &facts) {
    int dev = -1;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return gc_error(GC_DEVICE_ERROR, cudaGetErrorString(e));
    return device_facts(dev, facts);
}
int too_many_blocks() { return gc_error(GC_UNSUPPORTED, "more work than a grid has blocks"); }

}  // namespace

extern "C" {

int gc_b200_selective_scan_sizes(const gc_b200_scan_args *q, uint64_t *workspace, uint64_t *kept,
                                 uint64_t *backward_workspace) try {
    for (const uint64_t *p : {workspace, kept, backward_workspace})
        if (p == nullptr) return gc_error(GC_INVALID, "null size pointer");
    ScanCall c;
    int st = check_scan(q, c, false);
    if (st != GC_OK || (st = view_scan(q, c)) != GC_OK) return st;
    *workspace = *kept = *backward_workspace = 0;
    if (c.n == 0) return gc_error(GC_OK, "");
    DeviceFacts facts;
    if ((st = current_facts(facts)) != GC_OK) return st;
    *workspace = space_of(c, plan_scan(c, facts.sms, false), false).total();
    *kept = kept_bytes_of(c);
    *backward_workspace = space_of(c, plan_scan(c, facts.sms, true), true).total();
    return gc_error(GC_OK, "");
} catch (...) {
    return internal_error();
}

int gc_b200_selective_scan(const gc_b200_scan_args *q, gc_tensor *y, gc_tensor *state_out, void *kept,
                           uint64_t kept_bytes, void *workspace, uint64_t workspace_bytes, void *stream) try {
    ScanCall c;
    int st = check_scan(q, c, false);
    if (st != GC_OK) return st;
    if ((st = check_tokens(y, q->x, c, false)) != GC_OK) return st;
    if (state_out != nullptr && (st = check_state(state_out, q->x, c)) != GC_OK) return st;
    Strided out;
    if ((st = view_scan(q, c)) != GC_OK || (st = strided_of(y, c.y)) != GC_OK) return st;
    if (state_out != nullptr && (st = strided_of(state_out, out)) != GC_OK) return st;
    if (outputs_meet({range_of(c.y), range_of(out), {kept, kept_bytes}, {workspace, workspace_bytes}},
                     {range_of(c.x), range_of(c.dt), range_of(c.z), range_of(c.b), range_of(c.bc), range_of(q->a),
                      range_of(q->d), range_of(q->dt_bias), range_of(c.state), lengths_range(q, c)}))
        return gc_error(GC_INVALID, "outputs and workspaces must not overlap inputs or one another");
    if (c.n == 0) return gc_error(GC_OK, "");
    int dev = -1;
    if ((st = check_call({q->x, q->dt, q->z, q->a, q->b, q->c, q->d, q->dt_bias, q->state, y, state_out}, {q->lengths},
                         q->x->device_index, stream, dev)) != GC_OK)
        return st;
    if (c.l == 0 && state_out == nullptr) return gc_error(GC_OK, "");
    DeviceFacts facts;
    if ((st = device_facts(dev, facts)) != GC_OK) return st;
    ScanPlan plan = plan_scan(c, facts.sms, false);
    const ScanSpace space = space_of(c, plan, false);
    if ((st = check_workspace(workspace, workspace_bytes, space.total())) != GC_OK) return st;
    if (space.total() != 0 && (st = check_device_memory(workspace, q->x->device_index, dev)) != GC_OK) return st;
    if (kept != nullptr && kept_bytes_of(c) != 0) {
        if ((st = check_workspace(kept, kept_bytes, kept_bytes_of(c))) != GC_OK) return st;
        if ((st = check_device_memory(kept, q->x->device_index, dev)) != GC_OK) return st;
    }
    plan.vec = fours({&c.x, &c.dt, &c.z, &c.y}, c);
    plan.bvec = group_aligned(c.b, 4) && group_aligned(c.bc, 4);
    ScanParams P{};
    fill(P, q, c, plan, false);
    P.y = tokens_of(c.y, false);
    set_state_out(P, out);
    P.carry = static_cast<float *>(workspace);
    P.sums = reinterpret_cast<float *>(static_cast<char *>(workspace) + space.carry);
    P.kept = static_cast<float *>(kept);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (plan.segs > 1 && (st = launch(kCarry, plan, P, dev, facts, s, e)) != GC_OK) return st;
    if (e == cudaSuccess && (st = launch(kMain, plan, P, dev, facts, s, e)) != GC_OK) return st;
    return launched(e, PlanRecord::kSequence, "selective_scan", plan.blocks, kScanThreads, plan.vec ? 1 : 0, plan.lanes,
                    plan.per_lane, plan.segs, plan.segs > 1 ? 2 : 1);
} catch (...) {
    return internal_error();
}

int gc_b200_selective_scan_backward(const gc_b200_scan_args *q, const gc_tensor *dy, const gc_tensor *dstate_out,
                                    const void *kept, uint64_t kept_bytes, const gc_b200_scan_grads *g, void *workspace,
                                    uint64_t workspace_bytes, void *stream) try {
    ScanCall c;
    int st = check_scan(q, c, false);
    if (st != GC_OK) return st;
    if (g == nullptr) return gc_error(GC_INVALID, "null arguments");
    Strided dyv, dx, ddt, dz, db, dc, dlast, dfirst;
    if ((st = check_tokens(dy, q->x, c, false)) != GC_OK) return st;
    if ((st = check_tokens(g->x, q->x, c, false)) != GC_OK || (st = check_tokens(g->dt, q->x, c, false)) != GC_OK) return st;
    if ((g->z != nullptr) != (q->z != nullptr)) return gc_error(GC_INVALID, "the gate and its gradient come together");
    if (g->z != nullptr && (st = check_tokens(g->z, q->x, c, false)) != GC_OK) return st;
    for (const gc_tensor *t : {g->b, g->c})
        if (t != nullptr && (st = check_pairs(t, q->x, c, false)) != GC_OK) return st;
    if ((st = check_param(g->a, q->x, {c.c, c.states})) != GC_OK) return st;
    for (const gc_tensor *t : {g->d, g->dt_bias})
        if ((st = check_param(t, q->x, {c.c})) != GC_OK) return st;
    for (const gc_tensor *t : {dstate_out, static_cast<const gc_tensor *>(g->state)})
        if (t != nullptr && (st = check_state(t, q->x, c)) != GC_OK) return st;
    if ((st = view_scan(q, c)) != GC_OK) return st;
    const std::pair<const gc_tensor *, Strided *> views[] = {{dy, &dyv}, {g->x, &dx}, {g->dt, &ddt}, {g->z, &dz}, {g->b, &db},
                                                            {g->c, &dc}, {dstate_out, &dlast}, {g->state, &dfirst}};
    for (const auto &v : views)
        if (v.first != nullptr && (st = strided_of(v.first, *v.second)) != GC_OK) return st;
    for (const gc_tensor *t : {g->a, g->d, g->dt_bias})
        if ((st = check_dense(t, "parameters must be dense")) != GC_OK) return st;
    if (outputs_meet({range_of(dx), range_of(ddt), range_of(dz), range_of(db), range_of(dc), range_of(g->a), range_of(g->d),
                      range_of(g->dt_bias), range_of(dfirst), {workspace, workspace_bytes}},
                     {range_of(c.x), range_of(c.dt), range_of(c.z), range_of(c.b), range_of(c.bc), range_of(q->a),
                      range_of(q->d), range_of(q->dt_bias), range_of(c.state), range_of(dyv), range_of(dlast),
                      {kept, kept_bytes}, lengths_range(q, c)}))
        return gc_error(GC_INVALID, "outputs and workspace must not overlap inputs or one another");
    int dev = -1;
    if ((st = check_call({q->x, q->dt, q->z, q->a, q->b, q->c, q->d, q->dt_bias, q->state, dy, dstate_out, g->x, g->dt, g->a,
                          g->b, g->c, g->d, g->z, g->dt_bias, g->state},
                         {q->lengths}, q->x->device_index, stream, dev)) != GC_OK)
        return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (c.n == 0 || c.l == 0) {  // sums over nothing; the state's gradient passes through
        for (const gc_tensor *t : {g->a, g->d, g->dt_bias})
            if (t != nullptr && e == cudaSuccess) e = cudaMemsetAsync(t->data, 0, range_of(t).bytes, s);
        if (c.n == 0 || g->state == nullptr || e != cudaSuccess) return launched(e);
    }
    DeviceFacts facts;
    if ((st = device_facts(dev, facts)) != GC_OK) return st;
    ScanPlan plan = plan_scan(c, facts.sms, true);
    const ScanSpace space = space_of(c, plan, true);
    if ((st = check_workspace(workspace, workspace_bytes, space.total())) != GC_OK) return st;
    if ((st = check_device_memory(workspace, q->x->device_index, dev)) != GC_OK) return st;
    if ((st = check_workspace(kept, kept_bytes, kept_bytes_of(c))) != GC_OK) return st;
    if (kept_bytes_of(c) != 0 && (st = check_device_memory(kept, q->x->device_index, dev)) != GC_OK) return st;
    plan.vec = fours({&c.x, &c.dt, &c.z, &dyv, &dx, &ddt, &dz}, c);
    plan.bvec = group_aligned(c.b, 4) && group_aligned(c.bc, 4);
    ScanParams P{};
    fill(P, q, c, plan, false);
    P.dy = tokens_of(dyv, false);
    P.dx = tokens_of(dx, false);
    P.ddt = tokens_of(ddt, false);
    if (g->z != nullptr) P.dz = tokens_of(dz, false);
    if (dstate_out != nullptr && !dlast.empty) {
        P.dlast = reinterpret_cast<const float *>(dlast.data);
        P.dl_ldn = dlast.s[0];
        P.dl_ldc = dlast.s[1];
    }
    set_state_out(P, dfirst);
    P.kept = const_cast<float *>(static_cast<const float *>(kept));
    char *w = static_cast<char *>(workspace);
    P.carry = reinterpret_cast<float *>(w);
    P.sums = reinterpret_cast<float *>(w + space.carry);
    P.part_bc = reinterpret_cast<float *>(w + space.carry + space.sums);
    const bool sums_d = g->d != nullptr || g->dt_bias != nullptr;
    if (g->a != nullptr) P.part_a = reinterpret_cast<float *>(w + space.carry + space.sums + space.bc);
    if (sums_d) P.part_d = reinterpret_cast<float *>(w + space.carry + space.sums + space.bc + space.a);
    int launches = 1;
    if (plan.segs > 1) {
        if ((st = launch(kCarryBack, plan, P, dev, facts, s, e)) != GC_OK) return st;
        ++launches;
    }
    if (e == cudaSuccess && (st = launch(kGrad, plan, P, dev, facts, s, e)) != GC_OK) return st;
    if (e == cudaSuccess && c.l > 0 && (g->b != nullptr || g->c != nullptr)) {
        ScanJoinParams J{};
        J.part = P.part_bc;
        J.rows = c.n * c.l * c.groups;
        J.l = c.l;
        J.tiles = plan.grad_tiles;
        J.states = P.states;
        J.groups = P.groups;
        J.type = c.x.type;
        if (g->b != nullptr) J.db = pairs_of(db, false);
        if (g->c != nullptr) J.dc = pairs_of(dc, false);
        J.lengths = q->lengths;
        const wide blocks = (static_cast<wide>(J.rows) * 2 * J.states + kJoinThreads - 1) / kJoinThreads;
        if (blocks > INT32_MAX) return too_many_blocks();
        void *args[] = {&J};
        e = launch_pdl(reinterpret_cast<const void *>(&scan_join_kernel), dim3(static_cast<unsigned>(blocks)), dim3(kJoinThreads),
                       args, 0, s);
        ++launches;
    }
    for (int which = 0; which < 2 && e == cudaSuccess && c.l > 0; ++which) {
        if (which == 0 ? g->a == nullptr : !sums_d) continue;
        SumParams S{};
        S.part = which == 0 ? P.part_a : P.part_d;
        S.rows = c.n * plan.segs * plan.runs;
        S.cols = which == 0 ? c.c * c.states : c.c;
        S.planes = which == 0 ? 1 : 2;
        int i = 0;
        for (const gc_tensor *t : {which == 0 ? g->a : g->d, g->dt_bias}) {
            S.out[i] = t != nullptr ? t->data : nullptr;
            S.type[i] = t != nullptr ? elem_type(t->dtype) : kElemF32;
            S.mul[i++] = 1;
        }
        e = launch_sum_rows(S, s);
        ++launches;
    }
    return launched(e, PlanRecord::kSequence, "selective_scan_backward", plan.blocks, kScanThreads, plan.vec ? 1 : 0,
                    plan.lanes, plan.per_lane, plan.segs, launches);
} catch (...) {
    return internal_error();
}

int gc_b200_selective_scan_step(const gc_b200_scan_args *q, gc_tensor *y, gc_tensor *state_out, void *stream) try {
    ScanCall c;
    int st = check_scan(q, c, true);
    if (st != GC_OK) return st;
    if (q->lengths != nullptr) return gc_error(GC_INVALID, "a step has no lengths");
    if (q->state == nullptr || state_out == nullptr) return gc_error(GC_INVALID, "null tensor descriptor");
    if ((st = check_tokens(y, q->x, c, true)) != GC_OK || (st = check_state(state_out, q->x, c)) != GC_OK) return st;
    Strided out;
    if ((st = view_scan(q, c)) != GC_OK || (st = strided_of(y, c.y)) != GC_OK || (st = strided_of(state_out, out)) != GC_OK)
        return st;
    bool same = c.state.data == out.data;
    for (int i = 0; i < 3; ++i) same = same && c.state.s[i] == out.s[i];
    if (outputs_meet({range_of(c.y), range_of(out)},
                     {range_of(c.x), range_of(c.dt), range_of(c.z), range_of(c.b), range_of(c.bc), range_of(q->a),
                      range_of(q->d), range_of(q->dt_bias), same ? Range{nullptr, 0} : range_of(c.state)}))
        return gc_error(GC_INVALID, "outputs must not overlap inputs or one another (the new state may be the old one)");
    if (c.n == 0) return gc_error(GC_OK, "");
    int dev = -1;
    if ((st = check_call({q->x, q->dt, q->z, q->a, q->b, q->c, q->d, q->dt_bias, q->state, y, state_out}, {},
                         q->x->device_index, stream, dev)) != GC_OK)
        return st;
    DeviceFacts facts;
    if ((st = device_facts(dev, facts)) != GC_OK) return st;
    ScanPlan plan = plan_scan(c, facts.sms, false);
    plan.segs = 1;
    ScanParams P{};
    fill(P, q, c, plan, true);
    P.y = tokens_of(c.y, true);
    set_state_out(P, out);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    const int channels = 2 * kScanThreads / plan.lanes;  // of a block
    bool whole = plan.sp >= 4 && c.states == plan.sp && P.cpg % channels == 0 && c.n <= 65535 && q->z != nullptr &&
                 fours({&c.x, &c.dt, &c.z, &c.y}, c) && group_aligned(c.b, 4) && group_aligned(c.bc, 4);
    for (const gc_tensor *t : {q->a, q->d, q->dt_bias}) whole = whole && t != nullptr && t->dtype == GC_F32 && aligned16(t->data);
    for (const Strided *v : {static_cast<const Strided *>(&c.state), static_cast<const Strided *>(&out)})
        whole = whole && group_aligned(*v, 4) && v->s[1] == c.states;
    if (whole) {
        const ScanLaunch l = launch_of(kStepWhole, plan.type, plan.sp);
        void *args[] = {&P};
        e = launch_pdl(l.fn, dim3(static_cast<unsigned>(P.groups * P.tiles), static_cast<unsigned>(c.n)), dim3(l.threads), args, 0, s);
    } else if ((st = launch(kStep, plan, P, dev, facts, s, e)) != GC_OK) {
        return st;
    }
    return launched(e, PlanRecord::kSequence, "selective_scan_step", P.n * P.groups * P.tiles, kScanThreads, whole ? 1 : 0,
                    plan.lanes, plan.per_lane, 1, 1);
} catch (...) {
    return internal_error();
}

}  // extern "C"
