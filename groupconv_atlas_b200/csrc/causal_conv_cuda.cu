// gc_b200_causal_conv, its gradient and its form for one token: descriptor
// checks, plans and launches.  Nothing here allocates device memory,
// synchronizes or keeps anything of a call.
#include "groupconv.h"

#include <cuda_runtime.h>

#include <algorithm>

#include "host_util.h"
#include "kernel_causal_conv.cuh"
#include "sequence_util.cuh"

namespace {

using namespace gcb;

constexpr int kMostTaps = 8;

// Tensors of the data's type and device; dims of -1 are any.
int check_data_tensor(const gc_tensor *t, const gc_tensor *like, std::initializer_list<int64_t> dims) {
    const int rank = static_cast<int>(dims.size());
    int64_t count = 0;
    const int st = check_fields(t, rank, rank, count);
    if (st != GC_OK) return st;
    int i = 0;
    for (const int64_t d : dims)
        if (t->dims[i++] != d) return gc_error(GC_INVALID, "tensor dimensions differ");
    if (t->dtype != like->dtype) return gc_error(GC_INVALID, "tensor dtypes differ");
    if (t->device_index != like->device_index) return gc_error(GC_INVALID, "tensor device indices differ");
    return GC_OK;
}

struct ConvCall {
    Strided x, y, dy, state, state_out, dstate;
    int64_t n = 0, l = 1, c = 0, taps = 0;
};

bool known_activation(int a) {
    return a == GC_B200_ACT_NONE || a == GC_B200_ACT_RELU || a == GC_B200_ACT_RELU6 || a == GC_B200_ACT_SILU;
}

// x, weight and what has their dimensions.  step: x is (N, C).
int check_conv(const gc_tensor *x, const gc_tensor *weight, const gc_tensor *bias, ConvCall &call, bool step) {
    int64_t count = 0;
    int st = check_fields(x, step ? 2 : 3, step ? 2 : 3, count);
    if (st != GC_OK) return st;
    call.n = x->dims[0];
    call.l = step ? 1 : x->dims[1];
    call.c = x->dims[step ? 1 : 2];
    if (call.c < 1 || call.c > INT32_MAX / 16) return gc_error(GC_INVALID, "channel count out of range");
    if ((st = check_fields(weight, 2, 2, count)) != GC_OK) return st;
    call.taps = weight->dims[1];
    if (call.taps < 1) return gc_error(GC_INVALID, "the filter has no taps");
    if ((st = check_param(weight, x, {call.c, call.taps})) != GC_OK) return st;
    return check_param(bias, x, {call.c});
}
int check_layouts(const gc_tensor *weight, const gc_tensor *bias, int act, const ConvCall &call) {
    if (call.taps > kMostTaps) return gc_error(GC_UNSUPPORTED, "more than eight taps");
    if (!known_activation(act)) return gc_error(GC_UNSUPPORTED, "unknown activation");
    for (const gc_tensor *t : {weight, bias}) {
        const int st = check_dense(t, "parameters must be dense");
        if (st != GC_OK) return st;
    }
    return GC_OK;
}

bool empty_view(const Strided &v) { return v.data == nullptr || v.empty; }

// Whether the data can be taken so many elements at a time.
bool groups_of(std::initializer_list<const Strided *> views, int e) {
    for (const Strided *v : views)
        if (!empty_view(*v) && !group_aligned(*v, e)) return false;
    return true;
}
bool groups_of_four(std::initializer_list<const Strided *> views) { return groups_of(views, 4); }

void fill(ConvSeqParams &P, const ConvCall &call, const gc_tensor *weight, const gc_tensor *bias, int act,
          const int32_t *lengths, bool step) {
    P.n = call.n;
    P.l = call.l;
    P.c = static_cast<int>(call.c);
    P.taps = static_cast<int>(call.taps);
    P.w = weight->data;
    P.w_type = elem_type(weight->dtype);
    P.w_four = P.taps == 4 && aligned16(weight->data) ? 1 : 0;
    P.bias = bias != nullptr ? bias->data : nullptr;
    P.bias_type = bias != nullptr ? elem_type(bias->dtype) : kElemF32;
    P.act = act;
    P.lengths = lengths;
    P.x = call.x.data;
    P.x_ldn = call.x.s[0];
    P.x_ldt = step ? 0 : call.x.s[1];
    P.y = call.y.data;
    P.y_ldn = call.y.s[0];
    P.y_ldt = step ? 0 : call.y.s[1];
    P.dy = call.dy.data;
    P.dy_ldn = call.dy.s[0];
    P.dy_ldt = call.dy.s[1];
    if (!empty_view(call.state)) P.state = call.state.data;
    P.s_ldn = call.state.s[0];
    P.s_ldt = call.state.s[1];
    if (!empty_view(call.state_out)) P.state_out = call.state_out.data;
    P.so_ldn = call.state_out.s[0];
    P.so_ldt = call.state_out.s[1];
    if (!empty_view(call.dstate)) P.dstate = call.dstate.data;
    P.ds_ldn = call.dstate.s[0];
    P.ds_ldt = call.dstate.s[1];
}

enum ConvKernel { kForward, kBackward, kStep };
template <class T, int V, int KT, bool FULL, int ACT>
const void *conv_instance(ConvKernel k) {
    return k == kForward    ? reinterpret_cast<const void *>(&causal_conv_kernel<T, V, KT, FULL, ACT>)
           : k == kBackward ? reinterpret_cast<const void *>(&causal_conv_grad_kernel<T, V, KT, FULL, ACT>)
                            : reinterpret_cast<const void *>(&causal_conv_step_kernel<T, V, KT, FULL, ACT>);
}
template <class T, int V>
const void *conv_typed(ConvKernel k, int taps, int act) {
    if (taps > 4) return conv_instance<T, V, 8, false, -1>(k);
    if (taps < 4) return conv_instance<T, V, 4, false, -1>(k);
    if (act == GC_B200_ACT_SILU) return conv_instance<T, V, 4, true, kActSilu>(k);
    if (act == GC_B200_ACT_NONE) return conv_instance<T, V, 4, true, kActNone>(k);
    return conv_instance<T, V, 4, true, -1>(k);
}
template <class T>
const void *conv_eight(int act) {
    if (act == GC_B200_ACT_SILU) return reinterpret_cast<const void *>(&causal_conv_kernel<T, 8, 4, true, kActSilu>);
    if (act == GC_B200_ACT_NONE) return reinterpret_cast<const void *>(&causal_conv_kernel<T, 8, 4, true, kActNone>);
    return reinterpret_cast<const void *>(&causal_conv_kernel<T, 8, 4, true, -1>);
}
const void *conv_kernel(ConvKernel k, int type, bool vec, int taps, int act) {
    if (type == kElemF16) return vec ? conv_typed<__half, 4>(k, taps, act) : conv_typed<__half, 1>(k, taps, act);
    if (type == kElemBF16)
        return vec ? conv_typed<__nv_bfloat16, 4>(k, taps, act) : conv_typed<__nv_bfloat16, 1>(k, taps, act);
    return vec ? conv_typed<float, 4>(k, taps, act) : conv_typed<float, 1>(k, taps, act);
}

// Dynamic shared memory of a kernel's ring; the gradient's sums take its place.
size_t ring_bytes(int type, size_t v, int taps) {
    const size_t ring = kConvRing * kConvThreads * v * elem_size(type);
    return std::max(ring, (taps + 1) * v * kConvThreads * sizeof(float));
}
int opt_in_ring(int dev, const void *fn, size_t bytes, const DeviceFacts &facts) {
    return bytes > 40 * 1024 ? opt_in_smem(dev, fn, facts.smem_optin - 8192) : GC_OK;
}

// Tokens of a thread: 16 to 64, backwards 128, as many as leave so many threads; v:
// channels of a thread, four also where the forward kernel takes eight, which then has half
// of the threads.  Each thread loads its weights and the window in front of its stretch:
// shorter stretches were no faster (N8 L2048 C2048 bf16: forward the same at 32 and at 64,
// gradient 5 % more at 32).
int stretch_of(const ConvCall &call, int v, int sms, bool backward) {
    const long long threads = call.n * ceil_div(call.c, v), wanted = (backward ? 384LL : 768LL) * sms;
    long long stretch = backward ? 128 : 64;
    while (stretch > 16 && threads * ceil_div(call.l, stretch) < wanted) stretch /= 2;
    return static_cast<int>(stretch);
}

// The gradient's blocks: tiles of up to 32 vector columns, and for each as many
// blocks as fill the GPU, or as leave each worker 64 stretches, whose sums it adds up
// one after the other.
struct GradPlan {
    bool vec = false;
    int cols = 1, workers = 1, stretch = 8;
    long long tiles = 1, blocks_y = 1, segs = 1;
};
GradPlan plan_grad(const ConvCall &call, bool vec, int sms) {
    GradPlan p;
    p.vec = vec;
    const long long vcols = ceil_div(call.c, vec ? 4 : 1);
    p.tiles = ceil_div(vcols, 32);
    p.cols = static_cast<int>(ceil_div(vcols, p.tiles));
    p.workers = kConvThreads / p.cols;
    p.stretch = stretch_of(call, vec ? 4 : 1, sms, true);
    p.segs = ceil_div(call.l, p.stretch);
    const long long items = call.n * p.segs;
    p.blocks_y = std::max({1LL, std::min(ceil_div(items, p.workers), ceil_div(4LL * sms, p.tiles)),
                           ceil_div(items, static_cast<long long>(kSumRun) * p.workers)});
    return p;
}

int check_lengths(const int32_t *lengths) {
    return reinterpret_cast<uintptr_t>(lengths) % 4 == 0 ? GC_OK : gc_error(GC_INVALID, "lengths are not aligned");
}
Range range_of_lengths(const int32_t *lengths, int64_t n) { return {lengths, lengths != nullptr ? 4ull * n : 0}; }

int current_facts(DeviceFacts &facts) {
    int dev = -1;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return gc_error(GC_DEVICE_ERROR, cudaGetErrorString(e));
    return device_facts(dev, facts);
}

int check_states(std::initializer_list<std::pair<const gc_tensor *, Strided *>> states, const gc_tensor *x, const ConvCall &call) {
    for (const auto &s : states)
        if (s.first != nullptr) {
            const int st = check_data_tensor(s.first, x, {call.n, call.taps - 1, call.c});
            if (st != GC_OK) return st;
        }
    return GC_OK;
}
int view_states(std::initializer_list<std::pair<const gc_tensor *, Strided *>> states) {
    for (const auto &s : states)
        if (s.first != nullptr) {
            const int st = strided_of(s.first, *s.second);
            if (st != GC_OK) return st;
        }
    return GC_OK;
}

int check_grad_data(const gc_tensor *dy, const gc_tensor *x, const gc_tensor *weight, const gc_tensor *dx, ConvCall &call) {
    int st = check_conv(x, weight, nullptr, call, false);
    if (st != GC_OK) return st;
    for (const gc_tensor *t : {dy, dx})
        if ((st = check_data_tensor(t, x, {call.n, call.l, call.c})) != GC_OK) return st;
    if ((st = strided_of(x, call.x)) != GC_OK || (st = strided_of(dy, call.dy)) != GC_OK) return st;
    return strided_of(dx, call.y);
}
uint64_t grad_space(const GradPlan &p, const ConvCall &call) {
    return up16(static_cast<uint64_t>(p.blocks_y) * (call.taps + 1) * call.c * sizeof(float));
}

}  // namespace

extern "C" {

int gc_b200_causal_conv(const gc_tensor *x, const gc_tensor *weight, const gc_tensor *bias, const gc_tensor *state,
                        const int32_t *lengths, gc_tensor *y, gc_tensor *state_out, int activation, void *stream) try {
    ConvCall call;
    int st = check_conv(x, weight, bias, call, false);
    if (st != GC_OK) return st;
    if ((st = check_data_tensor(y, x, {call.n, call.l, call.c})) != GC_OK) return st;
    if ((st = check_states({{state, &call.state}, {state_out, &call.state_out}}, x, call)) != GC_OK) return st;
    if ((st = check_lengths(lengths)) != GC_OK) return st;
    if ((st = strided_of(x, call.x)) != GC_OK || (st = strided_of(y, call.y)) != GC_OK) return st;
    if ((st = view_states({{state, &call.state}, {state_out, &call.state_out}})) != GC_OK) return st;
    if (outputs_meet({range_of(call.y), range_of(call.state_out)},
                     {range_of(call.x), range_of(weight), range_of(bias), range_of(call.state), range_of_lengths(lengths, call.n)}))
        return gc_error(GC_INVALID, "outputs must not overlap inputs or one another");
    if ((st = check_layouts(weight, bias, activation, call)) != GC_OK) return st;
    if (call.n == 0) return gc_error(GC_OK, "");
    int dev = -1;
    if ((st = check_call({x, weight, bias, state, y, state_out}, {lengths}, x->device_index, stream, dev)) != GC_OK) return st;
    if (call.l == 0 && state_out == nullptr) return gc_error(GC_OK, "");
    DeviceFacts facts;
    if ((st = device_facts(dev, facts)) != GC_OK) return st;
    const bool vec = groups_of_four({&call.x, &call.y, &call.state, &call.state_out});
    ConvSeqParams P{};
    fill(P, call, weight, bias, activation, lengths, false);
    // Eight channels of 16 bits a thread where they lie on 16 bytes: 29 us against 36
    // with four at N8 L2048 C2048 (the gradient has no registers for eight).
    const bool eight = vec && call.x.type != kElemF32 && P.taps == 4 && groups_of({&call.x, &call.y, &call.state, &call.state_out}, 8);
    const int v = eight ? 8 : vec ? 4 : 1;
    P.vcols = P.c / v;
    P.stretch = stretch_of(call, vec ? 4 : 1, facts.sms, false);
    P.segs = std::max(1LL, ceil_div(call.l, P.stretch));
    const wide blocks = (static_cast<wide>(call.n) * P.segs * P.vcols + kConvThreads - 1) / kConvThreads;
    if (blocks > INT32_MAX) return gc_error(GC_UNSUPPORTED, "more work than a grid has blocks");
    P.small = blocks * kConvThreads <= UINT32_MAX ? 1 : 0;
    void *args[] = {&P};
    const void *fn = !eight                    ? conv_kernel(kForward, call.x.type, vec, P.taps, activation)
                     : call.x.type == kElemF16 ? conv_eight<__half>(activation)
                                               : conv_eight<__nv_bfloat16>(activation);
    const size_t smem = ring_bytes(call.x.type, v, 0);
    if ((st = opt_in_ring(dev, fn, smem, facts)) != GC_OK) return st;
    const cudaError_t e = launch_pdl(fn, dim3(static_cast<unsigned>(blocks)), dim3(kConvThreads), args, smem,
                                     reinterpret_cast<cudaStream_t>(stream));
    return launched(e, PlanRecord::kSequence, "causal_conv", static_cast<long long>(blocks), kConvThreads, vec ? 1 : 0,
                    P.vcols, P.stretch, P.segs, 1);
} catch (...) {
    return internal_error();
}

int gc_b200_causal_conv_backward_workspace(const gc_tensor *dy, const gc_tensor *x, const gc_tensor *weight,
                                           const gc_tensor *dx, uint64_t *bytes) try {
    if (bytes == nullptr) return gc_error(GC_INVALID, "null size pointer");
    ConvCall call;
    int st = check_grad_data(dy, x, weight, dx, call);
    if (st != GC_OK) return st;
    *bytes = 0;
    if (call.n == 0) return gc_error(GC_OK, "");
    DeviceFacts facts;
    if ((st = current_facts(facts)) != GC_OK) return st;
    // states that are aligned worse than the data need no more space than this
    *bytes = std::max(grad_space(plan_grad(call, true, facts.sms), call), grad_space(plan_grad(call, false, facts.sms), call));
    return gc_error(GC_OK, "");
} catch (...) {
    return internal_error();
}

int gc_b200_causal_conv_backward(const gc_tensor *dy, const gc_tensor *x, const gc_tensor *weight, const gc_tensor *bias,
                                 const gc_tensor *state, const gc_tensor *dstate_out, const int32_t *lengths,
                                 gc_tensor *dx, gc_tensor *dweight, gc_tensor *dbias, gc_tensor *dstate, int activation,
                                 void *workspace, uint64_t workspace_bytes, void *stream) try {
    ConvCall call;
    int st = check_grad_data(dy, x, weight, dx, call);
    if (st != GC_OK) return st;
    if ((st = check_param(bias, x, {call.c})) != GC_OK) return st;
    if ((st = check_param(dweight, x, {call.c, call.taps})) != GC_OK) return st;
    if ((st = check_param(dbias, x, {call.c})) != GC_OK) return st;
    if ((st = check_states({{state, &call.state}, {dstate_out, &call.dstate}, {dstate, &call.state_out}}, x, call)) != GC_OK)
        return st;
    if ((st = check_lengths(lengths)) != GC_OK) return st;
    if ((st = view_states({{state, &call.state}, {dstate_out, &call.dstate}, {dstate, &call.state_out}})) != GC_OK) return st;
    if (outputs_meet({range_of(call.y), range_of(dweight), range_of(dbias), range_of(call.state_out), {workspace, workspace_bytes}},
                     {range_of(call.x), range_of(call.dy), range_of(weight), range_of(bias), range_of(call.state),
                      range_of(call.dstate), range_of_lengths(lengths, call.n)}))
        return gc_error(GC_INVALID, "outputs and workspace must not overlap inputs or one another");
    if ((st = check_layouts(weight, bias, activation, call)) != GC_OK) return st;
    for (const gc_tensor *t : {static_cast<const gc_tensor *>(dweight), static_cast<const gc_tensor *>(dbias)})
        if ((st = check_dense(t, "parameters must be dense")) != GC_OK) return st;
    int dev = -1;
    if ((st = check_call({dy, x, weight, bias, state, dstate_out, dx, dweight, dbias, dstate}, {lengths}, x->device_index,
                         stream, dev)) != GC_OK)
        return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (call.n == 0) {  // sums over nothing
        for (const gc_tensor *t : {dweight, dbias})
            if (t != nullptr && e == cudaSuccess) e = cudaMemsetAsync(t->data, 0, range_of(t).bytes, s);
        return launched(e);
    }
    DeviceFacts facts;
    if ((st = device_facts(dev, facts)) != GC_OK) return st;
    const bool vec = groups_of_four({&call.x, &call.dy, &call.y, &call.state, &call.state_out, &call.dstate});
    const GradPlan plan = plan_grad(call, vec, facts.sms);
    const bool sums = dweight != nullptr || dbias != nullptr;
    if (sums) {
        if ((st = check_workspace(workspace, workspace_bytes, grad_space(plan, call))) != GC_OK) return st;
        if ((st = check_device_memory(workspace, x->device_index, dev)) != GC_OK) return st;
    }
    ConvSeqParams P{};
    fill(P, call, weight, bias, activation, lengths, false);
    P.vcols = P.c / (vec ? 4 : 1);
    P.stretch = plan.stretch;
    P.segs = std::max(1LL, plan.segs);  // a sequence of no tokens still passes its states' gradients on
    P.cols = plan.cols;
    P.workers = plan.workers;
    P.blocks_y = plan.blocks_y;
    P.part = sums ? static_cast<float *>(workspace) : nullptr;
    void *args[] = {&P};
    const long long grid = plan.tiles * plan.blocks_y;
    if (grid > INT32_MAX) return gc_error(GC_UNSUPPORTED, "more work than a grid has blocks");
    const void *fn = conv_kernel(kBackward, call.x.type, vec, P.taps, activation);
    const size_t smem = ring_bytes(call.x.type, vec ? 4 : 1, P.taps);
    if ((st = opt_in_ring(dev, fn, smem, facts)) != GC_OK) return st;
    e = launch_pdl(fn, dim3(static_cast<unsigned>(grid)), dim3(kConvThreads), args, smem, s);
    if (e == cudaSuccess && sums) {
        SumParams S{};
        S.part = P.part;
        S.rows = plan.blocks_y;
        S.cols = call.c;
        S.planes = P.taps + 1;
        for (int k = 0; k < P.taps; ++k) {
            S.out[k] = dweight != nullptr ? dweight->data : nullptr;
            S.type[k] = dweight != nullptr ? elem_type(dweight->dtype) : kElemF32;
            S.mul[k] = P.taps;
            S.add[k] = k;
        }
        S.out[P.taps] = dbias != nullptr ? dbias->data : nullptr;
        S.type[P.taps] = dbias != nullptr ? elem_type(dbias->dtype) : kElemF32;
        S.mul[P.taps] = 1;
        e = launch_sum_rows(S, s);
    }
    return launched(e, PlanRecord::kSequence, "causal_conv_backward", grid, kConvThreads, vec ? 1 : 0, P.cols, P.stretch,
                    P.segs, sums ? 2 : 1);
} catch (...) {
    return internal_error();
}

int gc_b200_causal_conv_step(const gc_tensor *x, const gc_tensor *weight, const gc_tensor *bias, const gc_tensor *state,
                             gc_tensor *y, gc_tensor *state_out, int activation, void *stream) try {
    ConvCall call;
    int st = check_conv(x, weight, bias, call, true);
    if (st != GC_OK) return st;
    if ((st = check_data_tensor(y, x, {call.n, call.c})) != GC_OK) return st;
    if (state == nullptr || state_out == nullptr) return gc_error(GC_INVALID, "null tensor descriptor");
    if ((st = check_states({{state, &call.state}, {state_out, &call.state_out}}, x, call)) != GC_OK) return st;
    if ((st = strided_of(x, call.x)) != GC_OK || (st = strided_of(y, call.y)) != GC_OK) return st;
    if ((st = view_states({{state, &call.state}, {state_out, &call.state_out}})) != GC_OK) return st;
    bool same = call.state.data == call.state_out.data;
    for (int i = 0; i < 3; ++i) same = same && call.state.s[i] == call.state_out.s[i];
    if (outputs_meet({range_of(call.y), range_of(call.state_out)},
                     {range_of(call.x), range_of(weight), range_of(bias), same ? Range{nullptr, 0} : range_of(call.state)}))
        return gc_error(GC_INVALID, "outputs must not overlap inputs or one another (the new state may be the old one)");
    if ((st = check_layouts(weight, bias, activation, call)) != GC_OK) return st;
    if (call.n == 0) return gc_error(GC_OK, "");
    int dev = -1;
    if ((st = check_call({x, weight, bias, state, y, state_out}, {}, x->device_index, stream, dev)) != GC_OK) return st;
    const bool vec = groups_of_four({&call.x, &call.y, &call.state, &call.state_out});
    ConvSeqParams P{};
    fill(P, call, weight, bias, activation, nullptr, true);
    P.vcols = P.c / (vec ? 4 : 1);
    const wide blocks = (static_cast<wide>(call.n) * P.vcols + kConvThreads - 1) / kConvThreads;
    if (blocks > INT32_MAX) return gc_error(GC_UNSUPPORTED, "more work than a grid has blocks");
    P.small = blocks * kConvThreads <= UINT32_MAX ? 1 : 0;
    void *args[] = {&P};
    const cudaError_t e = launch_pdl(conv_kernel(kStep, call.x.type, vec, P.taps, activation),
                                     dim3(static_cast<unsigned>(blocks)), dim3(kConvThreads), args, 0,
                                     reinterpret_cast<cudaStream_t>(stream));
    return launched(e, PlanRecord::kSequence, "causal_conv_step", static_cast<long long>(blocks), kConvThreads, vec ? 1 : 0,
                    P.vcols, 1, 1, 1);
} catch (...) {
    return internal_error();
}

}  // extern "C"
