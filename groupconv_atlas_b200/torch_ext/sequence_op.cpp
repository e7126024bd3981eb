// PyTorch front end of the operators on rows and sequences: layer_norm,
// causal_conv, selective_scan with their gradients, and the forms of the last
// two for one token.  As in conv_op.cpp outputs and workspaces come from
// PyTorch's allocator, calls go to the current stream, and errors come back as
// gc_status values.
#include "front_end.h"

#include <torch/csrc/autograd/variable.h>

#include <utility>

using namespace front_end;

namespace {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// Whether the library reads t as it lies: last axis dense, no two elements in
// the same place.
bool readable(const at::Tensor &t) {
    if (t.numel() == 0) return true;
    const int64_t last = t.dim() - 1;
    if (last >= 0 && t.size(last) > 1 && t.stride(last) != 1) return false;
    std::vector<std::pair<int64_t, int64_t>> axes;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1) axes.emplace_back(t.stride(i), t.size(i));
    std::sort(axes.begin(), axes.end());
    int64_t reach = 1;
    for (const auto &a : axes) {
        if (a.first < reach) return false;
        reach += (a.second - 1) * a.first;
    }
    return true;
}
at::Tensor as_read(const at::Tensor &t) { return !t.defined() || readable(t) ? t : t.contiguous(); }

// Rows of the last axis, evenly spaced, in at most four axes.
bool even_rows(const at::Tensor &t) {
    int64_t rows = 1, ld = 0;
    for (int64_t i = t.dim() - 2; i >= 0; --i) {
        if (t.size(i) > 1) {
            if (rows == 1) ld = t.stride(i);
            else if (t.stride(i) != ld * rows) return false;
        }
        rows *= t.size(i);
    }
    return true;
}
at::Tensor as_rows(const at::Tensor &t) { return t.numel() == 0 || (readable(t) && even_rows(t)) ? t : t.contiguous(); }

// A descriptor and a pointer to it, NULL for an undefined tensor.
struct Desc {
    gc_tensor t{};
    bool given = false;
    Desc() = default;
    explicit Desc(const at::Tensor &v) : given(v.defined()) {
        if (given) t = describe_view(v);
    }
    gc_tensor *get() { return given ? &t : nullptr; }
};

void check(int status) {
    if (status != GC_OK) fail(status);
}
at::Tensor dense_like(const at::Tensor &t) {
    return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous));
}
void *data_of(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

at::Tensor option(const c10::optional<at::Tensor> &t) { return t.value_or(at::Tensor()); }

bool any_wants_grad(std::initializer_list<at::Tensor> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor &t : tensors)
        if (wants_grad(t)) return true;
    return false;
}
void refuse_forward_mode(std::initializer_list<at::Tensor> tensors) {
    for (const at::Tensor &t : tensors) no_forward_mode(t);
}
template <class N>
std::shared_ptr<N> new_node() {
    return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}

// A tensor that the gradient needs, which may be none.
struct Saved {
    SavedVariable v;
    bool given = false;
    void set(const at::Tensor &t) {
        given = t.defined();
        if (given) v = SavedVariable(t, false);
    }
    at::Tensor get() const { return given ? v.unpack() : at::Tensor(); }
    void drop() {
        if (given) v.reset_data();
    }
};

// ---- lengths --------------------------------------------------------------------------
at::Tensor check_lengths(const c10::optional<at::Tensor> &lengths, const at::Tensor &x) {
    if (!lengths.has_value()) return at::Tensor();
    const at::Tensor &t = *lengths;
    if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong)
        throw std::invalid_argument("lengths must be int32 or int64");
    if (t.dim() != 1 || t.size(0) != x.size(0)) throw std::invalid_argument("lengths must have one element per sequence");
    if (t.device() != x.device()) throw std::invalid_argument("lengths must be on the data's device");
    if (t.scalar_type() == at::kLong) return t.clamp(0, INT32_MAX).to(at::kInt).contiguous();
    return t.contiguous();
}
const int32_t *lengths_ptr(const at::Tensor &t) { return t.defined() ? t.data_ptr<int32_t>() : nullptr; }

// ---- layer norm -----------------------------------------------------------------------
struct LayerNormGrad : torch::autograd::Node {
    Saved x_, gamma_, beta_;
    at::Tensor stats_;
    std::string name() const override { return "LayerNormGrad"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Saved *s : {&x_, &gamma_, &beta_}) s->drop();
    }
    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
        no_double_backward();
        const at::Tensor saved = x_.get();
        c10::OptionalDeviceGuard guard(saved.device());
        const at::Tensor x = as_rows(saved), dy = as_rows(grads[0]);
        at::Tensor gamma = gamma_.get(), beta = beta_.get(), dx = dense_like(x), dgamma, dbeta;
        if (gamma.defined()) gamma = gamma.contiguous();
        if (gamma.defined() && task_should_compute_output(1)) dgamma = dense_like(gamma);
        if (beta.defined() && task_should_compute_output(2)) dbeta = dense_like(beta);
        Desc xd(x), dyd(dy), dxd(dx), gd(gamma), sd(stats_), dgd(dgamma), dbd(dbeta);
        uint64_t bytes = 0;
        if (dgamma.defined() || dbeta.defined())
            check(gc_b200_layer_norm_backward_workspace(dyd.get(), xd.get(), dxd.get(), &bytes));
        const at::Tensor space = workspace_of(bytes, x);
        check(gc_b200_layer_norm_backward(dyd.get(), xd.get(), gd.get(), sd.get(), dxd.get(), dgd.get(), dbd.get(),
                                          data_of(space), bytes, stream_of(x)));
        return {dx, dgamma, dbeta};
    }
};

at::Tensor layer_norm(const at::Tensor &x, const c10::optional<at::Tensor> &gamma, const c10::optional<at::Tensor> &beta,
                      double eps) {
    no_tracing();
    if (x.dim() < 1) throw std::invalid_argument("input must have at least one axis");
    c10::OptionalDeviceGuard guard;
    if (x.is_cuda()) guard.reset_device(x.device());
    at::Tensor g = option(gamma), b = option(beta);
    refuse_forward_mode({x, g, b});
    if (g.defined()) g = g.contiguous();
    if (b.defined()) b = b.contiguous();
    const at::Tensor xi = as_rows(x.dim() > 4 ? x.flatten(0, -2) : x);
    const bool grad = any_wants_grad({xi, g, b});
    at::Tensor y = dense_like(xi), stats;
    const int64_t c = xi.size(-1), rows = c > 0 ? xi.numel() / c : 0;
    if (grad) stats = at::empty({rows, 2}, x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
    Desc xd(xi), yd(y), gd(g), bd(b), sd(stats);
    check(gc_b200_layer_norm(xd.get(), gd.get(), bd.get(), yd.get(), sd.get(), eps, stream_of(x)));
    if (grad) {
        auto node = new_node<LayerNormGrad>();
        node->set_next_edges(torch::autograd::collect_next_edges(xi, g, b));
        node->x_.set(xi);
        node->gamma_.set(g);
        node->beta_.set(b);
        node->stats_ = stats;
        torch::autograd::set_history(y, node);
    }
    return x.dim() > 4 ? y.view(x.sizes()) : y;
}

// ---- causal convolution ---------------------------------------------------------------
struct CausalConvGrad : torch::autograd::Node {
    Saved x_, w_, bias_, state_, lengths_;
    int64_t activation_ = 0;
    std::string name() const override { return "CausalConvGrad"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Saved *s : {&x_, &w_, &bias_, &state_, &lengths_}) s->drop();
    }
    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const at::Tensor dlast0 = grads.size() > 1 ? grads[1] : at::Tensor();
        if (!grads[0].defined() && !dlast0.defined()) return variable_list(4);
        no_double_backward();
        const at::Tensor saved = x_.get();
        c10::OptionalDeviceGuard guard(saved.device());
        const at::Tensor x = as_read(saved), w = w_.get().contiguous(), state = as_read(state_.get());
        const at::Tensor lengths = lengths_.given ? lengths_.get().contiguous() : at::Tensor();
        at::Tensor bias = bias_.get();
        if (bias.defined()) bias = bias.contiguous();
        const at::Tensor dy = grads[0].defined() ? as_read(grads[0]) : at::zeros(x.sizes(), x.options());
        const at::Tensor dlast = as_read(dlast0);
        at::Tensor dx = dense_like(x), dw, db, dstate;
        if (task_should_compute_output(1)) dw = dense_like(w);
        if (bias.defined() && task_should_compute_output(2)) db = dense_like(bias);
        if (state.defined() && task_should_compute_output(3)) dstate = dense_like(state);
        Desc xd(x), wd(w), bd(bias), sd(state), dyd(dy), dld(dlast), dxd(dx), dwd(dw), dbd(db), dsd(dstate);
        uint64_t bytes = 0;
        if (dw.defined() || db.defined())
            check(gc_b200_causal_conv_backward_workspace(dyd.get(), xd.get(), wd.get(), dxd.get(), &bytes));
        const at::Tensor space = workspace_of(bytes, x);
        check(gc_b200_causal_conv_backward(dyd.get(), xd.get(), wd.get(), bd.get(), sd.get(), dld.get(), lengths_ptr(lengths),
                                           dxd.get(), dwd.get(), dbd.get(), dsd.get(), static_cast<int>(activation_),
                                           data_of(space), bytes, stream_of(x)));
        return {dx, dw, db, dstate};
    }
};

std::pair<at::Tensor, at::Tensor> causal_conv(const at::Tensor &x, const at::Tensor &weight,
                                              const c10::optional<at::Tensor> &bias, int64_t activation,
                                              const c10::optional<at::Tensor> &state, const c10::optional<at::Tensor> &lengths,
                                              bool return_state) {
    no_tracing();
    if (x.dim() != 3) throw std::invalid_argument("input must be (N, L, C)");
    if (weight.dim() != 2 || weight.size(1) < 1) throw std::invalid_argument("weight must be (C, K)");
    c10::OptionalDeviceGuard guard;
    if (x.is_cuda()) guard.reset_device(x.device());
    at::Tensor b = option(bias), s = option(state);
    refuse_forward_mode({x, weight, b, s});
    const at::Tensor xi = as_read(x), w = weight.contiguous(), si = as_read(s), lens = check_lengths(lengths, x);
    if (b.defined()) b = b.contiguous();
    const bool grad = any_wants_grad({xi, w, b, si});
    at::Tensor y = dense_like(xi), last;
    if (return_state)
        last = at::empty({x.size(0), w.size(1) - 1, x.size(2)}, x.options().memory_format(at::MemoryFormat::Contiguous));
    Desc xd(xi), wd(w), bd(b), sd(si), yd(y), ld(last);
    check(gc_b200_causal_conv(xd.get(), wd.get(), bd.get(), sd.get(), lengths_ptr(lens), yd.get(), ld.get(),
                              static_cast<int>(activation), stream_of(x)));
    if (grad) {
        auto node = new_node<CausalConvGrad>();
        node->set_next_edges(torch::autograd::collect_next_edges(xi, w, b, si));
        node->x_.set(xi);
        node->w_.set(w);
        node->bias_.set(b);
        node->state_.set(si);
        node->lengths_.set(lens);
        node->activation_ = activation;
        torch::autograd::set_history(y, node);
        if (return_state) torch::autograd::set_history(last, node);
    }
    return {y, last};
}

// Steps write into a tensor of the caller's.
void prepare_step(std::initializer_list<at::Tensor> inputs, const at::Tensor &out) {
    refuse_forward_mode(inputs);
    no_forward_mode(out);
    if (any_wants_grad(inputs) || any_wants_grad({out}))
        throw std::runtime_error("a step has no gradient: call it under torch.no_grad()");
}
void wrote(const at::Tensor &t) {
    if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

at::Tensor causal_conv_step(const at::Tensor &x, const at::Tensor &weight, const at::Tensor &state,
                            const c10::optional<at::Tensor> &bias, int64_t activation,
                            const c10::optional<at::Tensor> &state_out) {
    no_tracing();
    if (x.dim() != 2) throw std::invalid_argument("input must be (N, C)");
    c10::OptionalDeviceGuard guard;
    if (x.is_cuda()) guard.reset_device(x.device());
    at::Tensor b = option(bias);
    const at::Tensor out = state_out.value_or(state);
    prepare_step({x, weight, b, state}, out);
    const at::Tensor xi = as_read(x), w = weight.contiguous();
    if (b.defined()) b = b.contiguous();
    at::Tensor y = dense_like(xi);
    Desc xd(xi), wd(w), bd(b), sd(state), yd(y), od(out);
    check(gc_b200_causal_conv_step(xd.get(), wd.get(), bd.get(), sd.get(), yd.get(), od.get(), static_cast<int>(activation),
                                   stream_of(x)));
    wrote(out);
    return y;
}

// ---- selective scan -------------------------------------------------------------------
// The operands in the order of the edges of the gradient's node.
enum { kX, kDt, kA, kB, kC, kD, kZ, kBias, kState, kOperands };
struct ScanDescs {
    Desc d[kOperands];
    gc_b200_scan_args args{};
    ScanDescs(const std::vector<at::Tensor> &t, const at::Tensor &lengths, bool softplus) {
        for (int i = 0; i < kOperands; ++i) d[i] = Desc(t[i]);
        args.x = d[kX].get();
        args.dt = d[kDt].get();
        args.a = d[kA].get();
        args.b = d[kB].get();
        args.c = d[kC].get();
        args.d = d[kD].get();
        args.z = d[kZ].get();
        args.dt_bias = d[kBias].get();
        args.state = d[kState].get();
        args.lengths = lengths_ptr(lengths);
        args.softplus = softplus ? 1 : 0;
    }
};
bool is_param(int i) { return i == kA || i == kD || i == kBias; }
std::vector<at::Tensor> scan_operands(std::vector<at::Tensor> t) {
    for (int i = 0; i < kOperands; ++i)
        if (t[i].defined()) t[i] = is_param(i) ? t[i].contiguous() : as_read(t[i]);
    return t;
}

struct SelectiveScanGrad : torch::autograd::Node {
    Saved saved_[kOperands], lengths_;
    at::Tensor kept_;
    uint64_t kept_bytes_ = 0;
    bool softplus_ = true;
    std::string name() const override { return "SelectiveScanGrad"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (Saved &s : saved_) s.drop();
        lengths_.drop();
        kept_.reset();
    }
    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const at::Tensor dlast0 = grads.size() > 1 ? grads[1] : at::Tensor();
        if (!grads[0].defined() && !dlast0.defined()) return variable_list(kOperands);
        no_double_backward();
        std::vector<at::Tensor> t(kOperands);
        for (int i = 0; i < kOperands; ++i) t[i] = saved_[i].get();
        c10::OptionalDeviceGuard guard(t[kX].device());
        t = scan_operands(t);
        const at::Tensor lengths = lengths_.given ? lengths_.get().contiguous() : at::Tensor();
        const at::Tensor dy = grads[0].defined() ? as_read(grads[0]) : at::zeros(t[kX].sizes(), t[kX].options());
        const at::Tensor dlast = as_read(dlast0);
        variable_list out(kOperands);
        for (int i = 0; i < kOperands; ++i)
            if (t[i].defined() && (i == kX || i == kDt || i == kZ || task_should_compute_output(i))) out[i] = dense_like(t[i]);
        ScanDescs q(t, lengths, softplus_);
        Desc g[kOperands];
        for (int i = 0; i < kOperands; ++i) g[i] = Desc(out[i]);
        const gc_b200_scan_grads gr{g[kX].get(), g[kDt].get(), g[kA].get(),    g[kB].get(),   g[kC].get(),
                                    g[kD].get(), g[kZ].get(),  g[kBias].get(), g[kState].get()};
        uint64_t forward = 0, kept = 0, bytes = 0;
        check(gc_b200_selective_scan_sizes(&q.args, &forward, &kept, &bytes));
        const at::Tensor space = workspace_of(bytes, t[kX]);
        Desc dyd(dy), dld(dlast);
        check(gc_b200_selective_scan_backward(&q.args, dyd.get(), dld.get(), data_of(kept_), kept_bytes_, &gr, data_of(space),
                                              bytes, stream_of(t[kX])));
        return out;
    }
};

std::pair<at::Tensor, at::Tensor> selective_scan(const at::Tensor &x, const at::Tensor &dt, const at::Tensor &a,
                                                 const at::Tensor &b, const at::Tensor &c, const c10::optional<at::Tensor> &d,
                                                 const c10::optional<at::Tensor> &z, const c10::optional<at::Tensor> &dt_bias,
                                                 bool softplus, const c10::optional<at::Tensor> &state,
                                                 const c10::optional<at::Tensor> &lengths, bool return_state) {
    no_tracing();
    if (x.dim() != 3) throw std::invalid_argument("input must be (N, L, C)");
    c10::OptionalDeviceGuard guard;
    if (x.is_cuda()) guard.reset_device(x.device());
    std::vector<at::Tensor> t = {x, dt, a, b.dim() == 3 ? b.unsqueeze(2) : b, c.dim() == 3 ? c.unsqueeze(2) : c,
                                 option(d), option(z), option(dt_bias), option(state)};
    for (const at::Tensor &v : t) no_forward_mode(v);
    t = scan_operands(t);
    const at::Tensor lens = check_lengths(lengths, x);
    bool grad = false;
    for (const at::Tensor &v : t) grad = grad || any_wants_grad({v});
    ScanDescs q(t, lens, softplus);
    uint64_t bytes = 0, kept_bytes = 0, backward = 0;
    check(gc_b200_selective_scan_sizes(&q.args, &bytes, &kept_bytes, &backward));
    at::Tensor y = dense_like(t[kX]), last, kept;
    const at::Tensor space = workspace_of(bytes, x);
    if (grad) kept = workspace_of(kept_bytes, x);
    if (return_state)
        last = at::empty({x.size(0), x.size(2), t[kB].size(3)},
                         x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
    Desc yd(y), ld(last);
    check(gc_b200_selective_scan(&q.args, yd.get(), ld.get(), data_of(kept), grad ? kept_bytes : 0, data_of(space), bytes,
                                 stream_of(x)));
    if (grad) {
        auto node = new_node<SelectiveScanGrad>();
        node->set_next_edges(torch::autograd::collect_next_edges(t[kX], t[kDt], t[kA], t[kB], t[kC], t[kD], t[kZ], t[kBias],
                                                                 t[kState]));
        for (int i = 0; i < kOperands; ++i) node->saved_[i].set(t[i]);
        node->lengths_.set(lens);
        node->kept_ = kept;
        node->kept_bytes_ = kept_bytes;
        node->softplus_ = softplus;
        torch::autograd::set_history(y, node);
        if (return_state) torch::autograd::set_history(last, node);
    }
    return {y, last};
}

at::Tensor selective_scan_step(const at::Tensor &x, const at::Tensor &dt, const at::Tensor &a, const at::Tensor &b,
                               const at::Tensor &c, const at::Tensor &state, const c10::optional<at::Tensor> &d,
                               const c10::optional<at::Tensor> &z, const c10::optional<at::Tensor> &dt_bias, bool softplus,
                               const c10::optional<at::Tensor> &state_out) {
    no_tracing();
    if (x.dim() != 2) throw std::invalid_argument("input must be (N, C)");
    c10::OptionalDeviceGuard guard;
    if (x.is_cuda()) guard.reset_device(x.device());
    const at::Tensor out = state_out.value_or(state);
    prepare_step({x, dt, a, b, c, state, option(d), option(z), option(dt_bias)}, out);
    std::vector<at::Tensor> t = scan_operands({x, dt, a, b.dim() == 2 ? b.unsqueeze(1) : b, c.dim() == 2 ? c.unsqueeze(1) : c,
                                               option(d), option(z), option(dt_bias), at::Tensor()});
    t[kState] = state;  // never a copy
    ScanDescs q(t, at::Tensor(), softplus);
    at::Tensor y = dense_like(t[kX]);
    Desc yd(y), od(out);
    check(gc_b200_selective_scan_step(&q.args, yd.get(), od.get(), stream_of(x)));
    wrote(out);
    return y;
}

}  // namespace

void bind_sequence_ops(pybind11::module_ &m) {
    m.def("layer_norm", &layer_norm, "gc_b200_layer_norm on the current CUDA stream, with its gradient");
    m.def("causal_conv", &causal_conv, "gc_b200_causal_conv on the current CUDA stream, with its gradient");
    m.def("causal_conv_step", &causal_conv_step, "gc_b200_causal_conv_step on the current CUDA stream");
    m.def("selective_scan", &selective_scan, "gc_b200_selective_scan on the current CUDA stream, with its gradient");
    m.def("selective_scan_step", &selective_scan_step, "gc_b200_selective_scan_step on the current CUDA stream");
}
