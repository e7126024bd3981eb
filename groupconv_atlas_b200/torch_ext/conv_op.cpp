// PyTorch front end of gc_cuda_conv for the torch.nn module: allocates the
// output with PyTorch's caching allocator and calls the C ABI on the current
// CUDA stream, all in C++, so that a substituted layer costs about as much
// host time per call as a cuDNN convolution.  The descriptors are built
// exactly as the reference's Python caller builds them (bench/api.py:71-83):
// element strides, the tensor's device and device index, float32 or float64.
// Errors come back as gc_status values with the library's thread-local
// message; nothing here computes a convolution.  conv_ex does the same for
// gc_b200_conv_ex (bias, activation, channels-last output); group_norm and
// dropout do it for gc_b200_group_norm and gc_b200_dropout and record their
// gradients with autograd.  sequence_op.cpp holds the operators on sequences.
#include "front_end.h"

using namespace front_end;

namespace {

// y = conv(x, w) with the layer's geometry; x must be 4-D.  Raises
// RuntimeError("gc_status <s>: <message>") on any non-OK status.
at::Tensor conv(const at::Tensor &x, const at::Tensor &w, int64_t cout, int64_t r, int64_t s, int64_t groups,
                int64_t sh, int64_t sw, int64_t ph, int64_t pw, int64_t dh, int64_t dw, int64_t implementation) {
    no_tracing();
    if (x.dim() != 4) throw std::invalid_argument("input must be 4-D NCHW");
    const gc_shape p{x.size(0), x.size(1), cout, x.size(2), x.size(3), r, s, groups, sh, sw, ph, pw, dh, dw};
    int64_t ho = 0, wo = 0;
    int st = gc_validate_shape(&p, &ho, &wo);
    if (st != GC_OK) throw std::runtime_error("gc_status " + std::to_string(st) + ": " + gc_last_error());
    // gc_cuda_conv requires the tensors' device to be the current device (as
    // nn.Conv2d runs on its input's device whatever the current one is).
    c10::OptionalDeviceGuard guard;
    if (x.is_cuda()) guard.reset_device(x.device());
    at::Tensor y = at::empty({p.n, cout, ho, wo}, x.options());
    const gc_tensor xd = describe(x), wd = describe(w);
    gc_tensor yd = describe(y);
    void *stream = x.is_cuda() ? static_cast<void *>(c10::cuda::getCurrentCUDAStream(x.get_device()).stream())
                               : nullptr;
    st = gc_cuda_conv(&p, &xd, &wd, &yd, static_cast<int>(implementation), stream);
    if (st != GC_OK) throw std::runtime_error("gc_status " + std::to_string(st) + ": " + gc_last_error());
    return y;
}

// y = act(conv(x, w) + bias) through gc_b200_conv_ex: bias optional, layout
// 0 (NCHW output) or 1 (channels-last output), activation GC_B200_ACT_*.
at::Tensor conv_ex(const at::Tensor &x, const at::Tensor &w, const c10::optional<at::Tensor> &bias, int64_t cout,
                   int64_t r, int64_t s, int64_t groups, int64_t sh, int64_t sw, int64_t ph, int64_t pw, int64_t dh,
                   int64_t dw, int64_t layout, int64_t activation) {
    no_tracing();
    if (x.dim() != 4) throw std::invalid_argument("input must be 4-D NCHW");
    const gc_shape p{x.size(0), x.size(1), cout, x.size(2), x.size(3), r, s, groups, sh, sw, ph, pw, dh, dw};
    int64_t ho = 0, wo = 0;
    int st = gc_validate_shape(&p, &ho, &wo);
    if (st != GC_OK) throw std::runtime_error("gc_status " + std::to_string(st) + ": " + gc_last_error());
    c10::OptionalDeviceGuard guard;
    if (x.is_cuda()) guard.reset_device(x.device());
    at::Tensor y = at::empty({p.n, cout, ho, wo}, x.options().memory_format(
                                                    layout == GC_B200_NHWC ? at::MemoryFormat::ChannelsLast
                                                                           : at::MemoryFormat::Contiguous));
    const gc_tensor xd = describe(x), wd = describe(w);
    gc_tensor yd = describe(y);
    gc_tensor bd{};
    if (bias.has_value()) bd = describe(*bias);
    void *stream = x.is_cuda() ? static_cast<void *>(c10::cuda::getCurrentCUDAStream(x.get_device()).stream())
                               : nullptr;
    st = gc_b200_conv_ex(&p, &xd, &wd, bias.has_value() ? &bd : nullptr, &yd, static_cast<int>(layout),
                         static_cast<int>(activation), stream);
    if (st != GC_OK) throw std::runtime_error("gc_status " + std::to_string(st) + ": " + gc_last_error());
    return y;
}


// ---- group norm and dropout -----------------------------------------------------

// Dense (N, C, ..) with the channels innermost, which is what channels_last
// means for rank 4 and what this library computes for ranks 2 and 3 too.
at::Tensor empty_channels_last(const at::Tensor &x) {
    std::vector<int64_t> strides(x.dim());
    int64_t expect = x.size(1);
    strides[1] = 1;
    for (int64_t i = x.dim() - 1; i >= 2; --i) {
        strides[i] = expect;
        expect *= std::max<int64_t>(x.size(i), 1);
    }
    strides[0] = expect;
    return at::empty_strided(x.sizes(), strides, x.options());
}

// Whether gc_b200_group_norm reads t as it lies: channel stride 1, evenly
// spaced pixels, images that do not interleave.
bool pixels_in_order(const at::Tensor &t) {
    if (t.size(1) > 1 && t.stride(1) != 1) return false;
    int64_t px = 1, ldp = t.size(1);
    for (int64_t i = t.dim() - 1; i >= 2; --i) {
        if (t.size(i) > 1) {
            if (px == 1) ldp = t.stride(i);
            else if (t.stride(i) != ldp * px) return false;
        }
        px *= t.size(i);
    }
    return ldp >= t.size(1) && (t.size(0) <= 1 || t.stride(0) >= (px - 1) * ldp + t.size(1));
}
at::Tensor in_order(const at::Tensor &t) {
    if (t.numel() == 0 || pixels_in_order(t)) return t;
    at::Tensor copy = empty_channels_last(t);
    copy.copy_(t);
    return copy;
}

// The dropout of one forward call and of its gradient.
struct Drop {
    gc_b200_dropout_args args{};
    at::Tensor used;  // the device words in effect, when the generator's are known only to a captured graph
    bool on = false;
};

// seed given: that seed and offset.  Otherwise torch's CUDA generator, which
// also works inside a graph capture (a replay draws anew); the top bit of the
// offset keeps these draws apart from torch's own, which count from 0.
Drop make_drop(const at::Tensor &x, double p, int64_t scope, const c10::optional<uint64_t> &seed, uint64_t offset,
               bool grad) {
    Drop d;
    d.on = p != 0.0;
    d.args.p = p;
    d.args.scope = static_cast<int32_t>(scope);
    if (!d.on) return d;
    if (seed.has_value()) {
        d.args.seed = *seed;
        d.args.offset = offset;
        return d;
    }
    if (!x.is_cuda()) return d;  // refused by the call
    auto *gen = at::get_generator_or_default<at::CUDAGeneratorImpl>(
        c10::nullopt, at::cuda::detail::getDefaultCUDAGenerator(x.get_device()));
    at::PhiloxCudaState state;
    {
        std::lock_guard<std::mutex> lock(gen->mutex_);
        state = gen->philox_cuda_state(4);
    }
    constexpr uint64_t kOwn = 1ull << 63;
    if (state.captured_) {
        d.args.seed_ptr = reinterpret_cast<const uint64_t *>(state.seed_.ptr);
        d.args.offset_ptr = reinterpret_cast<const uint64_t *>(state.offset_.ptr);
        d.args.offset = kOwn + state.offset_intragraph_;
        if (grad) {
            d.used = at::empty({2}, x.options().dtype(at::kLong).memory_format(at::MemoryFormat::Contiguous));
            d.args.used = reinterpret_cast<uint64_t *>(d.used.data_ptr<int64_t>());
        }
    } else {
        d.args.seed = state.seed_.val;
        d.args.offset = kOwn + state.offset_.val;
    }
    return d;
}

// The dropout again in the gradient: the words that were in effect.
Drop again(Drop d) {
    d.args.used = nullptr;
    if (d.used.defined()) {
        const uint64_t *w = reinterpret_cast<const uint64_t *>(d.used.data_ptr<int64_t>());
        d.args.seed = d.args.offset = 0;
        d.args.seed_ptr = w;
        d.args.offset_ptr = w + 1;
    }
    return d;
}

struct NormArgs {
    int64_t groups = 1, activation = 0;
    double eps = 0.0;
};

// One gc_b200_group_norm call; stats undefined for none.
at::Tensor norm_forward(const at::Tensor &x, const at::Tensor &gamma, const at::Tensor &beta, const NormArgs &a,
                        const Drop &drop, at::Tensor stats) {
    at::Tensor y = empty_channels_last(x);
    const gc_tensor xd = describe_view(x);
    gc_tensor yd = describe_view(y), gd{}, bd{}, sd{};
    if (gamma.defined()) gd = describe_view(gamma);
    if (beta.defined()) bd = describe_view(beta);
    if (stats.defined()) sd = describe_view(stats);
    // The resident path needs no workspace, so the call is tried without one
    // first; the query costs small calls a tenth of their host time.
    auto call = [&](void *space, uint64_t bytes) {
        return gc_b200_group_norm(&xd, gamma.defined() ? &gd : nullptr, beta.defined() ? &bd : nullptr, &yd,
                                  stats.defined() ? &sd : nullptr, a.groups, a.eps, static_cast<int>(a.activation),
                                  drop.on ? &drop.args : nullptr, space, bytes, stream_of(x));
    };
    int st = call(nullptr, 0);
    if (st == GC_INVALID) {
        uint64_t bytes = 0;
        if ((st = gc_b200_group_norm_workspace(&xd, &yd, a.groups, &bytes)) != GC_OK) fail(st);
        const at::Tensor space = workspace_of(bytes, x);
        st = call(space.defined() ? space.data_ptr() : nullptr, bytes);
    }
    if (st != GC_OK) fail(st);
    return y;
}

// The gradients are plain autograd nodes: a training step's host time counts,
// and a torch::autograd::Function's context costs several microseconds of it.
struct GroupNormGrad : torch::autograd::Node {
    torch::autograd::SavedVariable x_, gamma_, beta_;
    bool has_gamma_ = false, has_beta_ = false;
    at::Tensor stats_;
    NormArgs a_;
    Drop drop_;

    std::string name() const override { return "GroupNormGrad"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x_.reset_data();
        gamma_.reset_data();
        beta_.reset_data();
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
        no_double_backward();
        // Hooks on saved tensors may give them back with other strides (pinned
        // copies on the host are plain).
        const at::Tensor saved = x_.unpack();
        c10::OptionalDeviceGuard guard(saved.device());
        const at::Tensor x = in_order(saved), gamma = has_gamma_ ? gamma_.unpack().contiguous() : at::Tensor(),
                         beta = has_beta_ ? beta_.unpack().contiguous() : at::Tensor();
        const Drop drop = again(drop_);
        const at::Tensor dy = in_order(grads[0]);
        at::Tensor dx = empty_channels_last(x), dgamma, dbeta;
        if (has_gamma_ && task_should_compute_output(1)) dgamma = at::empty_like(gamma);
        if (has_beta_ && task_should_compute_output(2)) dbeta = at::empty_like(beta);
        const gc_tensor xd = describe_view(x), dyd = describe_view(dy), sd = describe_view(stats_);
        gc_tensor dxd = describe_view(dx), gd{}, bd{}, dgd{}, dbd{};
        if (has_gamma_) gd = describe_view(gamma);
        if (has_beta_) bd = describe_view(beta);
        if (dgamma.defined()) dgd = describe_view(dgamma);
        if (dbeta.defined()) dbd = describe_view(dbeta);
        uint64_t bytes = 0;
        int st = gc_b200_group_norm_backward_workspace(&dyd, &xd, &dxd, a_.groups, &bytes);
        if (st != GC_OK) fail(st);
        const at::Tensor space = workspace_of(bytes, x);
        st = gc_b200_group_norm_backward(
            &dyd, &xd, has_gamma_ ? &gd : nullptr, has_beta_ ? &bd : nullptr, &sd, &dxd,
            dgamma.defined() ? &dgd : nullptr, dbeta.defined() ? &dbd : nullptr, a_.groups,
            static_cast<int>(a_.activation), drop.on ? &drop.args : nullptr, space.defined() ? space.data_ptr() : nullptr,
            bytes, stream_of(x));
        if (st != GC_OK) fail(st);
        return {dx, dgamma, dbeta};
    }
};

at::Tensor group_norm(const at::Tensor &x, const c10::optional<at::Tensor> &gamma,
                      const c10::optional<at::Tensor> &beta, int64_t groups, double eps, int64_t activation, double p,
                      int64_t scope, const c10::optional<uint64_t> &seed, uint64_t offset) {
    no_tracing();
    if (x.dim() < 2 || x.dim() > 4) throw std::invalid_argument("input must have 2 to 4 axes (N, C, ..)");
    c10::OptionalDeviceGuard guard;
    if (x.is_cuda()) guard.reset_device(x.device());
    at::Tensor g = gamma.value_or(at::Tensor()), b = beta.value_or(at::Tensor());
    for (const at::Tensor &t : {x, g, b}) no_forward_mode(t);
    if (g.defined()) g = g.contiguous();
    if (b.defined()) b = b.contiguous();
    const bool grad = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(g) || wants_grad(b));
    const at::Tensor xi = in_order(x);
    const Drop drop = make_drop(x, p, scope, seed, offset, grad);
    const NormArgs a{groups, activation, eps};
    const bool whole = groups >= 1 && x.size(1) % groups == 0;  // else refused by the call, before stats of that size
    if (!grad || !whole) return norm_forward(xi, g, b, a, drop, at::Tensor());
    const at::Tensor stats =
        at::empty({x.size(0), groups, 2}, x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
    at::Tensor y = norm_forward(xi, g, b, a, drop, stats);
    auto node = std::shared_ptr<GroupNormGrad>(new GroupNormGrad(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(xi, g, b));
    node->x_ = torch::autograd::SavedVariable(xi, false);
    node->has_gamma_ = g.defined();
    node->has_beta_ = b.defined();
    if (g.defined()) node->gamma_ = torch::autograd::SavedVariable(g, false);
    if (b.defined()) node->beta_ = torch::autograd::SavedVariable(b, false);
    node->stats_ = stats;
    node->a_ = a;
    node->drop_ = drop;
    torch::autograd::set_history(y, node);
    return y;
}

// One gc_b200_dropout call on tensors that lie alike.
at::Tensor dropout_forward(const at::Tensor &x, const at::Tensor &residual, const Drop &drop) {
    at::Tensor y = at::empty_like(x);
    const gc_tensor xd = describe_view(x);
    gc_tensor yd = describe_view(y), rd{};
    if (residual.defined()) rd = describe_view(residual);
    const int st = gc_b200_dropout(&xd, residual.defined() ? &rd : nullptr, &yd, &drop.args, stream_of(x));
    if (st != GC_OK) fail(st);
    return y;
}

// `t` laid out like `like`, which is dense.
at::Tensor laid_out_like(const at::Tensor &t, const at::Tensor &like) {
    if (t.sizes() != like.sizes() || t.numel() == 0) return t;  // refused by the call, or nothing to lay out
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1 && t.stride(i) != like.stride(i)) {
            at::Tensor copy = at::empty_strided(like.sizes(), like.strides(), t.options());
            copy.copy_(t);
            return copy;
        }
    return t;
}

// Nothing of the data is kept: the gradient needs x's layout and the draws.
struct DropoutGrad : torch::autograd::Node {
    std::vector<int64_t> sizes_, strides_;
    Drop drop_;

    std::string name() const override { return "DropoutGrad"; }
    torch::autograd::variable_list apply(torch::autograd::variable_list &&grads) override {
        if (!grads[0].defined()) return {at::Tensor(), at::Tensor()};
        no_double_backward();
        c10::OptionalDeviceGuard guard(grads[0].device());
        at::Tensor dx;
        if (task_should_compute_output(0)) {
            // the mask goes by place in memory: dy has to lie as x did
            at::Tensor dy = grads[0];
            bool same = true;
            for (size_t i = 0; i < sizes_.size(); ++i) same = same && (sizes_[i] <= 1 || dy.stride(i) == strides_[i]);
            if (!same) {
                dy = at::empty_strided(sizes_, strides_, grads[0].options());
                dy.copy_(grads[0]);
            }
            dx = dropout_forward(dy, at::Tensor(), again(drop_));
        }
        return {dx, grads[0]};
    }
};

at::Tensor dropout(const at::Tensor &x, const c10::optional<at::Tensor> &residual, double p, int64_t scope,
                   const c10::optional<uint64_t> &seed, uint64_t offset) {
    no_tracing();
    if (x.dim() < 1 || x.dim() > 4) throw std::invalid_argument("input must have 1 to 4 axes");
    c10::OptionalDeviceGuard guard;
    if (x.is_cuda()) guard.reset_device(x.device());
    const at::Tensor r0 = residual.value_or(at::Tensor());
    no_forward_mode(x);
    no_forward_mode(r0);
    // dense in the order of its axes, else copied; channel decisions know two orders
    at::Tensor xi = x;
    const bool plain = x.is_contiguous();
    const bool last = x.dim() == 4 && x.is_contiguous(at::MemoryFormat::ChannelsLast);
    if (!plain && !last && (scope == GC_B200_DROP_CHANNEL || !x.is_non_overlapping_and_dense())) xi = x.contiguous();
    c10::optional<at::Tensor> r;
    if (r0.defined()) r = laid_out_like(r0, xi);
    const bool grad = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(r0));
    Drop drop = make_drop(x, p, scope, seed, offset, grad);
    const at::Tensor ri = r.value_or(at::Tensor());
    at::Tensor y = dropout_forward(xi, ri, drop);
    if (!grad) return y;
    auto node = std::shared_ptr<DropoutGrad>(new DropoutGrad(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(xi, ri));
    node->sizes_ = xi.sizes().vec();
    node->strides_ = xi.strides().vec();
    node->drop_ = drop;
    torch::autograd::set_history(y, node);
    return y;
}

}  // namespace

void bind_sequence_ops(pybind11::module_ &m);  // sequence_op.cpp

PYBIND11_MODULE(_gcb_torch, m) {
    m.doc() = "gc_cuda_conv for torch tensors: output allocation and the C ABI call in C++";
    m.def("conv", &conv, "y = gc_cuda_conv(x, w) on the current CUDA stream");
    m.def("conv_ex", &conv_ex, "y = act(conv(x, w) + bias) through gc_b200_conv_ex on the current CUDA stream");
    m.def("group_norm", &group_norm, "gc_b200_group_norm on the current CUDA stream, with its gradient");
    m.def("dropout", &dropout, "gc_b200_dropout on the current CUDA stream, with its gradient");
    bind_sequence_ops(m);
}
