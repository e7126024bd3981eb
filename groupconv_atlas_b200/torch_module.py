"""torch.nn front end: run a bias-free grouped Conv2d through gc_cuda_conv, or
a Conv2d -> BatchNorm2d -> ReLU/ReLU6 sequence through one gc_b200_conv_ex call.

Mirrors the reference's module substitution (``NativeDepthwise`` in
bench/module_run.py:215-230): the replacement keeps the convolution's weights,
allocates its output with torch, and calls the C ABI on the current stream.
The difference is the host path: a small C++ front end (torch_ext/conv_op.cpp,
built next to the library) allocates the output and calls the C ABI with no
Python in between, so a substituted layer costs about as much host time as a
cuDNN convolution and the block is competitive in synchronized (API) time, not
just in device time.  Without that front end the module falls back to ctypes
descriptors built once per input geometry (only their data pointers change per
call).  Both paths run the same CUDA kernels; outputs are computed on the GPU
only, and a missing library or an unsupported geometry raises NativeError.

Between convolutions: group_norm_act and B200GroupNormAct (GroupNorm ->
activation -> dropout as one gc_b200_group_norm call) and dropout and
B200Dropout (gc_b200_dropout), all with gradients through the C++ front end.
"""
from __future__ import annotations

import ctypes as ct

import torch

from . import api

def _cpp_conv():
    """The C++ front end's entry point (built next to the library by
    build.build_torch_ext), or None when it has not been built."""
    try:
        from . import _gcb_torch
    except ImportError:
        return None
    return _gcb_torch.conv


def _no_tracing():
    """A tracer would record the output's allocation alone (the C++ front end
    asks the same)."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError('this operation cannot be traced')


class B200Conv2d(torch.nn.Module):
    """Forward-only replacement of a bias-free ``torch.nn.Conv2d``."""

    def __init__(self, conv: torch.nn.Conv2d, native: api.Native | None = None, implementation: int = 3,
                 cpp: bool = True):
        super().__init__()
        if conv.bias is not None:
            raise ValueError('gc_cuda_conv has no bias term')
        if isinstance(conv.padding, str):
            raise ValueError('explicit integer padding required')
        self.native = native or api.Native()
        self.implementation = implementation
        self.register_buffer('weight', conv.weight.detach().contiguous().clone())
        self.geometry = dict(cin=conv.in_channels, cout=conv.out_channels, r=conv.kernel_size[0],
                             s=conv.kernel_size[1], groups=conv.groups, sh=conv.stride[0], sw=conv.stride[1],
                             ph=conv.padding[0], pw=conv.padding[1], dh=conv.dilation[0], dw=conv.dilation[1])
        self._cache = {}
        # The C++ front end allocates the output and calls gc_cuda_conv on the
        # current stream without Python in between (about 3 us less host time
        # per call than the ctypes path below, which serves when it is absent).
        self._op = _cpp_conv() if cpp else None
        g = self.geometry
        self._geo = (g['cout'], g['r'], g['s'], g['groups'], g['sh'], g['sw'], g['ph'], g['pw'], g['dh'], g['dw'])
        # gc_cuda_conv through a prototype taking plain addresses: the cached
        # descriptors are passed by address, which costs about half of what
        # ctypes' pointer-argument conversion does
        proto = ct.CFUNCTYPE(ct.c_int, ct.c_void_p, ct.c_void_p, ct.c_void_p, ct.c_void_p, ct.c_int, ct.c_void_p)
        self._fn = proto(ct.cast(self.native.lib.gc_cuda_conv, ct.c_void_p).value)
        # raw handle of the current stream; the public accessor builds a
        # Stream object per call, which costs more than the launch itself
        raw = getattr(torch._C, '_cuda_getCurrentRawStream', None)
        self._stream = (lambda dev: raw(dev)) if raw is not None else \
            (lambda dev: torch.cuda.current_stream(dev).cuda_stream)

    def _descriptors(self, x: torch.Tensor):
        """Per input geometry, device and dtype (input and weight): the
        convolution's Shape, its output size, the ctypes descriptors (only
        their data pointers change per call; their dtype and byte counts are
        part of the key) and their addresses."""
        key = (x.shape, x.get_device(), x.dtype, self.weight.dtype)
        entry = self._cache.get(key)
        if entry is None:
            shape = api.Shape(n=x.shape[0], h=x.shape[2], w=x.shape[3], **self.geometry)
            y = torch.empty(shape.output, device=x.device, dtype=x.dtype)
            descs = (api.cshape(shape), api.tensor(x), api.tensor(self.weight), api.tensor(y))
            entry = (shape, shape.output, descs, tuple(ct.addressof(d) for d in descs))
            self._cache[key] = entry
        return entry

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not x.is_contiguous():
            x = x.contiguous()
        if self._op is not None:
            try:
                return self._op(x, self.weight, *self._geo, self.implementation)
            except RuntimeError as e:
                text = str(e)
                if text.startswith('gc_status '):
                    status, _, message = text[len('gc_status '):].partition(': ')
                    raise api.NativeError(int(status), message) from None
                raise
        _no_tracing()
        if x.is_cuda and x.get_device() != torch.cuda.current_device():
            # gc_cuda_conv runs on the current device, which must hold the
            # tensors (nn.Conv2d runs on its input's device)
            with torch.cuda.device(x.device):
                return self.forward(x)
        _, out_shape, (_, xd, wd, yd), (pa, xa, wa, ya) = self._descriptors(x)
        y = x.new_empty(out_shape)
        xd.data = x.data_ptr()
        wd.data = self.weight.data_ptr()
        yd.data = y.data_ptr()
        status = self._fn(pa, xa, wa, ya, self.implementation, (self._stream(xd.device_index) if x.is_cuda else None))
        if status:
            self.native.check(status)
        return y


def _cpp_conv_ex():
    try:
        from . import _gcb_torch
    except ImportError:
        return None
    return getattr(_gcb_torch, 'conv_ex', None)


def _activation_name(act: torch.nn.Module | None) -> str:
    if act is None or isinstance(act, torch.nn.Identity):
        return 'none'
    if isinstance(act, torch.nn.ReLU6) or (isinstance(act, torch.nn.Hardtanh) and act.min_val == 0.0
                                           and act.max_val == 6.0):
        return 'relu6'
    if isinstance(act, torch.nn.ReLU):
        return 'relu'
    raise ValueError(f'activation {type(act).__name__} has no epilogue in gc_b200_conv_ex')


class B200ConvBNAct(torch.nn.Module):
    """Inference replacement of Conv2d -> BatchNorm2d -> ReLU/ReLU6 by ONE
    gc_b200_conv_ex call: the batch normalisation's running statistics are
    folded into the weights and a bias (w' = w * g / sqrt(var + eps),
    b' = beta + (b - mean) * g / sqrt(var + eps)) and the activation runs in
    the kernel's epilogue, so the three framework operations (three launches,
    three host paths) become one.  Eval mode only: the folded statistics are
    those at construction time."""

    def __init__(self, conv: torch.nn.Conv2d, bn: torch.nn.BatchNorm2d | None = None,
                 act: torch.nn.Module | None = None, native: api.Native | None = None):
        super().__init__()
        if isinstance(conv.padding, str):
            raise ValueError('explicit integer padding required')
        self.native = native or api.Native()
        w = conv.weight.detach().double()
        b = conv.bias.detach().double() if conv.bias is not None else torch.zeros(conv.out_channels,
                                                                                  dtype=torch.float64,
                                                                                  device=w.device)
        if bn is not None:
            scale = bn.weight.detach().double() / torch.sqrt(bn.running_var.detach().double() + bn.eps)
            w = w * scale[:, None, None, None]
            b = bn.bias.detach().double() + (b - bn.running_mean.detach().double()) * scale
        self.register_buffer('weight', w.float().contiguous())
        self.register_buffer('bias', b.float().contiguous())
        self.activation = _activation_name(act)
        self._act = api.ACTIVATIONS[self.activation]
        self.geometry = dict(cin=conv.in_channels, cout=conv.out_channels, r=conv.kernel_size[0],
                             s=conv.kernel_size[1], groups=conv.groups, sh=conv.stride[0], sw=conv.stride[1],
                             ph=conv.padding[0], pw=conv.padding[1], dh=conv.dilation[0], dw=conv.dilation[1])
        g = self.geometry
        self._geo = (g['cout'], g['r'], g['s'], g['groups'], g['sh'], g['sw'], g['ph'], g['pw'], g['dh'], g['dw'])
        self._op = _cpp_conv_ex()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        nhwc = x.is_contiguous(memory_format=torch.channels_last) and not x.is_contiguous()
        layout = api.NHWC if nhwc else api.NCHW
        if not nhwc and not x.is_contiguous():
            x = x.contiguous()
        if self._op is not None:
            try:
                return self._op(x, self.weight, self.bias, *self._geo, layout, self._act)
            except RuntimeError as e:
                text = str(e)
                if text.startswith('gc_status '):
                    status, _, message = text[len('gc_status '):].partition(': ')
                    raise api.NativeError(int(status), message) from None
                raise
        _no_tracing()
        shape = api.Shape(n=x.shape[0], h=x.shape[2], w=x.shape[3], **self.geometry)
        y = torch.empty(shape.output, device=x.device, dtype=x.dtype,
                        memory_format=torch.channels_last if nhwc else torch.contiguous_format)
        with torch.cuda.device(x.device):
            self.native.conv_ex(shape, x, self.weight, y, bias=self.bias, layout=layout, activation=self._act,
                                stream=torch.cuda.current_stream(x.device).cuda_stream)
        return y


def fuse_conv_bn_act(module: torch.nn.Module, predicate, native: api.Native | None = None) -> list[str]:
    """Replace every Sequential child whose first three members are Conv2d,
    BatchNorm2d and an activation (torchvision's Conv2dNormActivation, e.g.)
    and whose convolution satisfies predicate(conv) by one B200ConvBNAct;
    returns the dotted names replaced.  For inference (eval) models."""
    native = native or api.Native()
    replaced = []
    for name, child in list(module.named_modules()):
        for attr, sub in list(child._modules.items()):
            if not isinstance(sub, torch.nn.Sequential) or len(sub) < 2:
                continue
            conv, bn = sub[0], sub[1]
            act = sub[2] if len(sub) > 2 else None
            if not (isinstance(conv, torch.nn.Conv2d) and isinstance(bn, torch.nn.BatchNorm2d) and predicate(conv)):
                continue
            if len(sub) > 3:
                continue
            try:
                fused = B200ConvBNAct(conv, bn, act, native)
            except ValueError:
                continue
            child._modules[attr] = fused
            replaced.append(f'{name}.{attr}' if name else attr)
    return replaced


_ops = None


def _front_end():
    """The C++ front end, which these operators need: their gradients are
    recorded with autograd there."""
    global _ops
    if _ops is None:
        try:
            from . import _gcb_torch
        except ImportError as e:
            raise FileNotFoundError('the PyTorch front end is not built: '
                                    'groupconv_atlas_b200.build.build_torch_ext()') from e
        _ops = _gcb_torch
    return _ops


def _native_call(op, *args):
    try:
        return op(*args)
    except RuntimeError as e:
        text = str(e)
        if text.startswith('gc_status '):
            status, _, message = text[len('gc_status '):].partition(': ')
            raise api.NativeError(int(status), message) from None
        raise


def _scope_code(scope: str) -> int:
    code = api.DROP_SCOPES.get(scope)
    if code is None:
        raise ValueError(f"dropout scope must be one of {', '.join(api.DROP_SCOPES)}")
    return code


def group_norm_act(x: torch.Tensor, groups: int, weight: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, eps: float = 1e-5, activation: str = 'none',
                   dropout: float = 0.0, scope: str = 'element', seed: int | None = None,
                   offset: int = 0) -> torch.Tensor:
    """dropout(activation(group_norm(x))) as one gc_b200_group_norm call.

    x is (N, C), (N, C, L) or (N, C, H, W), float32, float16 or bfloat16, and is
    computed channels last: a channels_last tensor, or a channel slice of one,
    is read as it lies, anything else is copied first.  The result is dense and
    channels last.  weight and bias have C elements, float32 or x's type.
    activation is 'none', 'relu', 'relu6' or 'silu'.

    dropout is the probability of dropping, per 'element' or per 'channel' of
    an image (scope).  With a seed, the decisions are those of (seed, offset),
    see include/groupconv.h; without one they come from torch's CUDA generator,
    also inside a graph capture.  Differentiable once; the gradient draws the
    mask again, so none is stored."""
    act = api.NORM_ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(api.NORM_ACTIVATIONS)}")
    return _native_call((_ops or _front_end()).group_norm, x, weight, bias, groups, eps, act, dropout,
                        _scope_code(scope), seed, offset)


def dropout(x: torch.Tensor, p: float, residual: torch.Tensor | None = None, scope: str = 'element',
            seed: int | None = None, offset: int = 0) -> torch.Tensor:
    """[residual +] dropout(x) as one gc_b200_dropout call; x has one to four
    axes.  A decision goes by its element's place in memory (scope 'element')
    or by image and channel (scope 'channel'); a residual of other strides than
    x is copied first.  seed and offset as in group_norm_act."""
    return _native_call((_ops or _front_end()).dropout, x, residual, p, _scope_code(scope), seed, offset)


def _norm_activation_name(act: torch.nn.Module | None) -> str:
    return 'silu' if isinstance(act, torch.nn.SiLU) else _activation_name(act)


class B200GroupNormAct(torch.nn.Module):
    """GroupNorm -> activation -> dropout as one call, in training and
    inference.  Keeps the norm's own parameters (and their names) and the
    dropout (torch.nn.Dropout, or Dropout2d for whole channels) as its member
    ``drop``, whose own mode and probability decide."""

    def __init__(self, norm: torch.nn.GroupNorm, act: torch.nn.Module | None = None,
                 drop: torch.nn.Module | None = None):
        super().__init__()
        self.groups, self.eps = norm.num_groups, norm.eps
        self.weight, self.bias = norm.weight, norm.bias
        self.activation = _norm_activation_name(act)
        if drop is not None and not isinstance(drop, (torch.nn.Dropout, torch.nn.Dropout2d)):
            raise ValueError(f'{type(drop).__name__} has no epilogue in gc_b200_group_norm')
        self.drop = drop
        self.scope = 'channel' if isinstance(drop, torch.nn.Dropout2d) else 'element'
        self.training = norm.training

    @property
    def p(self) -> float:
        return 0.0 if self.drop is None else self.drop.p

    @p.setter
    def p(self, value: float) -> None:
        if self.drop is None:
            self.drop = torch.nn.Dropout().train(self.training)
        self.drop.p = value

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        drop = self.drop
        return group_norm_act(x, self.groups, self.weight, self.bias, self.eps, self.activation,
                              drop.p if drop is not None and drop.training else 0.0, self.scope)

    def extra_repr(self) -> str:
        return f'groups={self.groups}, eps={self.eps}, activation={self.activation}, p={self.p}, scope={self.scope}'


class B200Dropout(torch.nn.Module):
    """Dropout without a stored mask; forward(x, residual) also adds the
    residual, in evaluation too.  scope 'channel' drops whole channels."""

    def __init__(self, p: float = 0.5, scope: str = 'element'):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError('dropout probability must be between 0 and 1')
        _scope_code(scope)
        self.p, self.scope = p, scope

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return x if residual is None else residual + x
        return dropout(x, self.p, residual, self.scope)

    def extra_repr(self) -> str:
        return f'p={self.p}, scope={self.scope}'


def _plain(module: torch.nn.Module, kinds: tuple) -> bool:
    """One of these classes itself (a subclass may compute something else), and
    without hooks, which a fused call would not run."""
    return type(module) in kinds and not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks
                                          or module._backward_pre_hooks)


def fuse_norm_act(module: torch.nn.Module) -> list[str]:
    """In every Sequential, replace each GroupNorm with the activation (none,
    ReLU, ReLU6, SiLU) and the dropout (Dropout, Dropout2d) that follow it by
    one B200GroupNormAct; the members it takes over become Identity, so every
    other member keeps its name.  Subclasses of these, modules with hooks and
    Sequentials with a forward of their own, which may call their members in
    another order, stay as they are.  Returns the dotted names replaced.

    The replacement differs from torch's modules in three ways: it takes 2 to 4
    axes (a GroupNorm that sees (N, C, D, H, W) has to stay out of the fused
    module), its result is dense channels last, and of x's type, under autocast
    too, where torch's group_norm returns float32."""
    nn = torch.nn
    replaced = []
    for name, child in list(module.named_modules()):
        if not isinstance(child, nn.Sequential) or type(child).forward is not nn.Sequential.forward:
            continue
        members = list(child._modules.items())
        for at, (attr, norm) in enumerate(members):
            if not _plain(norm, (nn.GroupNorm,)):
                continue
            act = drop = None
            taken = []
            for follower, sub in members[at + 1:]:
                if drop is None and _plain(sub, (nn.Dropout, nn.Dropout2d)):
                    drop = sub
                elif drop is None and act is None and _plain(sub, (nn.ReLU, nn.ReLU6, nn.SiLU)):
                    act = sub
                else:
                    break
                taken.append(follower)
            child._modules[attr] = B200GroupNormAct(norm, act, drop)
            for follower in taken:
                child._modules[follower] = nn.Identity()
            replaced.append(f'{name}.{attr}' if name else attr)
    return replaced


def substitute(module: torch.nn.Module, predicate, native: api.Native | None = None) -> list[str]:
    """Replace every Conv2d child for which predicate(conv) is true; returns
    the dotted names replaced."""
    native = native or api.Native()
    replaced = []
    for name, child in list(module.named_modules()):
        for attr, sub in list(child._modules.items()):
            if isinstance(sub, torch.nn.Conv2d) and predicate(sub):
                child._modules[attr] = B200Conv2d(sub, native)
                replaced.append(f'{name}.{attr}' if name else attr)
    return replaced


def is_depthwise_3x3(conv: torch.nn.Conv2d) -> bool:
    return (conv.groups == conv.in_channels == conv.out_channels and conv.kernel_size == (3, 3)
            and conv.stride == (1, 1) and conv.padding == (1, 1) and conv.dilation == (1, 1)
            and conv.bias is None)


def is_depthwise(conv: torch.nn.Conv2d) -> bool:
    """Any depthwise convolution (groups == Cin == Cout), biased or not."""
    return conv.groups == conv.in_channels == conv.out_channels
