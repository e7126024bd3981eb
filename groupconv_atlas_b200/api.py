"""ctypes binding of the B200 ``libgroupconv.so``, shaped like the reference's.

Mirrors the reference's ``bench/api.py:1-158`` interface - ``Shape``,
``CShape``, ``Tensor``, ``tensor()``, ``cshape()``, ``native_int()``,
``NativeError``, ``Native`` and ``inputs()`` - with the same names, argument
meaning and error behaviour, so callers written against the reference bind
this library unchanged.  ``Native`` additionally binds the ``gc_b200_*``
extensions (kernel-family selection, launch plan, device status word).

Buffers are borrowed: every native call takes raw pointers and sizes from
numpy arrays or torch tensors and never keeps them.  Nothing here computes a
convolution; the CUDA library does, and a missing library is an error.
"""
from __future__ import annotations

import ctypes as ct
import dataclasses
import hashlib
import json
import operator
import os
from pathlib import Path

import numpy as np

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
LIBRARY = PACKAGE / 'libgroupconv.so'
FIELDS = ('n', 'cin', 'cout', 'h', 'w', 'r', 's', 'groups', 'sh', 'sw', 'ph', 'pw', 'dh', 'dw')

# Status codes (include/groupconv.h, reference csrc/common/groupconv.h:10-11).
GC_OK, GC_INVALID, GC_UNSUPPORTED, GC_DEVICE_ERROR, GC_UNAVAILABLE = range(5)
# Kernel families of gc_b200_conv.
AUTO, GENERAL, DIRECT_LDG, DIRECT_TMA, TF32X3, SMALL = range(6)
KERNELS = {'auto': AUTO, 'general': GENERAL, 'direct_ldg': DIRECT_LDG,
           'direct_tma': DIRECT_TMA, 'tf32x3': TF32X3, 'small': SMALL}
# Layouts of gc_b200_conv_ex.
NCHW, NHWC = 0, 1
LAYOUTS = {'nchw': NCHW, 'nhwc': NHWC}
# Activations of gc_b200_conv_ex.
ACT_NONE, ACT_RELU, ACT_RELU6 = 0, 1, 2
ACTIVATIONS = {'none': ACT_NONE, 'relu': ACT_RELU, 'relu6': ACT_RELU6}
# Activations of gc_b200_group_norm.
ACT_SILU = 3
NORM_ACTIVATIONS = {**ACTIVATIONS, 'silu': ACT_SILU}
# 16-bit element types of gc_b200_group_norm and gc_b200_dropout.
B200_F16, B200_BF16 = 16, 17
# What one decision of gc_b200_dropout covers.
DROP_ELEMENT, DROP_CHANNEL = 0, 1
DROP_SCOPES = {'element': DROP_ELEMENT, 'channel': DROP_CHANNEL}
STATUS_TMA_TIMEOUT = 0x1
STATUS_MMA_TIMEOUT = 0x2


@dataclasses.dataclass(frozen=True)
class Shape:
    """Convolution geometry; defaults and id hash as reference bench/api.py:15-52."""
    n: int = 1
    cin: int = 16
    cout: int = 16
    h: int = 16
    w: int = 16
    r: int = 3
    s: int = 3
    groups: int = 1
    sh: int = 1
    sw: int = 1
    ph: int = 1
    pw: int = 1
    dh: int = 1
    dw: int = 1

    @property
    def output(self):
        return (self.n, self.cout,
                (self.h + 2 * self.ph - self.dh * (self.r - 1) - 1) // self.sh + 1,
                (self.w + 2 * self.pw - self.dw * (self.s - 1) - 1) // self.sw + 1)

    @property
    def input(self):
        return (self.n, self.cin, self.h, self.w)

    @property
    def weight(self):
        return (self.cout, self.cin // self.groups, self.r, self.s)

    @property
    def cpg(self):
        return self.cin // self.groups

    @property
    def b_geometry(self):
        """3x3, stride 1, pad 1, dilation 1, Cin == Cout: the engine's fast path."""
        return (self.cin == self.cout and self.r == self.s == 3 and self.sh == self.sw == 1
                and self.ph == self.pw == 1 and self.dh == self.dw == 1)

    @property
    def id(self):
        key = {**dataclasses.asdict(self), 'dtype': 'float32', 'layout': 'NCHW', 'bias': False}
        digest = hashlib.sha256(json.dumps(key, sort_keys=True, separators=(',', ':')).encode())
        return 'gc_' + digest.hexdigest()[:16]

    def record(self):
        return {**dataclasses.asdict(self), 'shape_id': self.id, 'input_dims': self.input,
                'weight_dims': self.weight, 'output_dims': self.output, 'dtype': 'float32',
                'layout': 'NCHW', 'bias': False}

    @classmethod
    def from_record(cls, value):
        return cls(**{k: value[k] for k in FIELDS})


class CShape(ct.Structure):
    _fields_ = [(field, ct.c_int64) for field in FIELDS]


class Tensor(ct.Structure):
    _fields_ = [('data', ct.c_void_p), ('bytes', ct.c_uint64), ('dtype', ct.c_int32),
                ('device', ct.c_int32), ('device_index', ct.c_int32), ('rank', ct.c_int32),
                ('dims', ct.c_int64 * 4), ('strides', ct.c_int64 * 4)]


def native_int(value, bits=32):
    """Integral value in signed `bits` range, else ValueError (reference api.py:62-67)."""
    try:
        value = operator.index(value)
    except TypeError as exc:
        raise ValueError('native integers must be integral') from exc
    if not -(1 << (bits - 1)) <= value < (1 << (bits - 1)):
        raise ValueError(f'integer outside signed {bits}-bit range')
    return value


def cshape(shape):
    return CShape(*[native_int(getattr(shape, k), 64) for k in FIELDS])


def tensor(array):
    """Borrowed descriptor of a numpy array or torch tensor (reference api.py:71-83)."""
    if isinstance(array, np.ndarray):
        dtype = {np.dtype('float32'): 0, np.dtype('float64'): 1}.get(array.dtype, -1)
        ptr, size = array.ctypes.data, array.nbytes
        shape, strides = array.shape, tuple(s // array.itemsize for s in array.strides)
        device, index = 0, 0
    else:
        dtype = {'torch.float32': 0, 'torch.float64': 1}.get(str(array.dtype), -1)
        ptr, size = array.data_ptr(), array.numel() * array.element_size()
        shape, strides = tuple(array.shape), tuple(array.stride())
        device, index = (1, array.device.index or 0) if array.device.type == 'cuda' else (0, 0)
        if array.device.type not in ('cpu', 'cuda'):
            device = -1
    dims = (ct.c_int64 * 4)(*shape)
    strd = (ct.c_int64 * 4)(*strides)
    return Tensor(ptr, size, dtype, device, index, len(shape), dims, strd)


def view(array):
    """Descriptor for the entry points that also take float16 and bfloat16
    torch tensors and strided views: ``bytes`` covers the view from its first
    to its last element (rank at most 4)."""
    desc = tensor(array)
    desc.dtype = {'torch.float16': B200_F16, 'torch.bfloat16': B200_BF16}.get(str(array.dtype), desc.dtype)
    if 0 not in tuple(array.shape):
        span = 1 + sum((n - 1) * desc.strides[i] for i, n in enumerate(array.shape))
        desc.bytes = span * array.element_size() if hasattr(array, 'element_size') else span * array.itemsize
    return desc


class DropoutArgs(ct.Structure):
    """gc_b200_dropout_args; the three addresses are device words or None."""
    _fields_ = [('p', ct.c_double), ('seed', ct.c_uint64), ('offset', ct.c_uint64), ('seed_ptr', ct.c_void_p),
                ('offset_ptr', ct.c_void_p), ('used', ct.c_void_p), ('scope', ct.c_int32)]


def dropout_args(p, seed=0, offset=0, scope='element', seed_ptr=None, offset_ptr=None, used=None):
    scope = DROP_SCOPES.get(scope, scope) if isinstance(scope, str) else scope
    for value in (seed, offset):
        if not 0 <= operator.index(value) < 1 << 64:
            raise ValueError('seed and offset are unsigned 64-bit integers')
    return DropoutArgs(p, seed, offset, seed_ptr, offset_ptr, used, native_int(scope))


class ScanArgs(ct.Structure):
    """gc_b200_scan_args."""
    _fields_ = [(k, ct.POINTER(Tensor)) for k in ('x', 'dt', 'a', 'b', 'c', 'd', 'z', 'dt_bias', 'state')] + [
        ('lengths', ct.c_void_p), ('softplus', ct.c_int32)]


class ScanGrads(ct.Structure):
    """gc_b200_scan_grads."""
    _fields_ = [(k, ct.POINTER(Tensor)) for k in ('x', 'dt', 'a', 'b', 'c', 'd', 'z', 'dt_bias', 'state')]


def _pointers(struct, arrays):
    """A structure of descriptor pointers; the descriptors live as long as it does."""
    struct.descs = {k: view(a) for k, a in arrays.items() if a is not None}
    for k, d in struct.descs.items():
        setattr(struct, k, ct.pointer(d))
    return struct


def length_words(lengths, n):
    """Address of the lengths of n sequences, or None.  The library takes an address
    alone, so the tensor is looked at here."""
    if lengths is None:
        return None
    if str(lengths.dtype) != 'torch.int32' or tuple(lengths.shape) != (n,) or not lengths.is_contiguous():
        raise ValueError(f'lengths must be {n} dense int32 words')
    return lengths.data_ptr()


def scan_args(x, dt, a, b, c, d=None, z=None, dt_bias=None, state=None, lengths=None, softplus=True):
    """Arguments of the selective scan's calls, from borrowed device tensors."""
    args = _pointers(ScanArgs(), dict(x=x, dt=dt, a=a, b=b, c=c, d=d, z=z, dt_bias=dt_bias, state=state))
    args.lengths = length_words(lengths, x.shape[0])
    args.softplus = 1 if softplus else 0
    return args


class NativeError(RuntimeError):
    def __init__(self, status, message):
        self.status = status
        super().__init__(message)


class Native:
    """Loads ``libgroupconv.so`` and binds every ABI symbol (reference api.py:90-126).

    The default library is the in-tree build next to this file;
    ``$GROUPCONV_LIBRARY`` overrides it as in the reference.
    """

    def __init__(self, path=None):
        if path is None:
            path = os.environ.get('GROUPCONV_LIBRARY') or (str(LIBRARY) if LIBRARY.exists() else '')
        if not path:
            raise FileNotFoundError(
                'libgroupconv.so is not built: run python -m groupconv_atlas_b200.build')
        self.path = str(Path(path).resolve())
        self.lib = ct.CDLL(self.path)
        lib = self.lib
        lib.gc_last_error.restype = ct.c_char_p
        lib.gc_build_info.restype = ct.c_char_p
        lib.gc_abi_version.restype = ct.c_int
        if lib.gc_abi_version() != 1:
            raise RuntimeError('native ABI version mismatch')
        lib.gc_validate_shape.argtypes = [ct.POINTER(CShape), ct.POINTER(ct.c_int64), ct.POINTER(ct.c_int64)]
        lib.gc_validate_tensors.argtypes = [ct.POINTER(CShape)] + [ct.POINTER(Tensor)] * 3 + [ct.c_int, ct.c_int]
        lib.gc_cpu_conv.argtypes = [ct.POINTER(CShape)] + [ct.POINTER(Tensor)] * 3 + [ct.c_int, ct.c_int]
        lib.gc_cuda_conv.argtypes = [ct.POINTER(CShape)] + [ct.POINTER(Tensor)] * 3 + [ct.c_int, ct.c_void_p]
        lib.gc_opencl_create.argtypes = [ct.POINTER(ct.c_void_p)]
        lib.gc_opencl_info.argtypes = [ct.c_void_p]
        lib.gc_opencl_info.restype = ct.c_char_p
        lib.gc_opencl_upload.argtypes = [ct.c_void_p, ct.POINTER(CShape)] + [ct.POINTER(Tensor)] * 3
        lib.gc_opencl_run.argtypes = [ct.c_void_p, ct.c_int, ct.c_int, ct.POINTER(ct.c_double)]
        lib.gc_opencl_download.argtypes = [ct.c_void_p, ct.POINTER(Tensor)]
        lib.gc_opencl_destroy.argtypes = [ct.c_void_p]
        lib.gc_opencl_destroy.restype = None
        # B200 extensions.
        lib.gc_b200_conv.argtypes = [ct.POINTER(CShape)] + [ct.POINTER(Tensor)] * 3 + [ct.c_int, ct.c_void_p]
        lib.gc_b200_last_plan.restype = ct.c_char_p
        lib.gc_b200_device_status.argtypes = [ct.POINTER(ct.c_uint32), ct.c_int]
        lib.gc_b200_selftest_wait_timeout.argtypes = [ct.c_uint32, ct.c_void_p]
        lib.gc_b200_conv_ex.argtypes = [ct.POINTER(CShape)] + [ct.POINTER(Tensor)] * 4 + [ct.c_int, ct.c_int,
                                                                                              ct.c_void_p]
        ptr = ct.POINTER(Tensor)
        lib.gc_b200_group_norm_workspace.argtypes = [ptr] * 2 + [ct.c_int64, ct.POINTER(ct.c_uint64)]
        lib.gc_b200_group_norm.argtypes = ([ptr] * 5 + [ct.c_int64, ct.c_double, ct.c_int, ct.POINTER(DropoutArgs),
                                                        ct.c_void_p, ct.c_uint64, ct.c_void_p])
        lib.gc_b200_group_norm_backward_workspace.argtypes = [ptr] * 3 + [ct.c_int64, ct.POINTER(ct.c_uint64)]
        lib.gc_b200_group_norm_backward.argtypes = ([ptr] * 8 + [ct.c_int64, ct.c_int, ct.POINTER(DropoutArgs),
                                                                 ct.c_void_p, ct.c_uint64, ct.c_void_p])
        lib.gc_b200_dropout.argtypes = [ptr] * 3 + [ct.POINTER(DropoutArgs), ct.c_void_p]
        lib.gc_b200_layer_norm.argtypes = [ptr] * 5 + [ct.c_double, ct.c_void_p]
        lib.gc_b200_layer_norm_backward_workspace.argtypes = [ptr] * 3 + [ct.POINTER(ct.c_uint64)]
        lib.gc_b200_layer_norm_backward.argtypes = [ptr] * 7 + [ct.c_void_p, ct.c_uint64, ct.c_void_p]
        lib.gc_b200_causal_conv.argtypes = [ptr] * 4 + [ct.c_void_p] + [ptr] * 2 + [ct.c_int, ct.c_void_p]
        lib.gc_b200_causal_conv_backward_workspace.argtypes = [ptr] * 4 + [ct.POINTER(ct.c_uint64)]
        lib.gc_b200_causal_conv_backward.argtypes = ([ptr] * 6 + [ct.c_void_p] + [ptr] * 4 + [ct.c_int, ct.c_void_p,
                                                                                             ct.c_uint64, ct.c_void_p])
        lib.gc_b200_causal_conv_step.argtypes = [ptr] * 6 + [ct.c_int, ct.c_void_p]
        scan = ct.POINTER(ScanArgs)
        lib.gc_b200_selective_scan_sizes.argtypes = [scan] + [ct.POINTER(ct.c_uint64)] * 3
        lib.gc_b200_selective_scan.argtypes = [scan] + [ptr] * 2 + [ct.c_void_p, ct.c_uint64] * 2 + [ct.c_void_p]
        lib.gc_b200_selective_scan_backward.argtypes = ([scan] + [ptr] * 2 + [ct.c_void_p, ct.c_uint64, ct.POINTER(ScanGrads),
                                                                             ct.c_void_p, ct.c_uint64, ct.c_void_p])
        lib.gc_b200_selective_scan_step.argtypes = [scan] + [ptr] * 2 + [ct.c_void_p]
        lib.gc_b200_autotune.argtypes = [ct.POINTER(CShape)] + [ct.POINTER(Tensor)] * 3 + [ct.c_int, ct.c_void_p]
        lib.gc_b200_probe_ffma.argtypes = [ct.c_void_p, ct.c_int, ct.c_int, ct.c_void_p]
        lib.gc_b200_probe_ffma_flops.argtypes = [ct.c_int, ct.c_int]
        lib.gc_b200_probe_ffma_flops.restype = ct.c_longlong
        lib.gc_b200_probe_tf32_mma.argtypes = [ct.c_void_p, ct.c_int, ct.c_int, ct.c_void_p]
        lib.gc_b200_probe_tf32_mma_flops.argtypes = [ct.c_int, ct.c_int]
        lib.gc_b200_probe_tf32_mma_flops.restype = ct.c_longlong
        lib.gc_b200_probe_copy.argtypes = [ct.c_void_p, ct.c_void_p, ct.c_uint64, ct.c_int, ct.c_void_p]

    def check(self, status):
        if status:
            raise NativeError(status, self.lib.gc_last_error().decode())

    def cpu(self, shape, x, w, y, impl=0, threads=1):
        p, xd, wd, yd = cshape(shape), tensor(x), tensor(w), tensor(y)
        self.check(self.lib.gc_cpu_conv(ct.byref(p), ct.byref(xd), ct.byref(wd), ct.byref(yd),
                                        native_int(impl), native_int(threads)))
        return y

    @staticmethod
    def _stream(stream):
        stream = operator.index(stream)
        if not 0 <= stream < (1 << (ct.sizeof(ct.c_void_p) * 8)):
            raise ValueError('stream pointer out of range')
        return stream

    def cuda(self, shape, x, w, y, impl=0, stream=0):
        """gc_cuda_conv on borrowed device tensors; asynchronous on `stream`."""
        p, xd, wd, yd = cshape(shape), tensor(x), tensor(w), tensor(y)
        stream = self._stream(stream)
        self.check(self.lib.gc_cuda_conv(ct.byref(p), ct.byref(xd), ct.byref(wd), ct.byref(yd),
                                         native_int(impl), stream))
        return y

    def b200(self, shape, x, w, y, kernel=AUTO, stream=0):
        """gc_b200_conv: run one named kernel family (see KERNELS)."""
        kernel = KERNELS.get(kernel, kernel) if isinstance(kernel, str) else kernel
        p, xd, wd, yd = cshape(shape), tensor(x), tensor(w), tensor(y)
        stream = self._stream(stream)
        self.check(self.lib.gc_b200_conv(ct.byref(p), ct.byref(xd), ct.byref(wd), ct.byref(yd),
                                         native_int(kernel), stream))
        return y

    def conv_ex(self, shape, x, w, y, bias=None, layout='nchw', activation='none', stream=0):
        """gc_b200_conv_ex: optional bias (rank-1, Cout), activation ('none',
        'relu', 'relu6') and layout 'nchw' or 'nhwc' (x and y channels-last,
        e.g. torch.channels_last tensors)."""
        lay = LAYOUTS.get(layout, layout) if isinstance(layout, str) else layout
        act = ACTIVATIONS.get(activation, activation) if isinstance(activation, str) else activation
        p, xd, wd, yd = cshape(shape), tensor(x), tensor(w), tensor(y)
        bd = tensor(bias) if bias is not None else None
        self.check(self.lib.gc_b200_conv_ex(ct.byref(p), ct.byref(xd), ct.byref(wd),
                                            ct.byref(bd) if bd is not None else None, ct.byref(yd),
                                            native_int(lay), native_int(act), self._stream(stream)))
        return y

    def autotune(self, shape, x, w, y, candidates=8, stream=0):
        """gc_b200_autotune: time the planner's best candidates on these
        buffers once (synchronizing) and cache the fastest plan."""
        p, xd, wd, yd = cshape(shape), tensor(x), tensor(w), tensor(y)
        self.check(self.lib.gc_b200_autotune(ct.byref(p), ct.byref(xd), ct.byref(wd), ct.byref(yd),
                                             native_int(candidates), self._stream(stream)))
        return y

    @staticmethod
    def _views(*arrays):
        """Descriptors of the arrays that are given, and pointers (or None) to pass."""
        descs = [view(a) if a is not None else None for a in arrays]
        return descs, [ct.byref(d) if d is not None else None for d in descs]

    @staticmethod
    def _space(workspace):
        return (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())

    def group_norm_workspace(self, x, y, groups):
        """Bytes of device memory that group_norm needs for these tensors."""
        size = ct.c_uint64(0)
        _, ptrs = self._views(x, y)
        self.check(self.lib.gc_b200_group_norm_workspace(*ptrs, native_int(groups, 64), ct.byref(size)))
        return size.value

    def group_norm(self, x, y, groups, gamma=None, beta=None, eps=1e-5, activation='none', dropout=None, stats=None,
                   workspace=None, stream=0):
        """gc_b200_group_norm on borrowed channels-last device tensors:
        activation 'none', 'relu', 'relu6' or 'silu'; dropout from
        dropout_args(); stats an FP32 (N, groups, 2) tensor for the gradient;
        workspace a device tensor of group_norm_workspace() bytes."""
        act = NORM_ACTIVATIONS.get(activation, activation) if isinstance(activation, str) else activation
        _, (xp, gp, bp, yp, sp) = self._views(x, gamma, beta, y, stats)
        self.check(self.lib.gc_b200_group_norm(xp, gp, bp, yp, sp, native_int(groups, 64), eps, native_int(act),
                                               ct.byref(dropout) if dropout is not None else None,
                                               *self._space(workspace), self._stream(stream)))
        return y

    def group_norm_backward_workspace(self, dy, x, dx, groups):
        """Bytes of device memory that group_norm_backward needs for these tensors."""
        size = ct.c_uint64(0)
        _, ptrs = self._views(dy, x, dx)
        self.check(self.lib.gc_b200_group_norm_backward_workspace(*ptrs, native_int(groups, 64), ct.byref(size)))
        return size.value

    def group_norm_backward(self, dy, x, stats, dx, groups, gamma=None, beta=None, dgamma=None, dbeta=None,
                            activation='none', dropout=None, workspace=None, stream=0):
        """gc_b200_group_norm_backward: gradients of group_norm from its x,
        gamma, beta, activation, dropout and stored stats."""
        act = NORM_ACTIVATIONS.get(activation, activation) if isinstance(activation, str) else activation
        _, ptrs = self._views(dy, x, gamma, beta, stats, dx, dgamma, dbeta)
        self.check(self.lib.gc_b200_group_norm_backward(*ptrs, native_int(groups, 64), native_int(act),
                                                        ct.byref(dropout) if dropout is not None else None,
                                                        *self._space(workspace), self._stream(stream)))
        return dx

    def dropout(self, x, y, dropout, residual=None, stream=0):
        """gc_b200_dropout: y = [residual +] dropout(x) with dropout_args()."""
        _, (xp, rp, yp) = self._views(x, residual, y)
        self.check(self.lib.gc_b200_dropout(xp, rp, yp, ct.byref(dropout) if dropout is not None else None,
                                            self._stream(stream)))
        return y

    def layer_norm(self, x, y, gamma=None, beta=None, eps=1e-5, stats=None, stream=0):
        """gc_b200_layer_norm of the last axis of borrowed device tensors; stats
        an FP32 (rows, 2) tensor for the gradient."""
        _, (xp, gp, bp, yp, sp) = self._views(x, gamma, beta, y, stats)
        self.check(self.lib.gc_b200_layer_norm(xp, gp, bp, yp, sp, eps, self._stream(stream)))
        return y

    def layer_norm_backward_workspace(self, dy, x, dx):
        """Bytes of device memory that layer_norm_backward needs for these tensors."""
        size = ct.c_uint64(0)
        _, ptrs = self._views(dy, x, dx)
        self.check(self.lib.gc_b200_layer_norm_backward_workspace(*ptrs, ct.byref(size)))
        return size.value

    def layer_norm_backward(self, dy, x, stats, dx, gamma=None, dgamma=None, dbeta=None, workspace=None, stream=0):
        """gc_b200_layer_norm_backward: gradients from layer_norm's x, gamma and stats."""
        _, ptrs = self._views(dy, x, gamma, stats, dx, dgamma, dbeta)
        self.check(self.lib.gc_b200_layer_norm_backward(*ptrs, *self._space(workspace), self._stream(stream)))
        return dx

    def causal_conv(self, x, weight, y, bias=None, state=None, lengths=None, state_out=None, activation='none', stream=0):
        """gc_b200_causal_conv on borrowed device tensors: x, y (N, L, C), weight
        (C, K), states (N, K - 1, C), lengths N int32 words."""
        act = NORM_ACTIVATIONS.get(activation, activation) if isinstance(activation, str) else activation
        _, (xp, wp, bp, sp, yp, op) = self._views(x, weight, bias, state, y, state_out)
        self.check(self.lib.gc_b200_causal_conv(xp, wp, bp, sp, length_words(lengths, x.shape[0]), yp, op, native_int(act),
                                                self._stream(stream)))
        return y

    def causal_conv_backward_workspace(self, dy, x, weight, dx):
        """Bytes of device memory that causal_conv_backward needs for these tensors."""
        size = ct.c_uint64(0)
        _, ptrs = self._views(dy, x, weight, dx)
        self.check(self.lib.gc_b200_causal_conv_backward_workspace(*ptrs, ct.byref(size)))
        return size.value

    def causal_conv_backward(self, dy, x, weight, dx, bias=None, state=None, dstate_out=None, lengths=None, dweight=None,
                             dbias=None, dstate=None, activation='none', workspace=None, stream=0):
        """gc_b200_causal_conv_backward: gradients from causal_conv's arguments."""
        act = NORM_ACTIVATIONS.get(activation, activation) if isinstance(activation, str) else activation
        _, p = self._views(dy, x, weight, bias, state, dstate_out, dx, dweight, dbias, dstate)
        self.check(self.lib.gc_b200_causal_conv_backward(*p[:6], length_words(lengths, x.shape[0]), *p[6:], native_int(act),
                                                         *self._space(workspace), self._stream(stream)))
        return dx

    def causal_conv_step(self, x, weight, state, y, bias=None, state_out=None, activation='none', stream=0):
        """gc_b200_causal_conv_step: x, y (N, C); the state in place without state_out."""
        act = NORM_ACTIVATIONS.get(activation, activation) if isinstance(activation, str) else activation
        _, ptrs = self._views(x, weight, bias, state, y, state if state_out is None else state_out)
        self.check(self.lib.gc_b200_causal_conv_step(*ptrs, native_int(act), self._stream(stream)))
        return y

    def selective_scan_sizes(self, args):
        """(workspace, kept, workspace of the gradient) in bytes, for scan_args()."""
        sizes = [ct.c_uint64(0) for _ in range(3)]
        self.check(self.lib.gc_b200_selective_scan_sizes(ct.byref(args), *(ct.byref(s) for s in sizes)))
        return tuple(s.value for s in sizes)

    def selective_scan(self, args, y, state_out=None, kept=None, workspace=None, stream=0):
        """gc_b200_selective_scan with scan_args(); kept and workspace are device
        tensors of selective_scan_sizes() bytes."""
        _, (yp, op) = self._views(y, state_out)
        self.check(self.lib.gc_b200_selective_scan(ct.byref(args), yp, op, *self._space(kept), *self._space(workspace),
                                                   self._stream(stream)))
        return y

    def selective_scan_backward(self, args, dy, kept, grads, dstate_out=None, workspace=None, stream=0):
        """gc_b200_selective_scan_backward; grads: a dict of tensors by the names
        of scan_args()."""
        _, (gp, op) = self._views(dy, dstate_out)
        out = _pointers(ScanGrads(), grads)
        self.check(self.lib.gc_b200_selective_scan_backward(ct.byref(args), gp, op, *self._space(kept), ct.byref(out),
                                                            *self._space(workspace), self._stream(stream)))
        return grads

    def selective_scan_step(self, args, y, state_out=None, stream=0):
        """gc_b200_selective_scan_step; the state of scan_args() in place without state_out."""
        descs, (yp, op) = self._views(y, state_out)
        if state_out is None:
            op = args.state
        self.check(self.lib.gc_b200_selective_scan_step(ct.byref(args), yp, op, self._stream(stream)))
        return y

    def last_plan(self):
        return self.lib.gc_b200_last_plan().decode()

    def device_status(self, clear=True):
        """Synchronizes the current device and returns (and clears) its status word."""
        value = ct.c_uint32(0)
        self.check(self.lib.gc_b200_device_status(ct.byref(value), 1 if clear else 0))
        return value.value

    def selftest_wait_timeout(self, limit_us, stream=0):
        self.check(self.lib.gc_b200_selftest_wait_timeout(native_int(limit_us, 33), self._stream(stream)))

    # Peak-rate probes: each launches one kernel into caller-owned device
    # buffers (torch tensors here) and returns the work it does.
    def probe_ffma(self, out, blocks, iters, stream=0):
        """FFMA chains; returns the FLOPs of the launch."""
        self.check(self.lib.gc_b200_probe_ffma(ct.c_void_p(out.data_ptr()), native_int(blocks),
                                               native_int(iters), self._stream(stream)))
        return self.lib.gc_b200_probe_ffma_flops(native_int(blocks), native_int(iters))

    def probe_tf32_mma(self, status, blocks, iters, stream=0):
        """Back-to-back tcgen05 TF32 MMAs; returns the FLOPs of the launch."""
        self.check(self.lib.gc_b200_probe_tf32_mma(ct.c_void_p(status.data_ptr()), native_int(blocks),
                                                   native_int(iters), self._stream(stream)))
        return self.lib.gc_b200_probe_tf32_mma_flops(native_int(blocks), native_int(iters))

    def probe_copy(self, src, dst, blocks, stream=0):
        """Device copy src -> dst; returns the bytes moved (read + write)."""
        nbytes = src.numel() * src.element_size()
        self.check(self.lib.gc_b200_probe_copy(ct.c_void_p(src.data_ptr()), ct.c_void_p(dst.data_ptr()),
                                               nbytes, native_int(blocks), self._stream(stream)))
        return 2 * nbytes


def inputs(shape, seed=20260908):
    """Seeded FP32 inputs exactly as reference bench/api.py:156-158."""
    rng = np.random.default_rng(seed ^ int(shape.id[3:11], 16))
    return (rng.uniform(-1, 1, shape.input).astype(np.float32),
            rng.uniform(-1, 1, shape.weight).astype(np.float32))
