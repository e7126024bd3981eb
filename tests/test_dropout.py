"""gc_b200_dropout: a counter-based mask that is never stored, an optional
residual sum, and the gradient, against the definition in 64 bits."""
import ctypes as ct

import numpy as np
import pytest
import torch

from groupconv_atlas_b200 import api, torch_module
from tests.norm_helpers import HALF, TINY, U, assert_close, channels_last, keep_mask, philox

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}


def test_the_generator_is_philox():
    """Known answers of the published generator (Random123's kat_vectors):
    counter and key 0, all ones, and digits of pi."""
    words = lambda n, seed, offset: philox(8 * n, seed, offset).view('<u4').reshape(n, 4)[-1].tolist()
    assert words(1, 0, 0) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


def run(native, x, p, seed, offset, scope='element', residual=None, out=None, **words):
    y = torch.empty_like(x).fill_(float('nan')) if out is None else out
    native.dropout(x, y, api.dropout_args(p, seed, offset, scope, **words), residual,
                   torch.cuda.current_stream().cuda_stream)
    return y


def expected(x, p, seed, offset, scope, layout, residual=None):
    """(y, tolerance): one rounding of x * scale (and of the sum) in 32 bits,
    the scale's own, and the stored type's."""
    keep, scale = keep_mask(x.shape, p, seed, offset, scope, layout)
    v = torch.where(keep, x.double() * scale, torch.zeros((), dtype=torch.float64))
    y = v if residual is None else v + residual.double()
    return y, HALF[x.dtype] * y.abs() + TINY[x.dtype] + 3 * U * (v.abs() + y.abs()), keep


SHAPES = [(1,), (7,), (8,), (4099,), (3, 5), (1, 1, 1, 1), (2, 32, 7, 7), (3, 45, 5, 9), (2, 6, 1000), (5, 256, 9, 16),
          (1, 3, 301, 205)]


@pytest.mark.gpu
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: 'x'.join(map(str, s)))
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('layout', ['nchw', 'nhwc'])
@pytest.mark.parametrize('scope', ['element', 'channel'])
def test_values(native, torch_cuda, shape, dtype, layout, scope):
    if scope == 'channel' and len(shape) < 2:
        pytest.skip('no channel axis')
    g = torch.Generator().manual_seed(1)
    x = torch.randn(shape, generator=g).to(TYPES[dtype])
    r = torch.randn(shape, generator=g).to(TYPES[dtype])
    if layout == 'nhwc' and len(shape) > 1:
        x, r = channels_last(x), channels_last(r)
    order = layout if len(shape) > 1 else 'nchw'
    for p, residual in ((0.3, None), (0.3, r), (0.0, r), (1.0, r), (1.0, None)):
        want, tol, keep = expected(x, p, 2 ** 63 + 5, 2 ** 64 - 3, scope, order, residual)
        y = run(native, x.cuda(), p, 2 ** 63 + 5, 2 ** 64 - 3, scope, residual.cuda() if residual is not None else None)
        assert_close(y, want, tol, f'p={p} [{native.last_plan()}]')
        if residual is None:
            assert (y.cpu()[~keep] == 0).all() and not torch.signbit(y.cpu()[~keep]).any()


@pytest.mark.gpu
@pytest.mark.parametrize('p', [2.0 ** -18, 2.0 ** -16, 0.1, 0.5, 1 - 2.0 ** -16, 1 - 2.0 ** -18])
def test_probability_that_is_applied(native, torch_cuda, p):
    """The mask is the draws against round(65536 p), kept values scaled by what
    that probability leaves."""
    n = 1 << 18
    t = round(65536 * p)
    y = run(native, torch.ones(n, device='cuda'), p, 12, 34).cpu()
    keep = torch.from_numpy(philox(n, 12, 34) >= t)
    assert torch.equal(y != 0, keep if t < 65536 else torch.zeros(n, dtype=torch.bool))
    if keep.any() and t < 65536:
        assert abs(y[keep].double() - 65536 / (65536 - t)).max() <= U * 65536 / (65536 - t)


@pytest.mark.gpu
def test_masked_places_hide_infinities_and_nan(native, torch_cuda):
    keep, _ = keep_mask((4096,), 0.5, 1, 2, layout='nchw')
    x = torch.where(keep, torch.tensor(2.0), torch.tensor(float('nan')))
    x[~keep.clone() & (torch.arange(4096) % 2 == 0)] = float('inf')
    y = run(native, x.cuda(), 0.5, 1, 2).cpu()
    assert torch.equal(y, torch.where(keep, 4.0, 0.0))
    kept = torch.where(keep, torch.tensor(float('nan')), torch.tensor(1.0))
    assert torch.equal(torch.isnan(run(native, kept.cuda(), 0.5, 1, 2).cpu()), keep)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shift', [1, 2, 4])
def test_misaligned_views_and_guards(native, torch_cuda, dtype, shift):
    """Any element alignment; nothing outside the output is written."""
    n = 1003
    base = torch.randn(n + 16, generator=torch.Generator().manual_seed(3)).to(TYPES[dtype]).cuda()
    out = torch.full_like(base, 7.0)
    run(native, base[shift:shift + n], 0.4, 5, 6, out=out[shift:shift + n])
    want, tol, _ = expected(base[shift:shift + n].cpu(), 0.4, 5, 6, 'element', 'nchw')
    assert_close(out[shift:shift + n], want, tol)
    assert (out[:shift] == 7).all() and (out[shift + n:] == 7).all()


@pytest.mark.gpu
def test_device_words(native, torch_cuda):
    """Words added to seed and offset when the kernel runs; the pair in use
    written back; a captured call follows the words."""
    x = torch.randn(5000, generator=torch.Generator().manual_seed(4)).cuda()
    words = torch.tensor([11, 22], dtype=torch.int64, device='cuda')
    used = torch.zeros(2, dtype=torch.int64, device='cuda')
    at = dict(seed_ptr=words.data_ptr(), offset_ptr=words.data_ptr() + 8, used=used.data_ptr())
    y = run(native, x, 0.3, 100, 200, **at)
    assert torch.equal(y, run(native, x, 0.3, 111, 222)) and used.tolist() == [111, 222]
    back = dict(seed_ptr=used.data_ptr(), offset_ptr=used.data_ptr() + 8)
    assert torch.equal(run(native, x, 0.3, 0, 0, **back), y)
    out = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(native, x, 0.3, 100, 200, out=out, **at)
    for offset in (22, 23):
        words[1] = offset
        graph.replay()
        assert torch.equal(out, run(native, x, 0.3, 111, 200 + offset))


@pytest.mark.gpu
def test_places_past_32_bits(native, torch_cuda):
    """Counters above 2^32 elements (2^29 generator blocks): the last block of
    a tensor of 2^32 + 24 half-precision elements."""
    n = (1 << 32) + 24
    if torch.cuda.mem_get_info()[0] < 5 * n:
        pytest.skip('needs 20 GB of device memory')
    x = torch.ones(n, dtype=torch.bfloat16, device='cuda')
    y = torch.zeros_like(x)
    run(native, x, 0.5, 8, 9, out=y)
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    tail = y[-64:].cpu() != 0
    first = (n - 64) // 8
    c = [np.arange(first, first + 8, dtype=u) & low, np.arange(first, first + 8, dtype=u) >> u(32),
         np.full(8, 9, u), np.zeros(8, u)]
    for i in range(10):
        k0, k1 = u((8 + i * 0x9E3779B9) & 0xFFFFFFFF), u((i * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ k0, b & low, (a >> u(32)) ^ c[3] ^ k1, a & low]
    draws = np.stack(c, 1).astype('<u4').reshape(-1).view('<u2')
    assert torch.equal(tail, torch.from_numpy(draws >= 32768))
    assert abs(float((y[: 1 << 20] != 0).double().mean()) - 0.5) < 0.01


# Planes from a few elements to several vectors of a warp, images from one to
# thousands: each kernel of the channel decisions, with and without whole
# vectors, and places where a vector spans several planes.
CHANNEL_SHAPES = [(700, 24, 2, 2), (300, 20, 3, 5), (129, 64, 4, 4), (2000, 9, 1, 2), (513, 16), (37, 48, 11, 11),
                  (5, 48, 17, 31), (3, 45, 19, 29), (2, 1, 3, 7), (64, 3, 1, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize('shape', CHANNEL_SHAPES, ids=lambda s: 'x'.join(map(str, s)))
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('layout', ['nchw', 'nhwc'])
@pytest.mark.parametrize('shift', [0, 1])
def test_channel_decisions(native, torch_cuda, shape, dtype, layout, shift):
    g = torch.Generator().manual_seed(6)
    n = int(np.prod(shape))

    def place(t):  # behind `shift` elements of a guarded buffer
        b = torch.full((n + 16,), 7.0, dtype=TYPES[dtype], device='cuda')
        t = b[shift:shift + n].as_strided(t.shape, t.stride(), shift).copy_(t)
        return t, b

    x, r = (torch.randn(shape, generator=g).to(TYPES[dtype]) for _ in range(2))
    if layout == 'nhwc':
        x, r = channels_last(x), channels_last(r)
    for residual in (None, r):
        want, tol, keep = expected(x, 0.4, 3, 2 ** 40, 'channel', layout, residual)
        out, guard = place(torch.zeros_like(x))
        run(native, place(x)[0], 0.4, 3, 2 ** 40, 'channel', None if residual is None else place(residual)[0], out)
        assert_close(out, want, tol, native.last_plan())
        assert (guard[:shift] == 7).all() and (guard[shift + n:] == 7).all()
    pixels, size = n // shape[0] // shape[1], x.element_size()
    small = pixels * size < 512 if layout == 'nchw' else pixels * size * shape[1] <= 8192
    if shape[1] > 1:  # with one channel the two orders are one
        engine = 'element' if pixels == 1 else 'small_images' if small else 'planes' if layout == 'nchw' else 'channels_last'
        assert f'engine={engine} ' in native.last_plan()


def blocks_of_draws(first, count, seed, offset):
    """The draws of `count` generator blocks from block `first` on; seed and
    offset below 2^32."""
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    at = np.arange(first, first + count, dtype=u)
    c = [at & low, at >> u(32), np.full(count, offset, u), np.zeros(count, u)]
    for i in range(10):
        k0, k1 = u((seed + i * 0x9E3779B9) & 0xFFFFFFFF), u((i * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ k0, b & low, (a >> u(32)) ^ c[3] ^ k1, a & low]
    return torch.from_numpy(np.stack(c, 1).astype('<u4').reshape(-1).view('<u2').astype(np.int64))


def test_blocks_of_draws():
    assert torch.equal(blocks_of_draws(3, 4, 8, 9), torch.from_numpy(philox(56, 8, 9)[24:].astype(np.int64)))


@pytest.mark.gpu
@pytest.mark.parametrize('layout', ['nchw', 'nhwc'])
def test_small_images_past_32_bits(native, torch_cuda, layout):
    """Places above 2^32 of 2^28 + 2 images of 8 channels and 2 pixels."""
    n = (1 << 28) + 2
    if torch.cuda.mem_get_info()[0] < 5 * 16 * n:
        pytest.skip('needs 20 GB of device memory')
    x = torch.ones(16 * n, dtype=torch.bfloat16, device='cuda')
    x = x.view(n, 8, 1, 2) if layout == 'nchw' else x.view(n, 1, 2, 8).permute(0, 3, 1, 2)
    y = run(native, x, 0.5, 8, 9, 'channel')
    keep = (blocks_of_draws(n - 4, 4, 8, 9) >= 32768).view(4, 8, 1, 1).expand(4, 8, 1, 2)
    assert torch.equal(y[-4:].cpu() != 0, keep) and 'engine=small_images ' in native.last_plan()


# ---- the torch front end ----------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('scope', ['element', 'channel'])
def test_gradients(native, torch_cuda, dtype, scope):
    g = torch.Generator().manual_seed(6)
    x, r, dy = (channels_last(torch.randn((3, 20, 6, 7), generator=g).to(TYPES[dtype])) for _ in range(3))
    leaf, res = x.cuda().requires_grad_(), r.cuda().requires_grad_()
    y = torch_module.dropout(leaf, 0.4, res, scope, seed=5, offset=6)
    want, tol, _ = expected(x, 0.4, 5, 6, scope, 'nhwc', r)
    assert_close(y, want, tol, 'y')
    want, tol, _ = expected(dy, 0.4, 5, 6, scope, 'nhwc')
    for grad in (dy.cuda(), dy.contiguous().cuda()):  # a gradient that lies otherwise than x
        dx, dr = torch.autograd.grad(y, [leaf, res], grad, retain_graph=True)
        assert_close(dx, want, tol, 'dx')
        assert torch.equal(dr, grad)
    (dr,) = torch.autograd.grad(torch_module.dropout(x.cuda(), 0.4, res, scope, seed=5), res, dy.cuda())
    assert torch.equal(dr, dy.cuda())
    (dx,) = torch.autograd.grad(torch_module.dropout(leaf, 0.4, scope=scope, seed=5, offset=6), leaf, dy.cuda())
    assert_close(dx, want, tol, 'dx without a residual')


@pytest.mark.gpu
def test_layouts(native, torch_cuda):
    """Dense in any order of the axes: computed as it lies, gradient included;
    gaps and overlaps are copied first; a residual follows x."""
    x = torch.randn((4, 6, 5, 3), generator=torch.Generator().manual_seed(7)).cuda()
    for t in (x, x.to(memory_format=torch.channels_last), x.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0)):
        leaf = t.detach().requires_grad_()
        y = torch_module.dropout(leaf, 0.5, seed=1)
        assert y.stride() == t.stride()
        (dx,) = torch.autograd.grad(y, leaf, torch.ones_like(x))
        assert torch.equal(dx != 0, y != 0)
    sliced = x[:, ::2]
    assert torch.equal(torch_module.dropout(sliced, 0.5, seed=1), torch_module.dropout(sliced.contiguous(), 0.5, seed=1))
    leaf = x[:1].detach().requires_grad_()
    (dx,) = torch.autograd.grad(torch_module.dropout(leaf.expand(4, -1, -1, -1), 0.5, seed=1).sum(), leaf)
    assert dx.shape == leaf.shape
    last = x.to(memory_format=torch.channels_last)
    assert torch.equal(torch_module.dropout(last, 0.5, x, seed=1), torch_module.dropout(last, 0.5, last, seed=1))
    a = torch_module.dropout(x, 0.5, scope='channel', seed=1)
    assert torch.equal(a, torch_module.dropout(last, 0.5, scope='channel', seed=1))
    assert torch.equal(a, torch_module.dropout(x.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0), 0.5,
                                               scope='channel', seed=1))


@pytest.mark.gpu
def test_generator_and_module(native, torch_cuda):
    x = torch.ones((4, 16, 8, 8), device='cuda')
    drop = torch_module.B200Dropout(0.5)
    torch.manual_seed(1)
    a, b = drop(x), drop(x)
    torch.manual_seed(1)
    assert torch.equal(a, drop(x)) and not torch.equal(a, b)
    leaf = x.clone().requires_grad_()
    y = drop(leaf)
    assert torch.equal(torch.autograd.grad(y, leaf, torch.ones_like(y))[0], y.detach())
    leaf = x.clone().requires_grad_()  # autograd refuses a capture on leaves that an eager graph holds
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = drop(leaf)
        (dx,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    seen = []
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, y)
        seen.append(y.detach().clone())
    assert not torch.equal(*seen)
    channel = torch_module.B200Dropout(0.5, 'channel')(x)
    assert torch.equal(channel, channel[:, :, :1, :1].expand_as(channel))
    assert torch.equal(drop.eval()(x, x), 2 * x)


@pytest.mark.gpu
def test_empty_and_no_double_backward(native, torch_cuda):
    x = torch.empty((0, 4), device='cuda', requires_grad=True)
    y = torch_module.dropout(x, 0.5)
    assert y.shape == x.shape and torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    x = torch.ones(8, device='cuda', requires_grad=True)
    with pytest.raises(RuntimeError, match='not differentiable'):
        torch.autograd.grad(torch_module.dropout(x, 0.5).sum(), x, create_graph=True)


# ---- refusals (no device needed) ----------------------------------------------------------------
def test_refusals_without_a_device(native):
    arrays = [np.zeros((2, 3, 4, 5), np.float32) for _ in range(3)]
    x, r, y = (api.view(a) for a in arrays)
    for d in (x, r, y):
        d.device = 1
    copy = lambda d: type(d).from_buffer_copy(d)

    def call(x, y, residual=None, drop=api.dropout_args(0.5)):
        ref = lambda d: ct.byref(d) if d is not None else None
        return native.lib.gc_b200_dropout(ref(x), ref(residual), ref(y), ref(drop), None)

    assert call(None, y) == api.GC_INVALID and call(x, None) == api.GC_INVALID
    assert call(x, y, drop=None) == api.GC_INVALID
    assert call(x, x) == api.GC_INVALID and call(x, y, y) == api.GC_INVALID
    for field, value in (('device', 0), ('dtype', 9), ('rank', 0), ('rank', 5), ('device_index', 2), ('data', None),
                         ('bytes', 16), ('data', y.data + 1)):
        t = copy(y)
        setattr(t, field, value)
        assert call(x, t) == api.GC_INVALID, field
    t = copy(r)
    t.dims[3] = 4
    assert call(x, y, t) == api.GC_INVALID
    for p in (-1e-9, 1.0 + 1e-9, float('nan')):
        assert call(x, y, drop=api.dropout_args(p)) == api.GC_INVALID
    assert call(x, y, drop=api.dropout_args(0.5, scope=3)) == api.GC_INVALID
    t = copy(y)
    t.strides[0], t.strides[1] = 20, 40
    assert call(x, t) == api.GC_UNSUPPORTED  # other strides than x
    both = [copy(x), copy(y)]
    for d in both:
        d.strides[3], d.bytes = 2, 4096
    assert call(*both) == api.GC_UNSUPPORTED  # gaps
    both = [copy(x), copy(y)]
    for d in both:
        d.strides[0], d.strides[1], d.strides[2], d.strides[3] = 20, 40, 1, 4
    assert call(*both, drop=api.dropout_args(0.5, scope='channel')) == api.GC_UNSUPPORTED  # dense in a third order
    alive = [np.zeros(8, np.float32) for _ in range(2)]
    flat = [api.view(a) for a in alive]
    for d in flat:
        d.device = 1
    assert call(*flat, drop=api.dropout_args(0.5, scope='channel')) == api.GC_INVALID
    alive += [np.zeros((2, 3)) for _ in range(2)]
    f64 = [api.view(a) for a in alive[2:]]
    for d in f64:
        d.device = 1
    assert call(*f64) == api.GC_UNSUPPORTED
    empty = [copy(x), copy(y)]
    for d in empty:
        d.dims[2], d.data = 0, None
    assert call(*empty) == api.GC_OK
    with pytest.raises(api.NativeError):
        torch_module.dropout(torch.zeros(3), 0.5)
    with pytest.raises(ValueError):
        torch_module.B200Dropout(1.5)
    with pytest.raises(ValueError):
        torch_module.B200Dropout(0.5, 'row')
