"""gc_b200_group_norm and its gradient: channels-last group normalisation with
an activation and dropout in its epilogue, against the formulas in 64 bits."""
import ctypes as ct

import numpy as np
import pytest
import torch

from groupconv_atlas_b200 import api, torch_module
from tests.norm_helpers import (HALF, NormReference, assert_close, channels_last, keep_mask)

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}

# (dims, groups): one vector of channels and many, groups narrower and wider
# than a vector and straddling it, odd channel counts (one element at a time),
# single pixels, single elements, planes of one row, ranks 2 and 3, more
# channels than one block covers, planes over many chunks
SHAPES = [((1, 32, 7, 7), 8), ((2, 45, 5, 9), 9), ((3, 40, 11, 13), 4), ((2, 96, 1, 1), 1), ((1, 8, 1, 1), 8),
          ((5, 256, 9, 9), 32), ((2, 2056, 3, 3), 257), ((1, 1, 33, 17), 1), ((2, 64, 90, 70), 16), ((3, 24, 1, 50), 3),
          ((4, 48, 1000), 6), ((70, 64), 8), ((2, 16, 300, 2), 16), ((2, 30, 64, 65), 2), ((1, 512, 40, 3), 1),
          ((3, 7, 1), 7), ((1, 1040, 5, 6), 2), ((2, 128, 64, 64), 32),
          # more images than the GPU holds at once: a cluster takes several in turn
          ((600, 64, 4, 4), 4), ((900, 15, 5, 3), 5), ((1300, 24, 2, 2), 1), ((600, 64, 8, 8), 4), ((600, 63, 6, 6), 3)]

# Groups too large for shared memory, by vectors and by single elements.
SPLIT_SHAPES = [((1, 64, 300, 260), 1), ((2, 255, 100, 90), 1)]


def make(dims, dtype, seed=0, shift=0.5):
    g = torch.Generator().manual_seed(seed)
    c = dims[1]
    level = shift * torch.randn((1, c) + (1,) * (len(dims) - 2), generator=g)
    x = channels_last((torch.randn(dims, generator=g) * 1.5 + level).to(dtype))
    gamma = 1 + 0.3 * torch.randn(c, generator=g)
    beta = 0.3 * torch.randn(c, generator=g)
    dy = channels_last(torch.randn(dims, generator=g).to(dtype))
    return x, gamma, beta, dy


def space(nbytes):
    return torch.empty(nbytes, dtype=torch.uint8, device='cuda') if nbytes else None


def run_forward(native, x, groups, gamma, beta, eps=1e-5, act='none', drop=None, out=None):
    """The C ABI on the current stream: (y, stats), both filled with NaN before."""
    y = channels_last(torch.full(x.shape, float('nan'), dtype=x.dtype, device='cuda')) if out is None else out
    stats = torch.full((x.shape[0], groups, 2), float('nan'), device='cuda')
    ws = space(native.group_norm_workspace(x, y, groups))
    native.group_norm(x, y, groups, gamma, beta, eps, act, drop, stats, ws,
                      stream=torch.cuda.current_stream().cuda_stream)
    return y, stats


def run_backward(native, dy, x, stats, groups, gamma, beta, act='none', drop=None):
    dx = channels_last(torch.full(x.shape, float('nan'), dtype=x.dtype, device='cuda'))
    dgamma = torch.full_like(gamma, float('nan')) if gamma is not None else None
    dbeta = torch.full_like(beta, float('nan')) if beta is not None else None
    ws = space(native.group_norm_backward_workspace(dy, x, dx, groups))
    native.group_norm_backward(dy, x, stats, dx, groups, gamma, beta, dgamma, dbeta, act, drop, ws,
                               stream=torch.cuda.current_stream().cuda_stream)
    return dx, dgamma, dbeta


def check_step(native, x, gamma, beta, dy, groups, act, p=0.0, scope='element', seed=11, offset=5, eps=1e-5, label='',
               device_x=None, device_dy=None):
    """Forward and gradient through the C ABI against the 64-bit formulas."""
    keep, scale = (None, 1.0) if p == 0 else keep_mask(x.shape, p, seed, offset, scope)
    ref = NormReference(x, groups, gamma, beta, eps, act, keep, scale)
    dy = ref.away_from_kinks(dy)
    ref.backward(dy)
    drop = api.dropout_args(p, seed, offset, scope) if p else None
    put = lambda t: None if t is None else t.cuda()
    xd = put(x) if device_x is None else device_x
    if device_dy is None:
        dyd = put(dy)
    else:
        dyd = device_dy
        dyd.copy_(dy)
    gd, bd = put(gamma), put(beta)
    y, stats = run_forward(native, xd, groups, gd, bd, eps, act, drop)
    dx, dgamma, dbeta = run_backward(native, dyd, xd, stats, groups, gd, bd, act, drop)
    torch.cuda.synchronize()
    assert_close(y, ref.y, ref.tol_y, f'{label} y [{native.last_plan()}]')
    n = x.shape[0]
    kappa = ref.err.reshape(n, groups, -1)[..., 0]
    assert_close(stats[..., 0], ref.mean, kappa / ref.rstd, f'{label} mean')
    assert_close(stats[..., 1], ref.rstd, kappa * ref.rstd, f'{label} rstd')
    assert_close(dx, ref.dx, ref.tol_dx, f'{label} dx [{native.last_plan()}]')
    for name, got in (('dgamma', dgamma), ('dbeta', dbeta)):
        if got is not None:
            want, tol = getattr(ref, name), getattr(ref, 'tol_' + name)
            assert_close(got, want, tol + HALF[got.dtype] * want.abs() + 2.0 ** -25, f'{label} {name}')
    return y, stats, dx, dgamma, dbeta


@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups', SHAPES, ids=[f'{"x".join(map(str, d))}g{g}' for d, g in SHAPES])
@pytest.mark.parametrize('dtype', TYPES)
def test_forward_and_gradient(native, torch_cuda, dims, groups, dtype):
    x, gamma, beta, dy = make(dims, TYPES[dtype])
    check_step(native, x, gamma, beta, dy, groups, 'silu')


@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups', SPLIT_SHAPES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('p,scope,act', [(0.0, 'element', 'silu'), (0.25, 'element', 'none'), (0.25, 'channel', 'relu')])
def test_groups_that_are_read_twice(native, torch_cuda, dims, groups, dtype, p, scope, act):
    x, gamma, beta, dy = make(dims, TYPES[dtype], 20)
    check_step(native, x, gamma, beta, dy, groups, act, p, scope)
    assert 'split_backward' in native.last_plan()


# Many images of few pixels: one element a group, a vector's worth, none of
# these, as many as a warp holds, more groups than a block's threads.
SMALL_SHAPES = [((5000, 24, 2, 2), 3), ((3001, 40), 5), ((2003, 45, 3, 3), 5), ((30000, 8, 4, 5), 1), ((6000, 7), 7),
                ((1500, 600, 1), 300)]


@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups', SMALL_SHAPES, ids=[f'{"x".join(map(str, d))}g{g}' for d, g in SMALL_SHAPES])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('p,scope,act', [(0.0, 'element', 'silu'), (0.25, 'element', 'none'), (0.25, 'channel', 'relu6')])
def test_many_images_of_few_pixels(native, torch_cuda, dims, groups, dtype, p, scope, act):
    x, gamma, beta, dy = make(dims, TYPES[dtype], 22)
    check_step(native, x, gamma, beta, dy, groups, act, p, scope)
    assert 'small_backward' in native.last_plan()


@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups,path', [((600, 64, 8, 8), 4, 'resident'), ((900, 15, 5, 3), 5, ''),
                                              ((600, 63, 6, 6), 3, ''), ((600, 64, 4, 4), 4, '')])
@pytest.mark.parametrize('scope', ['element', 'channel'])
def test_dropout_of_many_images(native, torch_cuda, dims, groups, path, scope):
    x, gamma, beta, dy = make(dims, torch.bfloat16, 21)
    check_step(native, x, gamma, beta, dy, groups, 'silu', 0.5, scope)
    assert path in native.last_plan()


@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups', [((2, 40, 9, 11), 4), ((2, 45, 5, 9), 9)])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ['none', 'relu', 'relu6'])
def test_activations(native, torch_cuda, dims, groups, dtype, act):
    x, gamma, beta, dy = make(dims, TYPES[dtype], 1)
    check_step(native, x, 3 * gamma, beta, dy, groups, act)


@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups', [((2, 48, 9, 11), 6), ((3, 45, 5, 9), 5), ((4, 20, 30), 4), ((9, 64), 8)])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('scope', ['element', 'channel'])
@pytest.mark.parametrize('p', [0.25, 1.0])
def test_dropout_epilogue(native, torch_cuda, dims, groups, dtype, scope, p):
    x, gamma, beta, dy = make(dims, TYPES[dtype], 2)
    y, _, dx, _, _ = check_step(native, x, gamma, beta, dy, groups, 'silu', p, scope, seed=(3 << 40) + 7, offset=1 << 33)
    keep, _ = keep_mask(x.shape, p, (3 << 40) + 7, 1 << 33, scope)
    assert (y.cpu()[~keep] == 0).all()
    if p == 1.0:
        assert not y.any() and not dx.any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f16', 'bf16'])
def test_parameters_in_the_data_type_or_absent(native, torch_cuda, dtype):
    x, gamma, beta, dy = make((2, 64, 12, 10), TYPES[dtype], 3)
    check_step(native, x, gamma.to(x.dtype), beta.to(x.dtype), dy, 8, 'silu', label='both')
    check_step(native, x, None, None, dy, 8, 'silu', label='neither')
    check_step(native, x, gamma, None, dy, 8, 'none', label='gamma only')
    check_step(native, x, None, beta.to(x.dtype), dy, 8, 'relu', label='beta only')


@pytest.mark.gpu
@pytest.mark.parametrize('mean', [100.0, -4000.0])
@pytest.mark.parametrize('dims,groups', [((2, 32, 40, 40), 4), ((1, 45, 40, 40), 9), ((1, 16, 300, 200), 2)])
def test_a_mean_far_from_zero(native, torch_cuda, mean, dims, groups):
    """The variance comes from differences: sums of squares would lose it."""
    x, gamma, beta, dy = make(dims, torch.float32, 4)
    check_step(native, channels_last(x + mean), gamma, beta, dy, groups, 'none')


@pytest.mark.gpu
def test_an_outlier_in_first_place(native, torch_cuda):
    """The pivot of a run is its first value, here far from all others."""
    x, gamma, beta, dy = make((1, 32, 40, 40), torch.float32, 5)
    x[:, :, 0, 0] = 1e4
    check_step(native, x, gamma, beta, dy, 4, 'none')


@pytest.mark.gpu
def test_constant_groups_and_zero_eps(native, torch_cuda):
    x = channels_last(torch.full((2, 16, 5, 5), 3.25))
    y, stats = run_forward(native, x.cuda(), 4, None, None, 1e-5)
    assert not y.any() and (stats[..., 0] == 3.25).all()
    y, _ = run_forward(native, x.cuda(), 4, None, None, 0.0)
    assert torch.isnan(y).all()  # 0 * inf, as the formula says


@pytest.mark.gpu
@pytest.mark.parametrize('value', [float('nan'), float('inf'), float('-inf')])
@pytest.mark.parametrize('act', ['none', 'relu', 'relu6', 'silu'])
@pytest.mark.parametrize('c,groups', [(32, 4), (45, 9)])
def test_non_finite_values_stay_in_their_group(native, torch_cuda, value, act, c, groups):
    x, gamma, beta, _ = make((2, c, 6, 7), torch.float32, 6)
    clean, _ = run_forward(native, x.cuda(), groups, gamma.cuda(), beta.cuda(), act=act)
    bad = x.clone(memory_format=torch.preserve_format)
    bad[1, 0, 2, 3] = value
    y, _ = run_forward(native, bad.cuda(), groups, gamma.cuda(), beta.cuda(), act=act)
    cpg = c // groups
    assert torch.isnan(y[1, :cpg]).all()
    assert torch.equal(y[0], clean[0]) and torch.equal(y[1, cpg:], clean[1, cpg:])


@pytest.mark.gpu
def test_dropped_places_hide_non_finite_gradients(native, torch_cuda):
    x, gamma, beta, dy = make((1, 32, 8, 8), torch.float32, 7)
    keep, scale = keep_mask(x.shape, 0.5, 9, 1)
    ref = NormReference(x, 4, gamma, beta, act='silu', keep=keep, scale=scale).backward(dy)
    dy = torch.where(keep, dy, torch.tensor(float('inf')))
    drop = api.dropout_args(0.5, 9, 1)
    y, stats = run_forward(native, x.cuda(), 4, gamma.cuda(), beta.cuda(), act='silu', drop=drop)
    dx, dgamma, dbeta = run_backward(native, channels_last(dy).cuda(), x.cuda(), stats, 4, gamma.cuda(), beta.cuda(),
                                     'silu', drop)
    assert_close(dx, ref.dx, ref.tol_dx, 'dx')
    assert_close(dgamma, ref.dgamma, ref.tol_dgamma + HALF[torch.float32] * ref.dgamma.abs(), 'dgamma')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('start', [0, 16, 3])
def test_channel_slices_and_guarded_outputs(native, torch_cuda, dtype, start):
    """x and dy as channel slices of wider tensors (aligned and not), y as a
    slice of a buffer whose other channels stay as they were."""
    dt = TYPES[dtype]
    x, gamma, beta, dy = make((2, 48, 9, 7), dt, 8)
    wide_x = channels_last(torch.full((2, 80, 9, 7), 7.0, dtype=dt)).cuda()
    wide_dy = channels_last(torch.full((2, 80, 9, 7), 7.0, dtype=dt)).cuda()
    xs, dys = wide_x[:, start:start + 48], wide_dy[:, start:start + 48]
    xs.copy_(x)
    y0, *_ = check_step(native, x, gamma, beta, dy, 6, 'silu', device_x=xs, device_dy=dys)
    out = channels_last(torch.full((2, 80, 9, 7), 7.0, dtype=dt)).cuda()
    run_forward(native, xs, 6, gamma.cuda(), beta.cuda(), act='silu', out=out[:, start:start + 48])
    if start != 3:  # another path may round otherwise
        assert torch.equal(out[:, start:start + 48], y0)
    assert (out[:, :start] == 7).all() and (out[:, start + 48:] == 7).all()


@pytest.mark.gpu
def test_misaligned_base(native, torch_cuda):
    x, gamma, beta, dy = make((2, 32, 6, 6), torch.float32, 9)
    flat = torch.zeros(x.numel() + 1, device='cuda')
    xd = flat[1:].view(2, 6, 6, 32).permute(0, 3, 1, 2)
    xd.copy_(x)
    check_step(native, x, gamma, beta, dy, 4, 'silu', device_x=xd)


@pytest.mark.gpu
def test_results_are_reproducible_and_captured(native, torch_cuda):
    """Bitwise the same on repetition, on another stream and by graph replay."""
    x, gamma, beta, dy = (t.cuda() for t in make((3, 64, 40, 40), torch.bfloat16, 10))
    drop = api.dropout_args(0.2, 5, 6)

    def step():
        y, stats = run_forward(native, x, 8, gamma, beta, act='silu', drop=drop)
        return (y, *run_backward(native, dy, x, stats, 8, gamma, beta, 'silu', drop))

    first = step()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        second = step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
def test_offsets_past_32_bits(native, torch_cuda):
    """An image that starts more than 2^32 bytes and 2^31 elements into x: a
    batch view with a long image stride."""
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip('needs 16 GB of device memory')
    x, gamma, beta, dy = make((2, 32, 5, 5), torch.bfloat16, 11)
    stride = (1 << 31) + 1024
    base = torch.empty(stride + 32 * 25, dtype=torch.bfloat16, device='cuda')
    xd = base.as_strided((2, 32, 5, 5), (stride, 1, 160, 32))
    xd.copy_(x)
    check_step(native, x, gamma, beta, dy, 4, 'silu', device_x=xd)


@pytest.mark.gpu
def test_empty_batches_and_planes(native, torch_cuda):
    for dims in ((0, 16, 4, 4), (2, 16, 0, 4)):
        x = torch.empty(dims, device='cuda').to(memory_format=torch.channels_last).requires_grad_()
        w = torch.ones(16, device='cuda', requires_grad=True)
        y = torch_module.group_norm_act(x, 4, w, None, activation='silu')
        assert y.shape == x.shape
        dx, dw = torch.autograd.grad(y, [x, w], torch.empty_like(y))
        assert dx.shape == x.shape and not dw.any()


# ---- the torch front end ----------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_front_end_matches_the_c_abi(native, torch_cuda, dtype):
    x, gamma, beta, dy = (t.cuda() for t in make((2, 48, 10, 12), TYPES[dtype], 12))
    drop = api.dropout_args(0.3, 1 << 50, 77, 'channel')
    y, stats = run_forward(native, x, 6, gamma, beta, act='silu', drop=drop)
    grads = run_backward(native, dy, x, stats, 6, gamma, beta, 'silu', drop)
    leaves = [t.detach().requires_grad_() for t in (x, gamma, beta)]
    got = torch_module.group_norm_act(leaves[0], 6, leaves[1], leaves[2], activation='silu', dropout=0.3,
                                      scope='channel', seed=1 << 50, offset=77)
    assert got.is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(got, y)
    for a, b in zip(torch.autograd.grad(got, leaves, dy), grads):
        assert torch.equal(a, b)
    with torch.no_grad():
        again = torch_module.group_norm_act(*leaves[:1], 6, *leaves[1:], activation='silu', dropout=0.3,
                                            scope='channel', seed=1 << 50, offset=77)
    assert torch.equal(again, y)


@pytest.mark.gpu
def test_layouts_that_are_copied_first(native, torch_cuda):
    """Plain NCHW, transposed and expanded inputs, and gradients of any layout."""
    x, gamma, beta, dy = (t.cuda() for t in make((2, 24, 10, 12), torch.float32, 13))
    want = torch_module.group_norm_act(x, 4, gamma, beta, activation='silu')
    xr = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(torch_module.group_norm_act(xr, 4, gamma, beta, activation='silu'), xr, dy)
    for other in (x.contiguous(), x.transpose(2, 3).contiguous().transpose(2, 3),
                  channels_last(torch.cat([x, x], 2))[:, :, :10]):
        assert torch.equal(torch_module.group_norm_act(other, 4, gamma, beta, activation='silu'), want)
        leaf = other.detach().requires_grad_()
        out = torch_module.group_norm_act(leaf, 4, gamma, beta, activation='silu')
        assert torch.equal(torch.autograd.grad(out, leaf, dy.contiguous())[0], dx)
    row = x[:1].detach().requires_grad_()
    many = row.expand(5, -1, -1, -1)
    out = torch_module.group_norm_act(many, 4, gamma, beta)
    assert torch.equal(out[4], out[0])
    (drow,) = torch.autograd.grad(out.sum(0, keepdim=True), row, torch.ones_like(row))
    assert drow.shape == row.shape


@pytest.mark.gpu
def test_gradient_against_differences(native, torch_cuda):
    """(f(x + h v) - f(x - h v)) / 2h along a direction v, f = sum(w y) in 64
    bits from the FP32 result.  With |f|'s terms summed to F, the difference is
    good to F 2^-23 / 2h plus h^2 times the third derivative (of order F)."""
    x, gamma, beta, w = (t.cuda() for t in make((2, 32, 8, 8), torch.float32, 14))
    v = [channels_last(torch.randn(x.shape, generator=torch.Generator().manual_seed(1))).cuda(),
         torch.randn(32, generator=torch.Generator().manual_seed(2)).cuda(),
         torch.randn(32, generator=torch.Generator().manual_seed(3)).cuda()]
    leaves = [t.requires_grad_() for t in (x, gamma, beta)]
    f = lambda t: torch_module.group_norm_act(t[0], 4, t[1], t[2], activation='silu', dropout=0.2, seed=3, offset=4)
    grads = torch.autograd.grad(f(leaves), leaves, w)
    h = 2.0 ** -8
    for i in range(3):
        moved = [[t.detach() + s * h * v[i] if k == i else t.detach() for k, t in enumerate(leaves)] for s in (1, -1)]
        a, b = (f(m).double() * w.double() for m in moved)
        diff = ((a - b) / (2 * h)).sum()
        total = a.abs().sum()
        along = (grads[i].double() * v[i].double()).sum()
        assert abs(diff - along) <= total * (2.0 ** -23 / (2 * h) + 8 * h * h), (i, diff, along)


@pytest.mark.gpu
def test_generator_draws(native, torch_cuda):
    """Without a seed: torch's generator - reproducible, different from call to
    call, the gradient's mask the forward's; anew at each graph replay."""
    x = torch.ones((2, 32, 16, 16), device='cuda').to(memory_format=torch.channels_last)
    x = x + torch.randn_like(x)
    torch.manual_seed(5)
    f = lambda t: torch_module.group_norm_act(t, 4, dropout=0.5)
    a, b = f(x), f(x)
    torch.manual_seed(5)
    c = f(x)
    assert torch.equal(a, c) and not torch.equal(a, b)
    leaf = x.detach().requires_grad_()
    bias = torch.zeros(32, device='cuda', requires_grad=True)
    y = torch_module.group_norm_act(leaf, 4, None, bias, dropout=0.5)
    (db,) = torch.autograd.grad(y, bias, torch.ones_like(y))
    assert torch.equal(db, (y != 0).sum((0, 2, 3)) * 2.0)
    # captured: forward and gradient in one graph, new masks at each replay (on
    # leaves of its own: autograd refuses those that an eager graph holds)
    leaf, bias = x.detach().requires_grad_(), torch.zeros(32, device='cuda', requires_grad=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = torch_module.group_norm_act(leaf, 4, None, bias, dropout=0.5)
        (db,) = torch.autograd.grad(y, bias, torch.ones_like(y))
    masks = []
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        masks.append(y != 0)
        assert torch.equal(db, masks[-1].sum((0, 2, 3)) * 2.0)
    assert not torch.equal(*masks)


@pytest.mark.gpu
def test_probability_that_rounds_to_nothing(native, torch_cuda):
    x = make((2, 32, 6, 6), torch.float32, 16)[0].cuda()
    leaf = x.clone(memory_format=torch.preserve_format).requires_grad_()
    y = torch_module.group_norm_act(leaf, 4, dropout=1e-6)
    assert torch.equal(y, torch_module.group_norm_act(x, 4))
    assert torch.autograd.grad(y.sum(), leaf)[0].shape == x.shape


@pytest.mark.gpu
def test_expanded_gradients_and_strided_parameters(native, torch_cuda):
    x, gamma, beta, _ = (t.cuda() for t in make((2, 32, 6, 7), torch.float32, 17))
    leaf = x.requires_grad_()
    wide = torch.stack([gamma, gamma], 1)[:, 0].detach().requires_grad_()  # stride 2
    y = torch_module.group_norm_act(leaf, 4, wide, beta, activation='silu')
    dx, dw = torch.autograd.grad(y.sum(), [leaf, wide])
    z = torch_module.group_norm_act(leaf, 4, gamma.detach().requires_grad_(), beta, activation='silu')
    assert torch.equal(y, z)
    assert torch.equal(dx, torch.autograd.grad(z, leaf, torch.ones_like(z))[0]) and dw.shape == wide.shape


@pytest.mark.gpu
def test_changed_inputs_and_released_graphs_are_refused(native, torch_cuda):
    x = torch.randn((2, 8, 3, 3), device='cuda')
    leaf = x.clone().requires_grad_()
    mid = leaf * 1
    y = torch_module.group_norm_act(mid.to(memory_format=torch.channels_last).contiguous(memory_format=torch.channels_last), 2)
    torch.autograd.grad(y.sum(), leaf)
    with pytest.raises(RuntimeError, match='second time'):
        torch.autograd.grad(y.sum(), leaf)
    w = torch.ones(8, device='cuda', requires_grad=True)
    v = w * 1
    y = torch_module.group_norm_act(x, 2, v)
    v.add_(1)
    with pytest.raises(RuntimeError, match='inplace operation'):
        torch.autograd.grad(y.sum(), w)


@pytest.mark.gpu
def test_forward_mode_is_refused(native, torch_cuda):
    import torch.autograd.forward_ad as fwd
    x = torch.randn((2, 8, 3, 3), device='cuda', requires_grad=True)
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match='forward-mode'):
            torch_module.group_norm_act(fwd.make_dual(x, torch.ones_like(x)), 2)
        with pytest.raises(RuntimeError, match='forward-mode'):
            torch_module.dropout(fwd.make_dual(x, torch.ones_like(x)), 0.5)


FIRST_USE = """
import torch
from groupconv_atlas_b200 import torch_module
x = torch.randn(4, 64, 40, 40, device='cuda').to(memory_format=torch.channels_last)
w = torch.randn(4, 45, 30, 30, device='cuda').to(memory_format=torch.channels_last)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    a = [t.requires_grad_() for t in (x, w)]
    y = [torch_module.group_norm_act(a[0], 8, activation='silu', dropout=0.1),
         torch_module.group_norm_act(a[1], 9, activation='relu6'), torch_module.dropout(a[0], 0.2, scope='channel')]
    g = torch.autograd.grad(y, a, [torch.ones_like(t) for t in y])
graph.replay()
torch.cuda.synchronize()
assert all(bool(torch.isfinite(t).all()) for t in (*y, *g)) and bool(y[1].any())
"""


@pytest.mark.gpu
def test_first_use_inside_a_capture(native, torch_cuda):
    """Nothing that a first call sets up disturbs a capture."""
    import subprocess
    import sys
    done = subprocess.run([sys.executable, '-c', FIRST_USE], cwd=api.ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.gpu
def test_two_threads_and_streams(native, torch_cuda):
    """Calls of two host threads on streams of their own do not meet."""
    import threading
    inputs = [make((3, 64, 30, 30), torch.bfloat16, seed)[0].cuda() for seed in (18, 19)]
    want = [torch_module.group_norm_act(x, 8, activation='silu') for x in inputs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(50):
                got = torch_module.group_norm_act(inputs[i], 8, activation='silu')
                stream.synchronize()
                if not torch.equal(got, want[i]):
                    bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


@pytest.mark.gpu
def test_no_double_backward(native, torch_cuda):
    x = torch.randn((1, 8, 3, 3), device='cuda', requires_grad=True)
    y = torch_module.group_norm_act(x, 2)
    with pytest.raises(RuntimeError, match='not differentiable'):
        torch.autograd.grad(y.sum(), x, create_graph=True)


@pytest.mark.gpu
def test_another_device_than_the_current_one(native, torch_cuda):
    if torch.cuda.device_count() < 2:
        pytest.skip('needs two CUDA devices')
    x, gamma, beta, dy = (t.to('cuda:1') for t in make((2, 32, 6, 6), torch.float32, 15))
    torch.cuda.set_device(0)
    leaf = x.requires_grad_()
    y = torch_module.group_norm_act(leaf, 4, gamma, beta, activation='silu')
    (dx,) = torch.autograd.grad(y, leaf, dy)
    assert y.device == dx.device == x.device


# ---- modules ------------------------------------------------------------------------------------
def test_fuse_norm_act_replaces_and_keeps_names():
    nn = torch.nn
    model = nn.Sequential(nn.GroupNorm(2, 8), nn.SiLU(), nn.Dropout(0.1), nn.Conv2d(8, 8, 3),
                          nn.Sequential(nn.GroupNorm(4, 8), nn.ReLU6()), nn.GroupNorm(1, 8), nn.Tanh(),
                          nn.GroupNorm(8, 8), nn.Dropout2d(0.3), nn.SiLU())
    keys = list(model.state_dict())
    weight = model[0].weight
    assert torch_module.fuse_norm_act(model) == ['0', '5', '7', '4.0']
    assert list(model.state_dict()) == keys and model[0].weight is weight
    kinds = [(m.activation, m.p, m.scope) for m in (model[0], model[4][0], model[5], model[7])]
    assert kinds == [('silu', 0.1, 'element'), ('relu6', 0.0, 'element'), ('none', 0.0, 'element'),
                     ('none', 0.3, 'channel')]
    assert isinstance(model[6], nn.Tanh) and isinstance(model[9], nn.SiLU)  # a dropout before it stays in its order
    assert isinstance(model[1], nn.Identity) and isinstance(model[8], nn.Identity)
    with pytest.raises(ValueError):
        torch_module.B200GroupNormAct(nn.GroupNorm(2, 8), nn.Tanh())
    with pytest.raises(ValueError):
        torch_module.B200GroupNormAct(nn.GroupNorm(2, 8), nn.ReLU(), nn.AlphaDropout())


def residual_block(channels, groups, p):
    nn = torch.nn
    return nn.Sequential(nn.GroupNorm(groups, channels), nn.SiLU(), nn.Conv2d(channels, channels, 3, padding=1,
                                                                              groups=groups, bias=False),
                         nn.GroupNorm(groups, channels), nn.SiLU(), nn.Dropout(p),
                         nn.Conv2d(channels, channels, 3, padding=1, groups=groups, bias=False))


@pytest.mark.gpu
def test_residual_block_inference_with_this_library_s_convolutions(native, torch_cuda):
    """norm -> SiLU -> grouped 3x3 twice, channels last from end to end, every
    layer from this library, against the 64-bit model."""
    torch.manual_seed(3)
    block = residual_block(64, 16, 0.1).eval()
    x = torch.randn(2, 64, 20, 24, generator=torch.Generator().manual_seed(4))
    want = block.double()(x.double()) + x.double()
    block = block.float().cuda()
    assert torch_module.fuse_norm_act(block) == ['0', '3']
    for i in (2, 6):
        block[i] = torch_module.B200ConvBNAct(block[i], native=native)
    with torch.inference_mode():
        xd = x.cuda().to(memory_format=torch.channels_last)
        y = block(xd)
        assert y.is_contiguous(memory_format=torch.channels_last)
        y = torch_module.dropout(y, 0.0, residual=xd)
    # two convolutions of 36 products each behind two normalisations: a few
    # hundred roundings of values of order max|want|
    assert (y.cpu().double() - want).abs().max() <= 512 * 2.0 ** -24 * want.abs().max()


@pytest.mark.gpu
def test_residual_block_training_step(native, torch_cuda):
    """A training step of the fused block with dropout and the residual sum
    against the same step in 64 bits with the masks written out."""
    torch.manual_seed(6)
    block = residual_block(32, 8, 0.0).cuda()
    ref = residual_block(32, 8, 0.0).double()
    ref.load_state_dict({k: v.cpu().double() for k, v in block.state_dict().items()})
    x = channels_last(torch.randn(2, 32, 12, 10, generator=torch.Generator().manual_seed(7)))
    dy = channels_last(torch.randn(x.shape, generator=torch.Generator().manual_seed(8)))
    keep1, scale1 = keep_mask(x.shape, 0.2, 1, 2)
    keep2, scale2 = keep_mask(x.shape, 0.1, 3, 4, 'channel')

    xr = x.double().requires_grad_()
    h = ref[2](ref[1](ref[0](xr)))
    h = ref[4](ref[3](h)) * keep1.double() * scale1
    out = xr + ref[6](h) * keep2.double() * scale2
    names = [k for k, _ in ref.named_parameters()]
    want = torch.autograd.grad(out, [xr] + list(ref.parameters()), dy.double())

    xd = x.cuda().requires_grad_()
    old = torch.backends.cudnn.allow_tf32
    torch.backends.cudnn.allow_tf32 = False
    try:
        h = torch_module.group_norm_act(xd, 8, block[0].weight, block[0].bias, activation='silu')
        h = torch_module.group_norm_act(block[2](h), 8, block[3].weight, block[3].bias, activation='silu', dropout=0.2,
                                        seed=1, offset=2)
        got_out = torch_module.dropout(block[6](h), 0.1, residual=xd, scope='channel', seed=3, offset=4)
        got = torch.autograd.grad(got_out, [xd] + list(block.parameters()), dy.cuda())
    finally:
        torch.backends.cudnn.allow_tf32 = old
    # FP32 throughout, at most some 2000 roundings on the way of any value
    bound = lambda w: 2048 * 2.0 ** -24 * w.abs().max()
    assert (got_out.cpu().double() - out).abs().max() <= bound(out.detach())
    for name, a, b in zip(['x'] + names, got, want):
        assert (a.cpu().double() - b).abs().max() <= bound(b), name


# ---- refusals (no device needed: nothing is launched) ---------------------------------------------
def cpu_views(dims=(2, 8, 3, 3), dtype=api.GC_OK):
    """Descriptors of host memory marked as CUDA's: refused before any launch."""
    arrays = [np.zeros(dims, np.float32).transpose(0, 2, 3, 1).copy().transpose(0, 3, 1, 2) for _ in range(3)]
    descs = [api.view(a) for a in arrays]
    for d in descs:
        d.device = 1
    return arrays, descs


def call_norm(native, x, y, groups=2, eps=1e-5, act=0, gamma=None, beta=None, stats=None, drop=None):
    ref = lambda d: ct.byref(d) if d is not None else None
    return native.lib.gc_b200_group_norm(ref(x), ref(gamma), ref(beta), ref(y), ref(stats), groups, eps, act, ref(drop),
                                         None, 0, None)


def channel_vector(c, dtype=np.float32):
    a = np.ones(c, dtype)
    d = api.view(a)
    d.device = 1
    return a, d


def test_refusals_without_a_device(native):
    keepalive, (x, y, z) = cpu_views()
    bad = lambda d, **kw: [setattr(d, k, v) for k, v in kw.items()] and d
    copy = lambda d: type(d).from_buffer_copy(d)
    assert call_norm(native, None, y) == api.GC_INVALID
    assert call_norm(native, x, None) == api.GC_INVALID
    assert call_norm(native, bad(copy(x), rank=1), y) == api.GC_INVALID
    assert call_norm(native, bad(copy(x), rank=5), y) == api.GC_INVALID
    assert call_norm(native, bad(copy(x), device=0), y) == api.GC_INVALID
    assert call_norm(native, bad(copy(x), dtype=7), y) == api.GC_INVALID
    assert call_norm(native, x, bad(copy(y), dtype=api.B200_F16)) == api.GC_INVALID
    assert call_norm(native, x, bad(copy(y), device_index=1)) == api.GC_INVALID
    assert call_norm(native, bad(copy(x), data=None), y) == api.GC_INVALID
    assert call_norm(native, bad(copy(x), data=x.data + 2), y) == api.GC_INVALID
    assert call_norm(native, bad(copy(x), bytes=x.bytes - 4), y) == api.GC_INVALID
    assert call_norm(native, x, x) == api.GC_INVALID  # in place
    for groups in (0, -2, 3, 16):
        assert call_norm(native, x, y, groups=groups) == api.GC_INVALID
    for eps in (-1e-5, float('nan'), float('inf')):
        assert call_norm(native, x, y, eps=eps) == api.GC_INVALID
    for act in (-1, 4):
        assert call_norm(native, x, y, act=act) == api.GC_UNSUPPORTED
    for p in (-0.1, 1.1, float('nan')):
        assert call_norm(native, x, y, drop=api.dropout_args(p)) == api.GC_INVALID
    assert call_norm(native, x, y, drop=api.dropout_args(0.5, scope=2)) == api.GC_INVALID
    assert call_norm(native, x, y, drop=api.dropout_args(0.5, seed_ptr=64, used=64)) == api.GC_INVALID
    assert call_norm(native, x, y, drop=api.dropout_args(0.5, offset_ptr=72, used=64)) == api.GC_INVALID
    assert call_norm(native, x, y, drop=api.dropout_args(0.5, used=68)) == api.GC_INVALID
    for c, dtype in ((7, np.float32), (8, np.float64)):
        a, v = channel_vector(c, dtype)
        assert call_norm(native, x, y, gamma=v) == api.GC_INVALID
        assert call_norm(native, x, y, beta=v) == api.GC_INVALID
    a, v = channel_vector(16)
    v.dims[0], v.strides[0] = 8, 2
    assert call_norm(native, x, y, gamma=v) == api.GC_UNSUPPORTED
    stats = np.zeros((2, 2, 2), np.float32)
    s = api.view(stats)
    s.device = 1
    t = copy(s); t.dims[1] = 4
    assert call_norm(native, x, y, stats=t) == api.GC_INVALID
    t = copy(s); t.strides[0] = 8; t.bytes = 64
    assert call_norm(native, x, y, stats=t) == api.GC_UNSUPPORTED
    # layouts: plain NCHW, uneven pixels, images that interleave, FP64
    plain = np.zeros((2, 8, 3, 3), np.float32)
    nchw = api.view(plain)
    nchw.device = 1
    assert call_norm(native, nchw, y) == api.GC_UNSUPPORTED
    t = copy(x); t.strides[2] += 8; t.bytes = 4096
    assert call_norm(native, t, y) == api.GC_UNSUPPORTED
    t = copy(x); t.strides[0] = 8; t.bytes = 4096
    assert call_norm(native, t, y) == api.GC_UNSUPPORTED
    t = copy(x); t.strides[0] = 1 << 40
    assert call_norm(native, t, y) == api.GC_INVALID  # past the buffer
    wide = [copy(x), copy(y)]
    for d in wide:
        d.dtype = 1
    f64 = [np.zeros((2, 3, 3, 8)).transpose(0, 3, 1, 2) for _ in range(2)]
    wide = [api.view(a) for a in f64]
    for d in wide:
        d.device = 1
    assert call_norm(native, *wide) == api.GC_UNSUPPORTED
    t = copy(x); t.dims[0] = 1 << 60
    assert call_norm(native, t, y) == api.GC_INVALID
    # an empty batch is valid and needs no memory
    e = [copy(x), copy(y)]
    for d in e:
        d.dims[0], d.data = 0, None
    assert call_norm(native, *e) == api.GC_OK
    assert native.lib.gc_b200_group_norm_workspace(ct.byref(x), ct.byref(y), 2, None) == api.GC_INVALID


def test_front_end_refusals(native):
    x = torch.zeros(2, 8, 3, 3)
    with pytest.raises(api.NativeError) as err:
        torch_module.group_norm_act(x, 2)  # host memory
    assert err.value.status == api.GC_INVALID
    with pytest.raises(ValueError):
        torch_module.group_norm_act(x, 2, activation='tanh')
    with pytest.raises(ValueError):
        torch_module.group_norm_act(x, 2, dropout=0.5, scope='row')
    with pytest.raises(ValueError):
        torch_module.group_norm_act(torch.zeros(8), 2)
    with pytest.raises(TypeError):
        torch_module.group_norm_act(x, 2, dropout=0.5, seed=-1)
    with pytest.raises(ValueError):
        api.dropout_args(0.5, seed=1 << 64)


@pytest.mark.gpu
def test_device_refusals(native, torch_cuda):
    x = torch.randn((1, 8, 1000, 600), device='cuda').to(memory_format=torch.channels_last)
    y = torch.full_like(x, 7.0)
    need = native.group_norm_workspace(x, y, 2)
    assert need > 0
    for workspace in (None, space(need - 16), space(need + 16)[8:], torch.empty(need, dtype=torch.uint8).pin_memory()):
        with pytest.raises(api.NativeError) as err:
            native.group_norm(x, y, 2, workspace=workspace)
        assert err.value.status == api.GC_INVALID
    with pytest.raises(api.NativeError):
        native.group_norm(x, y, 2, workspace=x)
    with pytest.raises(api.NativeError):
        torch_module.group_norm_act(x, 2, torch.ones(8))  # parameters in host memory
    with pytest.raises(api.NativeError):
        torch_module.group_norm_act(x, 2, torch.ones(4, device='cuda'))
    with pytest.raises(api.NativeError) as err:
        torch_module.group_norm_act(x.double(), 2)
    assert err.value.status == api.GC_UNSUPPORTED
    torch.cuda.synchronize()
    assert (y == 7).all()
