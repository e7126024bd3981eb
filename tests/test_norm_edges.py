"""Group norm and dropout at the edges of their ranges: arguments far from zero,
several images a cluster, long sums, and calls that the front end refuses."""
import contextlib

import numpy as np
import pytest
import torch

from groupconv_atlas_b200 import api, torch_module
from tests.norm_helpers import HALF, K, TINY, U, NormReference, assert_close, keep_mask, philox
from tests.test_dropout import blocks_of_draws
from tests.test_group_norm import TYPES, check_step, make, run_backward, run_forward

# ---- arguments of SiLU far from zero --------------------------------------------------------------
# The resident path by vectors and by single elements, the small path, the split path.
FAR_SHAPES = [((2, 32, 6, 7), 4, 'resident'), ((2, 45, 5, 9), 9, 'resident'), ((5000, 24, 2, 2), 3, 'small'),
              ((1, 64, 300, 260), 1, 'split'), ((1, 255, 100, 90), 1, 'split')]
FAR = {0: -1e12, 3: -1e20, 5: -3e38, 6: 3e38, 9: 1e12, 10: -1e4, 12: 1e4}  # channel: beta


@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups,path', FAR_SHAPES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('params', ['f32', 'bf16'])
def test_silu_of_arguments_far_from_zero(native, torch_cuda, dims, groups, path, dtype, params):
    """Below -1e3 silu and its slope are 0 in every type, above 1e3 they are z
    and 1.  dx, dgamma and dbeta are therefore those of a beta of 40 in the high
    channels (where the slope differs from 1 by 2e-16) and of dy = 0 in the low
    ones."""
    if params == 'bf16' and dtype != 'bf16':
        pytest.skip('parameters are FP32 or of the data type')
    x, gamma, beta, dy = make(dims, TYPES[dtype], 30)
    gamma, beta = gamma.to(TYPES[params]), beta.to(TYPES[params])
    far = beta.clone()
    low, high = torch.zeros(dims[1], dtype=torch.bool), torch.zeros(dims[1], dtype=torch.bool)
    for c, value in FAR.items():
        far[c], beta[c] = value, 40.0 if value > 0 else 0.0
        (high if value > 0 else low)[c] = True
    dy[:, low] = 0
    ref = NormReference(x, groups, gamma, beta, 1e-5, 'silu').backward(dy)
    given = dy.clone(memory_format=torch.preserve_format)
    given[:, low] = 3.0  # what the slope has to hide
    y, stats = run_forward(native, x.cuda(), groups, gamma.cuda(), far.cuda(), act='silu')
    assert f'engine={path} ' in native.last_plan()
    dx, dgamma, dbeta = run_backward(native, given.cuda(), x.cuda(), stats, groups, gamma.cuda(), far.cuda(), 'silu')
    y, rest = y.cpu(), ~(low | high)
    assert (y[:, low] == 0).all()
    assert_close(y[:, rest], ref.y[:, rest], ref.tol_y[:, rest], 'y')
    for c in torch.nonzero(high).flatten().tolist():
        want = ref.xhat[:, c] * ref.gamma[:, c] + far[c].double()
        if x.dtype == torch.float16 and far[c] > 1e5:
            assert (y[:, c] == float('inf')).all()  # past the type's range
        else:
            tol = (HALF[x.dtype] + 16 * U) * want.abs() + ref.err[:, c] * ref.gamma[:, c].abs() * (ref.xhat[:, c].abs() + 1)
            assert_close(y[:, c], want, tol, f'y at {float(far[c])}')
    assert_close(dx, ref.dx, ref.tol_dx, f'dx [{native.last_plan()}]')
    for name, got in (('dgamma', dgamma), ('dbeta', dbeta)):
        want = getattr(ref, name)
        assert_close(got, want, getattr(ref, 'tol_' + name) + HALF[got.dtype] * want.abs() + 2.0 ** -25, name)


@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups,path', FAR_SHAPES)
@pytest.mark.parametrize('dtype', TYPES)
def test_silu_and_its_slope_over_the_whole_range(native, torch_cuda, dims, groups, path, dtype):
    """With gamma = 0, z is beta and dbeta the slope times the sum of dy (1 here).
    The exponential is off by 2 |z| u (the product with log2 e and that
    constant) and 4 u, the sum, product, reciprocal and products behind it by
    another 8 u: (2 |z| + 12) u of s and of 1 - s.  The sigmoid below 2^-126 is 0."""
    c, count = dims[1], int(np.prod(dims)) // dims[1]
    x = make(dims, TYPES[dtype], 31)[0].cuda()
    beta = torch.linspace(-110, 110, c)
    gamma = torch.zeros(c)
    y, stats = run_forward(native, x, groups, gamma.cuda(), beta.cuda(), act='silu')
    _, _, dbeta = run_backward(native, torch.ones_like(x), x, stats, groups, gamma.cuda(), beta.cuda(), 'silu')
    z = beta.double()
    s, t = torch.sigmoid(z), torch.sigmoid(-z)
    e = (2 * z.abs() + 12) * U
    tiny = 128 * 2.0 ** -126
    shape = (1, c) + (1,) * (len(dims) - 2)
    want = z * s
    tol = (e + HALF[x.dtype]) * want.abs() + tiny + TINY[x.dtype]
    assert_close(y, want.reshape(shape), tol.reshape(shape), 'y')
    slope = s * (1 + z * t)
    tol = s * (1 + 2 * z.abs() * t) * e + K * U * slope.abs() + tiny
    assert_close(dbeta / count, slope, tol + U * slope.abs(), 'dbeta')


@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups', [((2, 32, 6, 7), 4), ((2, 45, 5, 9), 9), ((5000, 24, 2, 2), 3)])
def test_silu_of_infinities(native, torch_cuda, dims, groups):
    """v / (1 + exp(-v)) is NaN at -inf and inf at inf; other channels are untouched."""
    x, gamma, beta, _ = make(dims, torch.float32, 32)
    ref = NormReference(x, groups, gamma, beta, act='silu')
    beta[1], beta[4] = float('-inf'), float('inf')
    y = run_forward(native, x.cuda(), groups, gamma.cuda(), beta.cuda(), act='silu')[0].cpu()
    assert torch.isnan(y[:, 1]).all() and (y[:, 4] == float('inf')).all()
    rest = [c for c in range(dims[1]) if c not in (1, 4)]
    assert_close(y[:, rest], ref.y[:, rest], ref.tol_y[:, rest], 'y')


@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups,path', [((4, 32, 6, 7), 4, 'resident'), ((4, 45, 5, 9), 9, 'resident'),
                                              ((5000, 24, 2, 2), 3, 'small'), ((2, 64, 300, 260), 1, 'split')])
@pytest.mark.parametrize('act', ['silu', 'none', 'relu'])
def test_dropped_channels_hide_infinite_arguments(native, torch_cuda, dims, groups, path, act):
    """dz is 0 where a place is dropped, whatever the slope there is (NaN for SiLU
    at an infinity): an image whose infinite channels are all dropped has the
    gradient that it has without them."""
    x, gamma, beta, dy = make(dims, torch.float32, 37)
    seed = 0
    while True:  # an image with both channels dropped
        keep, scale = keep_mask(x.shape, 0.5, seed, 3, 'channel')
        kept = keep[:, :, 0, 0]
        clean = ~kept[:, 2] & ~kept[:, 7]
        if clean.any():
            break
        seed += 1
    ref = NormReference(x, groups, gamma, beta, act=act, keep=keep, scale=scale)
    dy = ref.away_from_kinks(dy)
    ref.backward(dy)
    beta[2], beta[7] = float('-inf'), float('inf')
    drop = api.dropout_args(0.5, seed, 3, 'channel')
    y, stats = run_forward(native, x.cuda(), groups, gamma.cuda(), beta.cuda(), act=act, drop=drop)
    dx, _, _ = run_backward(native, dy.cuda(), x.cuda(), stats, groups, gamma.cuda(), beta.cuda(), act, drop)
    assert f'engine={path}_backward ' in native.last_plan()
    assert_close(y.cpu()[clean], ref.y[clean], ref.tol_y[clean], 'y')
    assert_close(dx.cpu()[clean], ref.dx[clean], ref.tol_dx[clean], 'dx')
    drop = api.dropout_args(1.0, seed, 3)
    y, stats = run_forward(native, x.cuda(), groups, gamma.cuda(), beta.cuda(), act=act, drop=drop)
    for t in (y, *run_backward(native, dy.cuda(), x.cuda(), stats, groups, gamma.cuda(), beta.cuda(), act, drop)):
        assert (t == 0).all()


# ---- clusters that take several images in turn ----------------------------------------------------
# (dims, groups, type, cluster of the forward pass or None where it takes one
# image, cluster of the gradient or None): 16-byte vectors and single elements
# (of 16 bits: copied through registers), clusters of one and of several.
ROUNDS = [((600, 64, 9, 9), 4, 'f32', None, 1), ((600, 96, 12, 11), 1, 'f32', 1, 2), ((600, 96, 12, 11), 1, 'bf16', None, 1),
          ((200, 64, 20, 21), 1, 'f32', None, 4), ((40, 96, 40, 40), 1, 'f32', 8, None),
          ((600, 96, 16, 16), 1, 'bf16', 1, 2), ((150, 64, 40, 40), 4, 'f16', 4, None),
          ((4000, 15, 5, 7), 1, 'f32', None, 1), ((4000, 15, 5, 7), 1, 'f16', None, 1), ((600, 255, 2, 3), 1, 'f32', 1, None),
          ((600, 255, 2, 3), 1, 'bf16', 1, None), ((150, 130, 9, 9), 2, 'f16', 1, None), ((600, 15, 28, 28), 1, 'f32', 4, None)]


def rounds_of(plan):
    """(engine, cluster, images that a cluster takes in turn)"""
    fields = dict(f.split('=') for f in plan.split())
    return fields['engine'], int(fields['cluster']), int(fields['rounds'])


@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups,dtype,forward,backward', ROUNDS)
@pytest.mark.parametrize('p,scope', [(0.0, 'element'), (0.25, 'element'), (0.25, 'channel')])
def test_clusters_that_take_several_images(native, torch_cuda, dims, groups, dtype, forward, backward, p, scope):
    """The tiles filled again during the second pass, exchange buffers in turn,
    statistics loaded for each image, parameter gradients added over images."""
    if p and dims[0] * dims[1] * dims[2] * dims[3] > 1 << 23:
        pytest.skip('the smaller shapes cover dropout')
    x, gamma, beta, dy = make(dims, TYPES[dtype], 33)
    run_forward(native, x.cuda(), groups, gamma.cuda(), beta.cuda(), act='silu', drop=api.dropout_args(p) if p else None)
    engine, cluster, rounds = rounds_of(native.last_plan())
    if forward is not None:
        assert engine == 'resident' and cluster == forward and rounds >= 2
    check_step(native, x, gamma, beta, dy, groups, 'silu', p, scope)
    engine, cluster, rounds = rounds_of(native.last_plan())
    if backward is not None:
        assert engine == 'resident_backward' and cluster == backward and rounds >= 2


# ---- long sums of one sign ------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('dims', [(593, 255, 45, 41), (297, 1024, 45, 40)], ids=['elements', 'vectors'])
def test_gradient_sums_over_long_chunks(native, torch_cuda, dims):
    """One chunk an image and one pixel lane a block: a thread adds 1800 products
    for each of its channels.  Added one after the other, these (of the value
    that a search found worst) are off by 450 half steps."""
    n, c, h, w = dims
    if torch.cuda.mem_get_info()[0] < 24 * n * c * h * w:
        pytest.skip('needs 14 GB of device memory')
    value = float.fromhex('0x1.171c02p0')
    g = torch.Generator(device='cuda').manual_seed(35)
    level = 2 * torch.randn(c, generator=g, device='cuda')
    x = (torch.randn((n, h, w, c), generator=g, device='cuda') + level).permute(0, 3, 1, 2)
    dy = torch.full((n, h, w, c), value, device='cuda').permute(0, 3, 1, 2)
    gamma, beta = torch.ones(c, device='cuda'), torch.zeros(c, device='cuda')
    _, stats = run_forward(native, x, 1, gamma, beta)
    dx, dgamma, dbeta = run_backward(native, dy, x, stats, 1, gamma, beta)
    assert 'engine=split_backward ' in native.last_plan()
    total = n * h * w
    assert_close(dbeta, torch.full((c,), total * value, dtype=torch.float64), torch.tensor((K + 1) * U * total * value))
    want = torch.zeros(c, dtype=torch.float64, device='cuda')
    tol = torch.zeros_like(want)
    for i in range(0, n, 27):
        part = x[i:i + 27].double()
        sigma, mean = (part.var((1, 2, 3), correction=0, keepdim=True) + 1e-5).sqrt(), part.mean((1, 2, 3), keepdim=True)
        xhat = (part - mean) / sigma
        err = K * U * (1 + part.abs().amax((1, 2, 3), keepdim=True) / sigma)  # as in norm_helpers
        want += value * xhat.sum((0, 2, 3))
        tol += value * (err * (xhat.abs() + 1) + K * U * xhat.abs()).sum((0, 2, 3))
    assert_close(dgamma, want.cpu(), (tol + U * want.abs()).cpu())


@pytest.mark.gpu
def test_gradient_sums_over_many_images(native, torch_cuda):
    """Rows of one channel, 1200 in turn for each thread of a wave of blocks, 256
    threads a block, 1184 blocks: sums that were added one after the other at
    each of the three levels."""
    n = 1200 * 256 * 1184
    if torch.cuda.mem_get_info()[0] < 24 * n:
        pytest.skip('needs 9 GB of device memory')
    value = float.fromhex('0x1.d114p0')
    x = torch.randn((n, 1), generator=torch.Generator(device='cuda').manual_seed(36), device='cuda')
    dy = torch.full((n, 1), value, device='cuda')
    gamma, beta = torch.ones(1, device='cuda'), torch.zeros(1, device='cuda')
    _, stats = run_forward(native, x, 1, gamma, beta)
    _, _, dbeta = run_backward(native, dy, x, stats, 1, gamma, beta)
    assert 'engine=small_backward ' in native.last_plan()
    assert_close(dbeta, torch.full((1,), n * value, dtype=torch.float64), torch.tensor(72 * U * n * value))


# ---- more than 2^32 elements ----------------------------------------------------------------------
def large(dims):
    """Random bf16 tensors of more than 2^32 elements, channels last: x, dy = 1."""
    count = int(np.prod(dims))
    if torch.cuda.mem_get_info()[0] < 12 * count:
        pytest.skip('needs 52 GB of device memory')
    shape = (dims[0], *dims[2:], dims[1])
    x = torch.randn(shape, generator=torch.Generator(device='cuda').manual_seed(38), dtype=torch.bfloat16, device='cuda')
    return x.movedim(-1, 1), torch.ones(shape, dtype=torch.bfloat16, device='cuda').movedim(-1, 1)


def tail_of_the_mask(dims, images, seed, offset):
    """keep of the last images, shaped like them: draws from their first place on."""
    place = int(np.prod(dims)) // dims[0]
    first = (dims[0] - images) * place
    draws = blocks_of_draws(first // 8, (images * place + 15) // 8, seed, offset)[first % 8:][:images * place]
    return (draws >= 32768).reshape(images, *dims[2:], dims[1]).movedim(-1, 1)


@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups,path', [((65537, 64, 32, 32), 4, 'resident'), ((268435461, 16), 2, 'small')])
def test_more_than_2_32_elements(native, torch_cuda, dims, groups, path):
    """The last images, their mask included; dbeta counts the kept places."""
    x, dy = large(dims)
    c = dims[1]
    gamma, beta = torch.ones(c, device='cuda'), torch.zeros(c, device='cuda')
    drop = api.dropout_args(0.5, 8, 9)
    y, stats = run_forward(native, x, groups, gamma, beta, act='silu', drop=drop)
    assert f'engine={path} ' in native.last_plan()
    dx, _, dbeta = run_backward(native, dy, x, stats, groups, gamma, beta, 'none', drop)
    assert f'engine={path}_backward ' in native.last_plan()
    keep = tail_of_the_mask(dims, 3, 8, 9)
    last = x[-3:].cpu()
    for act, got, want in (('silu', y, 'y'), ('none', dx, 'dx')):
        ref = NormReference(last, groups, act=act, keep=keep, scale=2.0).backward(torch.ones_like(last))
        assert_close(got[-3:], getattr(ref, want), getattr(ref, 'tol_' + want), want)
    kept = sum((part != 0).sum([d for d in range(part.dim()) if d != 1]) for part in y.split(1 << 22 if path == 'small' else 1 << 10))
    # a kept place whose activation is 0 or rounds to it: fewer than one in 2^10
    assert ((2 * kept <= dbeta * (1 + K * U)) & (dbeta <= 2 * kept * (1 + 2.0 ** -10))).all()


@pytest.mark.gpu
def test_an_image_of_more_than_2_32_elements(native, torch_cuda):
    """The split path: the last pixels, and both passes' sums over all of them."""
    dims, groups = (1, 8, 32769, 16384), 2
    x, dy = large(dims)
    gamma, beta = torch.ones(8, device='cuda'), torch.zeros(8, device='cuda')
    drop = api.dropout_args(0.5, 8, 9)
    y, stats = run_forward(native, x, groups, gamma, beta, drop=drop)
    assert 'engine=split ' in native.last_plan()
    dx, _, dbeta = run_backward(native, dy, x, stats, groups, gamma, beta, drop=drop)
    assert 'engine=split_backward ' in native.last_plan()
    rows = x[0].movedim(0, -1).reshape(-1, groups, 4)
    outs = y[0].movedim(0, -1).reshape(-1, groups, 4)
    parts = range(0, len(rows), 1 << 25)
    total = 4.0 * len(rows)
    mean = sum(rows[i:i + (1 << 25)].double().sum((0, 2)) for i in parts) / total
    var = sum((rows[i:i + (1 << 25)].double() - mean[:, None]).square().sum((0, 2)) for i in parts) / total
    rstd = (var + 1e-5).rsqrt()
    err = K * U * (1 + rows[:1 << 25].abs().max() * rstd)  # as in norm_helpers, for |x| up to the sample's largest
    assert ((stats[0, :, 0] - mean).abs() * rstd <= 2 * err).all() and ((stats[0, :, 1] / rstd - 1).abs() <= 2 * err).all()
    # s1 and s2 of dz = 2 keep, from the forward pass's own results: y = dz xhat
    # with a random rounding each
    s1 = sum(2.0 * (outs[i:i + (1 << 25)] != 0).sum((0, 2)) for i in parts) / total
    s2 = sum(outs[i:i + (1 << 25)].double().sum((0, 2)) for i in parts) / total
    count = 1 << 10
    first = len(rows) - count
    keep = (blocks_of_draws(first, count, 8, 9) >= 32768).view(count, groups, 4)
    mean, rstd, s1, s2 = (v.cpu()[:, None] for v in (mean, rstd, s1.double(), s2))
    xhat = (rows[-count:].cpu().double() - mean) * rstd
    dz = 2.0 * keep
    assert_close(outs[-count:], dz * xhat, HALF[x.dtype] * (dz * xhat).abs() + 2e-4)
    want = rstd * (dz - s1 - xhat * s2)
    assert_close(dx[0].movedim(0, -1).reshape(-1, groups, 4)[-count:], want, HALF[x.dtype] * want.abs() + 2e-4)
    assert ((dbeta.view(groups, 4).sum(1).double() / total).cpu() - s1[:, 0]).abs().max() <= 2.0 ** -10


# ---- repetition -----------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('dims,groups,path', [((32, 256, 28, 28), 32, 'resident'), ((200, 64, 28, 28), 1, 'resident'),
                                              ((5000, 24, 2, 2), 3, 'small'), ((2, 64, 300, 260), 1, 'split')])
@pytest.mark.parametrize('p', [0.0, 0.2])
def test_steps_repeat_bitwise(native, torch_cuda, dims, groups, path, p):
    """Whatever else the GPU does and whatever its caches hold: dgamma and dbeta
    too, in the parameters' 16-bit type."""
    x, gamma, beta, dy = (t.cuda() for t in make(dims, torch.bfloat16, 39))
    leaves = [t.requires_grad_() for t in (x, gamma.bfloat16(), beta.bfloat16())]
    busy, other = torch.empty(1 << 28, dtype=torch.uint8, device='cuda'), torch.cuda.Stream()
    want = None
    for i in range(24):
        if i % 3 == 1:
            busy.fill_(i)  # larger than the L2 cache
        if i % 3 == 2:
            other.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(other):
                busy.fill_(i)
        y = torch_module.group_norm_act(leaves[0], groups, *leaves[1:], activation='silu', dropout=p, seed=4, offset=5)
        if i == 0:
            assert f'engine={path} ' in native.last_plan()
        got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
        torch.cuda.synchronize()
        want = want or got
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# ---- saved tensors that come back with other strides ----------------------------------------------
HOOKS = {'host': lambda: torch.autograd.graph.save_on_cpu(),
         'pinned': lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
         'strided': lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.stack([t, t], -1)[..., 0])}


@pytest.mark.gpu
@pytest.mark.parametrize('hooks', HOOKS)
def test_hooks_on_saved_tensors(native, torch_cuda, hooks):
    x, gamma, beta, dy = (t.cuda() for t in make((2, 24, 6, 7), torch.float32, 34))
    grads = []
    for context in (contextlib.nullcontext, HOOKS[hooks]):
        leaves = [t.clone(memory_format=torch.preserve_format).requires_grad_() for t in (x, gamma, beta)]
        with context():
            y = torch_module.group_norm_act(leaves[0] * 1, 4, leaves[1] * 1, leaves[2] * 1, activation='silu')
        grads.append(torch.autograd.grad(y, leaves, dy))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


# ---- what the front end refuses -------------------------------------------------------------------
@pytest.mark.parametrize('grad', [True, False])
@pytest.mark.parametrize('operand', ['x', 'weight', 'bias', 'dropout x', 'residual'])
def test_forward_mode_of_any_operand_is_refused(native, operand, grad):
    """Duals whose primal requires no gradient too: their tangent would be lost.
    Refused before anything else, on the host's tensors as on the device's."""
    import torch.autograd.forward_ad as fwd
    x, w, b = torch.randn(2, 8, 3, 3), torch.ones(8), torch.zeros(8)
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        dual = lambda name, t: fwd.make_dual(t, torch.ones_like(t)) if name == operand else t
        with pytest.raises(RuntimeError, match='forward-mode'):
            if operand in ('dropout x', 'residual'):
                torch_module.dropout(dual('dropout x', x), 0.5, dual('residual', x.clone()))
            else:
                torch_module.group_norm_act(dual('x', x), 2, dual('weight', w), dual('bias', b))


@pytest.mark.parametrize('call', [lambda x: torch_module.group_norm_act(x, 2), lambda x: torch_module.dropout(x, 0.5)],
                         ids=['group_norm', 'dropout'])
def test_tracing_is_refused(native, call):
    """A traced graph would hold the output's allocation alone."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(2, 8, 3, 3)
    with pytest.raises(RuntimeError, match='cannot be traced'):
        torch.jit.trace(call, (x,))
    with pytest.raises(RuntimeError, match='cannot be traced'):
        make_fx(call)(x)


@pytest.mark.parametrize('front', [True, False], ids=['C++', 'ctypes'])
def test_tracing_of_a_convolution_is_refused(native, front):
    conv = torch_module.B200Conv2d(torch.nn.Conv2d(8, 8, 3, groups=2, bias=False), native, cpp=front)
    fused = torch_module.B200ConvBNAct(torch.nn.Conv2d(8, 8, 3, groups=2), native=native)
    if not front:
        fused._op = None
    for module in (conv, fused):
        with pytest.raises(RuntimeError, match='cannot be traced'):
            torch.jit.trace(module, (torch.randn(2, 8, 5, 5),))


@pytest.mark.parametrize('groups', [0, -2, 3, 16, 1 << 40, 1 << 60])
@pytest.mark.parametrize('grad', [True, False])
def test_group_counts_are_refused_by_status(native, groups, grad):
    """With a gradient wanted too, where statistics would be allocated first."""
    with pytest.raises(api.NativeError) as err:
        torch_module.group_norm_act(torch.zeros(2, 8, 3, 3, requires_grad=grad), groups)
    assert err.value.status == api.GC_INVALID


# ---- modules --------------------------------------------------------------------------------------
class OwnNorm(torch.nn.GroupNorm):
    def forward(self, x):
        return super().forward(x) + 1


class OwnReLU(torch.nn.ReLU):
    def forward(self, x):
        return super().forward(x) + 1


class OwnDropout(torch.nn.Dropout):
    def forward(self, x):
        return x


def test_fuse_norm_act_leaves_what_may_do_something_else():
    """Subclasses have a forward of their own, hooks expect to be called."""
    nn = torch.nn
    model = nn.Sequential(OwnNorm(2, 8), nn.ReLU(), nn.GroupNorm(2, 8), OwnReLU(), nn.GroupNorm(2, 8), nn.SiLU(),
                          OwnDropout(0.5), nn.GroupNorm(2, 8), nn.ReLU(), nn.GroupNorm(2, 8), nn.ReLU())
    model[8].register_forward_hook(lambda m, i, o: None)
    model[9].register_forward_pre_hook(lambda m, i: None)
    before = list(model)
    assert torch_module.fuse_norm_act(model) == ['2', '4', '7']
    for i in (0, 1, 3, 6, 8, 9, 10):
        assert model[i] is before[i]
    assert [model[i].activation for i in (2, 4, 7)] == ['none', 'silu', 'none']
    assert isinstance(model[5], nn.Identity)


class ActivationLast(torch.nn.Sequential):
    def forward(self, x):
        return self[1](self[2](self[0](x)))


class Named(torch.nn.Sequential):
    """A subclass that runs as Sequential does."""


def test_fuse_norm_act_leaves_sequentials_with_a_forward_of_their_own():
    nn = torch.nn
    members = lambda: (nn.GroupNorm(2, 8), nn.ReLU(), nn.Conv2d(8, 8, 1))
    model = nn.Sequential(ActivationLast(*members()), Named(*members()))
    assert torch_module.fuse_norm_act(model) == ['1.0']
    assert isinstance(model[0][1], nn.ReLU) and isinstance(model[1][1], nn.Identity)


@pytest.mark.parametrize('norm_mode', [True, False])
@pytest.mark.parametrize('drop_mode', [True, False])
def test_a_dropout_keeps_its_own_mode(monkeypatch, norm_mode, drop_mode):
    """Evaluation with the dropout left in training draws, as before the fusion."""
    nn = torch.nn
    seen = []
    monkeypatch.setattr(torch_module, 'group_norm_act',
                        lambda x, groups, w, b, eps, act, p, scope: seen.append((p, scope)) or x)
    drop = nn.Dropout2d(0.3)
    model = nn.Sequential(nn.GroupNorm(2, 8).train(norm_mode), nn.SiLU(), drop.train(drop_mode))
    keys = list(model.state_dict())
    torch_module.fuse_norm_act(model)
    assert model[0].training == norm_mode and list(model.state_dict()) == keys
    x = torch.zeros(1, 8, 2, 2)
    model(x)
    model.eval()(x)
    for m in model.modules():
        if isinstance(m, nn.Dropout2d):
            m.train()
    model(x)
    drop.p = 0.5
    model(x)
    model[0].p = 0.25
    model.train()(x)
    assert seen == [(0.3 if drop_mode else 0.0, 'channel'), (0.0, 'channel'), (0.3, 'channel'), (0.5, 'channel'),
                    (0.25, 'channel')]
    assert model[0].p == 0.25 and 'p=0.25' in model[0].extra_repr()


def test_a_norm_without_dropout_can_be_given_one():
    norm = torch_module.B200GroupNormAct(torch.nn.GroupNorm(2, 8).eval())
    assert norm.p == 0.0
    norm.p = 0.1
    assert norm.p == 0.1 and not norm.drop.training and norm.scope == 'element'


# ---- the generator --------------------------------------------------------------------------------
def philox_block(counter, key):
    """Philox4x32-10 of four counter words and two key words, with Python's integers."""
    (a, b, c, d), (k, m) = counter, key
    for _ in range(10):
        u, v = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = (v >> 32) ^ b ^ k, v & 0xFFFFFFFF, (u >> 32) ^ d ^ m, u & 0xFFFFFFFF
        k, m = (k + 0x9E3779B9) & 0xFFFFFFFF, (m + 0xBB67AE85) & 0xFFFFFFFF
    return [a, b, c, d]


def test_known_answers_of_the_generator():
    """The vectors published with Random123: zeros, ones, digits of pi."""
    ones = 0xFFFFFFFF
    assert philox_block([0] * 4, [0] * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert philox_block([ones] * 4, [ones] * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert philox_block([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0]) == [
        0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


@pytest.mark.parametrize('seed,offset', [(0, 0), (0x299f31d0a4093822, 0x0370734413198a2e), (1 << 32, 0), (1, 0),
                                         (0, 1 << 32), (0, 1), (2 ** 64 - 1, 2 ** 64 - 1)])
def test_draws_against_the_generator_s_blocks(seed, offset):
    """The oracle of the mask tests: key = seed, counter = (block, offset), each
    the low word first; half j % 2 of word j / 2 of a block is its draw j."""
    got = philox(8 * 3 + 5, seed, offset)
    low = 0xFFFFFFFF
    for j, draw in enumerate(got):
        words = philox_block([j // 8, 0, offset & low, offset >> 32], [seed & low, seed >> 32])
        assert draw == words[j % 8 // 2] >> 16 * (j % 2) & 0xFFFF
