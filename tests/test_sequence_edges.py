"""Layer norm, the causal convolution and the selective scan where calls can go
wrong: rows past 2^30 elements, long sums, values that are no numbers, what autograd
does around a call, first calls, calls of two threads."""
import contextlib
import subprocess
import sys
import threading

import pytest
import torch

from groupconv_atlas_b200 import api, torch_module
from tests import test_causal_conv, test_layer_norm, test_selective_scan
from tests.norm_helpers import HALF, U
from tests.sequence_helpers import LONG, ConvReference, ScanReference, assert_close
from tests.test_selective_scan import NAMES, TYPES, run


# ---- rows past 2^30 elements -------------------------------------------------------------------------
@pytest.mark.gpu
def test_a_row_of_almost_2_31_elements(native, torch_cuda):
    """The last columns within a block's step of 2^31.  A row of zeros: y is beta."""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip('needs 30 GB of device memory')
    c = 2 ** 31 - 1
    beta = torch.arange(c, device='cuda', dtype=torch.int32).remainder_(251).to(torch.bfloat16)
    y = torch_module.layer_norm(torch.zeros(1, c, device='cuda', dtype=torch.bfloat16), None, beta)
    assert 'kernel=layer_norm_long ' in api.Native().last_plan()
    assert torch.equal(y[0], beta)


@pytest.mark.gpu
def test_gradient_of_a_row_past_2_30_elements(native, torch_cuda):
    """Twice the row's length passes 31 bits: dbeta lies behind dgamma in the
    workspace.  x is 0 and dy +1 and -1 in turn, each thread's of one sign and
    as many: 2^21 + 2 in 32 bits, whose sums over threads cancel: dx is dy / sqrt(eps), dgamma 0, dbeta dy."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip('needs 60 GB of device memory')
    c, t = 2 ** 30 + 1024, torch.bfloat16
    x = torch.zeros(1, c, device='cuda', dtype=t, requires_grad=True)
    gamma, beta = torch.ones(c, device='cuda', dtype=t, requires_grad=True), torch.zeros(c, device='cuda', dtype=t, requires_grad=True)
    dy = torch.ones(1, c, device='cuda', dtype=t)
    dy[0, 1::2] = -1
    y = torch_module.layer_norm(x, gamma, beta, 2.0 ** -8)
    dx, dgamma, dbeta = torch.autograd.grad(y, (x, gamma, beta), dy)
    assert torch.equal(dbeta, dy[0]) and not dgamma.any() and torch.equal(dx, 16 * dy)


@pytest.mark.gpu
def test_gradient_of_a_scan_of_more_than_2_32_elements(native, torch_cuda):
    """Only the last 40 tokens of the last sequence are not zeros; in front of them x
    and dy are, so that the state and every gradient are."""
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip('needs 100 GB of device memory')
    n, l, ch = 2, 33000, 65540
    v = test_selective_scan.make(1, 40, ch, 1, 1, torch.bfloat16, 37)
    big = lambda t, fill: torch.full((n, l) + t.shape[2:], fill, dtype=t.dtype, device='cuda')
    q = {'x': big(v['x'], 0.0), 'dt': big(v['dt'], -1.0), 'b': big(v['b'], 1.0), 'c': big(v['c'], 1.0), 'a': v['a'].cuda()}
    for k in ('x', 'dt', 'b', 'c'):
        q[k][-1, -40:] = v[k][0].cuda()
    dy = big(v['dy'], 0.0)
    dy[-1, -40:] = v['dy'][0].cuda()
    leaves = {k: t.requires_grad_() for k, t in q.items()}
    y = run(v, leaves, True, None, False)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    ref = ScanReference(*(v[k] for k in NAMES[:5])).backward(v['dy'])
    for k in ('dt', 'c'):  # x and b in front receive what the tokens behind them pass back
        assert not grads[k][0].any() and not grads[k][1, :-40].any(), k
    assert not grads['x'][0].any() and not grads['b'][0].any()
    for k in ('x', 'dt', 'b', 'c'):
        assert_close(grads[k][-1:, -40:], getattr(ref, 'd' + k), getattr(ref, 'tol_d' + k) + 2.0 ** -40, k)
    assert_close(grads['a'], ref.da, ref.tol_da + HALF[torch.float32] * ref.da.abs() + 2.0 ** -25, 'a')


# ---- long sums --------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_rows_of_many_millions(native, torch_cuda):
    """Values of one size: a thread that adds its share of the squares, or of dy, one
    after the other in 32 bits is off by thousands of half steps (7700 and 5000 by
    arithmetic, of 32768 additions)."""
    v, c = float.fromhex('0x1.702dep0'), (1 << 24) + 3
    x = torch.full((1, c), v)
    x[0, ::2] = -v
    test_layer_norm.check(x, None, None, torch.full((1, c), v))


@pytest.mark.gpu
@pytest.mark.parametrize('c', [255, 257, 1001, 2047])
def test_constant_rows_of_large_values(native, torch_cuda, c):
    """Rows of one value, 2^100, and rstd = 2^30: the places of a row's first and last
    vector that are none of its columns count for nothing, though (0 - mean) rstd is
    infinite.  mean is exact, so xhat is 0: dx = rstd (dy - mean(dy)), its sum within
    2 c u of c for dy of -1 and 1 in turn and one 0."""
    x = torch.full((5, c), 2.0 ** 100, device='cuda').requires_grad_()
    gamma = torch.ones(c, device='cuda', requires_grad=True)
    dy = torch.ones(5, c, device='cuda')
    dy[:, ::2] = -1
    dy[:, 0] = 0
    y = torch_module.layer_norm(x, gamma, None, 2.0 ** -60)
    dx, dgamma = torch.autograd.grad(y, (x, gamma), dy)
    assert not y.any() and not dgamma.any()
    assert torch.equal(dx, 2.0 ** 30 * dy)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows', [1, 300, 100000])
def test_rows_of_one_column(native, torch_cuda, dtype, rows):
    """y is beta whatever x is, and dx exactly 0: dy gamma and its mean are rounded alike."""
    x, gamma, beta, dy = test_layer_norm.make((rows, 1), TYPES[dtype], 38)
    leaves = [t.cuda().requires_grad_() for t in (x, gamma, beta)]
    y = torch_module.layer_norm(*leaves)
    dx, dgamma, _ = torch.autograd.grad(y, leaves, dy.cuda())
    assert torch.equal(y, leaves[2].detach().to(y.dtype).expand_as(y)) and not dx.any() and not dgamma.any()


@pytest.mark.gpu
def test_parameters_of_a_long_scan(native, torch_cuda):
    """Steady states give dA, dD and ddt_bias sums of one value each, over segments of
    65536 tokens: added up in 32 bits tile after tile these would be off by more than
    1100 half steps.  Beside the sums' LONG u: a[t] = exp(-1) is off by 7 u, so the
    steady h and q = 1 / (1 - a) of what they add by at most (0.37 * 7 + 3) / 0.63 u < 9 u,
    their product with a and the slope's two terms by 2 * 9 + 7 + 6 < 32 u of terms whose
    difference is above a quarter of their sum: 128 u."""
    n, l, value = 3600, 65536, float.fromhex('0x1.d45a1cp0')
    one = lambda *shape: torch.ones(shape, device='cuda')
    names = ('x', 'dt', 'a', 'b', 'c', 'd', 'dt_bias')
    leaves = dict(zip(names, (one(n, l, 1), one(n, l, 1), -one(1, 1), one(n, l, 1, 1), one(n, l, 1, 1), one(1), 0 * one(1))))
    for t in leaves.values():
        t.requires_grad_()
    y = torch_module.selective_scan(*(leaves[k] for k in names[:5]), D=leaves['d'], dt_bias=leaves['dt_bias'], softplus=False)
    assert 'parts=1 ' in api.Native().last_plan()
    wanted = [leaves[k] for k in ('a', 'd', 'dt_bias')]
    da, dd, dbias = torch.autograd.grad(y, wanted, torch.full_like(y, value))
    a, h, q = torch.exp(torch.tensor(-1.0, dtype=torch.double)).item(), [0.0], [0.0]
    for _ in range(l):
        h.append(a * h[-1] + 1.0)
        q.append(a * q[-1] + value)
    m = [q[l - t] * a * h[t] for t in range(l)]  # q[t] a h[t - 1]
    want = {'da': sum(m), 'dd': l * value, 'dbias': sum(q[l - t] - m[t] for t in range(l))}
    for name, got in (('da', da), ('dd', dd), ('dbias', dbias)):
        w = n * want[name]
        assert abs(got.item() - w) <= (LONG + 128) * U * w, (name, got.item() / w - 1)


@pytest.mark.gpu
def test_runs_of_sequences_that_end_early(native, torch_cuda):
    """One segment of three runs of 512 tokens: sequences that end in each, and at
    their borders; the runs behind an end count as 0, whatever memory held."""
    n, l, ends = 4000, 1030, [1030, 1029, 1025, 1024, 1023, 513, 512, 511, 1, 0]
    v = test_selective_scan.make(len(ends), l, 8, 4, 1, torch.float32, 34)
    v['lengths'] = torch.tensor(ends, dtype=torch.int32)
    ref = ScanReference(*(v[k] for k in NAMES[:8]), True, v['state'], v['lengths']).backward(v['dy'], v['dlast'])
    params = ('a', 'd', 'dt_bias')
    many = lambda t: torch.cat([t, t.new_zeros((n - len(ends),) + t.shape[1:])]).cuda()
    q = {k: v[k].cuda() if k in params else many(v[k]) for k in NAMES}
    for k in params:
        q[k].requires_grad_()
    y, last = run(v, q, True, many(v['lengths']), True)
    assert 'parts=1 ' in api.Native().last_plan()
    spoiled = torch.full((1 << 28,), float('nan'), device='cuda')
    del spoiled
    grads = torch.autograd.grad([y, last], [q[k] for k in params], [many(v['dy']), many(v['dlast'])])
    for k, g in zip(params, grads):
        want, tol = getattr(ref, {'a': 'da', 'd': 'dd', 'dt_bias': 'ddt_bias'}[k]), getattr(ref, f'tol_d{k}')
        assert_close(g, want, tol + HALF[torch.float32] * want.abs() + 2.0 ** -25, k)


@pytest.mark.gpu
def test_weights_of_many_stretches(native, torch_cuda):
    """So many tokens that a block more than the GPU asks for takes part, each worker
    having 64 stretches; x and dy of one value each, so that dbias and each tap of dweight
    are their counts times a value (1.1015625, exact in bfloat16, and its square)."""
    if torch.cuda.mem_get_info()[0] < 70 << 30:
        pytest.skip('needs 70 GB of device memory')
    n, l, c, k, value = 5, 140000, 8192, 4, 1.1015625
    x = torch.full((n, l, c), value, device='cuda', dtype=torch.bfloat16).requires_grad_()
    w, b = torch.zeros(c, k, device='cuda', requires_grad=True), torch.zeros(c, device='cuda', requires_grad=True)
    y = torch_module.causal_conv(x, w, b)
    dw, db = torch.autograd.grad(y, (w, b), torch.full_like(y, value))
    count = torch.tensor([n * (l - (k - 1 - j)) for j in range(k)], dtype=torch.double)  # tap j reads zeros before token K - 1 - j
    assert_close(db, torch.full((c,), n * l * value, dtype=torch.double), torch.full((c,), LONG * U * n * l * value, dtype=torch.double))
    want = (count * value * value).expand(c, k)
    assert_close(dw, want, (LONG + 2) * U * want)


@pytest.mark.gpu
@pytest.mark.parametrize('states', [16, 64])
def test_pairs_of_many_channels(native, torch_cuda, states):
    """dB and dC are sums over 2^18 channels; of one value each they would be off by
    hundreds of half steps if blocks were added up one after the other in 32 bits.
    Each term is a product of few factors: 8 u beside the sums."""
    ch, value = 1 << 18, float.fromhex('0x1.141894p0')
    one = lambda *shape: torch.ones(shape, device='cuda')
    b, c = one(1, 1, 1, states).requires_grad_(), one(1, 1, 1, states).requires_grad_()
    y = torch_module.selective_scan(one(1, 1, ch), one(1, 1, ch), -one(ch, states), b, c, softplus=False)
    for g in torch.autograd.grad(y, [b, c], torch.full_like(y, value)):
        g = g.double().cpu()
        assert ((g - ch * value).abs() <= (LONG // 2 + 8) * U * ch * value).all(), g.reshape(-1)[0].item() / (ch * value) - 1


# ---- step sizes that are no numbers ----------------------------------------------------------------
def scan_with_gradient(v):
    leaves = {k: v[k].cuda().requires_grad_() for k in NAMES}
    y, last = run(v, leaves, True, None, True)
    grads = torch.autograd.grad([y, last], list(leaves.values()), [v['dy'].cuda(), v['dlast'].cuda()])
    return {'y': y.detach(), 'last': last.detach(), **{'d' + k: g for k, g in zip(NAMES, grads)}}


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(2, 100, 36, 16, 1), (2, 40, 33, 7, 3)])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('place', ['dt', 'dt_bias'])
@pytest.mark.parametrize('value', [float('nan'), float('inf'), -float('inf')])
@pytest.mark.parametrize('channel', [4, 5])
def test_step_sizes_stay_in_their_channel(native, torch_cuda, shape, dtype, place, value, channel):
    """Every other channel's results and gradients are those without the value (dB and
    dC are sums over channels).  A step size of 0, from -inf, leaves the state as it is."""
    v = test_selective_scan.make(*shape, TYPES[dtype], 31)
    ref = ScanReference(*(v[k] for k in NAMES[:8]), True, v['state']).backward(v['dy'], v['dlast'])
    clean = scan_with_gradient(v)
    v[place] = v[place].clone()
    if place == 'dt':
        v['dt'][1, 20, channel] = value
    else:
        v['dt_bias'][channel] = value
    got = scan_with_gradient(v)
    others = torch.arange(shape[2]) != channel
    for name in ('y', 'dx', 'ddt', 'dz'):
        assert_close(got[name].cpu()[..., others], getattr(ref, name)[..., others], getattr(ref, 'tol_' + name)[..., others] + 2.0 ** -40, name)
        if place == 'dt':
            assert torch.equal(got[name][0], clean[name][0]), name  # the other sequence
    for name in ('last', 'dstate'):
        assert_close(got[name].cpu()[:, others], getattr(ref, name)[:, others], getattr(ref, 'tol_' + name)[:, others] + 2.0 ** -40, name)
    for name in ('da', 'dd', 'ddt_bias'):
        want = getattr(ref, name)[others]
        tol = getattr(ref, 'tol_' + name)[others] + HALF[torch.float32] * want.abs() + 2.0 ** -25
        assert_close(got[name].cpu()[others], want, tol, name)
    own = got['y'][1, 20:, channel]
    assert torch.isfinite(own).all() if value == -float('inf') else not torch.isfinite(own).any()


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(3, 64, 16, 2), (3, 33, 7, 3)])  # every access whole, or not
@pytest.mark.parametrize('place', ['dt', 'dt_bias'])
@pytest.mark.parametrize('value', [float('nan'), float('inf'), -float('inf')])
@pytest.mark.parametrize('channel', [4, 5])
def test_step_sizes_of_a_token_stay_in_their_channel(native, torch_cuda, shape, place, value, channel):
    n, ch, s, groups = shape
    v = test_selective_scan.make(n, 1, ch, s, groups, torch.float32, 32)
    ref = ScanReference(*(v[k] for k in NAMES[:8]), True, v['state'])
    if place == 'dt':
        v['dt'][1, 0, channel] = value
    else:
        v['dt_bias'][channel] = value
    q = {k: t.cuda() for k, t in v.items()}
    state = q['state'].clone()
    y = torch_module.selective_scan_step(q['x'][:, 0], q['dt'][:, 0], q['a'], q['b'][:, 0], q['c'][:, 0], state, q['d'],
                                         q['z'][:, 0], q['dt_bias'])
    others = torch.arange(ch) != channel
    assert_close(y.cpu()[:, others], ref.y[:, 0, others], ref.tol_y[:, 0, others], 'y')
    assert_close(state.cpu()[:, others], ref.last[:, others], ref.tol_last[:, others], 'state')
    if value == -float('inf'):
        assert torch.equal(state[1, channel], q['state'][1, channel]) and torch.isfinite(y).all()
    else:
        assert not torch.isfinite(y[1, channel])


@pytest.mark.gpu
@pytest.mark.parametrize('states', [4, 16])
def test_growing_states_that_nothing_has_entered(native, torch_cuda, states):
    """A > 0: a segment's growth, exp(96) over 32 tokens, is infinite in 32 bits, and so
    is its product with nothing (0 inf) no number.  x is 0 but for the last tokens, dy but
    for the first."""
    n, l, ch = 2, 640, 8
    v = test_selective_scan.make(n, l, ch, states, 1, torch.float32, 39)
    v['dt'] = torch.ones_like(v['dt'])
    v['a'] = 3 * torch.rand(ch, states, generator=torch.Generator().manual_seed(40)).round()
    v['x'][:, :-12] = 0
    v['dy'][:, 12:] = 0
    ref = ScanReference(*(v[k] for k in NAMES[:7]), softplus=False).backward(v['dy'])
    leaves = {k: v[k].cuda().requires_grad_() for k in NAMES[:7]}
    y = run(v, leaves, False, None, False)
    assert 'parts=1 ' not in api.Native().last_plan()
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), v['dy'].cuda())))
    assert_close(y, ref.y, ref.tol_y, 'y')
    for k in ('x', 'dt', 'b', 'c', 'z'):
        assert_close(grads[k], getattr(ref, 'd' + k), getattr(ref, 'tol_d' + k) + 2.0 ** -40, k)
    for k in ('a', 'd'):
        want = getattr(ref, 'd' + k)
        assert_close(grads[k], want, getattr(ref, 'tol_d' + k) + HALF[torch.float32] * want.abs() + 2.0 ** -25, k)


@pytest.mark.gpu
@pytest.mark.parametrize('value', [float('nan'), float('inf'), -float('inf')])
@pytest.mark.parametrize('channel', [4, 5])
@pytest.mark.parametrize('op', ['gate', 'convolution'])
def test_arguments_of_silu_stay_in_their_channel(native, torch_cuda, op, value, channel):
    """silu's pairs share a reciprocal as well: the neighbour's values and gradients."""
    if op == 'gate':
        v = test_selective_scan.make(2, 40, 36, 16, 1, torch.float32, 35)
        ref = ScanReference(*(v[k] for k in NAMES[:8]), True, v['state']).backward(v['dy'], v['dlast'])
        v['z'][1, 20, channel] = value
        got = scan_with_gradient(v)
        names = ('y', 'dx', 'ddt', 'dz')
    else:
        v = test_causal_conv.make(2, 40, 36, 4, torch.float32, 36)
        ref = ConvReference(v['x'], v['w'], v['b'], 'silu').backward(v['dy'])
        v['x'][1, 20, channel] = value
        leaves = [v[k].cuda().requires_grad_() for k in ('x', 'w', 'b')]
        y = torch_module.causal_conv(*leaves, 'silu')
        got = {'y': y.detach(), 'dx': torch.autograd.grad(y, leaves, v['dy'].cuda())[0]}
        names = ('y', 'dx')
    others = torch.arange(36) != channel
    for name in names:
        assert_close(got[name].cpu()[..., others], getattr(ref, name)[..., others], getattr(ref, 'tol_' + name)[..., others] + 2.0 ** -40, name)
        assert_close(got[name][0], getattr(ref, name)[0], getattr(ref, 'tol_' + name)[0] + 2.0 ** -40, name)


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(3, 64, 16, 2), (3, 33, 7, 3)])
def test_infinite_decays_of_a_token(native, torch_cuda, shape):
    """A = -inf forgets the state, and with a step size of 0 leaves it as it is, in
    every kernel alike."""
    n, ch, s, groups = shape
    v = {k: t.cuda() for k, t in test_selective_scan.make(n, 1, ch, s, groups, torch.float32, 33).items()}
    v['a'][3] = -float('inf')
    v['dt'][0] = -300.0
    y, last = run(v, v, True, None, True)
    state = v['state'].clone()
    one = torch_module.selective_scan_step(v['x'][:, 0], v['dt'][:, 0], v['a'], v['b'][:, 0], v['c'][:, 0], state, v['d'],
                                           v['z'][:, 0], v['dt_bias'])
    assert torch.isfinite(one).all() and torch.equal(state[0], v['state'][0]) and torch.equal(last[0], v['state'][0])
    torch.testing.assert_close(one, y[:, 0], rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(state, last, rtol=1e-5, atol=1e-6)


# ---- what autograd does around a call --------------------------------------------------------------
def norm_call(t):
    return torch_module.layer_norm(t['x'], t['w'], t['b'])


def conv_call(t):
    return torch_module.causal_conv(t['x'], t['w'], t['b'], 'silu', t['state'], t['lengths'], True)


def scan_call(t):
    return run(t, {k: t[k] for k in NAMES}, True, t['lengths'], True)


def operands(op):
    """Tensors of a call on the host, all that it takes."""
    if op == 'norm':
        x, w, b, _ = test_layer_norm.make((3, 5, 24), torch.float32, 41)
        return {'x': x, 'w': w, 'b': b}
    v = test_causal_conv.make(2, 21, 12, 4, torch.float32, 42) if op == 'conv' else test_selective_scan.make(
        2, 70, 12, 8, 2, torch.float32, 43)
    return {k: t for k, t in v.items() if k not in ('dy', 'dlast')}


CALLS = {'norm': norm_call, 'conv': conv_call, 'scan': scan_call}
FLOATS = [(op, name) for op in CALLS for name, t in operands(op).items() if t.is_floating_point()]
HOOKS = {'host': lambda: torch.autograd.graph.save_on_cpu(),
         'pinned': lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
         'strided': lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.stack([t, t], -1)[..., 0])}


@pytest.mark.gpu
@pytest.mark.parametrize('op', CALLS)
@pytest.mark.parametrize('hooks', HOOKS)
def test_hooks_on_saved_tensors(native, torch_cuda, op, hooks):
    t = {k: v.cuda() for k, v in operands(op).items()}
    grads = []
    for context in (contextlib.nullcontext, HOOKS[hooks]):
        leaves = {k: v.clone().requires_grad_(v.is_floating_point()) for k, v in t.items()}
        with context():
            out = CALLS[op]({k: v * 1 for k, v in leaves.items()})
        out = out if isinstance(out, tuple) else (out,)
        seeds = [torch.cos(torch.arange(o.numel(), device='cuda').reshape(o.shape)).to(o.dtype) for o in out]
        grads.append(torch.autograd.grad(out, [v for v in leaves.values() if v.requires_grad], seeds))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize('grad', [True, False])
@pytest.mark.parametrize('op,name', FLOATS)
def test_forward_mode_of_any_operand_is_refused(native, op, name, grad):
    """Duals whose primal requires no gradient too: their tangent would be lost."""
    import torch.autograd.forward_ad as fwd
    t = operands(op)
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        t[name] = fwd.make_dual(t[name], torch.ones_like(t[name]))
        with pytest.raises(RuntimeError, match='forward-mode'):
            CALLS[op](t)


def token_calls(t, u, out=None):
    """The steps on the first token of operands('conv') and operands('scan')."""
    at = lambda v: v[:, 0]
    return {'conv': lambda: torch_module.causal_conv_step(at(t['x']), t['w'], t['state'], t['b'], 'silu', state_out=out),
            'scan': lambda: torch_module.selective_scan_step(at(u['x']), at(u['dt']), u['a'], at(u['b']), at(u['c']), u['state'],
                                                             u['d'], at(u['z']), u['dt_bias'], state_out=out)}


@pytest.mark.parametrize('op,name', [(op, n) for op, n in FLOATS if op != 'norm'] + [('conv', 'out'), ('scan', 'out')])
def test_forward_mode_of_steps_is_refused(native, op, name):
    """The tensor that a step writes its state to as well."""
    import torch.autograd.forward_ad as fwd
    t = {'conv': operands('conv'), 'scan': operands('scan')}
    out = torch.zeros_like(t[op]['state'])
    with fwd.dual_level(), torch.no_grad():
        if name == 'out':
            out = fwd.make_dual(out, torch.ones_like(out))
        else:
            t[op][name] = fwd.make_dual(t[op][name], torch.ones_like(t[op][name]))
        with pytest.raises(RuntimeError, match='forward-mode'):
            token_calls(t['conv'], t['scan'], out)[op]()


@pytest.mark.parametrize('op', CALLS)
def test_tracing_is_refused(native, op):
    """A traced graph would hold the outputs' allocations alone."""
    from torch.fx.experimental.proxy_tensor import make_fx
    t = operands(op)
    call = lambda x: CALLS[op]({**t, 'x': x})
    with pytest.raises(RuntimeError, match='cannot be traced'):
        torch.jit.trace(call, (t['x'],))
    with pytest.raises(RuntimeError, match='cannot be traced'):
        make_fx(call)(t['x'])


@pytest.mark.gpu
@pytest.mark.parametrize('op,name', FLOATS)
def test_function_transforms_are_refused(native, torch_cuda, op, name):
    """vmap and torch.func.grad hand in tensors without memory of their own."""
    t = {k: v.cuda() for k, v in operands(op).items()}

    def call(v):
        out = CALLS[op]({**t, name: v})
        return (out[0] if isinstance(out, tuple) else out).sum()
    with pytest.raises(RuntimeError):
        torch.func.vmap(call)(torch.stack([t[name]] * 2))
    with pytest.raises(RuntimeError):
        torch.func.grad(call)(t[name])
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize('op', ['conv', 'scan'])
def test_steps_under_vmap_are_refused(native, torch_cuda, op):
    """And leave the state as it was."""
    t, u = ({k: v.cuda() for k, v in operands(o).items()} for o in ('conv', 'scan'))
    q = t if op == 'conv' else u
    before = q['state'].clone()
    for name in [n for o, n in FLOATS if o == op and n != 'state']:
        def call(v):
            mine = {**q, name: v}
            return token_calls(mine if op == 'conv' else t, mine if op == 'scan' else u)[op]()
        with torch.no_grad(), pytest.raises(RuntimeError):
            torch.func.vmap(call)(torch.stack([q[name]] * 2))
        assert torch.equal(q['state'], before), name


# ---- first calls, calls of two threads --------------------------------------------------------------
FIRST_USE = """
import torch
from groupconv_atlas_b200 import torch_module as tm
r = lambda *s: torch.randn(s, device='cuda')
x, odd, w = r(64, 512), r(64, 501), r(16, 4)
u, dt, A, B, C = r(2, 200, 16), r(2, 200, 16), -r(16, 16).exp(), r(2, 200, 16), r(2, 200, 16)
long, half, cache, h = r(2, 9000), r(2, 64, 64).bfloat16(), r(2, 3, 16), r(2, 16, 16)
small = r(64, 16).bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    a = [t.requires_grad_() for t in (x, odd, long, u, half, small)]
    y = [tm.layer_norm(x), tm.layer_norm(odd), tm.layer_norm(long), tm.causal_conv(u, w), tm.causal_conv(half, r(64, 4).bfloat16()),
         tm.selective_scan(u, dt, A, B, C), tm.layer_norm(small)]
    g = torch.autograd.grad(y, a, [torch.ones_like(t) for t in y])
    with torch.no_grad():
        y += [tm.causal_conv_step(u[:, 0], w, cache), tm.selective_scan_step(u[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], h)]
graph.replay()
torch.cuda.synchronize()
assert all(bool(torch.isfinite(t).all()) for t in (*y, *g)) and all(bool(t.any()) for t in y)
"""


@pytest.mark.gpu
def test_first_use_inside_a_capture(native, torch_cuda):
    """Nothing that a first call sets up disturbs a capture."""
    done = subprocess.run([sys.executable, '-c', FIRST_USE], cwd=api.ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.gpu
def test_two_threads_and_streams(native, torch_cuda):
    """Training steps of two host threads on streams of their own do not meet."""
    sets = [{k: t.cuda() for k, t in test_selective_scan.make(2, 130, 24, 16, 1, torch.bfloat16, s).items()} for s in (44, 45)]
    weight = torch.randn(24, 4, device='cuda')

    def step(v):
        leaves = {k: v[k].detach().requires_grad_() for k in NAMES}
        u = torch_module.causal_conv(torch_module.layer_norm(leaves['x']), weight, activation='silu')
        y = run(v, {**leaves, 'x': u}, True, v['lengths'], False)
        return [y.detach(), *torch.autograd.grad(y, list(leaves.values()), v['dy'])]
    want = [step(v) for v in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                got = step(sets[i])
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


# ---- the block -------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('half', [torch.bfloat16, torch.float16])
def test_block_under_autocast(native, torch_cuda, half):
    """Parameters in 32 bits, branches in 16: new states fit the steps; prompts and
    tokens agree with the whole sequence.  Each of the few products of 16-bit values
    on the way is off by half a step of its factors: 2^-5 covers them at width 32."""
    torch.manual_seed(2)
    block = torch_module.B200SelectiveBlock(32, states=8, device='cuda')
    x = torch.randn(3, 20, 32, device='cuda')
    with torch.no_grad(), torch.autocast('cuda', half):
        want = block(x)
        states = block.new_states(3)
        for t in range(4):
            torch.testing.assert_close(block.step(x[:, t], states), want[:, t], rtol=2 ** -5, atol=2 ** -5)
        y, states = block.prefill(x[:, 4:10], None, states)
        torch.testing.assert_close(y, want[:, 4:10], rtol=2 ** -5, atol=2 ** -5)
        torch.testing.assert_close(block.step(x[:, 10], states), want[:, 10], rtol=2 ** -5, atol=2 ** -5)
    with torch.autocast('cuda', half):
        loss = block(x).square().mean()
    loss.backward()
    assert all(p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() and p.grad.any() for p in block.parameters())


@pytest.mark.gpu
def test_new_states_are_of_the_branch_s_type(native, torch_cuda):
    """The convolution's parameters may stay in 32 bits beside 16-bit projections."""
    block = torch_module.B200SelectiveBlock(16, states=4, device='cuda')
    for m in (block.norm, block.input, block.select, block.dt, block.output):
        m.to(torch.bfloat16)
    with torch.no_grad():
        x = torch.randn(2, 5, 16, device='cuda', dtype=torch.bfloat16)
        states = block.new_states(2)
        first = block.step(x[:, 0], states)
        torch.testing.assert_close(first, block(x)[:, 0], rtol=2 ** -5, atol=2 ** -5)


@pytest.mark.parametrize('default', [torch.float64, torch.bfloat16])
def test_scan_parameters_are_in_32_bits_whatever_the_default(default):
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        block = torch_module.B200SelectiveBlock(16, states=4, dtype=torch.float32)
        states = block.new_states(2)
    finally:
        torch.set_default_dtype(before)
    assert {p.dtype for p in block.parameters()} == {torch.float32} and {s.dtype for s in states} == {torch.float32}


@pytest.mark.parametrize('bad', [torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32),
                                 torch.zeros(4, dtype=torch.int32)[::2], torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2)])
def test_lengths_of_the_ctypes_calls(native, bad):
    """N dense words of 32 bits: the library cannot see what they are."""
    v = test_causal_conv.make(2, 9, 8, 4, torch.float32)
    u = test_selective_scan.make(2, 9, 8, 4, 2, torch.float32)
    with pytest.raises(ValueError):
        native.causal_conv(v['x'], v['w'], torch.empty_like(v['x']), lengths=bad)
    with pytest.raises(ValueError):
        native.causal_conv_backward(v['dy'], v['x'], v['w'], torch.empty_like(v['x']), lengths=bad)
    with pytest.raises(ValueError):
        api.scan_args(u['x'], u['dt'], u['a'], u['b'], u['c'], lengths=bad)
