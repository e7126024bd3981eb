"""gc_b200_selective_scan, its gradient and its form for one token against the
formulas in 64 bits, and the operators on sequences run together."""
import math

import pytest
import torch

from groupconv_atlas_b200 import api, torch_module
from tests.norm_helpers import HALF
from tests.sequence_helpers import ScanReference, assert_close

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}

# (N, L, channels, S, groups): one token, tiles and chunks of tokens that end
# early, every number of lanes, state counts between powers of two, channels that
# fill no block, groups of odd size (single elements), several segments, many
# sequences
SHAPES = [(1, 1, 4, 16, 1), (2, 2, 8, 1, 1), (2, 17, 36, 16, 1), (1, 33, 7, 4, 1), (2, 40, 132, 8, 2), (1, 50, 30, 12, 3),
          (2, 31, 20, 32, 1), (1, 70, 12, 64, 1), (1, 45, 10, 50, 2), (3, 16, 4, 3, 4), (1, 300, 40, 16, 1), (2, 200, 33, 7, 1),
          (40, 5, 24, 16, 1), (1, 260, 200, 1, 1), (1, 200, 150, 2, 2), (1, 64, 64, 16, 64)]
NAMES = ('x', 'dt', 'a', 'b', 'c', 'd', 'z', 'dt_bias', 'state')


def make(n, l, ch, s, groups, dtype, seed=0, params=torch.float32):
    g = torch.Generator().manual_seed(seed)
    r = lambda *shape: torch.randn(shape, generator=g)
    first = torch.exp(torch.rand(ch, generator=g) * math.log(100.0) + math.log(1e-3))
    return {'x': r(n, l, ch).to(dtype), 'dt': (0.5 * r(n, l, ch)).to(dtype),
            'a': (-torch.arange(1, s + 1) * torch.exp(0.2 * r(ch, s))).to(params),
            'b': r(n, l, groups, s).to(dtype), 'c': r(n, l, groups, s).to(dtype), 'd': (1 + 0.2 * r(ch)).to(params),
            'z': r(n, l, ch).to(dtype), 'dt_bias': (first + torch.log(-torch.expm1(-first))).to(params),
            'state': r(n, ch, s), 'dy': r(n, l, ch).to(dtype), 'dlast': r(n, ch, s),
            'lengths': torch.randint(0, l + 1, (n,), generator=g, dtype=torch.int32)}


def run(v, leaves, softplus, lengths, return_state):
    q = {k: leaves.get(k) for k in NAMES}
    return torch_module.selective_scan(q['x'], q['dt'], q['a'], q['b'], q['c'], D=q['d'], z=q['z'], dt_bias=q['dt_bias'],
                                       softplus=softplus, state=q['state'], lengths=lengths, return_state=return_state)


def check(v, without=(), softplus=True, lengths=False, on_gpu=None, label=''):
    """Forward and gradient; without: operands left out."""
    q = {k: None if k in without else v[k] for k in NAMES}
    lens = v['lengths'] if lengths else None
    ref = ScanReference(*(q[k] for k in NAMES[:8]), softplus, q['state'], lens)
    state = q['state'] is not None
    ref.backward(v['dy'], v['dlast'] if state else None)
    leaves = {k: ((on_gpu or {}).get(k, t.cuda())).detach().requires_grad_() for k, t in q.items() if t is not None}
    out = run(v, leaves, softplus, None if lens is None else lens.cuda(), state)
    y, last = out if state else (out, None)
    label += f' [{api.Native().last_plan()}]'
    assert y.dtype == v['x'].dtype and y.is_contiguous()
    assert_close(y, ref.y, ref.tol_y, f'y {label}')
    outs, given = ([y, last], [v['dy'].cuda(), v['dlast'].cuda()]) if state else ([y], [v['dy'].cuda()])
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), given)))
    if state:
        assert last.dtype == torch.float32
        assert_close(last, ref.last, ref.tol_last, f'state {label}')
        assert_close(grads['state'], ref.dstate, ref.tol_dstate + 2.0 ** -40, f'dstate {label}')
    for name, key in (('x', 'dx'), ('dt', 'ddt'), ('z', 'dz'), ('b', 'db'), ('c', 'dc')):
        if name in grads:
            assert_close(grads[name], getattr(ref, key), getattr(ref, 'tol_' + key) + 2.0 ** -40, f'{key} {label}')
    for name, key in (('a', 'da'), ('d', 'dd'), ('dt_bias', 'ddt_bias')):
        if name in grads:
            want = getattr(ref, key)
            assert_close(grads[name], want, getattr(ref, 'tol_' + key) + HALF[grads[name].dtype] * want.abs() + 2.0 ** -25,
                         f'{key} {label}')
    if lengths:
        for t in (y, grads['x'], grads['dt']):
            assert not (t.detach().cpu() * ~ref.inside).any()
        for t in (grads['b'], grads['c']):
            assert not (t.cpu() * ~ref.inside[..., None]).any()


@pytest.mark.gpu
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: 'x'.join(map(str, s)))
@pytest.mark.parametrize('dtype', TYPES)
def test_sequences(native, torch_cuda, shape, dtype):
    v = make(*shape, TYPES[dtype])
    check(v, without=('state',))
    check(v, lengths=True)


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(2, 37, 40, 16, 1), (1, 200, 18, 5, 2)])
@pytest.mark.parametrize('without', [('z',), ('d', 'dt_bias'), ('z', 'd', 'dt_bias', 'state')])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_operands_left_out(native, torch_cuda, shape, without, dtype):
    v = make(*shape, TYPES[dtype], 1)
    check(v, without)
    check(v, without, lengths=True)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f32', 'f16'])
def test_step_sizes_as_given(native, torch_cuda, dtype):
    """Without softplus, of either sign, with parameters of the data's type."""
    v = make(2, 70, 20, 16, 1, TYPES[dtype], 2, TYPES[dtype])
    v['dt'] = v['dt'] * 0.02
    v['dt_bias'] = (v['dt_bias'].float() * 0.001).to(TYPES[dtype])
    check(v, softplus=False)
    check(v, ('dt_bias', 'z'), softplus=False)


@pytest.mark.gpu
@pytest.mark.parametrize('lengths', [[0, 1, 2, 3], [200, 15, 300, -7], [0, 0, 0, 0], [16, 32, 64, 65], [199, 17, 128, 127]])
@pytest.mark.parametrize('c,groups', [(8, 1), (9, 3)])
def test_lengths(native, torch_cuda, lengths, c, groups):
    v = make(4, 200, c, 16, groups, torch.float32, 3)
    v['lengths'] = torch.tensor(lengths, dtype=torch.int32)
    check(v, lengths=True)
    leaves = {k: v[k].cuda() for k in NAMES}
    clean, last = run(v, leaves, True, v['lengths'].cuda(), True)
    for k in ('x', 'dt', 'b', 'c', 'z'):
        for i, e in enumerate(v['lengths'].clamp(0, 200).tolist()):
            leaves[k][i, e:] = float('nan')
    y, s = run(v, leaves, True, v['lengths'].long().cuda(), True)
    assert torch.equal(y, clean) and torch.equal(s, last)
    leaves = {k: t.requires_grad_() for k, t in leaves.items()}
    y, s = run(v, leaves, True, v['lengths'].cuda(), True)
    dy = v['dy'].cuda()
    for i, e in enumerate(v['lengths'].clamp(0, 200).tolist()):
        dy[i, e:] = float('inf')
    for g in torch.autograd.grad([y, s], list(leaves.values()), [dy, v['dlast'].cuda()]):
        assert torch.isfinite(g).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_layouts(native, torch_cuda, dtype):
    """Slices of the projections that give them, odd offsets, other orders (copied),
    broadcast operands."""
    t = TYPES[dtype]
    n, l, ch, s = 2, 37, 24, 16
    g = torch.Generator().manual_seed(5)
    for case in ('slices', 'odd', 'transposed', 'broadcast'):
        v = make(n, l, ch, s, 1, t, 4)
        gpu = {}
        if case in ('slices', 'odd'):
            at = 1 if case == 'odd' else 0
            for name in ('x', 'dt', 'z'):
                base = torch.randn((n, l, 2 * ch + 1), generator=g).to(t)
                v[name], gpu[name] = base[..., at:at + ch], base.cuda()[..., at:at + ch]
            base = torch.randn((n, l, 2 * s + 3), generator=g).to(t)
            for name, off in (('b', 3), ('c', 3 + s)):
                v[name], gpu[name] = (b[..., off:off + s].unsqueeze(2) for b in (base, base.cuda()))
        elif case == 'transposed':
            for name in ('x', 'dt', 'z'):
                base = torch.randn((n, ch, l), generator=g).to(t)
                v[name], gpu[name] = base.transpose(1, 2), base.cuda().transpose(1, 2)
            base = torch.randn((n, 1, s, l), generator=g).to(t)
            v['b'], gpu['b'] = (b.permute(0, 3, 1, 2) for b in (base, base.cuda()))
        else:
            for name in ('x', 'b'):
                v[name] = v[name][:1].expand_as(v[name])
                gpu[name] = v[name].cuda()[:1].expand_as(v[name])
            v['state'] = v['state'][:, :1].expand(n, ch, s)
            gpu['state'] = v['state'].cuda()[:, :1].expand(n, ch, s)
        check(v, lengths=True, on_gpu=gpu, label=case)


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(0, 5, 8, 4, 1), (3, 0, 8, 4, 2), (0, 0, 8, 4, 1)])
def test_nothing(native, torch_cuda, shape):
    v = make(*shape, torch.float32)
    leaves = {k: v[k].cuda().requires_grad_() for k in NAMES}
    y, last = run(v, leaves, True, None, True)
    assert y.shape == v['x'].shape and torch.equal(last, leaves['state'])
    grads = dict(zip(NAMES, torch.autograd.grad([y, last], list(leaves.values()), [v['dy'].cuda(), v['dlast'].cuda()])))
    assert torch.equal(grads['state'], v['dlast'].cuda())
    assert not any(grads[k].any() for k in NAMES if k != 'state')


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(1, 4, 16, 1), (5, 33, 16, 1), (3, 200, 7, 2), (2, 9, 64, 3), (300, 12, 1, 1), (2, 140, 32, 1),
                                   # blocks full of channels, as many states as lanes have: every access whole
                                   (7, 64, 16, 2), (2, 128, 4, 1), (3, 64, 8, 1), (2, 32, 32, 2), (2, 16, 64, 1)])
@pytest.mark.parametrize('dtype', TYPES)
def test_one_token(native, torch_cuda, shape, dtype):
    """Step by step against one call's reference, in place and to another tensor."""
    n, ch, s, groups = shape
    l = 5
    v = make(n, l, ch, s, groups, TYPES[dtype], 6)
    ref = ScanReference(*(v[k] for k in NAMES[:8]), True, v['state'])
    q = {k: v[k].cuda() for k in NAMES}
    results = []
    for out_of_place in (False, True):
        state = q['state'].clone()
        for t in range(l):
            new, before = (torch.empty_like(state) if out_of_place else None), state.clone()
            y = torch_module.selective_scan_step(q['x'][:, t], q['dt'][:, t], q['a'], q['b'][:, t], q['c'][:, t], state, q['d'],
                                                 q['z'][:, t], q['dt_bias'], state_out=new)
            assert_close(y, ref.y[:, t], ref.tol_y[:, t], f'y {t}')
            if out_of_place:
                assert torch.equal(state, before)
                state = new
        assert_close(state, ref.last, ref.tol_last, 'state')
        results.append(state)
    assert torch.equal(*results)
    y = torch_module.selective_scan_step(q['x'][:, 0], q['dt'][:, 0], q['a'], q['b'][:, 0], q['c'][:, 0], q['state'].clone())
    bare = ScanReference(*(v[k][:, :1] if k not in 'a' else v[k] for k in NAMES[:5]), state=v['state'])
    assert_close(y, bare.y[:, 0], bare.tol_y[:, 0])


@pytest.mark.gpu
def test_states_in_slices_of_a_cache(native, torch_cuda):
    v = make(3, 1, 20, 16, 1, torch.bfloat16, 7)
    q = {k: v[k].cuda() for k in NAMES}
    args = [q[k][:, 0] if k != 'a' else q[k] for k in NAMES[:5]]
    want = q['state'].clone()
    y = torch_module.selective_scan_step(*args, want)
    cache = torch.full((8, 24, 21), 7.0, device='cuda')
    part = cache[2:8:2, 2:22, 3:19]  # every second slot, rows of odd spacing
    part.copy_(q['state'])
    assert torch.equal(torch_module.selective_scan_step(*args, part), y) and torch.equal(part, want)
    part.fill_(7.0)
    assert (cache == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_prompts_in_pieces(native, torch_cuda, dtype):
    v = make(2, 190, 24, 16, 1, TYPES[dtype], 8)
    ref = ScanReference(*(v[k] for k in NAMES[:8]))
    q = {k: v[k].cuda() for k in NAMES}
    state, parts = None, []
    for a, e in ((0, 1), (1, 20), (20, 100), (100, 190)):
        piece = {k: q[k][:, a:e] if k in ('x', 'dt', 'b', 'c', 'z') else q[k] for k in NAMES if k != 'state'}
        piece['state'] = state
        y, state = run(v, piece, True, None, True)
        parts.append(y)
    assert_close(torch.cat(parts, 1), ref.y, ref.tol_y)
    assert_close(state, ref.last, ref.tol_last)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f32', 'f16'])
def test_extreme_step_sizes(native, torch_cuda, dtype):
    """softplus far from zero: no underflow trouble below, the argument itself
    above; decays of 0 and of 1."""
    v = make(2, 40, 12, 16, 1, TYPES[dtype], 9)
    v['dt'] = torch.linspace(-60, 60, 40).reshape(1, 40, 1).expand(2, 40, 12).contiguous().to(TYPES[dtype])
    v['dt_bias'] = torch.zeros(12)
    check(v)
    v['a'] = torch.zeros_like(v['a'])
    v['dt'] = v['dt'] * 0.1
    check(v)


@pytest.mark.gpu
def test_infinities_stay_in_their_channel(native, torch_cuda):
    v = make(2, 40, 36, 16, 1, torch.float32, 10)
    ref = ScanReference(*(v[k] for k in NAMES[:8]))
    v['x'][1, 20, 5] = float('inf')
    q = {k: v[k].cuda() for k in NAMES[:8]}
    y = run(v, q, True, None, False).cpu()
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[1, 20:, 5] = True
    assert not torch.isfinite(y[hit]).any()
    assert_close(y[~hit], ref.y[~hit], ref.tol_y[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize('segments', [False, True])
def test_long_sequences(native, torch_cuda, segments):
    """Two thousand tokens with decays close to 1, whose errors add up."""
    n, ch = (1, 8) if segments else (4000, 8)
    v = make(n, 2048, ch, 4, 1, torch.float32, 11)
    few = {k: v[k][:2] if v[k].shape[0] == n and k not in ('a', 'd', 'dt_bias') else v[k] for k in v}
    ref = ScanReference(*(few[k] for k in NAMES[:8]), True, few['state']).backward(few['dy'], few['dlast'])
    leaves = {k: v[k].cuda().requires_grad_() for k in NAMES}
    y, last = run(v, leaves, True, None, True)
    assert ('parts=1 ' in api.Native().last_plan()) != segments
    assert_close(y[:2], ref.y, ref.tol_y)
    assert_close(last[:2], ref.last, ref.tol_last)
    grads = dict(zip(NAMES, torch.autograd.grad([y, last], list(leaves.values()), [v['dy'].cuda(), v['dlast'].cuda()])))
    for name, key in (('x', 'dx'), ('dt', 'ddt'), ('z', 'dz'), ('b', 'db'), ('c', 'dc'), ('state', 'dstate')):
        assert_close(grads[name][:2], getattr(ref, key), getattr(ref, 'tol_' + key), key)


@pytest.mark.gpu
def test_more_than_32_bits_of_elements(native, torch_cuda):
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip('needs 80 GB of device memory')
    n, l, ch = 2, 33000, 65540
    v = make(1, 40, ch, 1, 1, torch.bfloat16, 12)
    big = lambda t, fill: torch.full((n, l) + t.shape[2:], fill, dtype=t.dtype, device='cuda')
    q = {'x': big(v['x'], 0.0), 'dt': big(v['dt'], -1.0), 'b': big(v['b'], 1.0), 'c': big(v['c'], 1.0), 'a': v['a'].cuda()}
    for k in ('x', 'dt', 'b', 'c'):
        q[k][-1, -40:] = v[k][0].cuda()
    y, last = run(v, q, True, None, True)
    ref = ScanReference(*(v[k] for k in NAMES[:5]))
    assert_close(y[-1:, -40:], ref.y, ref.tol_y)
    assert_close(last[-1:], ref.last, ref.tol_last)
    assert not y[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(2, 200, 24, 16, 1), (2, 37, 33, 7, 3), (64, 64, 64, 16, 1)])
def test_streams_graphs_and_repetition(native, torch_cuda, shape):
    v = {k: t.cuda() for k, t in make(*shape, torch.bfloat16, 13).items()}

    def step(x, dy):
        leaves = {k: (x if k == 'x' else v[k]).detach().requires_grad_() for k in NAMES}
        y, last = run(v, leaves, True, v['lengths'], True)
        return (y.detach(), last.detach(), *torch.autograd.grad([y, last], list(leaves.values()), [dy, v['dlast']]))
    want = step(v['x'], v['dy'])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(v['x'], v['dy'])
        again = step(v['x'], v['dy'])
        sx, sdy = torch.zeros_like(v['x']), torch.zeros_like(v['dy'])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(sx, sdy)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    for _ in range(2):
        sx.copy_(v['x'])
        sdy.copy_(v['dy'])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        sx.zero_()


@pytest.mark.gpu
def test_gradients_of_some_operands(native, torch_cuda):
    v = make(2, 30, 12, 8, 2, torch.float32, 14)
    full = {k: v[k].cuda().requires_grad_() for k in NAMES}
    want = dict(zip(NAMES, torch.autograd.grad(run(v, full, True, None, True), list(full.values()),
                                               [v['dy'].cuda(), v['dlast'].cuda()])))
    for name in NAMES:
        q = {k: v[k].cuda() for k in NAMES}
        q[name].requires_grad_()
        got, = torch.autograd.grad(run(v, q, True, None, True), q[name], [v['dy'].cuda(), v['dlast'].cuda()])
        assert torch.equal(got, want[name]), name
    # the last state alone
    only, = torch.autograd.grad(run(v, full, True, None, True)[1], full['state'], v['dlast'].cuda())
    ref = ScanReference(*(v[k] for k in NAMES[:8]), True, v['state']).backward(torch.zeros_like(v['dy']), v['dlast'])
    assert_close(only, ref.dstate, ref.tol_dstate)


@pytest.mark.gpu
def test_refusals_of_the_front_end(native, torch_cuda):
    v = {k: t.cuda() for k, t in make(2, 10, 8, 4, 2, torch.float32).items()}
    base = [v[k] for k in NAMES[:5]]

    def call(at=None, value=None, **kw):
        args = list(base)
        if at is not None:
            args[at] = value
        return torch_module.selective_scan(*args, **kw)
    wide = torch.randn(2, 10, 2, 65, device='cuda')
    for bad in (lambda: call(1, v['dt'][:, :9]), lambda: call(1, v['dt'].half()), lambda: call(2, v['a'][:, :3]),
                lambda: call(3, v['b'][..., :3]), lambda: call(3, v['b'][:, :, :1]), lambda: call(4, v['c'].half()),
                lambda: call(D=v['d'][:7]), lambda: call(z=v['z'][:1]), lambda: call(dt_bias=v['d'].double()),
                lambda: call(state=v['state'].half()), lambda: call(state=v['state'][:, :4]), lambda: call(0, v['x'].cpu()),
                lambda: call(2, v['a'].cpu()),
                lambda: torch_module.selective_scan(v['x'], v['dt'], torch.randn(8, 65, device='cuda'), wide, wide),
                lambda: torch_module.selective_scan(v['x'][..., :7], v['dt'][..., :7], v['a'][:7], v['b'], v['c'])):
        with pytest.raises(api.NativeError):
            bad()
    for bad in (lambda: call(0, v['x'][0]), lambda: call(lengths=v['lengths'][:1]), lambda: call(lengths=v['lengths'].cpu())):
        with pytest.raises(ValueError):
            bad()
    step = lambda state, out=None: torch_module.selective_scan_step(*(t[:, 0] if t.dim() > 2 else t for t in base), state,
                                                                    state_out=out)
    with pytest.raises(RuntimeError):
        step(v['state'].clone().requires_grad_())
    cache = torch.zeros(2, 9, 4, device='cuda')
    with pytest.raises(api.NativeError):
        step(cache[:, :8], cache[:, 1:])
    with pytest.raises(api.NativeError):
        step(torch.zeros(2, 4, 8, device='cuda').transpose(1, 2))
    leaf = v['x'].clone().requires_grad_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(call(0, leaf).sum(), leaf, create_graph=True)
    y = call(0, leaf)
    y.sum().backward(retain_graph=True)
    y.sum().backward()
    with pytest.raises(RuntimeError):
        y.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_block_in_training_prefill_and_steps(native, torch_cuda, dtype):
    """Layer norm, convolution and scan as a block runs them: prompts of several
    lengths, then tokens, against the whole sequences at once; gradients reach
    every parameter."""
    torch.manual_seed(1)
    block = torch_module.B200SelectiveBlock(48, states=8, device='cuda')
    x = torch.randn(3, 40, 48, device='cuda')
    if dtype == 'bf16':
        for m in (block.norm, block.input, block.conv, block.select, block.dt, block.output):
            m.to(torch.bfloat16)
        x = x.to(torch.bfloat16)
    tol = dict(rtol=1e-3, atol=1e-4) if dtype == 'f32' else dict(rtol=0.05, atol=0.1)
    want = block(x)
    want.float().square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any() for p in block.parameters())
    ends = [33, 1, 20]
    with torch.no_grad():
        y, states = block.prefill(x, torch.tensor(ends, device='cuda'))
        for i, e in enumerate(ends):
            torch.testing.assert_close(y[i, :e], want[i, :e], **tol)
        for t in range(7):
            rows = torch.arange(3, device='cuda')
            token = x[rows, torch.tensor(ends, device='cuda') + t]
            torch.testing.assert_close(block.step(token, states), want[rows, torch.tensor(ends, device='cuda') + t], **tol)
        states = block.new_states(3)
        first = block.step(x[:, 0], states)
        torch.testing.assert_close(first, want[:, 0], **tol)
        y, _ = block.prefill(x[:, 1:], None, states)
        torch.testing.assert_close(y, want[:, 1:], **tol)


def test_reference_gradient_against_differences():
    """The formulas that the GPU tests compare with, against difference quotients."""
    v = {k: t.double() if t.is_floating_point() else t for k, t in make(2, 9, 6, 3, 2, torch.float32, 15).items()}

    def value(**moved):
        q = {**v, **moved}
        r = ScanReference(*(q[k] for k in NAMES[:8]), True, q['state'], v['lengths'])
        return (v['dy'] * r.y).sum() + (v['dlast'] * r.last).sum()
    ref = ScanReference(*(v[k] for k in NAMES[:8]), True, v['state'], v['lengths']).backward(v['dy'], v['dlast'])
    for name, key in zip(NAMES, ('dx', 'ddt', 'da', 'db', 'dc', 'dd', 'dz', 'ddt_bias', 'dstate')):
        way = torch.randn(v[name].shape, generator=torch.Generator().manual_seed(16)).double()
        eps = 1e-5
        slope = (value(**{name: v[name] + eps * way}) - value(**{name: v[name] - eps * way})) / (2 * eps)
        assert abs(slope - (getattr(ref, key) * way).sum()) <= 1e-7 * (1 + abs(slope)), name
