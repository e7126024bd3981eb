"""gc_b200_causal_conv, its gradient and its form for one token against the
formulas in 64 bits."""
import pytest
import torch

from groupconv_atlas_b200 import api, torch_module
from tests.norm_helpers import HALF
from tests.sequence_helpers import ConvReference, assert_close

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}

# (N, L, C, K): one token, fewer tokens than taps, odd channels (single elements),
# one channel, whole and broken stretches of tokens, many sequences, more
# channels than a tile of columns
SHAPES = [(1, 1, 4, 4), (2, 2, 8, 4), (3, 17, 33, 3), (2, 9, 1, 2), (1, 200, 64, 4), (2, 65, 132, 4), (40, 7, 20, 4),
          (2, 70, 1000, 4), (3, 40, 12, 1), (2, 30, 24, 5), (2, 50, 7, 8), (1, 64, 516, 8), (2, 33, 260, 2), (1, 1000, 16, 4)]


def make(n, l, c, k, dtype, seed=0, params=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    params = params or dtype
    return {'x': r(n, l, c).to(dtype), 'w': (r(c, k) / k ** 0.5).to(params), 'b': (0.2 * r(c)).to(params),
            'state': r(n, k - 1, c).to(dtype), 'dy': r(n, l, c).to(dtype), 'dlast': r(n, k - 1, c).to(dtype),
            'lengths': torch.randint(0, l + 1, (n,), generator=g, dtype=torch.int32)}


def check(v, act='silu', bias=True, state=False, lengths=False, device_x=None, label=''):
    b, s, lens = v['b'] if bias else None, v['state'] if state else None, v['lengths'] if lengths else None
    ref = ConvReference(v['x'], v['w'], b, act, s, lens)
    dy = ref.away_from_kinks(v['dy'])
    ref.backward(dy, v['dlast'] if state else None)
    x = (v['x'].cuda() if device_x is None else device_x).detach().requires_grad_()
    w = v['w'].cuda().requires_grad_()
    bd = b.cuda().requires_grad_() if bias else None
    sd = s.cuda().requires_grad_() if state else None
    lens = lens.cuda() if lengths else None
    out = torch_module.causal_conv(x, w, bd, act, sd, lens, return_state=state)
    y, last = out if state else (out, None)
    label += f' [{api.Native().last_plan()}]'
    assert y.dtype == x.dtype and y.is_contiguous()
    assert_close(y, ref.y, ref.tol_y, f'y {label}')
    leaves = [t for t in (x, w, bd, sd) if t is not None]
    grads = torch.autograd.grad([y, last] if state else [y], leaves, [dy.cuda(), v['dlast'].cuda()] if state else [dy.cuda()])
    got = dict(zip([k for k, t in zip(('dx', 'dw', 'db', 'dstate'), (x, w, bd, sd)) if t is not None], grads))
    assert_close(got['dx'], ref.dx, ref.tol_dx, f'dx {label}')
    for name in ('dw', 'db'):
        if name in got:
            want = getattr(ref, name)
            assert_close(got[name], want, getattr(ref, 'tol_' + name) + HALF[got[name].dtype] * want.abs() + 2.0 ** -25, f'{name} {label}')
    if state:
        assert torch.equal(last.detach().cpu().double(), ref.last)
        assert_close(got['dstate'], ref.dstate, ref.tol_dstate, f'dstate {label}')
    if lengths:
        assert not (y.detach().cpu() * ~ref.inside).any() and not (got['dx'].cpu() * ~ref.inside).any()


@pytest.mark.gpu
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: 'x'.join(map(str, s)))
@pytest.mark.parametrize('dtype', TYPES)
def test_sequences(native, torch_cuda, shape, dtype):
    v = make(*shape, TYPES[dtype])
    check(v)
    check(v, state=True, lengths=True)


@pytest.mark.gpu
@pytest.mark.parametrize('act', ['none', 'relu', 'relu6', 'silu'])
@pytest.mark.parametrize('params', ['f32', 'f16'])
def test_activations_and_parameters(native, torch_cuda, act, params):
    v = make(2, 21, 40, 4, torch.float16, 1, TYPES[params])
    for key in ('x', 'state'):
        v[key] = v[key] * 4
    check(v, act)
    check(v, act, bias=False, lengths=True)


@pytest.mark.gpu
@pytest.mark.parametrize('lengths', [[0, 1, 2, 3], [40, 4, 100, -7], [0, 0, 0, 0], [39, 8, 16, 17]])
@pytest.mark.parametrize('c', [8, 9])
def test_lengths(native, torch_cuda, lengths, c):
    """None, one, fewer tokens than taps, all; values outside 0..L; what lies
    behind an end is not read."""
    v = make(4, 40, c, 4, torch.float32, 2)
    v['lengths'] = torch.tensor(lengths, dtype=torch.int32)
    ends = v['lengths'].clamp(0, 40)
    check(v, state=True, lengths=True)
    x, w, b = v['x'].cuda(), v['w'].cuda(), v['b'].cuda()
    clean, last = torch_module.causal_conv(x, w, b, 'silu', lengths=v['lengths'].cuda(), return_state=True)
    for bad in (float('nan'), float('inf')):
        for i, e in enumerate(ends.tolist()):
            x[i, e:] = bad
        for kind in (torch.int32, torch.int64):
            y, s = torch_module.causal_conv(x, w, b, 'silu', lengths=v['lengths'].to(kind).cuda(), return_state=True)
            assert torch.equal(y, clean) and torch.equal(s, last)
    leaf = x.requires_grad_()
    dy = v['dy'].cuda()
    for i, e in enumerate(ends.tolist()):
        dy[i, e:] = float('nan')
    dx, = torch.autograd.grad(torch_module.causal_conv(leaf, w, b, 'silu', lengths=v['lengths'].cuda()), leaf, dy)
    assert torch.isfinite(dx).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_layouts(native, torch_cuda, dtype):
    """Channel slices, odd offsets, tokens before sequences, other orders (copied)."""
    for shape, view in [((2, 30, 64), lambda t: t[..., :32]), ((2, 30, 64), lambda t: t[..., 3:35]),
                        ((30, 2, 32), lambda t: t.transpose(0, 1)), ((2, 32, 30), lambda t: t.transpose(1, 2)),
                        ((2, 60, 32), lambda t: t[:, ::2]), ((1, 30, 32), lambda t: t.expand(2, 30, 32))]:
        v = make(2, 30, 32, 4, TYPES[dtype], 4)
        base = torch.randn(shape, generator=torch.Generator().manual_seed(5)).to(TYPES[dtype])
        v['x'] = view(base)
        check(v, state=True, lengths=True, device_x=view(base.cuda()), label=str(shape))


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(0, 5, 8), (3, 0, 8), (0, 0, 8)])
def test_nothing(native, torch_cuda, shape):
    n, l, c = shape
    v = make(n, l, c, 4, torch.float32)
    x, w, b, s = (v[k].cuda().requires_grad_() for k in ('x', 'w', 'b', 'state'))
    y, last = torch_module.causal_conv(x, w, b, 'silu', s, return_state=True)
    assert y.shape == shape and torch.equal(last, s)
    grads = torch.autograd.grad([y, last], [x, w, b, s], [v['dy'].cuda(), v['dlast'].cuda()])
    assert not grads[1].any() and not grads[2].any() and torch.equal(grads[3], v['dlast'].cuda())


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(1, 4, 4), (5, 33, 3), (3, 1000, 4), (7, 12, 1), (2, 20, 6), (2, 9, 8), (300, 64, 2)])
@pytest.mark.parametrize('dtype', TYPES)
def test_one_token(native, torch_cuda, shape, dtype):
    """A step is the sequence's next token: bitwise the same as in one call, in
    place and to another tensor."""
    n, c, k = shape
    v = make(n, 6, c, k, TYPES[dtype], 6)
    x, w, b, s = (v[key].cuda() for key in ('x', 'w', 'b', 'state'))
    want, last = torch_module.causal_conv(x, w, b, 'silu', s, return_state=True)
    for out_of_place in (False, True):
        state = s.clone()
        for t in range(6):
            new = torch.empty_like(state) if out_of_place else None
            before = state.clone()
            y = torch_module.causal_conv_step(x[:, t], w, state, b, 'silu', state_out=new)
            assert torch.equal(y, want[:, t])
            if out_of_place:
                assert torch.equal(state, before)
                state = new
        assert torch.equal(state, last)


@pytest.mark.gpu
def test_states_in_slices_of_a_cache(native, torch_cuda):
    v = make(3, 1, 40, 4, torch.bfloat16, 7)
    x, w, s = v['x'][:, 0].cuda(), v['w'].cuda(), v['state'].cuda()
    want = s.clone()
    y = torch_module.causal_conv_step(x, w, want)
    cache = torch.full((8, 5, 48), 7.0, device='cuda', dtype=torch.bfloat16)
    part = cache[2:5, 1:4, 4:44]
    part.copy_(s)
    assert torch.equal(torch_module.causal_conv_step(x, w, part), y) and torch.equal(part, want)
    part.fill_(7.0)
    assert (cache == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_prompts_in_pieces(native, torch_cuda, dtype):
    v = make(3, 90, 24, 4, TYPES[dtype], 8)
    x, w, b = (v[k].cuda() for k in ('x', 'w', 'b'))
    want, last = torch_module.causal_conv(x, w, b, 'silu', return_state=True)
    state, parts = None, []
    for a, e in ((0, 1), (1, 3), (3, 50), (50, 90)):
        y, state = torch_module.causal_conv(x[:, a:e], w, b, 'silu', state, return_state=True)
        parts.append(y)
    assert torch.equal(torch.cat(parts, 1), want) and torch.equal(state, last)


@pytest.mark.gpu
def test_infinities_reach_what_they_multiply(native, torch_cuda):
    """An infinite input makes K results of its channel infinite or NaN, and no
    others; K below the kernel's own number of taps."""
    for k in (1, 2, 3, 4, 6):
        v = make(2, 40, 12, k, torch.float32, 9)
        ref = ConvReference(v['x'], v['w'], v['b'])
        x = v['x'].clone()
        x[1, 20, 5] = float('inf')
        y = torch_module.causal_conv(x.cuda(), v['w'].cuda(), v['b'].cuda()).cpu()
        hit = torch.zeros_like(y, dtype=torch.bool)
        hit[1, 20:20 + k, 5] = True
        assert not torch.isfinite(y[hit]).any()
        assert_close(y[~hit], ref.y[~hit], ref.tol_y[~hit], f'K {k}')


@pytest.mark.gpu
def test_more_than_32_bits_of_elements(native, torch_cuda):
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip('needs 60 GB of device memory')
    n, l, c = 3, 350001, 4100
    v = make(1, 80, c, 4, torch.bfloat16, 10)
    x = torch.zeros(n, l, c, dtype=torch.bfloat16, device='cuda')
    x[-1, -80:] = v['x'][0].cuda()
    x.requires_grad_()
    w = v['w'].cuda().requires_grad_()
    y = torch_module.causal_conv(x, w, None, 'silu')
    dy = torch.zeros_like(y)
    dy[-1, -80:] = v['dy'][0].cuda()
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    ref = ConvReference(v['x'], v['w'], None, 'silu').backward(v['dy'])
    assert_close(y[-1:, -80:], ref.y, ref.tol_y)
    assert_close(dx[-1:, -80:], ref.dx, ref.tol_dx)
    assert_close(dw, ref.dw, ref.tol_dw + HALF[dw.dtype] * ref.dw.abs() + 2.0 ** -25)
    assert not dx[:-1].any() and not y[:-1].any()


@pytest.mark.gpu
@pytest.mark.parametrize('c', [64, 33])
def test_streams_graphs_and_repetition(native, torch_cuda, c):
    v = {k: t.cuda() for k, t in make(3, 200, c, 4, torch.bfloat16, 11).items()}

    def step(x, dy):
        leaves = [t.detach().requires_grad_() for t in (x, v['w'], v['b'], v['state'])]
        y, last = torch_module.causal_conv(*leaves[:3], 'silu', leaves[3], v['lengths'], True)
        return (y.detach(), last.detach(), *torch.autograd.grad([y, last], leaves, [dy, v['dlast']]))
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
def test_module(native, torch_cuda):
    conv = torch.nn.Conv1d(24, 24, 4, groups=24, padding=3).cuda()
    x = torch.randn(2, 30, 24, device='cuda')
    want = torch.nn.functional.silu(conv(x.transpose(1, 2))[..., :30]).transpose(1, 2)
    fused = torch_module.B200CausalConv1d(conv, torch.nn.SiLU())
    torch.testing.assert_close(fused(x), want, rtol=1e-4, atol=1e-5)
    y, state = fused(x[:, :20], return_state=True)
    with torch.no_grad():
        torch.testing.assert_close(fused.step(x[:, 20], state), want[:, 20], rtol=1e-4, atol=1e-5)
    for bad in (torch.nn.Conv1d(24, 24, 4), torch.nn.Conv1d(24, 24, 4, groups=24, padding=1),
                torch.nn.Conv1d(24, 24, 9, groups=24), torch.nn.Conv1d(24, 24, 4, groups=24, stride=2),
                torch.nn.Conv1d(24, 24, 4, groups=24, dilation=2)):
        with pytest.raises(ValueError):
            torch_module.B200CausalConv1d(bad)


@pytest.mark.gpu
def test_refusals_of_the_front_end(native, torch_cuda):
    v = {k: t.cuda() for k, t in make(2, 10, 8, 4, torch.float32).items()}
    x, w, s = v['x'], v['w'], v['state']
    call = torch_module.causal_conv
    for bad in (lambda: call(x, w[:7]), lambda: call(x, w.half()), lambda: call(x, w, v['b'][:3]),
                lambda: call(x, w, state=s[:, :2]), lambda: call(x, w, state=s.half()), lambda: call(x.double(), w.double()),
                lambda: call(x, torch.randn(8, 9, device='cuda')), lambda: call(x.cpu(), w), lambda: call(x, w.cpu())):
        with pytest.raises(api.NativeError):
            bad()
    for bad in (lambda: call(x[0], w), lambda: call(x, w[0]), lambda: call(x, w, activation='gelu'),
                lambda: call(x, w, lengths=v['lengths'][:1]), lambda: call(x, w, lengths=v['lengths'].float()),
                lambda: call(x, w, lengths=v['lengths'].cpu()), lambda: torch_module.causal_conv_step(x, w, s)):
        with pytest.raises(ValueError):
            bad()
    step = torch_module.causal_conv_step
    with pytest.raises(RuntimeError):
        step(x[:, 0].clone().requires_grad_(), w, s)
    cache = torch.zeros(2, 4, 8, device='cuda')
    with pytest.raises(api.NativeError):  # shifted by a token: neither the state itself nor apart from it
        step(x[:, 0], w, cache[:, :3], state_out=cache[:, 1:])
    with pytest.raises(api.NativeError):  # a state that would be copied
        step(x[:, 0], w, torch.zeros(2, 8, 3, device='cuda').transpose(1, 2))
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(call(leaf, w).sum(), leaf, create_graph=True)
    state = s.clone()
    y = call(leaf, w, state=state)
    with torch.no_grad():
        step(x[:, 0], w, state)  # writes what the gradient needs
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_reference_gradient_against_differences():
    """The formulas that the GPU tests compare with, against difference quotients."""
    v = {k: t.double() if t.is_floating_point() else t for k, t in make(2, 9, 3, 4, torch.float32, 12).items()}
    dy, dlast = v['dy'], v['dlast']

    def value(**moved):
        q = {**v, **moved}
        r = ConvReference(q['x'], q['w'], q['b'], 'silu', q['state'], v['lengths'])
        return (torch.where(r.inside, dy, 0.0) * r.y).sum() + (dlast * r.last).sum()
    ref = ConvReference(v['x'], v['w'], v['b'], 'silu', v['state'], v['lengths']).backward(dy, dlast)
    for name, grad in (('x', ref.dx), ('w', ref.dw), ('b', ref.db), ('state', ref.dstate)):
        way = torch.randn(v[name].shape, generator=torch.Generator().manual_seed(13)).double()
        eps = 1e-5
        slope = (value(**{name: v[name] + eps * way}) - value(**{name: v[name] - eps * way})) / (2 * eps)
        assert abs(slope - (grad * way).sum()) <= 1e-7 * (1 + abs(slope)), name
