"""Calls of the operators on sequences that meet: one tensor in several places,
steps captured into a graph, many short sequences, calls on two streams."""
import pytest
import torch

from groupconv_atlas_b200 import torch_module
from tests.test_selective_scan import NAMES, check, make, run


@pytest.mark.gpu
def test_one_tensor_in_several_places(native, torch_cuda):
    """x also as step sizes and gate, B also as C: the gradients add up."""
    v = {k: t.cuda() for k, t in make(2, 70, 24, 16, 1, torch.float32, 21).items()}
    places = {'x': 'x', 'dt': 'x', 'z': 'x', 'b': 'b', 'c': 'b'}
    apart = {k: v[places.get(k, k)].clone().requires_grad_() for k in NAMES}
    want = run(v, apart, True, v['lengths'], False)
    grads = dict(zip(NAMES, torch.autograd.grad(want, list(apart.values()), v['dy'])))
    once = {k: v[k].clone().requires_grad_() for k in ('x', 'b')}
    shared = {k: once[places[k]] if k in places else v[k] for k in NAMES}
    y = run(v, shared, True, v['lengths'], False)
    assert torch.equal(y, want)
    dx, db = torch.autograd.grad(y, [once['x'], once['b']], v['dy'])
    for got, parts in ((dx, ('x', 'dt', 'z')), (db, ('b', 'c'))):
        parts = torch.stack([grads[k].double() for k in parts])
        # at most two sums in 32 bits, each off by half a step of a partial sum
        assert ((got.double() - parts.sum(0)).abs() <= 2 * 2.0 ** -24 * 1.001 * parts.abs().sum(0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(5, 33, 7, 3), (4, 64, 16, 1)])
def test_captured_steps(native, torch_cuda, dtype, shape):
    """The convolution's and the scan's step as one graph, replayed token by token,
    beside the same calls made one by one."""
    n, ch, s, groups = shape
    l, taps = 6, 4
    v = {k: t.cuda() for k, t in make(n, l, ch, s, groups, dtype, 22).items()}
    weight, bias = torch.randn(ch, taps, device='cuda'), torch.randn(ch, device='cuda')
    first = torch.randn(n, taps - 1, ch, device='cuda').to(dtype)

    def token(t, x, dt, b, c, z):
        return [a.copy_(v[k][:, t]) for a, k in ((x, 'x'), (dt, 'dt'), (b, 'b'), (c, 'c'), (z, 'z'))]

    def step(x, dt, b, c, z, before, h):
        u = torch_module.causal_conv_step(x, weight, before, bias, 'silu')
        return torch_module.selective_scan_step(u, dt, v['a'], b, c, h, v['d'], z, v['dt_bias'])
    inputs = [torch.empty_like(v[k][:, 0]) for k in ('x', 'dt', 'b', 'c', 'z')]
    states = first.clone(), v['state'].clone()
    want = [step(*token(t, *inputs), *states) for t in range(l)]
    replayed = first.clone(), v['state'].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out = step(*inputs, *replayed)
    torch.cuda.current_stream().wait_stream(side)
    for t in range(l):
        token(t, *inputs)
        graph.replay()
        assert torch.equal(out, want[t])
    assert all(torch.equal(a, b) for a, b in zip(replayed, states))


@pytest.mark.gpu
def test_many_short_sequences(native, torch_cuda):
    """More partial sums of the parameters than 256."""
    check(make(300, 3, 9, 5, 1, torch.float32, 23), lengths=True)
    check(make(513, 2, 8, 16, 2, torch.bfloat16, 24))


@pytest.mark.gpu
def test_calls_on_two_streams(native, torch_cuda):
    """Training steps at once on two streams, each with workspaces of its own."""
    sets = [{k: t.cuda() for k, t in make(2, 300, 40, 16, 1, torch.bfloat16, s).items()} for s in (25, 26)]

    def step(v):
        leaves = {k: v[k].detach().requires_grad_() for k in NAMES}
        u = torch_module.layer_norm(leaves['x'])
        y = run(v, {**leaves, 'x': u}, True, v['lengths'], False)
        return [y.detach(), *torch.autograd.grad(y, list(leaves.values()), v['dy'])]
    want = [step(v) for v in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(4):
        got = []
        for v, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(step(v))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
