"""gc_b200_layer_norm and its gradient against the formulas in 64 bits.  A row is
an image of one pixel and one group: the tolerances are those of group norm."""
import pytest
import torch

from groupconv_atlas_b200 import api, torch_module
from tests.norm_helpers import HALF, NormReference, assert_close

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}

# (rows, row length): one element, less than a vector, a vector, teams of several
# to a warp, a warp with one, two and four vectors a lane, blocks as teams, odd
# lengths (single elements, four and sixteen a thread), rows for which a block
# needs two and four vectors a thread, rows too long for registers, more rows
# than one turn of the blocks
SHAPES = [(1, 1), (3, 3), (5, 8), (70, 16), (33, 40), (257, 96), (50, 256), (19, 384), (21, 512), (40, 768), (9, 1024),
          (17, 1001), (6, 2048), (3, 2056), (4, 4096), (5, 4104), (3, 8192), (2, 8200), (3, 129), (4, 2047), (3, 6001),
          (2, 9001), (2, 20000), (20000, 12), (9000, 33), (2500, 600),
          # odd lengths in aligned vectors: one, two and four a thread, a warp and blocks as teams, rows of every
          # place within 16 bytes, more than one turn
          (11, 259), (300, 515), (1700, 333), (70, 1023), (33, 4095), (9, 2053), (5000, 135), (40, 510), (23, 254)]


def make(shape, dtype, seed=0, params=torch.float32):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]
    x = (torch.randn(shape, generator=g) * 1.5 + 0.5 * torch.randn(c, generator=g)).to(dtype)
    gamma, beta = (1 + 0.3 * torch.randn(c, generator=g)).to(params), (0.3 * torch.randn(c, generator=g)).to(params)
    return x, gamma, beta, torch.randn(shape, generator=g).to(dtype)


def check(x, gamma, beta, dy, eps=1e-5, device_x=None, device_dy=None, label=''):
    """Through the front end, with its gradient; leaves on the GPU."""
    c = x.shape[-1]
    ref = NormReference(x.reshape(-1, c), 1, gamma, beta, eps).backward(dy.reshape(-1, c))
    leaves = [(x.cuda() if device_x is None else device_x).detach().requires_grad_()]
    leaves += [t.cuda().requires_grad_() for t in (gamma, beta) if t is not None]
    given = [t is not None for t in (gamma, beta)]
    w, b = (leaves[1 + sum(given[:i])] if given[i] else None for i in (0, 1))
    y = torch_module.layer_norm(leaves[0], w, b, eps)
    plan = api.Native().last_plan()
    grads = torch.autograd.grad(y, leaves, dy.cuda() if device_dy is None else device_dy)
    assert y.dtype == x.dtype and y.is_contiguous() and y.shape == x.shape
    assert_close(y.reshape(-1, c), ref.y, ref.tol_y, f'{label} y [{plan}]')
    assert_close(grads[0].reshape(-1, c), ref.dx, ref.tol_dx, f'{label} dx')
    for name, got in zip([n for n, ok in zip(('dgamma', 'dbeta'), given) if ok], grads[1:]):
        want = getattr(ref, name)
        assert_close(got, want, getattr(ref, 'tol_' + name) + HALF[got.dtype] * want.abs() + 2.0 ** -25, f'{label} {name}')
    return y, grads


@pytest.mark.gpu
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: 'x'.join(map(str, s)))
@pytest.mark.parametrize('dtype', TYPES)
def test_rows(native, torch_cuda, shape, dtype):
    check(*make(shape, TYPES[dtype]))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['f16', 'bf16'])
@pytest.mark.parametrize('c', [96, 1001])
def test_parameters_of_the_data_type_and_none(native, torch_cuda, dtype, c):
    x, gamma, beta, dy = make((40, c), TYPES[dtype], 1, TYPES[dtype])
    check(x, gamma, beta, dy)
    check(x, gamma, None, dy)
    check(x, None, beta, dy)
    check(x, None, None, dy)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_layouts(native, torch_cuda, dtype):
    """Row slices, odd offsets, the pixels of a channels_last image, other orders
    (copied), one to six axes."""
    t = TYPES[dtype]
    for shape, view in [((7, 5, 200), lambda v: v[..., :96]), ((7, 5, 200), lambda v: v[..., 1:97]),
                        ((9, 101), lambda v: v[:, 3:99]), ((2, 96, 5, 4), lambda v: v.permute(0, 2, 3, 1)),
                        ((6, 8, 96), lambda v: v.transpose(0, 1)), ((96, 30), lambda v: v.t()), ((96,), lambda v: v),
                        ((2, 1, 3, 2, 2, 96), lambda v: v), ((1, 96), lambda v: v.expand(5, 96))]:
        g = torch.Generator().manual_seed(3)
        base = torch.randn(shape, generator=g).to(t)
        if len(shape) == 4:
            base = base.contiguous(memory_format=torch.channels_last)
        x = view(base)
        _, gamma, beta, _ = make((1, 96), t)
        dy = torch.randn(x.shape, generator=g).to(t)
        wide = torch.randn(x.shape[:-1] + (100,), generator=g).to(t).cuda()  # a gradient with rows of its own spacing
        wide[..., :96] = dy.cuda()
        check(x, gamma, beta, dy, device_x=view(base.cuda()), device_dy=wide[..., :96], label=str(shape))


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(0, 16), (3, 0, 16), (0, 1001)])
def test_no_rows(native, torch_cuda, shape):
    x, gamma, beta, dy = make(shape, torch.float32)
    leaves = [t.cuda().requires_grad_() for t in (x, gamma, beta)]
    y = torch_module.layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    assert y.shape == shape and grads[0].shape == shape and not grads[1].any() and not grads[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize('c', [40, 1001, 4096, 20000])
def test_infinities_stay_in_their_row(native, torch_cuda, c):
    x, gamma, beta, dy = make((6, c), torch.float32, 5)
    ref = NormReference(x, 1, gamma, beta)
    x[1, c // 2], x[4, 0] = float('inf'), float('nan')
    y = torch_module.layer_norm(x.cuda(), gamma.cuda(), beta.cuda()).cpu()
    assert torch.isnan(y[[1, 4]]).all()
    rest = [0, 2, 3, 5]
    assert_close(y[rest], ref.y[rest], ref.tol_y[rest])


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(300, 96), (40, 1001), (64, 2048), (3, 9000)])
@pytest.mark.parametrize('level', [1000.0, -3e4])
def test_rows_far_from_zero(native, torch_cuda, shape, level):
    """The variance is of differences from the mean; the tolerance grows with
    max|x| / sigma and no further."""
    x, gamma, beta, dy = make(shape, torch.float32, 6)
    check(x + level, gamma, beta, dy)


@pytest.mark.gpu
@pytest.mark.parametrize('c', [96, 1001])
def test_long_sums_of_one_sign(native, torch_cuda, c):
    """dbeta over rows whose dy is one value: added one after the other in 32 bits
    these would be off by hundreds of half steps."""
    value, rows = float.fromhex('0x1.171c02p0'), 200000
    x = torch.randn((rows, c), generator=torch.Generator(device='cuda').manual_seed(1), device='cuda').requires_grad_()
    w, b = torch.ones(c, device='cuda', requires_grad=True), torch.zeros(c, device='cuda', requires_grad=True)
    y = torch_module.layer_norm(x, w, b)
    _, dbeta = torch.autograd.grad(y, [x, b], torch.full_like(y, value))
    want = torch.full((c,), rows * value, dtype=torch.float64)
    assert_close(dbeta, want, 256 * 2.0 ** -24 * want)


@pytest.mark.gpu
def test_more_than_32_bits_of_elements(native, torch_cuda):
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip('needs 60 GB of device memory')
    rows, c = (1 << 21) + 5, 2056
    g = torch.Generator(device='cuda').manual_seed(2)
    x = torch.empty(rows, c, device='cuda', dtype=torch.bfloat16)
    x[:] = 0.25
    x[-70:] = torch.randn(70, c, generator=g, device='cuda').to(x.dtype)
    x.requires_grad_()
    w = torch.ones(c, device='cuda', requires_grad=True)
    y = torch_module.layer_norm(x, w)
    dy = torch.zeros_like(y)
    dy[-70:] = torch.randn(70, c, generator=g, device='cuda').to(x.dtype)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    ref = NormReference(x[-70:].detach().cpu(), 1).backward(dy[-70:].cpu())
    assert_close(y[-70:], ref.y, ref.tol_y)
    assert_close(dx[-70:], ref.dx, ref.tol_dx)
    assert_close(dw, ref.dgamma, ref.tol_dgamma + HALF[torch.float32] * ref.dgamma.abs() + 2.0 ** -25)
    assert not dx[:-70].any()


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(500, 96), (300, 1001), (40, 4096)])
def test_streams_graphs_and_repetition(native, torch_cuda, shape):
    """Bitwise the same on another stream, in a replayed graph with new inputs, and
    beside other work."""
    x, gamma, beta, dy = (t.cuda() for t in make(shape, torch.bfloat16, 8))

    def step(x, dy):
        leaves = [t.detach().requires_grad_() for t in (x, gamma, beta)]
        y = torch_module.layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    want = step(x, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            again = step(x, dy)
        sx, sdy = torch.zeros_like(x), torch.zeros_like(dy)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(sx, sdy)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    for _ in range(2):
        sx.copy_(x)
        sdy.copy_(dy)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        sx.zero_()


@pytest.mark.gpu
def test_modules(native, torch_cuda):
    model = torch.nn.Sequential(torch.nn.LayerNorm(48), torch.nn.Linear(48, 24), torch.nn.LayerNorm(24, bias=False),
                                torch.nn.LayerNorm((3, 24)), torch.nn.LayerNorm(24, elementwise_affine=False)).cuda()
    keys = list(model.state_dict())
    x = torch.randn(5, 3, 48, device='cuda')
    want = model(x)
    assert torch_module.substitute_layer_norm(model) == ['0', '2', '4']
    assert list(model.state_dict()) == keys and isinstance(model[3], torch.nn.LayerNorm)
    torch.testing.assert_close(model(x), want, rtol=1e-4, atol=1e-5)
    with pytest.raises(ValueError):
        model[0](x[..., :24])


@pytest.mark.gpu
def test_refusals_of_the_front_end(native, torch_cuda):
    x = torch.randn(4, 16, device='cuda')
    w = torch.ones(16, device='cuda')
    for bad in (dict(weight=torch.ones(15, device='cuda')), dict(weight=w.half()), dict(bias=w.cpu()), dict(eps=-1.0),
                dict(eps=float('nan'))):
        with pytest.raises(api.NativeError):
            torch_module.layer_norm(x, **bad)
    for t in (x.double(), x.int(), x.cpu(), x[:, :0]):
        with pytest.raises(api.NativeError):
            torch_module.layer_norm(t)
    y = torch_module.layer_norm(x.requires_grad_(), w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda t: torch_module.layer_norm(t, w), (x.detach(),))
    y = torch_module.layer_norm(x, w)
    with torch.no_grad():
        x += 1
    with pytest.raises(RuntimeError):  # what the gradient needs has changed
        y.sum().backward()
