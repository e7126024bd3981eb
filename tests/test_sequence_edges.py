"""Layer norm, the causal convolution and the selective scan where calls can go
wrong: rows past 2^30 elements, long sums, values that are no numbers, what autograd
does around a call, first calls, calls of two threads."""
import pytest
import torch

from groupconv_atlas_b200 import api, torch_module
from tests import test_layer_norm


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
