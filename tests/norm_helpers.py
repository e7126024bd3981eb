"""Plain 64-bit forms of group normalisation and dropout, and the tolerances of
their GPU tests.

Tolerances.  u = 2^-24 is half a step of the kernels' 32-bit arithmetic, h half a
step of the stored type relative to the value.  A kernel's sum adds at most
about 64 values one after the other before partial sums are joined in trees, and
the variance is built from differences, so mean and standard deviation are off by
at most K u (1 + max|x| / sigma) relative to sigma, K = 256 (64 additions, the
squares' doubling of it, and a factor 2 for the trees).  That moves z by
  e_z = K u (1 + max|x| / sigma) (|gamma| (|xhat| + 1) + |beta|).
act is Lipschitz with 1.1 (SiLU; 1 for the others), act' with 0.5 (SiLU; the
tests give elements of the others that lie within e_z of a kink a dy of 0).
"""
import numpy as np
import torch

U = 2.0 ** -24
K = 256
# Half a step relative to the value; results in the subnormal range of float16
# are off by at most half of its smallest step.
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def philox(count, seed, offset):
    """`count` 16-bit draws of Philox4x32-10."""
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    blocks = np.arange((count + 7) // 8, dtype=u)
    c = [blocks & low, blocks >> u(32), np.full_like(blocks, offset & 0xFFFFFFFF), np.full_like(blocks, offset >> 32)]
    for i in range(10):
        k0 = u((seed + i * 0x9E3779B9) & 0xFFFFFFFF)
        k1 = u(((seed >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ k0, b & low, (a >> u(32)) ^ c[3] ^ k1, a & low]
    return np.stack(c, 1).astype('<u4').reshape(-1).view('<u2')[:count]


def keep_mask(shape, p, seed, offset, scope='element', layout='nhwc'):
    """(keep, 1 / (1 - q)): keep is shaped like the tensor, (N, C, ..)."""
    t = round(65536 * p)
    scale = 65536 / (65536 - t) if t < 65536 else 0.0
    n, c, rest = shape[0], shape[1] if len(shape) > 1 else 1, tuple(shape[2:])
    if scope == 'channel':
        keep = torch.from_numpy(philox(n * c, seed, offset) >= t).reshape((n, c) + (1,) * len(rest))
        return keep.expand(shape), scale
    keep = torch.from_numpy(philox(int(np.prod(shape)), seed, offset) >= t)
    if layout == 'nhwc':
        return keep.reshape((n,) + rest + (c,)).movedim(-1, 1), scale
    return keep.reshape(shape), scale


def activation(name, z):
    if name == 'relu':
        return z.clamp(min=0)
    if name == 'relu6':
        return z.clamp(0, 6)
    return z * torch.sigmoid(z) if name == 'silu' else z


def activation_slope(name, z):
    if name == 'relu':
        return (z > 0).double()
    if name == 'relu6':
        return ((z > 0) & (z < 6)).double()
    if name == 'silu':
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    return torch.ones_like(z)


class NormReference:
    """Forward, gradient and tolerances in 64 bits; tensors on the CPU."""

    def __init__(self, x, groups, gamma=None, beta=None, eps=1e-5, act='none', keep=None, scale=1.0):
        self.dtype, self.act, self.groups = x.dtype, act, groups
        shape = (1, -1) + (1,) * (x.dim() - 2)
        n, c = x.shape[:2]
        x = x.double()
        self.gamma = gamma.double().reshape(shape) if gamma is not None else torch.ones(c).double().reshape(shape)
        self.beta = beta.double().reshape(shape) if beta is not None else torch.zeros(c).double().reshape(shape)
        v = x.reshape(n, groups, -1)
        mean = v.mean(2, keepdim=True)
        var = (v - mean).square().mean(2, keepdim=True)
        sigma = (var + eps).sqrt()
        self.mean, self.rstd = mean[..., 0], 1 / sigma[..., 0]
        self.sigma = sigma.expand_as(v).reshape(x.shape)
        self.xhat = ((v - mean) / sigma).reshape(x.shape)
        kappa = (v.abs().amax(2, keepdim=True) / sigma).expand_as(v).reshape(x.shape)
        self.err = K * U * (1 + kappa)  # of xhat, relative to |xhat| + 1
        self.z = self.xhat * self.gamma + self.beta
        self.e_z = self.err * (self.gamma.abs() * (self.xhat.abs() + 1) + self.beta.abs())
        self.factor = torch.full_like(x, 1.0) if keep is None else keep.double() * scale
        self.y = activation(act, self.z) * self.factor
        # + 8 u |y|: the exponential, the division and the scaling
        self.tol_y = HALF[self.dtype] * self.y.abs() + (1.1 * self.e_z + 8 * U * self.y.abs()) * self.factor + TINY[self.dtype]

    def group_mean(self, v):
        n = v.shape[0]
        g = v.reshape(n, self.groups, -1)
        return g.mean(2, keepdim=True).expand_as(g).reshape(v.shape)

    def away_from_kinks(self, dy):
        """dy with zeros where the activation's slope may go either way."""
        kinks = {'relu': [0.0], 'relu6': [0.0, 6.0]}.get(self.act, [])
        dy = dy.clone()
        for k in kinks:
            dy[(self.z - k).abs() <= self.e_z] = 0
        return dy

    def backward(self, dy):
        dy = dy.double() * self.factor
        dz = dy * activation_slope(self.act, self.z)
        e_dz = dy.abs() * (0.5 * self.e_z * (self.act == 'silu') + 12 * U)
        axes = (0,) + tuple(range(2, dy.dim()))
        self.dbeta, self.dgamma = dz.sum(axes), (dz * self.xhat).sum(axes)
        e_t = e_dz * self.xhat.abs() + dz.abs() * self.err * (self.xhat.abs() + 1)
        self.tol_dbeta = (e_dz + K * U * dz.abs()).sum(axes)
        self.tol_dgamma = (e_t + K * U * (dz * self.xhat).abs()).sum(axes)
        g = dz * self.gamma
        s1, s2 = self.group_mean(g), self.group_mean(g * self.xhat)
        self.dx = (g - s1 - self.xhat * s2) / self.sigma
        e_g = e_dz * self.gamma.abs()
        e_s1 = self.group_mean(e_g + K * U * g.abs())
        e_s2 = self.group_mean(e_t * self.gamma.abs() + K * U * (g * self.xhat).abs())
        parts = g.abs() + s1.abs() + (self.xhat * s2).abs()
        self.tol_dx = HALF[self.dtype] * self.dx.abs() + TINY[self.dtype] + (
            e_g + e_s1 + self.xhat.abs() * e_s2 + self.err * (self.xhat.abs() + 1) * s2.abs()
            + (self.err + 8 * U) * parts) / self.sigma
        return self


def assert_close(got, want, tol, label=''):
    got = got.detach().cpu().double()
    want, tol = want.expand_as(got), tol.expand_as(got)
    assert not torch.isnan(got).any(), f'{label}: NaN in the result'
    over = (got - want).abs() - tol
    worst = int(over.argmax()) if over.numel() else 0
    assert over.numel() == 0 or over.max() <= 0, (
        f'{label}: {int((over > 0).sum())} of {over.numel()} outside, worst at {worst}: '
        f'{got.reshape(-1)[worst]} for {want.reshape(-1)[worst]}, tolerance {tol.reshape(-1)[worst]}')


def channels_last(t):
    """Dense with the channels innermost, ranks 2 to 4."""
    return t.movedim(1, -1).contiguous().movedim(-1, 1)
