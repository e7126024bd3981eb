"""Plain 64-bit forms of the causal convolution and the selective scan with their
gradients, and the tolerances of their GPU tests.

Tolerances.  u = 2^-24 is half a step of the kernels' 32-bit arithmetic, h half a
step of the stored type relative to the value.  Every bound is carried through the
formulas to first order, beside the values:
  sum of k products   k u sum |products|, beside what the factors are off by
  exp2                4 u of the value (the instruction is good to 2^-22), beside
                      its argument's error: |arg| 3 u for the product with A log2(e)
  sigmoid and SiLU    (2 |z| + 12) u of s and of 1 - s: the argument's product with
                      log2(e), the exponential, sum, reciprocal and products
  softplus            (2 |v| + 24) u of the value: the sum dt + bias moves it by
                      |v| u (its slope is at most its value for negative arguments),
                      the exponential by |v| u + 4 u, reciprocal, series and
                      products by 16 u
  state               E[t] = a E[t - 1] + |h[t - 1]| e_a + |b| e_b + 3 u (|a h| + |b|)
  segments            a sequence's state may be formed over segments: the sum of a
                      segment's deltas is off by at most L u relative, which moves
                      its decay, exp(A sum), by at most L u max(x exp(-x)) < 0.4 L u
Long sums over tokens add at most 512 values one after the other (64 of a stretch,
256 of a block's workers, what a worker takes in turn) before 64-bit sums join them.
"""
import torch

from tests import norm_helpers
from tests.norm_helpers import HALF, TINY, U, activation, activation_slope

LONG = 512


def sigmoid_error(z):
    return (2 * z.abs() + 12) * U


def silu_slope_error(z):
    s = torch.sigmoid(z)
    return s * (1 + 2 * z.abs() * (1 - s)) * sigmoid_error(z)


def act_errors(name, v, e_v):
    """Of act(v) and act'(v)."""
    if name != 'silu':
        return e_v, torch.zeros_like(v)  # away from the kinks
    s = torch.sigmoid(v)
    return 1.1 * e_v + (v * s).abs() * (sigmoid_error(v) + 2 * U), 0.5 * e_v + silu_slope_error(v)


def rounded(value, error, dtype):
    return error + HALF.get(dtype, 0.0) * (value.abs() + error) + TINY.get(dtype, 0.0)


def assert_close(got, want, tol, label=''):
    """As norm_helpers', but float16 ends at 65504: from 65520 on, half a step beyond,
    a value rounds to infinity, and may where its error reaches that."""
    got = got.detach().cpu()
    if got.dtype == torch.float16:
        want, tol = want.expand(got.shape), tol.expand(got.shape)
        over = torch.isinf(got) & (want.abs() + tol >= 65520) & (torch.sign(got) == torch.sign(want))
        got = torch.where(over, want, got.double())
    norm_helpers.assert_close(got, want, tol, label)


def inside_mask(n, l, lengths):
    if lengths is None:
        return torch.ones(n, l, 1, dtype=torch.bool)
    return (torch.arange(l) < lengths.cpu().clamp(0, l)[:, None])[..., None]


class ConvReference:
    """x (N, L, C), weight (C, K); tensors on the CPU."""

    def __init__(self, x, weight, bias=None, act='none', state=None, lengths=None):
        self.dtype, self.act = x.dtype, act
        n, l, c = x.shape
        k = weight.shape[1]
        self.inside = inside_mask(n, l, lengths)
        self.ends = self.inside[..., 0].sum(1)
        x = torch.where(self.inside, x.double(), 0.0)
        self.w = weight.double()
        b = bias.double() if bias is not None else torch.zeros(c, dtype=torch.double)
        first = state.double() if state is not None else torch.zeros(n, k - 1, c, dtype=torch.double)
        self.u = torch.cat([first, x], 1)
        self.v = b.expand(n, l, c).clone()
        size = b.abs().expand(n, l, c).clone()
        for j in range(k):
            self.v += self.w[:, j] * self.u[:, j:j + l]
            size += (self.w[:, j] * self.u[:, j:j + l]).abs()
        self.e_v = (k + 1) * U * size
        y = torch.where(self.inside, activation(act, self.v), 0.0)
        self.e_act, self.e_slope = act_errors(act, self.v, self.e_v)
        self.y, self.tol_y = y, rounded(y, self.e_act, self.dtype) * self.inside
        self.last = torch.stack([self.u[i, e:e + k - 1] for i, e in enumerate(self.ends.tolist())]) if n else first

    def away_from_kinks(self, dy):
        dy = dy.clone()
        for kink in {'relu': [0.0], 'relu6': [0.0, 6.0]}.get(self.act, []):
            dy[(self.v - kink).abs() <= self.e_v] = 0
        return dy

    def backward(self, dy, dlast=None):
        n, l, c = self.v.shape
        k = self.w.shape[1]
        dy = torch.where(self.inside, dy.double(), 0.0)
        g = dy * activation_slope(self.act, self.v)
        e_g = dy.abs() * (self.e_slope + 2 * U * activation_slope(self.act, self.v).abs())
        du, e_du = torch.zeros_like(self.u), torch.zeros_like(self.u)
        self.dw, self.tol_dw = torch.zeros_like(self.w), torch.zeros_like(self.w)
        for j in range(k):
            du[:, j:j + l] += g * self.w[:, j]
            e_du[:, j:j + l] += (e_g + (k + 2) * U * g.abs()) * self.w[:, j].abs()
            u = self.u[:, j:j + l]
            self.dw[:, j] = (g * u).sum((0, 1))
            self.tol_dw[:, j] = (e_g * u.abs() + LONG * U * (g * u).abs()).sum((0, 1))
        self.db, self.tol_db = g.sum((0, 1)), (e_g + LONG * U * g.abs()).sum((0, 1))
        if dlast is not None:
            for i, e in enumerate(self.ends.tolist()):
                du[i, e:e + k - 1] += dlast[i].double()
                e_du[i, e:e + k - 1] += 2 * U * dlast[i].double().abs()
        self.dx = torch.where(self.inside, du[:, k - 1:], 0.0)
        self.tol_dx = rounded(self.dx, torch.where(self.inside, e_du[:, k - 1:], 0.0), self.dtype)
        self.dstate = du[:, :k - 1]
        self.tol_dstate = rounded(self.dstate, e_du[:, :k - 1], self.dtype)
        return self


class ScanReference:
    """x, dt, z (N, L, C), a (C, S), b, c (N, L, G, S); tensors on the CPU."""

    def __init__(self, x, dt, a, b, c, d=None, z=None, dt_bias=None, softplus=True, state=None, lengths=None):
        self.dtype = x.dtype
        n, l, ch = x.shape
        self.groups, s = b.shape[2], b.shape[3]
        inside = self.inside = inside_mask(n, l, lengths)
        put = lambda t: torch.where(inside.reshape(inside.shape + (1,) * (t.dim() - 3)), t.double(), 0.0)
        self.x, self.a = put(x), a.double()
        self.b, self.c = (put(t).repeat_interleave(ch // self.groups, 2) for t in (b, c))  # (N, L, C, S)
        bias = dt_bias.double() if dt_bias is not None else torch.zeros(ch, dtype=torch.double)
        self.d = d.double() if d is not None else torch.zeros(ch, dtype=torch.double)
        raw = put(dt) + bias
        if softplus:
            self.delta, self.slope = torch.logaddexp(raw, torch.zeros_like(raw)), torch.sigmoid(raw)
            self.e_delta, self.e_dslope = (2 * raw.abs() + 24) * U, (2 * raw.abs() + 12) * U  # relative
        else:
            self.delta, self.slope = raw, torch.ones_like(raw)
            self.e_delta, self.e_dslope = torch.full_like(raw, U), torch.zeros_like(raw)
            if dt_bias is not None:  # the sum may cancel
                self.e_delta = U * (1 + (put(dt).abs() + bias.abs()) / raw.abs().clamp(min=1e-300))
        self.delta = torch.where(inside, self.delta, 0.0)
        arg = self.delta[..., None] * self.a
        self.decay = torch.exp(arg)
        self.e_a = self.decay * (arg.abs() * (self.e_delta[..., None] + 3 * U) + 4 * U)
        self.u = self.delta * self.x
        add = self.u[..., None] * self.b
        e_add = add.abs() * (self.e_delta[..., None] + 2 * U)
        h = state.double() if state is not None else torch.zeros(n, ch, s, dtype=torch.double)
        e_h = torch.zeros_like(h)
        hs, es = [h], [e_h]
        for t in range(l):
            e_h = (self.decay[:, t] * e_h + h.abs() * self.e_a[:, t] + e_add[:, t]
                   + 3 * U * ((self.decay[:, t] * h).abs() + add[:, t].abs()))
            h = self.decay[:, t] * h + add[:, t]
            hs.append(h)
            es.append(e_h)
        self.h, self.e_h = torch.stack(hs, 1), torch.stack(es, 1)  # (N, L + 1, C, S)
        self.e_h += 0.4 * l * U * self.h.abs().amax(1, keepdim=True) * (l > 64)
        self.last, self.tol_last = self.h[:, -1], self.e_h[:, -1]
        v = (self.h[:, 1:] * self.c).sum(-1)
        e_v = ((self.e_h[:, 1:] + (s + 2) * U * self.h[:, 1:].abs()) * self.c.abs()).sum(-1) + 3 * U * (self.d * self.x).abs()
        self.v, self.e_v = v + self.d * self.x, e_v + 2 * U * v.abs()
        self.z = put(z) if z is not None else None
        self.gate = self.z * torch.sigmoid(self.z) if z is not None else torch.ones_like(self.v)
        self.e_gate = self.gate.abs() * (sigmoid_error(self.z) + U) if z is not None else torch.zeros_like(self.v)
        self.y = torch.where(inside, self.v * self.gate, 0.0)
        e_y = self.e_v * self.gate.abs() + self.v.abs() * self.e_gate + U * self.y.abs()
        self.tol_y = rounded(self.y, e_y, self.dtype) * inside

    def backward(self, dy, dlast=None):
        n, l, ch, s = self.b.shape
        dy = torch.where(self.inside, dy.double(), 0.0)
        f = dy * self.gate
        e_f = dy.abs() * self.e_gate + U * f.abs()
        if self.z is not None:
            sg = torch.sigmoid(self.z)
            slope = sg * (1 + self.z * (1 - sg))
            self.dz = dy * self.v * slope
            e = dy.abs() * (self.e_v * slope.abs() + self.v.abs() * (silu_slope_error(self.z) + 3 * U * slope.abs()))
            self.tol_dz = rounded(self.dz, e, self.dtype)
        q = dlast.double() if dlast is not None else torch.zeros(n, ch, s, dtype=torch.double)
        e_q = torch.zeros_like(q)
        qs, es = [None] * l, [None] * l
        for t in reversed(range(l)):
            add = f[:, t, :, None] * self.c[:, t]
            e_add = (e_f[:, t, :, None] + 2 * U * f[:, t, :, None].abs()) * self.c[:, t].abs()
            q, e_q = q + add, e_q + e_add + 2 * U * q.abs()
            qs[t], es[t] = q, e_q
            e_q = self.decay[:, t] * e_q + q.abs() * (self.e_a[:, t] + 2 * U * self.decay[:, t])
            q = self.decay[:, t] * q
        if l > 64:
            e_q = e_q + 0.4 * l * U * torch.stack(qs, 1).abs().amax(1)
        self.dstate, self.tol_dstate = q, e_q
        empty = torch.zeros(n, 0, ch, s, dtype=torch.double)
        qs, es = (torch.stack(v, 1) if l else empty for v in (qs, es))
        if l > 64:
            es = es + 0.4 * l * U * qs.abs().amax(1, keepdim=True)
        before, e_before = self.h[:, :-1], self.e_h[:, :-1]
        m = qs * self.decay * before
        e_m = (self.decay * (es * before.abs() + qs.abs() * e_before) + (qs * before).abs() * self.e_a + 3 * U * m.abs())
        live = self.inside[..., None]
        m, e_m = m * live, e_m * live
        du, e_du = (qs * self.b).sum(-1), ((es + (s + 2) * U * qs.abs()) * self.b.abs()).sum(-1)
        self.dx = torch.where(self.inside, self.delta * du + self.d * f, 0.0)
        e = self.delta.abs() * (e_du + du.abs() * (self.e_delta + 2 * U)) + self.d.abs() * (e_f + 2 * U * f.abs())
        self.tol_dx = rounded(self.dx, e * self.inside, self.dtype)
        dd, e_dd = (m * self.a).sum(-1), ((e_m + (s + 4) * U * m.abs()) * self.a.abs()).sum(-1)
        ddelta, e_ddelta = dd + self.x * du, e_dd + self.x.abs() * (e_du + 3 * U * du.abs()) + 2 * U * dd.abs()
        self.ddt = torch.where(self.inside, ddelta * self.slope, 0.0)
        e_ddt = (e_ddelta + ddelta.abs() * (self.e_dslope + 2 * U)) * self.slope * self.inside
        self.tol_ddt = rounded(self.ddt, e_ddt, self.dtype)
        self.ddt_bias = self.ddt.sum((0, 1))
        self.tol_ddt_bias = (e_ddt + LONG * U * self.ddt.abs()).sum((0, 1))
        self.dd = (f * self.x).sum((0, 1))
        self.tol_dd = (e_f * self.x.abs() + LONG * U * (f * self.x).abs()).sum((0, 1))
        md = m * self.delta[..., None]
        self.da = md.sum((0, 1))
        self.tol_da = (e_m * self.delta.abs()[..., None] + md.abs() * (self.e_delta[..., None] + LONG * U)).sum((0, 1))
        into = qs * live
        per = ch // self.groups
        join = lambda t: t.reshape(n, l, self.groups, per, s).sum(3)
        add = into * self.u[..., None]
        self.db = join(add)
        self.tol_db = rounded(self.db, join(es * live * self.u.abs()[..., None]
                                            + add.abs() * (self.e_delta[..., None] + (LONG + 2) * U)), self.dtype)
        add = self.h[:, 1:] * f[..., None]
        self.dc = join(add)
        self.tol_dc = rounded(self.dc, join(self.e_h[:, 1:] * f.abs()[..., None] + self.h[:, 1:].abs() * e_f[..., None]
                                            + (LONG + 2) * U * add.abs()), self.dtype)
        return self
