"""Workloads of the group-normalisation and dropout operators: inputs, plain forms, exact results.

A case is one call (``op`` "norm" or "dropout") or one training step (``step`` true: the call and
its gradients).  With ``own`` false, ``run`` computes the operator from elementary torch
operations in 32 bits; with ``own`` true it calls ``groupconv_atlas_b200.torch_module``.

Definitions
  norm     x [N, C, H, W] channels last in G groups of C / G channels;
           mean, var over a group's channels and pixels (biased), z = (x - mean) / sqrt(var + eps)
           * gamma + beta, a = activation(z), then dropout.
  dropout  y = [residual +] (keep ? x / (1 - q) : 0), q = t / 65536, t = round(65536 p);
           keep = draw(j) >= t, with j the element's place in memory order, or n * C + c where
           the scope is the channel.  draw(j): 16 bits of Philox4x32-10 (Salmon, Moraes, Dror,
           Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with the seed as its key and
           the counter (j // 8, offset): half j % 2 (the low one first) of word (j % 8) // 2.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


def _norm(name, n, c, h, w, groups, dtype, act, step=False, p=0.0, scope='element', params='float32'):
    return {'name': name, 'op': 'norm', 'n': n, 'c': c, 'h': h, 'w': w, 'groups': groups, 'dtype': dtype,
            'params': params, 'act': act, 'step': step, 'p': p, 'scope': scope}


def _dropout(name, n, c, h, w, dtype, p, step=False, residual=False, scope='element', layout='nhwc'):
    return {'name': name, 'op': 'dropout', 'n': n, 'c': c, 'h': h, 'w': w, 'dtype': dtype, 'p': p, 'step': step,
            'residual': residual, 'scope': scope, 'layout': layout}


def listed():
    return [
        # one image after a small grouped layer: the call's latency
        _norm('norm small', 1, 32, 56, 56, 8, 'float32', 'silu'),
        # a batch of mid-network feature maps at inference, half precision
        _norm('norm bf16 batch', 32, 256, 56, 56, 32, 'bfloat16', 'silu'),
        # early layers: few channels, large planes, the type of the convolutions
        _norm('norm f32 planes', 16, 64, 112, 112, 16, 'float32', 'relu'),
        # odd plane sizes, groups that are no power of two, parameters in the input's type
        _norm('norm f16 odd planes', 4, 144, 57, 55, 12, 'float16', 'none', params='float16'),
        # a channel count whose pixels are not 16-byte aligned
        _norm('norm f32 odd channels', 2, 45, 29, 31, 9, 'float32', 'relu6'),
        # one high-resolution image: a group's pixels outgrow any on-chip memory
        _norm('norm bf16 large image', 1, 128, 512, 512, 32, 'bfloat16', 'silu'),
        # training: late layers of a residual network, all in half precision
        _norm('norm step bf16', 32, 256, 28, 28, 32, 'bfloat16', 'silu', step=True, params='bfloat16'),
        # training with one group over all channels (a layer norm over the image)
        _norm('norm step f32 one group', 8, 96, 56, 56, 1, 'float32', 'silu', step=True),
        # training with channel dropout, the last and smallest planes
        _norm('norm step f16 7x7', 64, 512, 7, 7, 32, 'float16', 'silu', step=True, p=0.2, scope='channel'),
        # training at high resolution: norm, activation and dropout of a residual block
        _norm('norm step bf16 dropout', 8, 128, 256, 256, 16, 'bfloat16', 'silu', step=True, p=0.1),
        # the smallest dropout: its latency
        _dropout('dropout small', 1, 32, 56, 56, 'float32', 0.2),
        # a residual branch's dropout and its gradient
        _dropout('dropout step bf16 residual', 32, 256, 56, 56, 'bfloat16', 0.1, step=True, residual=True),
    ]


def draw(rng):
    def log_int(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    most = 3 << 23  # elements of x: no dearer than the largest listed case in any type
    dtype = rng.choice(['float32', 'bfloat16', 'float16'])
    p, scope = rng.choice([0.0, 0.1, 0.2, 0.5]), rng.choice(['element', 'element', 'channel'])
    if rng.random() < 0.7:
        groups = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 32])
        c = groups * log_int(1, max(1, 1024 // groups))
        h, w = log_int(4, 320), log_int(4, 320)
        n = log_int(1, max(1, min(128, most // (c * h * w))))
        while n * c * h * w > most:
            h, w = (h + 1) // 2, (w + 1) // 2
        case = _norm('', n, c, h, w, groups, dtype, rng.choice(['none', 'silu', 'silu']), rng.random() < 0.5, p, scope,
                     rng.choice(['float32', dtype]))
        if not case['step']:
            case['act'] = rng.choice(['none', 'relu', 'relu6', 'silu'])
    else:
        c, h, w = log_int(1, 1024), log_int(1, 320), log_int(1, 320)
        n = log_int(1, max(1, min(128, most // (c * h * w))))
        while n * c * h * w > most:
            h, w = (h + 1) // 2, (w + 1) // 2
        case = _dropout('', n, c, h, w, dtype, p or 0.3, rng.random() < 0.5, rng.random() < 0.5, scope,
                        rng.choice(['nhwc', 'nchw']))
    del case['name']
    return case


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dtype = DTYPES[case['dtype']]
    n, c, h, w = case['n'], case['c'], case['h'], case['w']

    def image():
        v = torch.randn((n, h, w, c), generator=g, device='cuda')
        if case['op'] == 'norm':  # a convolution's outputs: every channel has its own level and spread
            v = v * (0.5 + torch.rand(c, generator=g, device='cuda')) + 0.3 * torch.randn(c, generator=g, device='cuda')
        return v

    def put(v):
        v = v.to(dtype).permute(0, 3, 1, 2)
        return v.contiguous() if case.get('layout') == 'nchw' else v

    state = {'case': case, 'seed': seed * 0x9E3779B97F4A7C15 % (1 << 64), 'offset': 3 * seed + 1}
    state['x'] = put(image())
    if case['step']:
        state['dy'] = put(torch.randn((n, h, w, c), generator=g, device='cuda'))
    if case['op'] == 'norm':
        pt = DTYPES[case['params']]
        state['gamma'] = (1 + 0.2 * torch.randn(c, generator=g, device='cuda')).to(pt)
        state['beta'] = (0.2 * torch.randn(c, generator=g, device='cuda')).to(pt)
    elif case['residual']:
        state['residual'] = put(torch.randn((n, h, w, c), generator=g, device='cuda'))
    if case['step']:
        for name in ('x', 'gamma', 'beta', 'residual'):
            if name in state:
                state[name].requires_grad_()
    return state


def _philox(blocks, seed, offset, device):
    """[blocks, 4] words of Philox4x32-10, as int64."""
    mask, half = 0xFFFFFFFF, 0xFFFF

    def mul(a, m):  # high and low word of a * m, in pieces that stay below 2^63
        low = a * (m & half)
        high = a * (m >> 16) + (low >> 16)
        return high >> 16, ((high & half) << 16) | (low & half)

    at = torch.arange(blocks, device=device)
    c0, c1 = at & mask, at >> 32
    c2, c3 = torch.full_like(at, offset & mask), torch.full_like(at, offset >> 32)
    k0, k1 = seed & mask, seed >> 32
    for _ in range(10):
        h0, l0 = mul(c0, 0xD2511F53)
        h1, l1 = mul(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack([c0, c1, c2, c3], 1)


def _keep(state):
    """Truth values shaped like the data in memory order, and 1 / (1 - q)."""
    case = state['case']
    n, c, h, w = case['n'], case['c'], case['h'], case['w']
    t = round(65536 * case['p'])
    nhwc = case.get('layout', 'nhwc') == 'nhwc'
    count = n * c if case['scope'] == 'channel' else n * c * h * w
    words = _philox((count + 7) // 8, state['seed'], state['offset'], state['x'].device)
    keep = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:count] >= t
    if case['scope'] == 'channel':
        keep = keep.reshape(n, c, 1, 1)
    else:
        keep = keep.reshape(n, h, w, c).permute(0, 3, 1, 2) if nhwc else keep.reshape(n, c, h, w)
    return keep, 65536 / (65536 - t)


def _plain_dropout(state):
    case, dtype = state['case'], state['x'].dtype
    keep, scale = _keep(state)
    zero = torch.zeros((), device=keep.device)
    y = torch.where(keep, state['x'].float() * scale, zero)
    if case['residual']:
        y = y + state['residual'].float()
    out = {'y': y.to(dtype)}
    if case['step']:
        out['dx'] = torch.where(keep, state['dy'].float() * scale, zero).to(dtype)
        if case['residual']:
            out['dresidual'] = state['dy']
    return out


def _plain_norm(state):
    case, x = state['case'], state['x']
    n, c, h, w = x.shape
    groups, pt = case['groups'], state['gamma'].dtype
    xf = x.permute(0, 2, 3, 1).float().reshape(n, h * w, groups, c // groups)
    mean = xf.mean((1, 3), keepdim=True)
    d = xf - mean
    rstd = torch.rsqrt((d * d).mean((1, 3), keepdim=True) + EPS)
    xhat = (d * rstd).reshape(n, h * w, c)
    gamma, beta = state['gamma'].float(), state['beta'].float()
    z = xhat * gamma + beta
    if case['act'] == 'silu':
        s = 1 / (1 + torch.exp(-z))
        a = z * s
    else:
        s = None
        a = z if case['act'] == 'none' else z.clamp(0) if case['act'] == 'relu' else z.clamp(0, 6)
    keep = None
    if case['p'] > 0:
        keep, scale = _keep(state)
        keep = keep.permute(0, 2, 3, 1).reshape(n, -1, c)
        zero = torch.zeros((), device=x.device)
        a = torch.where(keep, a * scale, zero)

    def back(v):
        return v.to(x.dtype).reshape(n, h, w, c).permute(0, 3, 1, 2)

    out = {'y': back(a)}
    if case['step']:
        dz = state['dy'].permute(0, 2, 3, 1).float().reshape(n, h * w, c)
        if keep is not None:
            dz = torch.where(keep, dz * scale, zero)
        if s is not None:
            dz = dz * (s * (1 + z * (1 - s)))
        out['dgamma'] = (dz * xhat).sum((0, 1)).to(pt)
        out['dbeta'] = dz.sum((0, 1)).to(pt)
        gz = (dz * gamma).reshape(n, h * w, groups, c // groups)
        xg = xhat.reshape(gz.shape)
        s1 = gz.mean((1, 3), keepdim=True)
        s2 = (gz * xg).mean((1, 3), keepdim=True)
        out['dx'] = back((rstd * (gz - s1 - xg * s2)).reshape(n, h * w, c))
    return out


def _own(state):
    from groupconv_atlas_b200 import torch_module
    case = state['case']
    if case['op'] == 'dropout':
        y = torch_module.dropout(state['x'], case['p'], residual=state.get('residual'), scope=case['scope'],
                                 seed=state['seed'], offset=state['offset'])
        names = [k for k in ('x', 'residual') if k in state]
    else:
        y = torch_module.group_norm_act(state['x'], case['groups'], state['gamma'], state['beta'], EPS,
                                        activation=case['act'], dropout=case['p'], scope=case['scope'],
                                        seed=state['seed'], offset=state['offset'])
        names = ['x', 'gamma', 'beta']
    out = {'y': y.detach()}
    if case['step']:
        grads = torch.autograd.grad(y, [state[k] for k in names], state['dy'])
        out |= {'d' + k: v for k, v in zip(names, grads)}
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain_dropout(state) if state['case']['op'] == 'dropout' else _plain_norm(state)


def work(case):
    size = 2 if case['dtype'] != 'float32' else 4
    count = case['n'] * case['c'] * case['h'] * case['w']
    if case['op'] == 'dropout':
        tensors = 2 + case['residual'] + (2 if case['step'] else 0)
        return {'bytes': size * count * tensors, 'flops': count * (2 + case['step'])}
    params = case['c'] * (2 if case['params'] != 'float32' else 4)
    # statistics, scale and shift, activation; the gradient's sums and its result
    return {'bytes': size * count * (4 if case['step'] else 2) + params * (4 if case['step'] else 2),
            'flops': count * (26 if case['step'] else 10)}


def exact(case, seed):
    """The definition in 64 bits, over [N, G, C/G, H, W] views; the draws with numpy's 64-bit integers."""
    state = prepare(case, seed)
    with torch.no_grad():
        x = state['x'].detach().double()
        n, c, h, w = x.shape
        factor = None
        if case['p'] > 0:
            count = n * c * (1 if case['scope'] == 'channel' else h * w)
            t = round(65536 * case['p'])
            bits = _draws(count, state['seed'], state['offset'])
            factor = torch.from_numpy((bits >= t).astype(np.float32)).cuda().double() / (1 - t / 65536)
            if case['scope'] == 'channel':
                factor = factor.reshape(n, c, 1, 1)
            elif case.get('layout') == 'nchw':
                factor = factor.reshape(n, c, h, w)
            else:
                factor = factor.reshape(n, h, w, c).permute(0, 3, 1, 2)
        dy = state['dy'].double() if case['step'] else None
        if case['op'] == 'dropout':
            out = {'y': x * factor + (state['residual'].detach().double() if case['residual'] else 0)}
            if case['step']:
                out['dx'] = dy * factor
                if case['residual']:
                    out['dresidual'] = dy
            return out
        view = (n, case['groups'], c // case['groups'], h, w)
        var, mean = torch.var_mean(x.reshape(view), (2, 3, 4), unbiased=False, keepdim=True)
        sigma = torch.sqrt(var + EPS)
        gamma = state['gamma'].detach().double().reshape(1, c, 1, 1)
        unit = ((x.reshape(view) - mean) / sigma).reshape(x.shape)
        z = unit * gamma + state['beta'].detach().double().reshape(1, c, 1, 1)
        slope = None
        if case['act'] == 'silu':
            sig = torch.sigmoid(z)
            y, slope = z * sig, sig + z * sig * (1 - sig)
        else:
            y = z if case['act'] == 'none' else torch.clamp(z, 0, math.inf if case['act'] == 'relu' else 6)
        out = {'y': y if factor is None else y * factor}
        if case['step']:
            if factor is not None:
                dy = dy * factor
            if slope is not None:
                dy = dy * slope
            out['dgamma'] = (dy * unit).sum((0, 2, 3))
            out['dbeta'] = dy.sum((0, 2, 3))
            flow = (dy * gamma).reshape(view)
            unit = unit.reshape(view)
            flow = flow - flow.mean((2, 3, 4), keepdim=True) - unit * (flow * unit).mean((2, 3, 4), keepdim=True)
            out['dx'] = (flow / sigma).reshape(x.shape)
        return out


def _draws(count, seed, offset):
    """`count` 16-bit draws, from numpy's 64-bit products."""
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    blocks = np.arange((count + 7) // 8, dtype=u)
    ctr = [blocks & low, blocks >> u(32), np.full_like(blocks, offset & 0xFFFFFFFF), np.full_like(blocks, offset >> 32)]
    for i in range(10):
        key = [u((seed + i * 0x9E3779B9) & 0xFFFFFFFF), u(((seed >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF)]
        a, b = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        ctr = [(b >> u(32)) ^ ctr[1] ^ key[0], b & low, (a >> u(32)) ^ ctr[3] ^ key[1], a & low]
    words = np.stack(ctr, 1).astype('<u4')
    return words.reshape(-1).view('<u2')[:count]
