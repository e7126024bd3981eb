"""Workloads of layer norm, the causal depthwise convolution and the selective scan: inputs, plain
forms, exact results.

A case is one call (``mode`` "forward"), one training step ("step": the call and its gradients) or
one token of every sequence ("token").  With ``own`` false, ``run`` computes the operator from
elementary torch operations; with ``own`` true it calls ``groupconv_atlas_b200.torch_module``.

Definitions (sequences lie as [N, L, C], tokens by channels)
  norm   y = (x - mean) / sqrt(var + eps) * gamma + beta over the last axis of x, var biased.
  conv   v[t, c] = bias[c] + sum_k weight[c, k] u[t + k, c], u = the K - 1 inputs of `state` (0 without
         one), then x;  y = v or v / (1 + exp(-v));  the new state is the last K - 1 inputs.
  scan   delta = softplus(dt + dt_bias);  h[t] = exp(delta[t] A) h[t-1] + delta[t] x[t] B[t], a state of
         S numbers for each channel, h[-1] = `state` (0 without one);  v[t] = C[t] . h[t] + D x[t];
         y = v z / (1 + exp(-z)), or v without z.  Channel c reads group c // (channels / G) of B, C.
  With lengths, a sequence ends there: what lies behind it is not read, results there are 0 and the
  new state is the one at its end.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


def _norm(name, rows, c, dtype, mode='forward', params='float32'):
    return {'name': name, 'op': 'norm', 'rows': rows, 'c': c, 'dtype': dtype, 'mode': mode, 'params': params}


def _conv(name, n, l, c, k, dtype, mode='forward', act='silu', lengths=False, state=False):
    return {'name': name, 'op': 'conv', 'n': n, 'l': l, 'c': c, 'k': k, 'dtype': dtype, 'mode': mode, 'act': act,
            'lengths': lengths, 'state': state}


def _scan(name, n, l, c, s, dtype, mode='forward', groups=1, gate=True, lengths=False, state=False):
    return {'name': name, 'op': 'scan', 'n': n, 'l': l, 'c': c, 's': s, 'dtype': dtype, 'mode': mode, 'groups': groups,
            'gate': gate, 'lengths': lengths, 'state': state}


def listed():
    return [
        # one image's feature map behind a depthwise layer: the call's latency
        _norm('norm small', 14 * 14, 384, 'bfloat16'),
        # a batch of prompts in front of a projection
        _norm('norm bf16 prompts', 16384, 2048, 'bfloat16'),
        # training, first stage of an image network: many short rows, the type of the convolutions
        _norm('norm step f32 stage', 32 * 56 * 56, 96, 'float32', 'step'),
        # training, rows whose length is no multiple of anything, parameters in the input's type
        _norm('norm step bf16 odd', 8191, 1001, 'bfloat16', 'step', params='bfloat16'),
        # one token of each of a batch's sequences: latency
        _conv('conv token f16', 32, 1, 2048, 4, 'float16', 'token'),
        # prompts of several lengths, continued from their states, odd channels
        _conv('conv f32 odd prompts', 3, 1021, 333, 3, 'float32', act='none', lengths=True, state=True),
        # training on long sequences
        _conv('conv step bf16', 8, 2048, 2048, 4, 'bfloat16', 'step'),
        # one token of each of a batch's sequences
        _scan('scan token bf16', 64, 1, 4096, 16, 'bfloat16', 'token'),
        # one long prompt: few channels to work on at a time
        _scan('scan bf16 long prompt', 1, 8192, 2048, 16, 'bfloat16'),
        # training on long sequences
        _scan('scan step bf16', 4, 2048, 2048, 16, 'bfloat16', 'step'),
        # training on images, rows of patches as sequences
        _scan('scan step f16 images', 16, 196, 384, 16, 'float16', 'step'),
        # prompts of several lengths, several groups, odd sizes, no gate
        _scan('scan f32 odd prompts', 5, 777, 330, 12, 'float32', groups=3, gate=False, lengths=True, state=True),
    ]


def draw(rng):
    def log_int(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    dtype = rng.choice(['float32', 'bfloat16', 'float16'])
    op = rng.choice(['norm', 'conv', 'scan', 'scan'])
    if op == 'norm':
        c = log_int(1, 8192)
        case = _norm('', log_int(1, max(1, min(1 << 17, (1 << 24) // c))), c, dtype, rng.choice(['forward', 'step']),
                     rng.choice(['float32', dtype]))
    else:
        mode = rng.choice(['forward', 'step', 'token'])
        if op == 'conv':
            c, k = log_int(1, 8192), rng.choice([1, 2, 3, 4, 4, 5, 8])
            most = (1 << 24) // c
        else:
            groups = rng.choice([1, 1, 2, 3, 4])
            s = rng.choice([16, 16, 1, 4, 7, 8, 12, 32, 50, 64])
            c = groups * log_int(1, 4096 // groups)
            most = (1 << 27) // (c * s)
        if mode == 'token':
            n, l = log_int(1, max(1, min(256, most))), 1
        else:
            l = log_int(1, max(1, min(8192, most)))
            n = log_int(1, max(1, min(64, most // l)))
        lengths = mode != 'token' and rng.random() < 0.3
        if op == 'conv':
            case = _conv('', n, l, c, k, dtype, mode, rng.choice(['none', 'silu']), lengths, mode == 'forward' and rng.random() < 0.5)
        else:
            case = _scan('', n, l, c, s, dtype, mode, groups, rng.random() < 0.7, lengths, mode == 'forward' and rng.random() < 0.5)
    del case['name']
    return case


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dtype, step = DTYPES[case['dtype']], case['mode'] == 'step'

    def randn(*shape, scale=1.0, level=0.0):
        return torch.randn(shape, generator=g, device='cuda') * scale + level

    def uniform(*shape):
        return torch.rand(shape, generator=g, device='cuda')

    state = {'case': case}
    c = case['c']
    if case['op'] == 'norm':
        pt = DTYPES[case['params']]
        # every channel has its own level and spread
        state['x'] = (randn(case['rows'], c) * (0.5 + uniform(c)) + randn(c, scale=0.3)).to(dtype)
        state['gamma'], state['beta'] = randn(c, scale=0.2, level=1.0).to(pt), randn(c, scale=0.2).to(pt)
        if step:
            state['dy'] = randn(case['rows'], c).to(dtype)
        wanted = ['x', 'gamma', 'beta']
    else:
        n, l, token = case['n'], case['l'], case['mode'] == 'token'
        both = randn(n, l, 2 * c).to(dtype)  # one projection gives the branch and its gate
        if case['lengths']:
            state['lengths'] = torch.randint(0, l + 1, (n,), generator=g, device='cuda', dtype=torch.int32)
        if case['op'] == 'conv':
            state['x'] = both[..., :c]
            state['weight'] = randn(c, case['k'], scale=1 / math.sqrt(case['k'])).to(dtype)
            state['bias'] = randn(c, scale=0.1).to(dtype)
            if case['state'] or token:
                state['state'] = randn(n, case['k'] - 1, c).to(dtype)
            wanted = ['x', 'weight', 'bias']
        else:
            s, groups = case['s'], case['groups']
            state['x'] = randn(n, l, c).to(dtype)
            state['dt'] = randn(n, l, c, scale=0.5).to(dtype)
            parts = randn(n, l, 2 * groups * s).to(dtype)  # one projection gives B and C
            state['B'] = parts[..., :groups * s].unflatten(-1, (groups, s))
            state['C'] = parts[..., groups * s:].unflatten(-1, (groups, s))
            state['A'] = -(torch.arange(1, s + 1, device='cuda') * torch.exp(randn(c, s, scale=0.2)))
            state['D'] = randn(c, scale=0.2, level=1.0)
            first = torch.exp(uniform(c) * math.log(100.0) + math.log(1e-3))  # the step sizes that training starts from
            state['dt_bias'] = first + torch.log(-torch.expm1(-first))
            wanted = ['x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias']
            if case['gate']:
                state['z'] = both[..., c:]
                wanted.append('z')
            if case['state'] or token:
                state['state'] = randn(n, c, s, scale=0.5)
        if token:
            for name in ('x', 'dt', 'z', 'B', 'C'):
                if name in state:
                    state[name] = state[name][:, 0]
            state['new_state'] = torch.empty_like(state['state'])
        if step:
            state['dy'] = randn(n, l, c).to(dtype)
    if step:
        state['wanted'] = wanted
        for name in wanted:
            state[name].requires_grad_()
    return state


def _inside(state):
    """[N, L, 1] truth values: tokens of the sequences; None where every token is one."""
    if 'lengths' not in state:
        return None
    at = torch.arange(state['case']['l'], device=state['x'].device)
    return (at < state['lengths'][:, None])[..., None]


def _only(inside, v):
    return v if inside is None else torch.where(inside, v, torch.zeros((), dtype=v.dtype, device=v.device))


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _plain_norm(state):
    x, gamma, beta = state['x'], state['gamma'].float(), state['beta'].float()
    d = x.float() - x.float().mean(-1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS)
    xhat = d * rstd
    out = {'y': (xhat * gamma + beta).to(x.dtype)}
    if 'dy' in state:
        dy = state['dy'].float()
        g = dy * gamma
        out['dx'] = (rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))).to(x.dtype)
        out['dgamma'] = (dy * xhat).sum(0).to(state['gamma'].dtype)
        out['dbeta'] = dy.sum(0).to(state['beta'].dtype)
    return out


def _plain_conv(state):
    case, x, dtype, w = state['case'], state['x'], state['x'].dtype, state['weight'].float()
    n, c, k = case['n'], case['c'], case['k']
    token, inside = case['mode'] == 'token', _inside(state)
    xf = x.float()[:, None] if token else _only(inside, x.float())
    before = state['state'].float() if 'state' in state else torch.zeros(n, k - 1, c, device=x.device)
    u = torch.cat([before, xf], 1)
    windows = u.unfold(1, k, 1)
    v = (windows * w).sum(-1) + state['bias'].float()
    y = v * _sigmoid(v) if case['act'] == 'silu' else v
    out = {'y': (y[:, 0] if token else _only(inside, y)).to(dtype)}
    if token:
        out['state'] = u[:, 1:].to(dtype)
    elif 'state' in state:
        end = state['lengths'].long() if inside is not None else torch.full((n,), case['l'], device=x.device)
        at = (end[:, None] + torch.arange(k - 1, device=x.device))[..., None].expand(n, k - 1, c)
        out['state'] = u.gather(1, at).to(dtype)
    if 'dy' in state:
        dv = _only(inside, state['dy'].float())
        if case['act'] == 'silu':
            s = _sigmoid(v)
            dv = dv * (s * (1 + v * (1 - s)))
        out['dweight'] = (dv[..., None] * windows).sum((0, 1)).to(dtype)
        out['dbias'] = dv.sum((0, 1)).to(dtype)
        later = torch.cat([dv, torch.zeros(n, k - 1, c, device=x.device)], 1).unfold(1, k, 1)
        out['dx'] = _only(inside, (later * w.flip(1)).sum(-1)).to(dtype)
    return out


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] along axis 1 from h[-1] = 0, by doubling."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _plain_scan(state):
    case, dtype = state['case'], state['x'].dtype
    n, l, c, s, groups = case['n'], case['l'], case['c'], case['s'], case['groups']
    inside = _inside(state)

    def tokens(name):
        v = state[name].float()
        return v[:, None] if case['mode'] == 'token' else v

    x, A = _only(inside, tokens('x')), state['A'].float()
    B, C = (torch.where(inside[..., None], tokens(k), 0.0) if inside is not None else tokens(k) for k in ('B', 'C'))
    B, C = (v.repeat_interleave(c // groups, 2) for v in (B, C))  # [N, L, C, S]
    raw = tokens('dt') + state['dt_bias'].float()
    delta = _only(inside, raw.clamp(min=0) + torch.log1p(torch.exp(-raw.abs())))
    a = torch.exp(delta[..., None] * A)
    b = (delta * x)[..., None] * B
    first = state['state'] if 'state' in state else torch.zeros(n, c, s, device=x.device)
    b[:, 0] += a[:, 0] * first
    h = _recurrence(a, b)
    v = (h * C).sum(-1) + state['D'].float() * x
    y = v
    if case['gate']:
        z = _only(inside, tokens('z'))
        sz = _sigmoid(z)
        y = v * (z * sz)
    y = _only(inside, y)
    out = {'y': (y[:, 0] if case['mode'] == 'token' else y).to(dtype)}
    if 'state' in state:
        out['state'] = h[:, -1]
    if 'dy' in state:
        dv = _only(inside, state['dy'].float())
        if case['gate']:
            out['dz'] = (dv * v * (sz * (1 + z * (1 - sz)))).to(dtype)
            dv = dv * (z * sz)
        decay = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
        dh = _recurrence(decay.flip(1), (dv[..., None] * C).flip(1)).flip(1)
        before = torch.cat([first[:, None], h[:, :-1]], 1)
        moved = dh * a * before
        du = (dh * B).sum(-1)
        ddelta = (moved * A).sum(-1) + x * du
        draw_ = _only(inside, ddelta * _sigmoid(raw))
        out['dx'] = _only(inside, delta * du + state['D'].float() * dv).to(dtype)
        out['ddt'] = draw_.to(dtype)
        out['ddt_bias'] = draw_.sum((0, 1))
        out['dA'] = (moved * delta[..., None]).sum((0, 1))
        out['dD'] = (dv * x).sum((0, 1))
        out['dB'] = _only(None if inside is None else inside[..., None], (dh * (delta * x)[..., None]).unflatten(2, (groups, -1)).sum(3)).to(dtype)
        out['dC'] = (h * dv[..., None]).unflatten(2, (groups, -1)).sum(3).to(dtype)
    return out


def _own(state):
    from groupconv_atlas_b200 import torch_module as ops
    case = state['case']
    token = case['mode'] == 'token'
    if case['op'] == 'norm':
        out = {'y': ops.layer_norm(state['x'], state['gamma'], state['beta'], EPS)}
    elif case['op'] == 'conv':
        if token:
            y = ops.causal_conv_step(state['x'], state['weight'], state['state'], state['bias'], activation=case['act'],
                                     state_out=state['new_state'])
            out = {'y': y, 'state': state['new_state']}
        elif 'state' in state:
            y, last = ops.causal_conv(state['x'], state['weight'], state['bias'], activation=case['act'],
                                      state=state['state'], lengths=state.get('lengths'), return_state=True)
            out = {'y': y, 'state': last}
        else:
            out = {'y': ops.causal_conv(state['x'], state['weight'], state['bias'], activation=case['act'],
                                        lengths=state.get('lengths'))}
    else:
        names = ('x', 'dt', 'A', 'B', 'C')
        if token:
            y = ops.selective_scan_step(*(state[k] for k in names), state['state'], D=state['D'], z=state.get('z'),
                                        dt_bias=state['dt_bias'], softplus=True, state_out=state['new_state'])
            out = {'y': y, 'state': state['new_state']}
        elif 'state' in state:
            y, last = ops.selective_scan(*(state[k] for k in names), D=state['D'], z=state.get('z'),
                                         dt_bias=state['dt_bias'], softplus=True, state=state['state'],
                                         lengths=state.get('lengths'), return_state=True)
            out = {'y': y, 'state': last}
        else:
            out = {'y': ops.selective_scan(*(state[k] for k in names), D=state['D'], z=state.get('z'),
                                           dt_bias=state['dt_bias'], softplus=True, lengths=state.get('lengths'))}
    if 'dy' in state:
        grads = torch.autograd.grad(out['y'], [state[k] for k in state['wanted']], state['dy'])
        out = {'y': out['y'].detach()} | {'d' + k: v for k, v in zip(state['wanted'], grads)}
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {'norm': _plain_norm, 'conv': _plain_conv, 'scan': _plain_scan}[state['case']['op']](state)


def work(case):
    size, step = 2 if case['dtype'] != 'float32' else 4, case['mode'] == 'step'
    if case['op'] == 'norm':
        count, params = case['rows'] * case['c'], case['c'] * (2 if case['params'] != 'float32' else 4)
        return {'bytes': size * count * (4 if step else 2) + params * (4 if step else 2), 'flops': count * (20 if step else 8)}
    n, l, c = case['n'], case['l'], case['c']
    count = n * l * c
    lengths = 4 * n if case['lengths'] else 0
    carried = (2 if case['state'] or case['mode'] == 'token' else 0) * n * c  # states read and written
    if case['op'] == 'conv':
        k = case['k']
        return {'bytes': size * (count * (4 if step else 2) + c * (k + 1) * (2 if step else 1) + carried * (k - 1)) + lengths,
                'flops': count * ((6 * k + 16) if step else (2 * k + 5))}
    s, pairs = case['s'], n * l * case['groups'] * case['s']
    tensors = 3 + case['gate']  # x, dt, z and y
    if step:
        tensors = 5 + 2 * case['gate'] + 1  # also dy, dx, ddt, dz
    params = 4 * c * (s + 2) * (2 if step else 1)
    # per state: the exponential, its argument, two products and sums; the gradient's repeat these and take seven more
    return {'bytes': size * (count * tensors + 2 * pairs * (2 if step else 1)) + params + 4 * carried * s + lengths,
            'flops': count * (s * (26 if step else 7) + (40 if step else 14))}


def exact(case, seed):
    """The definitions in 64 bits: sums of shifted products, and the recurrence one token after the other."""
    state = prepare(case, seed)
    with torch.no_grad():
        values = {k: v.detach().double() for k, v in state.items() if torch.is_tensor(v) and v.is_floating_point()}
        if case['op'] == 'norm':
            return _exact_norm(case, values)
        lengths = state.get('lengths')
        ends = lengths.tolist() if lengths is not None else [case['l']] * case['n']
        return (_exact_conv if case['op'] == 'conv' else _exact_scan)(case, values, ends)


def _exact_norm(case, v):
    x, gamma = v['x'], v['gamma']
    var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    sigma = torch.sqrt(var + EPS)
    unit = (x - mean) / sigma
    out = {'y': torch.addcmul(v['beta'], unit, gamma)}
    if 'dy' in v:
        flow = v['dy'] * gamma
        out['dx'] = (flow - flow.mean(1, keepdim=True) - unit * (flow * unit).mean(1, keepdim=True)) / sigma
        out['dgamma'], out['dbeta'] = torch.einsum('rc,rc->c', v['dy'], unit), v['dy'].sum(0)
    return out


def _exact_conv(case, v, ends):
    n, l, c, k = case['n'], case['l'], case['c'], case['k']
    token, silu = case['mode'] == 'token', case['act'] == 'silu'
    x = v['x'].reshape(n, l, c)
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    last, dw, db = torch.zeros(n, k - 1, c).to(x), torch.zeros_like(v['weight']), torch.zeros_like(v['bias'])
    for i, end in enumerate(ends):
        line = torch.zeros(k - 1 + end, c).to(x)
        if 'state' in v:
            line[:k - 1] = v['state'][i]
        line[k - 1:] = x[i, :end]
        last[i] = line[end:]
        pre = v['bias'].expand(end, c).clone()
        for j in range(k):
            pre += line[j:j + end] * v['weight'][:, j]
        sig = torch.sigmoid(pre)
        y[i, :end] = pre * sig if silu else pre
        if 'dy' in v:
            flow = v['dy'][i, :end]
            if silu:
                flow = flow * (sig + pre * sig * (1 - sig))
            back = torch.zeros_like(line)
            for j in range(k):
                back[j:j + end] += flow * v['weight'][:, j]
                dw[:, j] += (flow * line[j:j + end]).sum(0)
            db += flow.sum(0)
            dx[i, :end] = back[k - 1:]
    if token:
        return {'y': y[:, 0], 'state': last}
    out = {'y': y}
    if 'state' in v:
        out['state'] = last
    return out | {'dweight': dw, 'dbias': db, 'dx': dx} if 'dy' in v else out


def _exact_scan(case, v, ends):
    n, l, c, s, groups = case['n'], case['l'], case['c'], case['s'], case['groups']
    x = v['x'].reshape(n, l, c)
    of = torch.arange(c, device=x.device) // (c // groups)  # a channel's group
    Bs, Cs = (v[k].reshape(n, l, groups, s) for k in ('B', 'C'))
    raw = v['dt'].reshape(n, l, c) + v['dt_bias']
    delta = torch.logaddexp(raw, torch.zeros_like(raw))
    inside = torch.arange(l, device=x.device) < torch.tensor(ends, device=x.device)[:, None]  # [N, L]
    h = v['state'].clone() if 'state' in v else torch.zeros(n, c, s).to(x)
    grad = 'dy' in v
    kept = torch.empty(l + 1, n, c, s).to(x) if grad else None
    out = torch.zeros_like(x)
    for t in range(l):
        if grad:
            kept[t] = h
        after = torch.exp(delta[:, t, :, None] * v['A']) * h + (delta[:, t] * x[:, t])[..., None] * Bs[:, t][:, of]
        h = torch.where(inside[:, t, None, None], after, h)
        out[:, t] = torch.where(inside[:, t, None], torch.einsum('ncs,ncs->nc', h, Cs[:, t][:, of]), 0.0)
    out += torch.where(inside[..., None], v['D'] * x, 0.0)
    gate = None
    ungated = out
    if case['gate']:
        z = v['z'].reshape(n, l, c)
        gate = z * torch.sigmoid(z)
        out = torch.where(inside[..., None], ungated * gate, 0.0)
    if case['mode'] == 'token':
        return {'y': out[:, 0], 'state': h}
    result = {'y': out}
    if 'state' in v:
        result['state'] = h
    if not grad:
        return result
    kept[l] = h
    flow = torch.where(inside[..., None], v['dy'], 0.0)
    if gate is not None:
        sig = torch.sigmoid(z)
        result['dz'] = flow * ungated * (sig + gate * (1 - sig))
        flow = flow * gate
    dA, dB, dC = torch.zeros_like(v['A']), torch.zeros_like(Bs), torch.zeros_like(Cs)
    dx, ddelta, back = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(h)
    for t in reversed(range(l)):
        live = inside[:, t, None, None]
        back_t = back + flow[:, t, :, None] * Cs[:, t][:, of]
        decay = torch.exp(delta[:, t, :, None] * v['A'])
        through = torch.where(live, back_t * decay * kept[t], 0.0)
        dA += torch.einsum('ncs,nc->cs', through, delta[:, t])
        into = torch.where(live, back_t, 0.0)
        du = torch.einsum('ncs,ncs->nc', into, Bs[:, t][:, of])
        dx[:, t] = du * delta[:, t]
        ddelta[:, t] = torch.einsum('ncs,cs->nc', through, v['A']) + du * x[:, t]
        dB[:, t] = (into * (delta[:, t] * x[:, t])[..., None]).unflatten(1, (groups, -1)).sum(2)
        dC[:, t] = (kept[t + 1] * flow[:, t, :, None]).unflatten(1, (groups, -1)).sum(2)
        back = torch.where(live, back_t * decay, back)
    ddt = ddelta * torch.sigmoid(raw)
    return result | {'dx': dx + flow * v['D'], 'ddt': ddt, 'ddt_bias': ddt.sum((0, 1)), 'dA': dA, 'dB': dB, 'dC': dC,
                     'dD': torch.einsum('nlc,nlc->c', flow, torch.where(inside[..., None], x, 0.0))}
