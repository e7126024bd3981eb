"""Host side of layer norm, the causal convolution and the selective scan against
a stand-in for the CUDA runtime (fake_cudart.cpp): refusals, plans of many sizes,
failed launches and memory that runs out.  No GPU; each test in a process of its
own, with the stand-in preloaded."""
import os
import subprocess
import sys

import pytest

from groupconv_atlas_b200 import api, build

SETUP = """
import ctypes as ct
import itertools
from groupconv_atlas_b200 import api
fake = ct.CDLL(FAKE)
flag = lambda name: ct.c_int.in_dll(fake, name)
native = api.Native()
lib, ref = native.lib, ct.byref
PLACE = 1 << 44
OK, INVALID, UNSUPPORTED, DEVICE = api.GC_OK, api.GC_INVALID, api.GC_UNSUPPORTED, api.GC_DEVICE_ERROR
SIZE = {0: 4, 1: 8, 16: 2, 17: 2}


def tensor(dims, place, dtype=0, strides=None, offset=0):
    t = api.Tensor()
    if strides is None:
        strides = [1] * len(dims)
        for i in range(len(dims) - 2, -1, -1):
            strides[i] = strides[i + 1] * max(dims[i + 1], 1)
    count = 1
    for n in dims:
        count *= n
    span = 0 if 0 in dims else max(count, 1 + sum((n - 1) * s for n, s in zip(dims, strides)))
    t.data, t.bytes, t.dtype, t.device, t.rank = place * PLACE + offset, span * SIZE.get(dtype, 4), dtype, 1, len(dims)
    for i, (n, s) in enumerate(zip(dims, strides)):
        t.dims[i], t.strides[i] = n, s
    return t


def p(t):
    return ref(t) if t is not None else None


class Norm:
    def __init__(self, dims=(6, 40), dtype=0):
        c, rows = dims[-1], 1
        for n in dims[:-1]:
            rows *= n
        self.x, self.y, self.dy, self.dx = (tensor(dims, i, dtype) for i in (1, 2, 3, 4))
        self.gamma, self.beta, self.dgamma, self.dbeta = (tensor((c,), i) for i in (5, 6, 7, 8))
        self.stats, self.eps, self.space = tensor((rows, 2), 9), 1e-5, (10 * PLACE, PLACE)

    def forward(self):
        return lib.gc_b200_layer_norm(p(self.x), p(self.gamma), p(self.beta), p(self.y), p(self.stats), self.eps, None)

    def size(self):
        n = ct.c_uint64(7)
        return lib.gc_b200_layer_norm_backward_workspace(p(self.dy), p(self.x), p(self.dx), ref(n)), n.value

    def backward(self):
        return lib.gc_b200_layer_norm_backward(p(self.dy), p(self.x), p(self.gamma), p(self.stats), p(self.dx), p(self.dgamma),
                                               p(self.dbeta), *self.space, None)


class Conv:
    def __init__(self, n=2, l=9, c=8, k=4, dtype=0):
        self.x, self.y, self.dy, self.dx = (tensor((n, l, c), i, dtype) for i in (1, 2, 3, 4))
        self.x1, self.y1 = (tensor((n, c), i, dtype) for i in (1, 2))
        self.w, self.dw, self.b, self.db = tensor((c, k), 5), tensor((c, k), 6), tensor((c,), 7), tensor((c,), 8)
        self.state, self.out, self.dstate, self.dlast = (tensor((n, k - 1, c), i, dtype) for i in (9, 10, 11, 12))
        self.lengths, self.act, self.space = 13 * PLACE, 3, (14 * PLACE, PLACE)

    def forward(self):
        return lib.gc_b200_causal_conv(p(self.x), p(self.w), p(self.b), p(self.state), self.lengths, p(self.y), p(self.out),
                                       self.act, None)

    def size(self):
        n = ct.c_uint64(7)
        return lib.gc_b200_causal_conv_backward_workspace(p(self.dy), p(self.x), p(self.w), p(self.dx), ref(n)), n.value

    def backward(self):
        return lib.gc_b200_causal_conv_backward(p(self.dy), p(self.x), p(self.w), p(self.b), p(self.state), p(self.dlast),
                                                self.lengths, p(self.dx), p(self.dw), p(self.db), p(self.dstate), self.act,
                                                *self.space, None)

    def step(self):
        return lib.gc_b200_causal_conv_step(p(self.x1), p(self.w), p(self.b), p(self.state), p(self.y1), p(self.out), self.act,
                                            None)


class Scan:
    def __init__(self, n=2, l=9, c=8, s=16, g=2, dtype=0):
        token = lambda i: tensor((n, l, c), i, dtype)
        pairs = lambda i: tensor((n, l, g, s), i, dtype)
        self.q = dict(x=token(1), dt=token(2), a=tensor((c, s), 3), b=pairs(4), c=pairs(5), d=tensor((c,), 6), z=token(7),
                      dt_bias=tensor((c,), 8), state=tensor((n, c, s), 9))
        self.g = dict(x=token(21), dt=token(22), a=tensor((c, s), 23), b=pairs(24), c=pairs(25), d=tensor((c,), 26), z=token(27),
                      dt_bias=tensor((c,), 28), state=tensor((n, c, s), 29))
        self.one = {k: tensor([t.dims[i] for i in range(t.rank) if i != 1], i + 1, dtype) if k in ('x', 'dt', 'b', 'c', 'z') else t
                    for i, (k, t) in enumerate(self.q.items())}
        self.y, self.y1, self.dy, self.out, self.dlast = token(10), tensor((n, c), 10, dtype), token(11), tensor((n, c, s), 12), tensor((n, c, s), 13)
        self.lengths, self.kept, self.space = 14 * PLACE, (15 * PLACE, PLACE), (16 * PLACE, PLACE)

    def args(self, q, lengths):
        a = api.ScanArgs()
        for k, t in q.items():
            if t is not None:
                setattr(a, k, ct.pointer(t))
        a.lengths, a.softplus = lengths, 1
        return a

    def sizes(self):
        n = [ct.c_uint64(7) for _ in range(3)]
        return lib.gc_b200_selective_scan_sizes(ref(self.args(self.q, self.lengths)), *map(ref, n)), *(v.value for v in n)

    def forward(self):
        return lib.gc_b200_selective_scan(ref(self.args(self.q, self.lengths)), p(self.y), p(self.out), *self.kept, *self.space,
                                          None)

    def backward(self):
        grads = api.ScanGrads()
        for k, t in self.g.items():
            if t is not None:
                setattr(grads, k, ct.pointer(t))
        return lib.gc_b200_selective_scan_backward(ref(self.args(self.q, self.lengths)), p(self.dy), p(self.dlast), *self.kept,
                                                   ref(grads), *self.space, None)

    def step(self):
        return lib.gc_b200_selective_scan_step(ref(self.args(self.one, None)), p(self.y1), p(self.out), None)


CALLS = [Norm().forward, Norm().backward, Conv().forward, Conv().backward, Conv().step, Scan().forward, Scan().backward, Scan().step]


def expect(status, call, what=''):
    got = call()
    got = got[0] if isinstance(got, tuple) else got
    assert got == status, (what, got, native.lib.gc_last_error())
"""


@pytest.fixture(scope='module')
def run(native, tmp_path_factory):
    """Runs code with the stand-in; its output."""
    fake = tmp_path_factory.mktemp('fake') / 'fake_cudart.so'
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(build.nvcc()))), 'include')
    subprocess.run(['g++', '-O1', '-std=c++17', '-shared', '-fPIC', f'-I{cuda}', '-o', str(fake),
                    os.path.join(os.path.dirname(__file__), 'fake_cudart.cpp')], check=True)

    def call(code):
        done = subprocess.run([sys.executable, '-c', f'FAKE = {str(fake)!r}\n' + SETUP + code], cwd=api.ROOT,
                              capture_output=True, text=True, timeout=300, env=dict(os.environ, LD_PRELOAD=str(fake)))
        assert done.returncode == 0, done.stdout[-1000:] + done.stderr[-3000:]
        return done.stdout
    return call


def test_every_size_has_a_plan(run):
    """No size of the ranges stops the process or is refused; workspaces of the
    sizes given suffice, a byte less does not."""
    run("""
for dims in [(1, 1), (3, 7), (5, 8), (1000000, 12), (70000, 33), (7, 96), (3, 1001), (2, 2048), (9, 4104), (4, 8192), (1, 8200),
             (2, 100000), (0, 5), (2, 3, 4, 96), (17,), (1 << 30, 64)]:
    for dtype in (0, 16, 17):
        v = Norm(dims, dtype)
        expect(OK, v.forward, dims)
        st, need = v.size()
        assert st == OK and need < 1 << 33
        v.space = (10 * PLACE, need)
        expect(OK, v.backward, dims)
        if need:
            v.space = (10 * PLACE, need - 1)
            expect(INVALID, v.backward, dims)
            v.dgamma = v.dbeta = None
            expect(OK, v.backward, dims)
for n, l, c, k in itertools.product((0, 1, 3, 500), (0, 1, 2, 63, 64, 1000, 70000), (1, 3, 4, 33, 128, 1000, 8192), (1, 4, 5, 8)):
    for dtype in (0, 17):
        v = Conv(n, l, c, k, dtype)
        for call in (v.forward, v.step):
            expect(OK, call, (n, l, c, k))
        st, need = v.size()
        assert st == OK
        v.space = (14 * PLACE, need)
        expect(OK, v.backward, (n, l, c, k))
for n, l, (g, per), s in itertools.product((0, 1, 3, 200), (0, 1, 15, 64, 65, 1000, 70000), ((1, 1), (1, 40), (3, 7), (2, 2048)),
                                           (1, 2, 3, 4, 7, 16, 33, 64)):
    v = Scan(n, l, g * per, s, g, 17)
    st, w, kept, back = v.sizes()
    assert st == OK
    v.kept, v.space = (15 * PLACE, kept), (16 * PLACE, w)
    expect(OK, v.forward, (n, l, g, per, s))
    v.space = (16 * PLACE, back)
    expect(OK, v.backward, (n, l, g, per, s))
    expect(OK, v.step, (n, l, g, per, s))
    if n and back:
        v.space = (16 * PLACE, back - 16)
        if l:
            expect(INVALID, v.backward)
    if n and kept:
        v.space, v.kept = (16 * PLACE, PLACE), (15 * PLACE, kept - 1)
        expect(INVALID, v.forward)
        expect(INVALID, v.backward)
""")


def test_refusals_of_layer_norm(run):
    run("""
def both(status, change, forward=True, backward=True):
    v = Norm()
    change(v)
    if forward:
        expect(status, v.forward, change)
    if backward:
        expect(status, v.backward, change)
def put(**kw):
    return lambda v: v.__dict__.update(kw)
both(INVALID, put(x=None))
both(INVALID, put(y=None), backward=False)
both(INVALID, put(dy=None), forward=False)
both(INVALID, put(x=tensor((5, 40), 1)))
both(INVALID, put(x=tensor((6, 40), 1, 16)))
both(INVALID, put(gamma=tensor((39,), 5)))
both(INVALID, put(gamma=tensor((40,), 5, 16)))
both(INVALID, put(gamma=tensor((40, 1), 5)))
both(INVALID, put(dbeta=tensor((41,), 8)), forward=False)
both(INVALID, put(stats=tensor((7, 2), 9)))
both(INVALID, put(stats=tensor((6, 2), 9, 16)))
both(INVALID, put(stats=tensor((6, 2), 9, offset=4)))
both(INVALID, put(stats=None), forward=False)
for eps in (-1.0, float('nan'), float('inf')):
    both(INVALID, put(eps=eps), backward=False)
both(INVALID, put(y=tensor((6, 40), 1, offset=64)), backward=False)       # over the input
both(INVALID, put(dx=tensor((6, 40), 3)), forward=False)
both(INVALID, put(stats=tensor((6, 2), 2)), backward=False)               # over the output
both(INVALID, put(space=(7 * PLACE, 1 << 20)), forward=False)             # over dgamma
both(INVALID, put(space=(10 * PLACE + 8, PLACE)), forward=False)          # not aligned
both(INVALID, put(space=(None, 0)), forward=False)
wide = lambda i, s: put(**{('x', 'y', 'dy', 'dx')[i - 1]: tensor((6, 40), i, strides=s)})
both(OK, wide(1, (64, 1)))
both(OK, wide(2, (41, 1)), backward=False)
both(UNSUPPORTED, wide(1, (80, 2)))
both(UNSUPPORTED, wide(1, (39, 1)))
both(UNSUPPORTED, wide(1, (0, 1)))
both(UNSUPPORTED, wide(1, (-40, 1)))
both(UNSUPPORTED, put(gamma=tensor((40,), 5, strides=(2,))))
both(UNSUPPORTED, put(stats=tensor((6, 2), 9, strides=(3, 1))))
v = Norm((2, 3, 40))
v.x = tensor((2, 3, 40), 1, strides=(200, 40, 1))
expect(UNSUPPORTED, v.forward)
f64 = Norm((6, 40), 1)
expect(UNSUPPORTED, f64.forward)
for dims in ((40, 0), (1, 1, 1, 1, 4)):
    v = Norm((6, 40))
    v.x = v.y = api.Tensor()
    expect(INVALID, v.forward)
short = Norm()
short.x.bytes -= 4
expect(INVALID, short.forward)
expect(INVALID, short.backward)
""")


def test_refusals_of_the_convolution(run):
    run("""
def try_all(status, change, calls=('forward', 'backward', 'step')):
    v = Conv()
    change(v)
    for name in calls:
        expect(status, getattr(v, name), (change, name))
def put(**kw):
    return lambda v: v.__dict__.update(kw)
FB, F, B, S = ('forward', 'backward'), ('forward',), ('backward',), ('step',)
try_all(INVALID, put(x=None, x1=None))
try_all(INVALID, put(w=None))
try_all(INVALID, put(w=tensor((7, 4), 5)))
try_all(INVALID, put(w=tensor((8, 0), 5)))
try_all(INVALID, put(w=tensor((8, 4), 5, 16)))
try_all(INVALID, put(b=tensor((7,), 7)))
try_all(INVALID, put(y=tensor((2, 8, 8), 2), y1=tensor((2, 9), 2), dx=tensor((2, 9, 9), 4)))
try_all(INVALID, put(state=tensor((2, 4, 8), 9)))
try_all(INVALID, put(state=tensor((2, 3, 8), 9, 16)))
try_all(INVALID, put(out=tensor((2, 2, 8), 10)), ('forward', 'step'))
try_all(INVALID, put(dlast=tensor((2, 2, 8), 10)), B)
try_all(INVALID, put(lengths=13 * PLACE + 2), FB)
try_all(INVALID, put(out=tensor((2, 3, 8), 9, offset=32)), S)             # a state moved by a token
try_all(OK, put(out=tensor((2, 3, 8), 9)), S)                             # the state itself
try_all(INVALID, put(out=tensor((2, 3, 8), 9)), F)
try_all(INVALID, put(out=tensor((2, 3, 8), 9, strides=(24, 8, 1)), state=tensor((2, 3, 8), 9, strides=(48, 8, 1))), S)
try_all(INVALID, put(state=None), S)
try_all(INVALID, put(out=None), S)
try_all(OK, put(state=None, out=None), FB)
try_all(INVALID, put(y=tensor((2, 9, 8), 1), y1=tensor((2, 8), 1), dx=tensor((2, 9, 8), 1)))
try_all(INVALID, put(y=tensor((2, 9, 8), 13)), F)                         # over the lengths
try_all(INVALID, put(dw=tensor((8, 4), 8)), B)                            # over dbias
try_all(INVALID, put(space=(14 * PLACE, 64)), B)
try_all(OK, put(space=(None, 0), dw=None, db=None), B)
try_all(UNSUPPORTED, put(act=4))
try_all(UNSUPPORTED, put(w=tensor((8, 4), 5, strides=(1, 8))))
try_all(UNSUPPORTED, put(x=tensor((2, 9, 8), 1, strides=(72, 1, 9)), x1=tensor((2, 8), 1, strides=(1, 2))))
try_all(UNSUPPORTED, put(x=tensor((2, 9, 8), 1, strides=(0, 8, 1)), x1=tensor((2, 8), 1, strides=(0, 1))))
nine = Conv(k=9)
for call in (nine.forward, nine.backward, nine.step):
    expect(UNSUPPORTED, call)
f64 = Conv(dtype=1)
for call in (f64.forward, f64.backward, f64.step):
    expect(UNSUPPORTED, call)
""")


def test_refusals_of_the_scan(run):
    run("""
def try_all(status, change, calls=('sizes', 'forward', 'backward')):
    v = Scan()
    change(v)
    for name in calls:
        expect(status, getattr(v, name), (change, name))
def q(**kw):
    return lambda v: v.q.update(kw)
def g(**kw):
    return lambda v: v.g.update(kw)
def put(**kw):
    return lambda v: v.__dict__.update(kw)
F, B, S, FB = ('forward',), ('backward',), ('step',), ('forward', 'backward')
for name in ('x', 'dt', 'a', 'b', 'c'):
    try_all(INVALID, q(**{name: None}))
for name in ('d', 'dt_bias', 'state'):
    try_all(OK, q(**{name: None}))
try_all(INVALID, q(z=None), B)                                             # the gate's gradient without a gate
try_all(OK, lambda v: (v.q.update(z=None), v.g.update(z=None)))
try_all(INVALID, g(z=None), B)
try_all(INVALID, g(x=None), B)
try_all(INVALID, g(dt=None), B)
try_all(OK, lambda v: v.g.update(a=None, b=None, c=None, d=None, dt_bias=None, state=None), B)
try_all(INVALID, q(dt=tensor((2, 8, 8), 2)))
try_all(INVALID, q(dt=tensor((2, 9, 8), 2, 17)))
try_all(INVALID, q(b=tensor((2, 9, 3, 16), 4)))
try_all(INVALID, q(c=tensor((2, 9, 2, 15), 5)))
try_all(INVALID, q(a=tensor((8, 15), 3)))
try_all(INVALID, q(a=tensor((8, 16), 3, 17)))
try_all(INVALID, q(state=tensor((2, 8, 16), 9, 17)))
try_all(INVALID, q(state=tensor((2, 8, 15), 9)))
try_all(INVALID, put(lengths=14 * PLACE + 1))
try_all(INVALID, put(y=tensor((2, 9, 8), 4)), F)                           # over B
try_all(INVALID, put(out=tensor((2, 8, 16), 9)), F)                        # over the first state
try_all(INVALID, put(kept=(10 * PLACE, PLACE)), F)                         # over y
try_all(INVALID, put(kept=(15 * PLACE, 100)), FB)
try_all(INVALID, put(kept=(15 * PLACE + 4, PLACE)), FB)
try_all(OK, put(kept=(None, 0)), F)
try_all(INVALID, put(kept=(None, 0)), B)
try_all(INVALID, put(space=(None, 0)), B)
try_all(INVALID, put(space=(15 * PLACE, PLACE)), B)                        # over what was kept
try_all(INVALID, g(dt=tensor((2, 9, 8), 21)), B)                           # two gradients in one place
try_all(UNSUPPORTED, q(b=tensor((2, 9, 2, 16), 4, strides=(288, 32, 1, 2))))
try_all(UNSUPPORTED, q(x=tensor((2, 9, 8), 1, strides=(0, 8, 1))))
try_all(UNSUPPORTED, q(a=tensor((8, 16), 3, strides=(1, 8))))
wide = Scan(s=65)
for call in (wide.sizes, wide.forward, wide.backward, wide.step):
    expect(UNSUPPORTED, call)
f64 = Scan(dtype=1)
expect(UNSUPPORTED, f64.sizes)
expect(INVALID, lambda: lib.gc_b200_selective_scan_sizes(None, *[ref(ct.c_uint64())] * 3))
expect(INVALID, lambda: lib.gc_b200_selective_scan_sizes(ref(Scan().args(Scan().q, None)), None, None, None))
v = Scan()
expect(OK, v.step)
v.out = v.one['state']
expect(OK, v.step)
v.out = tensor((2, 8, 16), 9, offset=64)
expect(INVALID, v.step)
v.out = None
expect(INVALID, v.step)
v = Scan()
v.one['state'] = None
expect(INVALID, v.step)
""")


def test_the_last_plan_is_that_of_a_successful_call(run):
    run("""
plans = []
for call in CALLS:
    expect(OK, call)
    plans.append(native.last_plan().split()[0])
assert plans == ['kernel=' + k for k in ('layer_norm', 'layer_norm_backward', 'causal_conv', 'causal_conv_backward',
                                         'causal_conv_step', 'selective_scan', 'selective_scan_backward', 'selective_scan_step')], plans
flag('fake_launch_error').value = 2
for call in CALLS[:-1]:
    expect(DEVICE, call)
    assert native.last_plan().startswith('kernel=selective_scan_step ')
""")


def test_memory_that_runs_out_is_a_status(run):
    run("""
import threading
calls = CALLS + [Norm().size, Conv().size, Scan().sizes]
for no_memory in (0, 1):
    for call in calls:
        got = []

        def work():  # a thread of its own: its message slot is empty
            flag('fake_throw').value, flag('fake_no_memory').value = 1, no_memory
            st = call()
            flag('fake_throw').value = flag('fake_no_memory').value = 0
            got.append(st[0] if isinstance(st, tuple) else st)
            got.append(native.lib.gc_last_error())
        thread = threading.Thread(target=work)
        thread.start()
        thread.join()
        assert got == [DEVICE, b'' if no_memory else b'host resources exhausted'], (got, call)
for call in calls:
    expect(OK, call)
""")
