"""Host side of group norm and dropout against a stand-in for the CUDA runtime
(fake_cudart.cpp): what a failed launch or an allocation that fails leaves
behind.  No GPU; each test in a process of its own, with the stand-in preloaded."""
import os
import subprocess
import sys

import pytest

from groupconv_atlas_b200 import api, build

SETUP = """
import ctypes as ct
from groupconv_atlas_b200 import api
fake = ct.CDLL(FAKE)
flag = lambda name: ct.c_int.in_dll(fake, name)
native = api.Native()
lib, ref = native.lib, ct.byref


def tensor(dims, base):  # channels last, FP32
    t = api.Tensor()
    n, c, h, w = dims
    t.data, t.bytes, t.device, t.rank = base, 4 * n * c * h * w, 1, 4
    for i, (size, stride) in enumerate(zip(dims, (h * w * c, 1, w * c, c))):
        t.dims[i], t.strides[i] = size, stride
    return t


def stats(n, groups, base):
    t = api.Tensor()
    t.data, t.bytes, t.device, t.rank = base, 8 * n * groups, 1, 3
    for i, (size, stride) in enumerate(zip((n, groups, 2), (2 * groups, 2, 1))):
        t.dims[i], t.strides[i] = size, stride
    return t


PLACE = 1 << 40


def forward(dims, groups, drop=None):
    x, y = tensor(dims, PLACE), tensor(dims, 2 * PLACE)
    return lib.gc_b200_group_norm(ref(x), None, None, ref(y), None, groups, 1e-5, 3, None, 6 * PLACE, PLACE, None)


def backward(dims, groups):
    x, dy, dx = (tensor(dims, (i + 1) * PLACE) for i in range(3))
    return lib.gc_b200_group_norm_backward(ref(dy), ref(x), None, None, ref(stats(dims[0], groups, 4 * PLACE)), ref(dx),
                                           None, None, groups, 3, None, 6 * PLACE, PLACE, None)


def dropout(dims):
    x, y = tensor(dims, PLACE), tensor(dims, 2 * PLACE)
    return lib.gc_b200_dropout(ref(x), None, ref(y), ref(api.dropout_args(0.5)), None)


RESIDENT, SMALL, SPLIT = ((2, 32, 6, 7), 4), ((5000, 24, 2, 2), 3), ((1, 64, 300, 260), 1)
CALLS = [lambda a=a, f=f: f(*a) for a in (RESIDENT, SMALL, SPLIT) for f in (forward, backward)]
CALLS.append(lambda: dropout((2, 32, 6, 7)))
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


def test_the_last_plan_is_that_of_a_successful_call(run):
    run("""
plans = []
for call in CALLS:
    assert call() == 0, native.lib.gc_last_error()
    plans.append(native.last_plan())
assert [p.split('engine=')[1].split()[0] for p in plans] == [
    'resident', 'resident_backward', 'small', 'small_backward', 'split', 'split_backward', 'element'], plans
before = flag('fake_launches').value
flag('fake_launch_error').value = 2
for call in CALLS[:-1]:
    assert call() == api.GC_DEVICE_ERROR and native.last_plan() == plans[-1], native.last_plan()
flag('fake_launch_error').value = 0
assert CALLS[0]() == 0
flag('fake_launch_error').value = 2
assert CALLS[-1]() == api.GC_DEVICE_ERROR and native.last_plan() == plans[0]
assert flag('fake_launches').value == before + 1
""")


def test_memory_that_runs_out_is_a_status(run):
    """No exception and no abort leaves an entry point, also where the message
    itself finds no memory."""
    run("""
import threading
calls = CALLS + [lambda: lib.gc_b200_group_norm_workspace(ref(tensor(*RESIDENT[:1], PLACE)), ref(tensor(*RESIDENT[:1], 2 * PLACE)),
                                                          4, ref(ct.c_uint64())),
                 lambda: lib.gc_b200_group_norm_backward_workspace(
                     *(ref(tensor(*RESIDENT[:1], (i + 1) * PLACE)) for i in range(3)), 4, ref(ct.c_uint64()))]
for no_memory in (0, 1):
    for call in calls:
        got = []

        def work():  # a thread of its own: its message slot is empty
            flag('fake_throw').value, flag('fake_no_memory').value = 1, no_memory
            got.append(call())
            flag('fake_throw').value = flag('fake_no_memory').value = 0
            got.append(native.lib.gc_last_error())
        thread = threading.Thread(target=work)
        thread.start()
        thread.join()
        assert got == [api.GC_DEVICE_ERROR, b'' if no_memory else b'host resources exhausted'], got
assert CALLS[0]() == 0
""")


def test_plans_of_many_shapes_are_bounded(run):
    """A program whose shapes never repeat keeps a bounded number of plans."""
    run("""
def use(first, count):
    for n in range(first, first + count):
        assert forward((n, 8, 2, 1), 2) == 0
    return flag('fake_live').value
use(1, 100)
start = use(1, 100)
assert use(1000, 12000) - start <= 5000, flag('fake_live').value - start
assert use(20000, 6000) - start <= 5000
""")


def test_outputs_over_the_generator_s_words_are_refused(run):
    """Seed and offset words are inputs: the kernels read them while others of
    their blocks already write."""
    run("""
def norm(drop, workspace=6 * PLACE):
    x, y = tensor((2, 32, 6, 7), PLACE), tensor((2, 32, 6, 7), 2 * PLACE)
    return lib.gc_b200_group_norm(ref(x), None, None, ref(y), ref(stats(2, 4, 3 * PLACE)), 4, 1e-5, 3, ref(drop),
                                  workspace, PLACE, None)
def grad(drop):
    x, dy, dx = (tensor((2, 32, 6, 7), (i + 1) * PLACE) for i in range(3))
    dgamma, dbeta = api.Tensor(), api.Tensor()
    for t, base in ((dgamma, 4 * PLACE), (dbeta, 4 * PLACE + 4096)):
        t.data, t.bytes, t.device, t.rank, t.dims[0], t.strides[0] = base, 128, 1, 1, 32, 1
    return lib.gc_b200_group_norm_backward(ref(dy), ref(x), None, None, ref(stats(2, 4, 5 * PLACE)), ref(dx), ref(dgamma),
                                           ref(dbeta), 4, 3, ref(drop), 6 * PLACE, PLACE, None)
def drop(args):
    x, y = tensor((2, 32, 6, 7), PLACE), tensor((2, 32, 6, 7), 2 * PLACE)
    return lib.gc_b200_dropout(ref(x), None, ref(y), ref(args), None)
size = 4 * 2 * 32 * 6 * 7
places = {norm: [2 * PLACE, 2 * PLACE + size - 8, 3 * PLACE + 8, 6 * PLACE + 800, 7 * PLACE - 8, 8 * PLACE],
          grad: [3 * PLACE + 8, 4 * PLACE + 120, 4 * PLACE + 4096, 6 * PLACE, 8 * PLACE], drop: [2 * PLACE + size - 8, 8 * PLACE]}
for call, at in places.items():
    for word in ('seed_ptr', 'offset_ptr'):
        for p in at:
            got = call(api.dropout_args(0.5, used=8 * PLACE, **{word: p}))
            assert got == api.GC_INVALID, (call.__name__, word, hex(p), got)
        for p in (9 * PLACE, 8 * PLACE + 16, 8 * PLACE - 8):
            assert call(api.dropout_args(0.5, used=8 * PLACE, **{word: p})) == 0, native.lib.gc_last_error()
""")
