"""Plans of the operators on sequences at sizes that no test can run, against the
stand-in for the CUDA runtime."""
from tests.test_sequence_host import run


def test_a_worker_of_the_convolution_takes_at_most_64_stretches(run):
    """What a worker adds up in 32 bits, of sequences of any number and length: 128
    tokens of a stretch and 64 stretches, before partial results are joined."""
    run("""
for n, l, c, k, dtype in [(8, 2048, 2048, 4, 17), (3, 1021, 333, 3, 0), (64, 1 << 20, 33, 4, 0), (1, 1 << 28, 4, 4, 17),
                          (1000, 70000, 129, 8, 16), (1 << 22, 200, 7, 1, 0), (4, 1 << 20, 8192, 4, 17), (5, 140000, 8192, 4, 17)]:
    v = Conv(n, l, c, k, dtype)
    st, need = v.size()
    assert st == OK
    v.space = (14 * PLACE, need)
    expect(OK, v.backward, (n, l, c, k))
    plan = dict(p.split('=') for p in native.last_plan().split()[1:])
    cols, stretch, segs, grid = (int(plan[name]) for name in ('lanes', 'per_lane', 'parts', 'grid'))
    vcols = c // 4 if plan['vec'] == '1' else c
    blocks = grid // -(-vcols // cols)  # of a tile of columns
    assert stretch <= 128 and segs == -(-l // stretch)
    assert n * segs <= 64 * blocks * (256 // cols), (n, l, c, k, native.last_plan())
""")
