"""The transformer-block operators at the edges of their ranges: values that
are not finite or far from 1, sums that cancel, features of very different
sizes, long contractions, expired waits, and arguments that a call refuses.
Tolerances as in test_gpu_ops.py unless a test derives its own."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mlipcpp_b200 as mb  # noqa: E402
from test_gpu_ops import DTYPES, IDS, act64, c_of, gen, rand, unit  # noqa: E402

if torch.cuda.is_available():
    from mlipcpp_b200 import ops

ACTS = ("identity", "sigmoid", "silu", "gelu", "gelu_tanh", "relu")
# rows, in, out: the few-row kernels, one tile, a divided contraction
PATHS = [(4, 64, 40), (150, 64, 72), (150, 2560, 72)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(37, 512), (37, 300), (37, 301), (700, 2048), (3, 16384)], ids=str)
def test_no_gate_whatever_its_stride(dtype, shape):
    """From C, a gate that is not there is 1 also where its stride is that of
    a gate for every row: the same bits as with a stride of 0."""
    m, d = shape
    g = gen(m + d)
    r, y, ds, do = (rand(g, m, d, dtype=dtype) for _ in range(4))
    w, pw = rand(g, d, dtype=dtype, mean=1), rand(g, d, dtype=dtype, mean=1)

    def run(ldgate, backward):
        a, b = torch.zeros_like(r), torch.zeros_like(r)
        dw, dpw = torch.zeros_like(w), torch.zeros_like(w)
        at = lambda *t: [s.data_ptr() for s in t]  # noqa: E731
        args = ops._NORM.pack(ops._DTYPES[dtype], 1, 2, m, d, 0.5, 1e-5, *at(r, y, w), 0, *at(pw), 0, 0, d, d, ldgate,
                              *(at(a, b) if not backward else (0, 0)), d, d, *at(ds, do), d, d,
                              *(at(a, b, dw) + [0] + at(dpw) + [0, 0] if backward else (0,) * 7), d, d, d)
        ops._call("residual_norm", args, 0, backward)
        return a, b, dw, dpw

    for backward in (False, True):
        want = run(0, backward)
        assert want[0].abs().max() > 0
        for ldgate in (d, d + 8, 1):
            for s, t in zip(run(ldgate, backward), want):
                assert torch.equal(s, t)
    # no rows: a gradient of gates for each row has no elements to write
    guard = torch.full((d,), 7.0, dtype=dtype, device="cuda")
    args = ops._NORM.pack(ops._DTYPES[dtype], 1, 0, 0, d, 1.0, 1e-5, *(0,) * 7, d, d, d, 0, 0, d, d, 0, 0, d, d,
                          *(0,) * 6, guard.data_ptr(), d, d, d)
    ops._call("residual_norm", args, 0, True)
    assert (guard == 7).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 256), (40, 64), (4100, 2048), (3000, 520)], ids=str)
def test_expired_norm_wait_is_reported(dtype, shape):
    """Rows whose copies never come: their waits run out, the status says so
    once, and the next call is whole."""
    m, d = shape
    g = gen(m)
    r, y, gate = (rand(g, m, d, dtype=dtype) for _ in range(3))
    w = rand(g, d, dtype=dtype, mean=1)

    def run():
        s, o = ops.residual_norm(r, y, w, post_weight=w, gate=gate, post_norm="layer")
        return [s, o, *[t for t in ops.residual_norm_backward(r, y, r, y, w, post_weight=w, gate=gate, post_norm="layer")
                        if t is not None]]

    want = run()
    ops.check_status()
    L = mb.lib()
    for call in (lambda: ops.residual_norm(r, y, w), lambda: ops.residual_norm_backward(r, y, r, y, w)):
        assert L.mlipcpp_b200_set_wait_bound_ns(1_000_000) == mb.OK
        try:
            assert L.mlipcpp_b200_inject_norm_stall() == mb.OK
            call()
            with pytest.raises(mb.MLIPError) as e:
                ops.check_status()
            assert e.value.code == mb.COMPUTATION
        finally:
            assert L.mlipcpp_b200_set_wait_bound_ns(0) == mb.OK
        ops.check_status()
        for a, b in zip(run(), want):
            assert torch.equal(a, b)
    ops.check_status()


def test_expired_norm_wait_fails_the_prediction(model_file):
    """A norm of a pre-norm model that gives up a wait fails that prediction,
    and no operator call of someone else; the model stays usable."""
    from mlipcpp_b200 import workloads as wl
    p, s = mb.Predictor(model_file("pet-mad-s-gated")), wl.si_diamond(2, seed=3)
    args = (s.positions, s.numbers, s.cell)
    want = p.predict(*args)
    ops.check_status()
    L = mb.lib()
    assert L.mlipcpp_b200_set_wait_bound_ns(1_000_000) == mb.OK
    try:
        assert L.mlipcpp_b200_inject_norm_stall() == mb.OK
        with pytest.raises(mb.MLIPError) as e:
            p.predict(*args)
        assert e.value.code == mb.COMPUTATION
    finally:
        assert L.mlipcpp_b200_set_wait_bound_ns(0) == mb.OK
    ops.check_status()
    got = p.predict(*args)
    assert got.energy == want.energy and (got.forces == want.forces).all()
