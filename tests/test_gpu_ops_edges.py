"""The transformer-block operators at the edges of their ranges: values that
are not finite or far from 1, sums that cancel, features of very different
sizes, long contractions, expired waits, and arguments that a call refuses.
Tolerances as in test_gpu_ops.py unless a test derives its own."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mlipcpp_b200 as mb  # noqa: E402
from test_gpu_ops import DTYPES, IDS, act64, c_of, check_gated, gen, rand, unit  # noqa: E402

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


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", PATHS, ids=str)
def test_nan_reaches_the_results(dtype, act, shape):
    """A NaN in x, a weight or a bias makes exactly the results and gradients
    NaN that it makes NaN in float64."""
    m, k, n = shape
    g = gen(m + k)
    clean = [rand(g, m, k, dtype=dtype), rand(g, n, k, dtype=dtype, std=k ** -0.5),
             rand(g, n, k, dtype=dtype, std=k ** -0.5), rand(g, n, dtype=dtype), rand(g, n, dtype=dtype)]
    dy = rand(g, m, n, dtype=dtype)
    for i, at in ((0, (2, 5)), (1, (7, 9)), (3, (11,))):
        t = [c.clone() for c in clean]
        t[i][at] = float("nan")
        x, w, v, b, c = t
        X, W, V, B, C, D = (s.double() for s in (*t, dy))
        a, da = act64(act, X @ W.T + B)
        z = X @ V.T + C
        # (an activation has no derivative at NaN: relu's is 0, the others' NaN)
        dz, dg, dv = D * da, D * z * da, D * a
        for got, ref, what in (
                (ops.linear(x, w, b, act), a, "y"),
                (ops.gated_linear(x, w, v, b, c, act), a * z, "h"),
                *zip(ops.linear_backward(dy, x, w, b, act), (dz @ W, dz.T @ X, dz.sum(0)), ("dx", "dw", "db")),
                *zip(ops.gated_linear_backward(dy, x, w, v, b, c, act),
                     (dg @ W + dv @ V, dg.T @ X, dv.T @ X, dg.sum(0), dv.sum(0)),
                     ("dx", "dw_gate", "dw_value", "db_gate", "db_value"))):
            assert torch.equal(got.isnan(), ref.isnan()), (i, what, int(got.isnan().sum()), int(ref.isnan().sum()))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", PATHS, ids=str)
def test_activations_far_out(dtype, act, shape):
    """Where an activation has reached its limits (|z| >= 100): 0, 1 or z, and
    a derivative of 0 or 1, up to one rounding and, in f32, what the 22 bits of a
    product's operands leave.  z is one element of x times 1, the value half 1."""
    m, k, n = shape
    far = [100.0, 2e3, 5e4] if dtype == torch.float16 else [100.0, 2e3, 1e6, 1e10, 1e12, 1e13, 1e18, 1e20, 1e30, 1e36, 3e38]
    far = torch.tensor(far, device="cuda").to(dtype)
    z = torch.cat([far, -far])
    w, v = torch.zeros(n, k, dtype=dtype, device="cuda"), torch.zeros(n, k, dtype=dtype, device="cuda")
    w[0, 0] = 1
    c = torch.ones(n, dtype=dtype, device="cuda")
    u = 1.01 * unit(dtype) + (2.0 ** -22 if dtype == torch.float32 else 0)
    for i in range(0, len(z), m):
        zi = z[i:i + m]
        x = torch.zeros(m, k, dtype=dtype, device="cuda")
        x[:len(zi), 0] = zi
        a, da = act64(act, zi.double())
        one = torch.zeros(m, n, dtype=dtype, device="cuda")
        one[:, 0] = 1
        rows = slice(0, len(zi))
        for got, ref, what in (
                (ops.linear(x, w, None, act)[rows, 0], a, "y"),
                (ops.linear_backward(one, x, w, None, act)[0][rows, 0], da, "dx"),
                (ops.gated_linear(x, w, v, None, c, act)[rows, 0], a, "h"),
                (ops.gated_linear_backward(one, x, w, v, None, c, act)[0][rows, 0], da, "gated dx")):
            # p = 1 / (1 + e^-z) is 0 or 1 to 2^-126 here
            assert ((got.double() - ref).abs() <= u * ref.abs() + 1e-30).all(), (what, zi, got, ref)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(5, 640, 529), (3000, 640, 529), (200, 2500, 72)], ids=str)
def test_relu_of_sums_that_cancel(dtype, shape):
    """Two terms of 2^12 that cancel leave a third one of 2^-24 or -2^-24,
    which is below the last bit of a 32-bit sum: the derivative is the third
    term's."""
    m, k, f = shape
    g = gen(7 * m + k)
    x, w = rand(g, m, k, dtype=dtype), rand(g, f, k, dtype=dtype, std=k ** -0.5)
    x[:, 0] = x[:, 1] = 1
    x[:, 2] = 2.0 ** -10
    x[::2, 2] = -2.0 ** -10
    w[5::40] = 0
    w[5::40, 0], w[5::40, 1], w[5::40, 2] = 2.0 ** 12, -2.0 ** 12, 2.0 ** -14
    dy = rand(g, m, f, dtype=dtype)
    zero, v = torch.zeros(f, dtype=dtype, device="cuda"), rand(g, f, k, dtype=dtype, std=k ** -0.5)
    dz = dy.double() * (x.double() @ w.double().T > 0)
    # each term counts whole or not at all
    db = ops.linear_backward(dy, x, w, zero, "relu")[2]
    assert ((db.double() - dz.sum(0)).abs() <= unit(dtype) * dz.sum(0).abs() + 2.0 ** -18 * dz.abs().sum(0))[5::40].all()
    dbg = ops.gated_linear_backward(dy, x, w, v, zero, None, "relu")[3]
    t = dz * (x.double() @ v.double().T)
    # (the value's own sum is good to c_of of its terms)
    e = (dz.abs() * (x.double().abs() @ v.double().abs().T)).sum(0) * c_of(k, dtype)
    assert ((dbg.double() - t.sum(0)).abs() <= unit(dtype) * t.sum(0).abs() + e + 2.0 ** -15 * t.abs().sum(0))[5::40].all()


@pytest.mark.parametrize("m", [150, 700])
def test_f32_features_of_different_sizes(m):
    """f32 products keep their accuracy in every row and column on its own:
    weights whose output features, and weights and inputs whose input
    features, lie up to 2^-36 below the largest of their matrix.

    The bound is c_of of the terms' magnitude, per element of each result: a
    feature's scale multiplies all terms of its row or column alike, and along
    a contraction the sizes of both factors fall together, so that a block's
    largest elements meet."""
    k, n = 200, 300
    g = gen(m)
    f32 = torch.float32
    fall = 2.0 ** torch.linspace(0, -36, n, device="cuda").round()
    wide = 2.0 ** torch.linspace(0, -36, k, device="cuda").round()

    def mixed(t, perm_seed):
        return t[torch.randperm(len(t), generator=gen(perm_seed)).cuda()]

    rows, cols = mixed(fall, 1), mixed(wide, 2)
    x = rand(g, m, k, dtype=f32) * cols
    w = rand(g, n, k, dtype=f32) * rows[:, None] * cols
    v = rand(g, n, k, dtype=f32) * rows[:, None] * cols
    dy = rand(g, m, n, dtype=f32)
    c = c_of(max(m, 2 * n), f32) + 2.0 ** -22
    X, W, V, D = (t.double() for t in (x, w, v, dy))

    def check(got, a, b, what):
        ref, s = a @ b, a.abs() @ b.abs()
        bad = (got.double() - ref).abs() / s
        assert (bad <= c).all(), (what, bad.max().item(), c)

    check(ops.linear(x, w), X, W.T, "y")
    dx, dw, _ = ops.linear_backward(dy, x, w)
    check(dx, D, W, "dx")
    check(dw, D.T, X, "dw")
    # with one projection the identity of the other: h = (x Wg^T) (x Wv^T)
    h = ops.gated_linear(x, w, v, None, None, "identity")
    gate, value = X @ W.T, X @ V.T
    sg, sv = X.abs() @ W.abs().T, X.abs() @ V.abs().T
    assert ((h.double() - gate * value).abs() <= c * (sg * value.abs() + gate.abs() * sv + c * sg * sv)
            + 2.0 ** -22 * (gate * value).abs()).all()
    gdx, dwg, dwv, _, _ = ops.gated_linear_backward(dy, x, w, v, None, None, "identity")
    dg, dv = D * value, D * gate
    eg, ev = D.abs() * sv * c + 2.0 ** -22 * dg.abs(), D.abs() * sg * c + 2.0 ** -22 * dv.abs()
    for got, ref, tol, what in (
            (gdx, dg @ W + dv @ V, (c * dg.abs() + eg) @ W.abs() + (c * dv.abs() + ev) @ V.abs(), "gated dx"),
            (dwg, dg.T @ X, (c * dg.abs() + eg).T @ X.abs(), "dw_gate"),
            (dwv, dv.T @ X, (c * dv.abs() + ev).T @ X.abs(), "dw_value")):
        assert ((got.double() - ref).abs() <= tol).all(), (what, ((got.double() - ref).abs() / tol).max().item())


def test_long_f16_contraction():
    """A weight's gradient over 2^20 tokens: the additions of one accumulator
    lose at most half a rounding of the result in all, however long the
    contraction is.  All elements of dy^T x are the same sum of equal terms."""
    m, n = 1 << 20, 2304
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    f16 = torch.float16
    a, b, scale = 1 + 37 / 1024, 1 + 101 / 1024, 2.0 ** -14
    x, dy = torch.full((m, n), a, dtype=f16, device="cuda"), torch.full((m, n), b, dtype=f16, device="cuda")
    dw = ops.linear_backward(dy, x, x[:n], scale=scale, needs=(False, True, False))[1]
    ref = m * a * b * scale
    u = unit(f16)
    assert (dw.double() - ref).abs().max().item() <= 1.5 * u * (1 + u) * ref


def test_long_f16_projection():
    """Both projections with more inputs than one accumulator takes, over more
    tiles than there are SMs."""
    g, f16 = gen(33), torch.float16
    m, k, f = 2000, 33000, 2700
    x, dh = rand(g, m, k, dtype=f16), rand(g, m, f, dtype=f16)
    wg, wv = rand(g, f, k, dtype=f16, std=k ** -0.5), rand(g, f, k, dtype=f16, std=k ** -0.5)
    check_gated(x, wg, wv, None, dh[0], "silu", dh)


def test_forward_mode_is_refused():
    """The operators have no forward-mode derivatives: a dual tensor is turned
    down instead of losing its tangent."""
    from torch.autograd import forward_ad
    x, w = torch.randn(20, 32, device="cuda"), torch.randn(32, 32, device="cuda")
    calls = [lambda a, b: ops.linear(a, b), lambda a, b: ops.gated_linear(a, b, w), lambda a, b: ops.residual_norm(a, b[:20]),
             lambda a, b: ops.linear_backward(x, a, b), lambda a, b: ops.linear(x, w, residual=a, bias=b[0])]
    with forward_ad.dual_level():
        dx, dw = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        for call in calls:
            for a, b in ((dx, w), (x, dw)):
                with pytest.raises(mb.MLIPError):
                    call(a, b)
            call(x, w)
    for call in calls:
        call(x, w)


def test_every_expired_wait_is_reported_once():
    """Waits given up between, beside and after checks, on two streams: each
    check tells whether there were any since the last one."""
    L = mb.lib()
    r = torch.randn(40, 256, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def expire(stream):
        with torch.cuda.stream(stream):
            assert L.mlipcpp_b200_inject_norm_stall() == mb.OK
            ops.residual_norm(r)
        stream.synchronize()

    def failed(stream):
        with torch.cuda.stream(stream):
            try:
                ops.check_status()
            except mb.MLIPError as e:
                assert e.code == mb.COMPUTATION
                return True
        return False

    assert L.mlipcpp_b200_set_wait_bound_ns(1_000_000) == mb.OK
    try:
        for a in streams:
            for b in streams:
                assert not failed(b)
                expire(a)
                assert failed(b) and not failed(a) and not failed(b)
                expire(a)
                expire(b)
                assert failed(a) and not failed(b)
    finally:
        assert L.mlipcpp_b200_set_wait_bound_ns(0) == mb.OK
    assert not failed(streams[0])


@pytest.mark.parametrize("m", [1, 8, 16])
def test_long_f16_rows(m):
    """The same of a few rows with 2^22 inputs."""
    k, n = 1 << 22, 40
    f16 = torch.float16
    a, b, scale = 1 + 37 / 1024, 1 + 101 / 1024, 2.0 ** -16
    x, w = torch.full((m, k), a, dtype=f16, device="cuda"), torch.full((n, k), b, dtype=f16, device="cuda")
    y = ops.linear(x, w, scale=scale)
    ref, u = k * a * b * scale, unit(f16)
    assert (y.double() - ref).abs().max().item() <= 1.5 * u * (1 + u) * ref


def test_long_f16_tokens():
    """Both weights' gradients over more tokens than one accumulator takes,
    over more tiles than there are SMs."""
    g, f16 = gen(34), torch.float16
    m, k, f = 40000, 1024, 3000
    x, dh = rand(g, m, k, dtype=f16), rand(g, m, f, dtype=f16, std=2.0 ** -6)
    wg, wv = rand(g, f, k, dtype=f16, std=k ** -0.5), rand(g, f, k, dtype=f16, std=k ** -0.5)
    check_gated(x, wg, wv, None, None, "gelu_tanh", dh)
