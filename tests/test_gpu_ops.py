"""The transformer-block operators (mlipcpp_b200.ops) against their
definitions in float64, elementwise.

The tolerances are bounds, worked out per element from the rounding steps:
  * a result of type t is rounded once: u |ref|, u = finfo(t).eps / 2;
  * a product of K terms in 16 bits has exact terms and at most K / 16 + 4
    truncating additions of its partial sums, each losing at most 2^-23 of
    S = |x| |w|^T: c(K) S with c = (K / 16 + 4) 2^-23; with few rows the
    terms are added with FMAs, at most K / 32 + 16 in a row, 2^-24 each,
    which c(K) covers twice over;
  * in f32 each operand has 22 bits (2^-22 of it each, lo lo dropped) and
    every 128 terms are 24 truncating additions, joined with rounded ones:
    c = 2^-20 + (24 + K / 128) 2^-23 relative to the block maxima's products,
    taken as 4 times that of S (a block's largest element against its mean);
  * |act'| <= 1.13 and |act''| <= 1.6 for every activation but relu, whose
    derivative jumps: an element closer to 0 than its error may count whole;
  * gradients that enter a product are rounded to t: u of each term.
Fast exponentials and reciprocals are good to 2^-20."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mlipcpp_b200 as mb  # noqa: E402

if torch.cuda.is_available():
    from mlipcpp_b200 import ops

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]
L1, L2 = 1.13, 1.6


def unit(t):
    return torch.finfo(t).eps / 2


def c_of(k, dtype):
    if dtype == torch.float32:
        return 4 * (2.0 ** -20 + (24 + k / 128) * 2.0 ** -23)
    return (k / 16 + 4) * 2.0 ** -23


def act64(name, z):
    """(act, act') in float64."""
    if name == "identity":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "gelu":
        p = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        a = 2 * math.sqrt(2 / math.pi)
        p = torch.sigmoid(a * (z + 0.044715 * z ** 3))
        return z * p, p + z * p * (1 - p) * a * (1 + 3 * 0.044715 * z * z)
    p = torch.sigmoid(z)
    return (p, p * (1 - p)) if name == "sigmoid" else (z * p, p * (1 + z * (1 - p)))


def rand(g, *shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * std + mean).to(dtype).cuda()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def close(got, ref, tol, what):
    got = got.double()
    assert got.shape == ref.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    # twice the smallest step of the type, for results that underflow
    tol = tol + 2.0 ** -24
    bad = (got - ref).abs() > tol
    if bad.any():
        i = ((got - ref).abs() / tol).argmax().item()
        i = np.unravel_index(i, tuple(ref.shape))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst at {i}: {got[i].item()} vs "
                             f"{ref[i].item()} (tolerance {tol[i].item():.3g})")


def dense(x, w, b, dtype):
    """(x w^T + b, bound of its error) in float64."""
    z = x @ w.T
    s = x.abs() @ w.abs().T
    e = c_of(x.shape[1], dtype) * s
    if b is not None:
        z = z + b
        e = e + 2.0 ** -23 * (s + b.abs())
    return z, e


def d_of(*ts):
    return [None if t is None else t.double() for t in ts]


# (rows, in, out): one row, the few-row kernel and its end, one past a tile,
# odd sizes, widths of one, several tiles of every kind
SHAPES = [(1, 64, 64), (1, 1, 1), (3, 257, 130), (8, 1000, 96), (9, 64, 64), (31, 129, 65), (128, 128, 128),
          (129, 192, 257), (200, 1, 7), (257, 333, 1), (300, 2050, 136), (1000, 512, 520), (4101, 136, 1100),
          (2500, 1030, 600)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("bias", [False, True])
def test_gated_linear(shape, dtype, bias):
    m, k, f = shape
    act = ops.ACTIVATIONS[(m + k) % 6]
    g = gen(m * 7 + k)
    x, wg, wv = rand(g, m, k, dtype=dtype), rand(g, f, k, dtype=dtype, std=k ** -0.5), \
        rand(g, f, k, dtype=dtype, std=k ** -0.5)
    bg, bv = (rand(g, f, dtype=dtype), rand(g, f, dtype=dtype)) if bias else (None, None)
    check_gated(x, wg, wv, bg, bv, act, rand(g, m, f, dtype=dtype))


def check_gated(x, wg, wv, bg, bv, act, dh):
    dtype, u = x.dtype, unit(x.dtype)
    h = ops.gated_linear(x, wg, wv, bg, bv, act)
    X, G, V, BG, BV, D = d_of(x, wg, wv, bg, bv, dh)
    z, ez = dense(X, G, BG, dtype)
    v, ev = dense(X, V, BV, dtype)
    a, da = act64(act, z)
    ea = L1 * ez + 2.0 ** -20 * (a.abs() + z.abs())
    close(h, a * v, u * (a * v).abs() * 1.01 + ea * v.abs() + (a.abs() + ea) * ev + 2.0 ** -22 * (a * v).abs(), "h")
    got = ops.gated_linear_backward(dh, x, wg, wv, bg, bv, act)
    dg, dv = D * v * da, D * a
    eda = L2 * ez + 2.0 ** -19 * (1 + z.abs())
    if act == "relu":
        eda = ((z.abs() <= ez).double()) * 1.0
    edg = D.abs() * (v.abs() * eda + L1 * ev) + (u + 2.0 ** -21) * dg.abs() + 2.0 ** -25
    edv = D.abs() * ea + (u + 2.0 ** -21) * dv.abs() + 2.0 ** -25
    check_products(got[0], [(dg, edg, G), (dv, edv, V)], dtype, "dx")
    for i, (t, e) in enumerate(((dg, edg), (dv, edv))):
        check_products(got[1 + i], [(t.T, e.T, X)], dtype, ("dw_gate", "dw_value")[i])
        if (bg, bv)[i] is not None:
            check_sum(got[3 + i], t, e, dtype, ("db_gate", "db_value")[i])
        else:
            assert got[3 + i] is None


def check_products(got, terms, dtype, what):
    """got = sum of a @ b over terms (a, error of a, b)."""
    ref = sum(a @ b for a, _, b in terms)
    k = sum(a.shape[1] for a, _, _ in terms)
    tol = sum(e @ b.abs() + c_of(k, dtype) * (a.abs() @ b.abs()) for a, e, b in terms)
    close(got, ref, tol + unit(dtype) * (ref.abs() + tol), what)


def check_sum(got, t, e, dtype, what):
    tol = e.sum(0) + t.abs().sum(0) * (t.shape[0] / 64 + 32) * 2.0 ** -24
    close(got, t.sum(0), tol + unit(dtype) * (t.sum(0).abs() + tol), what)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("act", ["identity", "gelu", "silu"])
def test_linear(shape, dtype, act):
    m, k, n = shape
    g = gen(m * 5 + k)
    x, w = rand(g, m, k, dtype=dtype), rand(g, n, k, dtype=dtype, std=k ** -0.5)
    full = (m + n) % 2 == 0
    b, r, scale = (rand(g, n, dtype=dtype), rand(g, m, n, dtype=dtype), 0.5) if full else (None, None, 1.0)
    check_linear(x, w, b, act, r, scale, rand(g, m, n, dtype=dtype))


def check_linear(x, w, b, act, r, scale, dy):
    dtype, u = x.dtype, unit(x.dtype)
    y = ops.linear(x, w, b, act, r, scale)
    X, W, B, R, D = d_of(x, w, b, r, dy)
    z, ez = dense(X, W, B, dtype)
    a, da = act64(act, z)
    ref = scale * a + (0 if r is None else R)
    tol = abs(scale) * (L1 * ez + 2.0 ** -20 * (a.abs() + z.abs()))
    close(y, ref, tol + u * (ref.abs() + tol) + 2.0 ** -23 * ref.abs(), "y")
    got = ops.linear_backward(dy, x, w, b, act, scale)
    dz = scale * D * da
    if act == "identity":
        ed = 2.0 ** -23 * dz.abs()
    else:
        ed = abs(scale) * D.abs() * (L2 * ez + 2.0 ** -19 * (1 + z.abs())) + (u + 2.0 ** -21) * dz.abs() + 2.0 ** -25
    check_products(got[0], [(dz, ed, W)], dtype, "dx")
    check_products(got[1], [(dz.T, ed.T, X)], dtype, "dw")
    if b is not None:
        check_sum(got[2], dz, ed, dtype, "db")
    else:
        assert got[2] is None


def norm64(kind, t, eps):
    """(normalised rows, 1 / sigma, largest |t| / sigma of the row)."""
    if kind == "none":
        return t, torch.ones_like(t[:, :1]), t.abs()
    c = t - t.mean(1, keepdim=True) if kind == "layer" else t
    inv = 1 / ((c * c).mean(1, keepdim=True) + eps).sqrt()
    return c * inv, inv, t.abs().amax(1, keepdim=True) * inv


def norm_back64(kind, dn, n, inv):
    if kind == "none":
        return dn
    d = dn - n * (dn * n).mean(1, keepdim=True)
    return inv * (d - dn.mean(1, keepdim=True) if kind == "layer" else d)


NORM_SHAPES = [(1, 1), (1, 64), (5, 7), (9, 256), (17, 300), (64, 512), (33, 513), (40, 1024), (7, 1500), (21, 2048),
               (6, 4096), (3, 5000), (2, 8192), (2, 16384), (700, 40)]
NORM_HOW = [("rms", "none", None), ("rms", "rms", "channel"), ("layer", "layer", "row"), ("none", "rms", None),
            ("layer", "none", "channel")]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("how", NORM_HOW, ids=str)
def test_residual_norm(shape, dtype, how):
    check_norm(shape, dtype, how, bias=shape[0] % 2 == 1)


def check_norm(shape, dtype, how, bias, offset=0.0):
    """Rounding: a sum over a row adds at most 32 numbers in turn and then in
    trees, 2^-19 of its terms' magnitude at most, so a mean is off by 2^-19 of
    the row's largest element and a normalised element by 2^-18 of (largest
    element / sigma) + itself; the gradients are linear in these."""
    m, d = shape
    kind, post, gated = how
    scale, eps, u = 0.75, 1e-5, unit(dtype)
    g = gen(m + d)
    r, y = rand(g, m, d, dtype=dtype, mean=offset), rand(g, m, d, dtype=dtype)
    w = rand(g, d, dtype=dtype, std=0.2, mean=1) if kind != "none" else None
    b = rand(g, d, dtype=dtype) if bias and w is not None else None
    pw = rand(g, d, dtype=dtype, std=0.2, mean=1) if post != "none" else None
    pb = rand(g, d, dtype=dtype) if bias and pw is not None else None
    gate = {None: None, "channel": rand(g, d, dtype=dtype), "row": rand(g, m, d, dtype=dtype)}[gated]
    ds, do = rand(g, m, d, dtype=dtype), rand(g, m, d, dtype=dtype)
    args = (r, y, w, b, pw, pb, gate, scale, kind, post, eps)
    stream, out = ops.residual_norm(*args)
    R, Y, W, B, PW, PB, GT, DS, DO = d_of(r, y, w, b, pw, pb, gate, ds, do)
    one = torch.ones(1, d, dtype=torch.float64, device="cuda")
    e18 = 2.0 ** -18
    pn, pinv, pbig = norm64(post, Y, eps)
    epn = e18 * (pbig + pn.abs()) if post != "none" else torch.zeros_like(pn)
    PWv, GTv = (one if PW is None else PW), (one if GT is None else GT)
    uu = pn * PWv + (0 if PB is None else PB)
    eu = epn * PWv.abs() + 2.0 ** -22 * (uu.abs() + (pn * PWv).abs())
    s = scale * R + GTv * uu
    es = eu * GTv.abs() + 2.0 ** -22 * (s.abs() + (GTv * uu).abs() + (scale * R).abs())
    close(stream, s, u * (s.abs() + es) + es, "stream")
    n, inv, big = norm64(kind, s, eps)
    # an element's own error, the row's through the mean and sigma
    rowe = (es.amax(1, keepdim=True)) * inv
    en = e18 * (big + n.abs()) + 4 * rowe * (1 + n.abs()) if kind != "none" else es
    Wv = one if W is None else W
    o = n * Wv + (0 if B is None else B)
    eo = en * Wv.abs() + 2.0 ** -22 * (o.abs() + (n * Wv).abs())
    close(out, o, u * (o.abs() + eo) + eo, "out")

    got = ops.residual_norm_backward(ds, do, *args)
    dn = DO * Wv
    dxs = norm_back64(kind, dn, n, inv)
    gs = DS + dxs
    ndn = dn.abs().mean(1, keepdim=True) * (1 + n.abs()) + (dn * n).abs().mean(1, keepdim=True) * n.abs() + dn.abs()
    rel = (en.amax(1, keepdim=True) + 2.0 ** -17)  # relative error of n, sigma and the means
    egs = 8 * rel * inv * (ndn + n.abs().amax(1, keepdim=True) * ndn.amax(1, keepdim=True)) + 2.0 ** -21 * gs.abs() \
        if kind != "none" else 2.0 ** -21 * (gs.abs() + dn.abs())
    close(got.residual, scale * gs, (scale * egs + u * (scale * gs).abs()) * 1.01, "dresidual")
    du = gs * GTv
    edu = egs * GTv.abs() + 2.0 ** -22 * du.abs()
    dp = du * PWv
    edp = edu * PWv.abs() + 2.0 ** -22 * dp.abs()
    dy = norm_back64(post, dp, pn, pinv)
    if post != "none":
        ndp = dp.abs().mean(1, keepdim=True) * (1 + pn.abs()) + (dp * pn).abs().mean(1, keepdim=True) * pn.abs() + dp.abs()
        prel = epn.amax(1, keepdim=True) + 2.0 ** -17
        edy = 8 * prel * pinv * (ndp + pn.abs().amax(1, keepdim=True) * ndp.amax(1, keepdim=True)) \
            + pinv * (edp + (edp.mean(1, keepdim=True) * (1 + pn.abs() * pn.abs().amax(1, keepdim=True))))
    else:
        edy = edp
    close(got.y, dy, (edy + u * dy.abs()) * 1.01, "dy")
    vectors = {"weight": (w, DO * n, DO.abs() * en), "bias": (b, DO, 0 * DO),
               "post_weight": (pw, du * pn, edu * pn.abs() + du.abs() * epn), "post_bias": (pb, du, edu)}
    if gated == "channel":
        vectors["gate"] = (gate, gs * uu, egs * uu.abs() + gs.abs() * eu)
    for name, (t, term, e) in vectors.items():
        if t is None:
            assert getattr(got, name) is None
        else:
            check_sum(getattr(got, name), term, e + 2.0 ** -22 * term.abs(), dtype, name)
    if gated == "row":
        ref, e = gs * uu, egs * uu.abs() + gs.abs() * eu
        close(got.gate, ref, (e + u * ref.abs()) * 1.01, "dgate")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norm_far_from_zero(kind, dtype):
    """A mean far above the spread: the variance is taken about the mean."""
    check_norm((20, 640), dtype, (kind, "none", None), True, offset=30.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_norm_constant_rows(dtype):
    """Rows of zeros and of one value: sigma is sqrt(eps), nothing overflows."""
    r = torch.zeros(3, 96, dtype=dtype, device="cuda")
    r[1] = 2.0
    for kind in ("rms", "layer"):
        s, o = ops.residual_norm(r, norm=kind)
        assert torch.equal(s, r)
        assert (o[0] == 0).all()
        # 2 / sqrt(4 + eps) is 1 to 2^-19; a constant row about its mean is 0
        ref = 1.0 if kind == "rms" else 0.0
        assert (o[1].double() - ref).abs().max().item() <= unit(dtype) + 2.0 ** -18
        g = ops.residual_norm_backward(None, torch.ones_like(r), r, norm=kind)
        assert torch.isfinite(g.residual).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_strided_and_unaligned(dtype):
    """Row strides beyond the rows, odd starts and odd strides."""
    g = gen(3)
    big = rand(g, 300, 513, dtype=dtype)
    wb = rand(g, 220, 400, dtype=dtype, std=0.05)
    for m in (5, 150):
        for x in (big[:m, :136], big[:m, 1:137], big[:2 * m:2, 8:144], big.T[:m, :136]):
            dh = big[100:100 + m, 200:300]
            check_gated(x, wb[:100, :136], wb[100:200, 3:139], None, wb[0, :100], "silu", dh)
            check_linear(x, wb[:100, 5:141], wb[1, :100], "gelu", big[:m, 300:400], 0.5, dh)
        a = big[:m, 1:129]
        s, o = ops.residual_norm(a, big[:m, 130:258], wb[0, 1:129], norm="layer")
        s2, o2 = ops.residual_norm(a.contiguous(), big[:m, 130:258].contiguous(), wb[0, 1:129].clone(), norm="layer")
        assert torch.equal(s, s2) and (o.double() - o2.double()).abs().max() <= 2.0 ** -17 + 4 * unit(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_expanded_gradient_and_leading_dimensions(dtype):
    g = gen(4)
    x, w = rand(g, 2, 3, 20, 64, dtype=dtype), rand(g, 48, 64, dtype=dtype, std=0.1)
    y = ops.linear(x, w)
    assert y.shape == (2, 3, 20, 48)
    assert torch.equal(y.reshape(-1, 48), ops.linear(x.reshape(-1, 64), w))
    one = torch.ones(1, device="cuda", dtype=dtype).expand(2, 3, 20, 48)
    dx, dw, _ = ops.linear_backward(one, x, w)
    ex, ew, _ = ops.linear_backward(one.contiguous(), x, w)
    assert torch.equal(dx, ex) and torch.equal(dw, ew) and dx.shape == x.shape


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m", [3, 64])
def test_same_tensor_twice(dtype, m):
    """One weight for both projections, and x as its own residual."""
    g = gen(5)
    x, w = rand(g, m, 96, dtype=dtype), rand(g, 96, 96, dtype=dtype, std=0.1)
    check_gated(x, w, w, None, None, "silu", rand(g, m, 96, dtype=dtype))
    check_linear(x, w, None, "identity", x, 1.0, x)
    a = ops.residual_norm(x, x, w[0], w[0])
    b = ops.residual_norm(x, x.clone(), w[0].clone(), w[0].clone())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_no_rows(dtype):
    x, w = torch.empty(0, 64, dtype=dtype, device="cuda"), torch.ones(32, 64, dtype=dtype, device="cuda")
    b = torch.ones(32, dtype=dtype, device="cuda")
    assert ops.gated_linear(x, w, w, b, b).shape == (0, 32)
    assert ops.linear(x, w, b).shape == (0, 32)
    dh = torch.empty(0, 32, dtype=dtype, device="cuda")
    dx, *grads = ops.gated_linear_backward(dh, x, w, w, b, b)
    assert dx.shape == (0, 64) and all((t == 0).all() for t in grads)
    dx, *grads = ops.linear_backward(dh, x, w, b)
    assert dx.shape == (0, 64) and all((t == 0).all() for t in grads)
    v = torch.ones(64, dtype=dtype, device="cuda")
    s, o = ops.residual_norm(x, x, v, v, v, v, v, post_norm="rms")
    assert s.shape == o.shape == (0, 64)
    g = ops.residual_norm_backward(x, x, x, x, v, v, v, v, v, post_norm="rms")
    assert all((t == 0).all() for t in g[2:])


def test_f32_large_and_small_values():
    """Rows, weights and features of very different sizes: each row keeps its
    own scale, and a weight far below its matrix's largest keeps 2^-40 of it."""
    g = gen(8)
    x = rand(g, 140, 200, dtype=torch.float32) * (10.0 ** torch.linspace(-18, 18, 140, device="cuda"))[:, None]
    w = rand(g, 72, 200, dtype=torch.float32)
    y = ops.linear(x, w)
    ref = x.double() @ w.double().T
    s = x.double().abs() @ w.double().abs().T
    assert ((y.double() - ref).abs() <= (c_of(200, torch.float32) + 2.0 ** -24) * s).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m", [4, 40])
def test_nan_stays_in_its_row(dtype, m):
    """A NaN or an infinity in one row of x reaches no other row."""
    g = gen(9)
    x, w = rand(g, m, 256, dtype=dtype), rand(g, 160, 256, dtype=dtype, std=0.06)
    clean = ops.gated_linear(x, w[:80], w[80:])
    for v in (float("nan"), float("inf")):
        z = x.clone()
        z[2, 5] = v
        h = ops.gated_linear(z, w[:80], w[80:])
        keep = torch.arange(m, device="cuda") != 2
        assert torch.equal(h[keep], clean[keep])
        assert not torch.isfinite(h[2]).any()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gradients_against_differences(dtype):
    """Directional derivatives of each operator's sum against central
    differences of the float64 definition."""
    g = gen(11)
    m, k, f = 37, 72, 56
    x, wg, wv = rand(g, m, k, dtype=dtype), rand(g, f, k, dtype=dtype, std=0.1), rand(g, f, k, dtype=dtype, std=0.1)
    dh = rand(g, m, f, dtype=dtype)

    def loss(X, G, V):
        a, _ = act64("silu", X @ G.T)
        return (D * a * (X @ V.T)).sum()

    X, G, V, D = d_of(x, wg, wv, dh)
    got = ops.gated_linear_backward(dh, x, wg, wv)[:3]
    for i, t in enumerate((X, G, V)):
        step = torch.randn(t.shape, generator=gen(20 + i), dtype=torch.float64).cuda()
        args = [X, G, V]
        h = 1e-6
        args[i] = t + h * step
        hi = loss(*args)
        args[i] = t - h * step
        diff = ((hi - loss(*args)) / (2 * h)).item()
        # the bound of a rounded gradient: two roundings of each of its terms,
        # here a sum of independent ones; 8 standard deviations
        sd = 2 * unit(dtype) * (got[i].double().abs() * step.abs()).pow(2).sum().sqrt().item()
        assert abs((got[i].double() * step).sum().item() - diff) <= 8 * sd + 1e-4 * max(1.0, abs(diff)), i


def block(x, r, p, backward=None):
    """norm -> gated projection -> projection onto the stream, through autograd."""
    stream, u = ops.residual_norm(r, x, p["n"], post_weight=p["pn"], gate=p["g"], post_norm="rms")
    return ops.linear(ops.gated_linear(u, p["wg"], p["wv"], p["bg"]), p["wo"], p["bo"], residual=stream)


def plain_block(x, r, p):
    def rms(t, w):
        return t / (t.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w
    stream = r + p["g"] * rms(x, p["pn"])
    u = rms(stream, p["n"])
    h = torch.nn.functional.silu(u @ p["wg"].T + p["bg"]) * (u @ p["wv"].T)
    return stream + h @ p["wo"].T + p["bo"]


def block_inputs(seed, dtype, rows=(2, 75), d=136, f=200):
    g = gen(seed)
    p = {"n": rand(g, d, dtype=dtype, std=0.1, mean=1), "pn": rand(g, d, dtype=dtype, std=0.1, mean=1),
         "g": rand(g, d, dtype=dtype), "wg": rand(g, f, d, dtype=dtype, std=d ** -0.5),
         "wv": rand(g, f, d, dtype=dtype, std=d ** -0.5), "bg": rand(g, f, dtype=dtype, std=0.1),
         "wo": rand(g, d, f, dtype=dtype, std=f ** -0.5), "bo": rand(g, d, dtype=dtype, std=0.1)}
    return rand(g, *rows, d, dtype=dtype), rand(g, *rows, d, dtype=dtype), p


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_block_and_its_gradients(dtype):
    """The three together, as a block runs them, against float64 autograd.
    Each of the five roundings between the operators (u, h, out and the
    gradients of the same) enters every result once, as do the products'
    own; relative to the largest result, 16 u covers them."""
    x, r, p = block_inputs(31, dtype)
    leaves = [t.clone().requires_grad_() for t in (x, r, *p.values())]
    y = block(leaves[0], leaves[1], dict(zip(p, leaves[2:])))
    gy = rand(gen(32), *y.shape, dtype=dtype)
    grads = torch.autograd.grad(y, leaves, gy)
    exact = [t.double().requires_grad_() for t in (x, r, *p.values())]
    y64 = plain_block(exact[0], exact[1], dict(zip(p, exact[2:])))
    ref = torch.autograd.grad(y64, exact, gy.double())
    tol = 16 * unit(dtype) + 2.0 ** -18
    for a, b in zip((y, *grads), (y64, *ref)):
        assert a.dtype == dtype and a.shape == b.shape
        assert (a.double() - b).norm() <= tol * b.norm()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_graph_capture(dtype):
    """Forward and backward captured and replayed on new inputs, beside two
    graphs that share nothing, equal the eager calls bit for bit."""
    x, r, p = block_inputs(41, dtype, rows=(150,))
    gy = rand(gen(42), 150, 136, dtype=dtype)

    def step():
        stream, u = ops.residual_norm(r, x, p["n"], post_weight=p["pn"], gate=p["g"], post_norm="rms")
        h = ops.gated_linear(u, p["wg"], p["wv"], p["bg"])
        dh, dwo, dbo = ops.linear_backward(gy, h, p["wo"], p["bo"])
        du, *dw = ops.gated_linear_backward(dh, u, p["wg"], p["wv"], p["bg"])
        g = ops.residual_norm_backward(gy, du, r, x, p["n"], post_weight=p["pn"], gate=p["g"], post_norm="rms")
        return [stream, u, h, dwo, dbo, *[t for t in dw if t is not None], *[t for t in g if t is not None]]

    step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for seed in (43, 44):
        nx, nr, _ = block_inputs(seed, dtype, rows=(150,))
        x.copy_(nx)
        r.copy_(nr)
        want = [t.clone() for t in step()]
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_streams(dtype):
    """Calls on two streams at once, many times over: each has its own
    workspace, and results do not depend on timing."""
    x, r, p = block_inputs(51, dtype, rows=(700,))
    gy = rand(gen(52), 700, 200, dtype=dtype)
    want = [t for t in ops.gated_linear_backward(gy, x, p["wg"], p["wv"], p["bg"]) if t is not None]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([t for t in ops.gated_linear_backward(gy, x, p["wg"], p["wv"], p["bg"]) if t is not None])
    torch.cuda.synchronize()
    for res in got:
        for a, b in zip(res, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_needs(dtype):
    """Only the wanted gradients, equal to those of the whole call."""
    x, r, p = block_inputs(61, dtype, rows=(90,))
    dh = rand(gen(62), 90, 200, dtype=dtype)
    full = ops.gated_linear_backward(dh, x, p["wg"], p["wv"], p["bg"], p["bg"])
    for i in range(5):
        one = ops.gated_linear_backward(dh, x, p["wg"], p["wv"], p["bg"], p["bg"], needs=[j == i for j in range(5)])
        assert [t is not None for t in one] == [j == i for j in range(5)]
        assert torch.equal(one[i], full[i])
    g = rand(gen(63), 90, 136, dtype=dtype)
    args = (r, x, p["n"], p["pn"], p["pn"], p["n"], p["g"])
    whole = ops.residual_norm_backward(g, g, *args, post_norm="layer")
    for i in range(7):
        one = ops.residual_norm_backward(g, g, *args, post_norm="layer", needs=[j == i for j in range(7)])
        assert torch.equal(one[i], whole[i])
    # a missing upstream gradient is a zero one
    zero = torch.zeros_like(g)
    for a, b in ((None, g), (g, None)):
        x1 = ops.residual_norm_backward(a, b, *args, post_norm="layer")
        x2 = ops.residual_norm_backward(zero if a is None else a, zero if b is None else b, *args, post_norm="layer")
        for s, t in zip(x1, x2):
            assert (s.double() - t.double()).abs().max() <= 4 * unit(dtype) * max(1.0, t.abs().max().item())


def test_small_workspace_is_refused():
    """A workspace a byte too small changes nothing."""
    x, w = torch.randn(40, 64, device="cuda"), torch.randn(32, 64, device="cuda")
    h = torch.full((40, 32), 7.0, device="cuda")
    args = ops._GATED.pack(0, 2, 40, 64, 32, x.data_ptr(), w.data_ptr(), w.data_ptr(), 0, 0, 64, 64, 64, h.data_ptr(),
                           32, 0, 32, 0, 0, 0, 0, 0, 64, 64, 64)
    need = mb.lib().mlipcpp_b200_gated_linear_workspace(args, False)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert mb.lib().mlipcpp_b200_gated_linear(args, ws.data_ptr(), need - 1, None) == mb.INVALID_PARAMETER
    torch.cuda.synchronize()
    assert (h == 7).all()
    assert mb.lib().mlipcpp_b200_gated_linear(args, ws.data_ptr(), need, None) == mb.OK
    ops.check_status()
    assert not (h == 7).any()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_beyond_the_call_stay(dtype):
    """Output rows and columns around the call's are left as they were."""
    g = gen(71)
    x, w = rand(g, 133, 64, dtype=dtype), rand(g, 70, 64, dtype=dtype, std=0.1)
    for m in (3, 133):
        for pad in (0, 3, 10):
            y = torch.full((140, 70 + pad + 3), 5.0, dtype=dtype, device="cuda")
            ld, es = y.stride(0), y.element_size()
            args = ops._LINEAR.pack(ops._DTYPES[dtype], 0, m, 64, 70, 1.0, x.data_ptr(), w.data_ptr(), 0, 0, 64, 64, 70,
                                    y.data_ptr() + pad * es, ld, 0, 70, 0, 0, 0, 64, 64)
            ops._call("linear", args, 0, False)
            assert (y[m:] == 5).all() and (y[:, :pad] == 5).all() and (y[:, pad + 70:] == 5).all()
            assert torch.equal(y[:m, pad:pad + 70], ops.linear(x[:m], w))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m", [150, 4101])
def test_expired_wait_is_reported(dtype, m):
    """With a bound of a nanosecond on every wait the pipelines give up: the
    call's status says so once, and the next call is whole again."""
    x, r, p = block_inputs(81, dtype, rows=(m,), f=1100)
    want = ops.gated_linear(x, p["wg"], p["wv"], p["bg"])
    ops.check_status()
    L = mb.lib()
    assert L.mlipcpp_b200_set_wait_bound_ns(1) == mb.OK
    try:
        ops.gated_linear(x, p["wg"], p["wv"], p["bg"])
        with pytest.raises(mb.MLIPError) as e:
            ops.check_status()
        assert e.value.code == mb.COMPUTATION
    finally:
        assert L.mlipcpp_b200_set_wait_bound_ns(0) == mb.OK
    ops.check_status()
    assert torch.equal(ops.gated_linear(x, p["wg"], p["wv"], p["bg"]), want)
    ops.check_status()


def test_offsets_past_32_bits():
    """Rows that start beyond 2^31 elements: the last rows of a long call are
    those of a short one."""
    m, d, n = 1_100_000, 2048, 64
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    bf = torch.bfloat16
    x = torch.empty(m, d, dtype=bf, device="cuda").normal_()
    w, v = rand(gen(91), n, d, dtype=bf, std=0.02), rand(gen(92), d, dtype=bf, std=0.1, mean=1)
    tail = slice(m - 300, m)
    y = ops.linear(x, w)
    assert (y[tail].double() - x[tail].double() @ w.double().T).abs().max() <= 0.05
    dx, dw, _ = ops.linear_backward(y, x, w)
    assert torch.equal(dx[tail], ops.linear_backward(y[tail], x[tail], w, needs=(True, False, False))[0])
    ref = sum(y[i:i + 100_000].float().T.double() @ x[i:i + 100_000].double() for i in range(0, m, 100_000))
    # 22 split sums of 50,000 tokens each in 3,125 truncating additions, then
    # one rounding: 2^-9 of an element, 2^-11 of the largest
    assert ((dw.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -11 * ref.abs().max()).all()
    del dx, dw, y
    s, o = ops.residual_norm(x, x, v, norm="rms", post_norm="rms")
    s2, o2 = ops.residual_norm(x[tail], x[tail], v, norm="rms", post_norm="rms")
    assert torch.equal(s[tail], s2) and torch.equal(o[tail], o2)
    g = ops.residual_norm_backward(None, o, x, x, v, norm="rms", post_norm="rms", needs=(True, False, True) + (False,) * 4)
    g2 = ops.residual_norm_backward(None, o2, x[tail], x[tail], v, norm="rms", post_norm="rms")
    assert torch.equal(g.residual[tail], g2.residual)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(3000, 640, 529), (200, 2500, 72)], ids=str)
def test_relu_near_zero(dtype, shape):
    """The derivative's side where z is next to 0 is that of float64: every
    other weight row is chosen so that z is 0 up to its last bits."""
    m, k, f = shape
    g = gen(101)
    x, w = rand(g, m, k, dtype=dtype), rand(g, f, k, dtype=dtype, std=k ** -0.5)
    x[:, 1] = x[:, 0]
    w[::2, 1] = -w[::2, 0]          # two large terms that cancel
    w[::2, 2:] *= 2.0 ** -7
    dy = rand(g, m, f, dtype=dtype)
    z = x.double() @ w.double().T
    dz = dy.double() * (z > 0)
    db = ops.linear_backward(dy, x, w, torch.zeros(f, dtype=dtype, device="cuda"), "relu")[2]
    # no term may be missing or too many: each is a whole dy, the rounding of
    # the sums far less than the smallest that counts
    err = (db.double() - dz.sum(0)).abs()
    assert (err <= unit(dtype) * dz.sum(0).abs() + 2.0 ** -18 * dz.abs().sum(0)).all()
    v = rand(g, f, k, dtype=dtype, std=k ** -0.5)
    dbg = ops.gated_linear_backward(dy, x, w, v, torch.zeros(f, dtype=dtype, device="cuda"), None, "relu")[3]
    t = dz * (x.double() @ v.double().T)
    assert ((dbg.double() - t.sum(0)).abs() <= unit(dtype) * t.sum(0).abs() + 2.0 ** -15 * t.abs().sum(0)).all()


def test_relu_rows_of_zeros_and_of_other_scales():
    """Blocks of zeros, and blocks next to 0 as a whole, cost and give what
    others do."""
    g = gen(102)
    m, k, f = 2048, 256, 512
    x, w = rand(g, m, k, dtype=torch.float32), rand(g, f, k, dtype=torch.float32, std=k ** -0.5)
    x[100:900] = 0
    x[901:1500] *= 2.0 ** -30
    dy = rand(g, m, f, dtype=torch.float32)
    dx, dw, db = ops.linear_backward(dy, x, w, torch.zeros(f, device="cuda"), "relu")
    z = x.double() @ w.double().T
    dz = dy.double() * (z > 0)
    assert (dx.double()[100:900] == 0).all()
    for a, b in ((db, dz.sum(0)), (dx, dz @ w.double()), (dw, dz.T @ x.double())):
        assert ((a.double() - b).norm() / b.norm()) <= 2.0 ** -10  # (a flip among 2^18 would be 2^-9)
