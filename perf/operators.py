"""Cases of the transformer-block operators (mlipcpp_b200.ops): the gated
feed-forward projection, the dense layer with its epilogue, and the residual
update between two norms, each forward and backward.

`run` computes a case in plain 32-bit torch operations, or, when `own` is
true, through the framework's operators.  `exact` gives the same outputs in
64 bits.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTS = ("identity", "sigmoid", "silu", "gelu", "gelu_tanh", "relu")


def _ops():
    """mlipcpp_b200.ops (the package's folder name is no identifier, so it is loaded by path)."""
    if "mlipcpp_b200" not in sys.modules:
        folder = os.path.join(ROOT, "mlip.cpp_b200")
        spec = importlib.util.spec_from_file_location(
            "mlipcpp_b200", os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        module = importlib.util.module_from_spec(spec)
        sys.modules["mlipcpp_b200"] = module
        spec.loader.exec_module(module)
    from mlipcpp_b200 import ops
    return ops


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def _gated(way, dtype, m, k, f, act="silu", bias=False):
    return {"op": "gated_linear", "way": way, "dtype": dtype, "m": m, "k": k, "f": f, "act": act, "bias": bias}


def _linear(way, dtype, m, k, n, act="identity", bias=True, residual=False, scale=1.0):
    return {"op": "linear", "way": way, "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "bias": bias,
            "residual": residual, "scale": scale}


def _norm(way, dtype, m, d, norm="rms", post="none", gate="none", bias=False, scale=1.0):
    return {"op": "residual_norm", "way": way, "dtype": dtype, "m": m, "d": d, "norm": norm, "post": post,
            "gate": gate, "bias": bias, "scale": scale}


def listed():
    return [
        # one new token of one sequence: all of it is reading the two weights
        {"name": "gated_token_bf16", **_gated("forward", "bf16", 1, 2048, 5632)},
        # a ragged prompt at odd widths
        {"name": "gated_prompt_f16", **_gated("forward", "f16", 777, 1000, 1331, act="gelu_tanh", bias=True)},
        # one training step's tokens: every gradient
        {"name": "gated_train_bf16", **_gated("backward", "bf16", 8192, 1024, 4096)},
        # the 65,202 tokens (1,728 atoms, 63,474 edges) of the 1,728-atom fcc cell at d = 512
        {"name": "gated_atoms_f32", **_gated("forward", "f32", 65202, 512, 1024, bias=True)},
        # the 19,390 tokens of the 512-atom cell: the gradient that forces need, and the weights'
        {"name": "gated_atoms_back_f32", **_gated("backward", "f32", 19390, 512, 1024, bias=True)},
        # the projection back, for the next tokens of four sequences
        {"name": "linear_token_bf16", **_linear("forward", "bf16", 4, 5632, 2048, bias=False, residual=True)},
        # a ragged prompt whose rows start on odd addresses
        {"name": "linear_prompt_f16", **_linear("forward", "f16", 1500, 643, 770, act="gelu")},
        # one training step's tokens through the projection back
        {"name": "linear_train_bf16", **_linear("backward", "bf16", 8192, 4096, 1024)},
        # the projection back of the 65,202 tokens, onto their residual
        {"name": "linear_atoms_f32", **_linear("forward", "f32", 65202, 1024, 512, residual=True)},
        # one new token between two blocks
        {"name": "norm_token_bf16", **_norm("forward", "bf16", 1, 2048)},
        # a long prompt, norms on both sides and a gate for each channel
        {"name": "norm_prompt_f16", **_norm("forward", "f16", 16383, 4096, post="rms", gate="channel", scale=0.5)},
        # one training step's tokens, norms on both sides
        {"name": "norm_train_bf16", **_norm("backward", "bf16", 8192, 4096, post="rms", gate="channel")},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _width(rng, lo, hi):
    """A width: half of them multiples of 128, the others any."""
    n = _log(rng, lo, hi)
    return max(128, n // 128 * 128) if rng.random() < 0.5 else n


def draw(rng):
    top = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(("gated_linear", "linear", "residual_norm"))
        way = rng.choice(("forward", "backward"))
        dtype = rng.choice(tuple(DTYPES))
        m = _log(rng, 1, 16384)
        if op == "gated_linear":
            case = _gated(way, dtype, m, _width(rng, 64, 2048), _width(rng, 64, 5632), rng.choice(ACTS),
                          rng.random() < 0.5)
        elif op == "linear":
            case = _linear(way, dtype, m, _width(rng, 64, 5632), _width(rng, 64, 2048), rng.choice(ACTS),
                           rng.random() < 0.5, rng.random() < 0.5, rng.choice((1.0, 0.25)))
        else:
            case = _norm(way, dtype, m, _width(rng, 64, 4096), rng.choice(("rms", "layer")),
                         rng.choice(("none", "rms", "layer")), rng.choice(("none", "channel", "row")),
                         rng.random() < 0.5, rng.choice((1.0, 0.5)))
        if work(case)["flops"] <= top:
            return case


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
EPS = 1e-5


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, device="cuda", generator=g) * std + mean).to(dt)

    def gradient(m, n):
        """A loss's gradient: tokens of uneven weight, the last 1 in 16 padding without any."""
        t = torch.randn(m, n, device="cuda", generator=g) * torch.exp(0.5 * torch.randn(m, 1, device="cuda", generator=g))
        if m >= 16:
            t[m - m // 16:] = 0
        return (t * 0.25).to(dt)

    s = dict(case)
    m, back = case["m"], case["way"] == "backward"
    if case["op"] == "gated_linear":
        k, f = case["k"], case["f"]
        s["x"] = normal(m, k)
        s["w_gate"], s["w_value"] = normal(f, k, std=k ** -0.5), normal(f, k, std=k ** -0.5)
        s["b_gate"], s["b_value"] = (normal(f, std=0.1), normal(f, std=0.1)) if case["bias"] else (None, None)
        s["dh"] = gradient(m, f) if back else None
    elif case["op"] == "linear":
        k, n = case["k"], case["n"]
        s["x"], s["w"] = normal(m, k), normal(n, k, std=k ** -0.5)
        s["b"] = normal(n, std=0.1) if case["bias"] else None
        s["r"] = normal(m, n, std=2.0) if case["residual"] else None
        s["dy"] = gradient(m, n) if back else None
    else:
        d = case["d"]
        # a residual stream has a few channels far above the others
        channel = torch.exp(0.7 * torch.randn(d, device="cuda", generator=g))
        s["r"] = (torch.randn(m, d, device="cuda", generator=g) * channel).to(dt)
        s["y"] = normal(m, d)
        s["weight"] = normal(d, std=0.1, mean=1.0)
        s["bias"] = normal(d, std=0.1) if case["bias"] else None
        post = case["post"] != "none"
        s["post_weight"] = normal(d, std=0.1, mean=1.0) if post else None
        s["post_bias"] = normal(d, std=0.1) if post and case["bias"] else None
        s["gate"] = {"none": None, "channel": normal(d, std=0.2, mean=0.5) if case["gate"] == "channel" else None,
                     "row": normal(m, d, std=0.2, mean=0.5) if case["gate"] == "row" else None}[case["gate"]]
        s["ds"] = gradient(m, d) if back else None
        s["do"] = gradient(m, d) if back else None
    return s


# --------------------------------------------------------------------------
# Plain forms (32 bits, rounded once at the end)
# --------------------------------------------------------------------------
def _f(t):
    return None if t is None else t.float()


def _act(name, z):
    """Activation and its derivative."""
    if name == "identity":
        return z, torch.ones_like(z)
    if name == "relu":
        on = (z > 0).float()
        return z * on, on
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    p = 1 / (1 + torch.exp(-z))
    if name == "sigmoid":
        return p, p * (1 - p)
    return z * p, p * (1 + z * (1 - p))


def _dense(x, w, b):
    z = x @ w.t()
    return z if b is None else z + b


def _plain_gated(s):
    dt = s["x"].dtype
    x, wg, wv = _f(s["x"]), _f(s["w_gate"]), _f(s["w_value"])
    g, v = _dense(x, wg, _f(s["b_gate"])), _dense(x, wv, _f(s["b_value"]))
    a, da = _act(s["act"], g)
    if s["way"] == "forward":
        return (a * v).to(dt)
    dh = _f(s["dh"])
    dg, dv = dh * v * da, dh * a
    out = [dg @ wg + dv @ wv, dg.t() @ x, dv.t() @ x]
    if s["bias"]:
        out += [dg.sum(0), dv.sum(0)]
    return [t.to(dt) for t in out]


def _plain_linear(s):
    dt = s["x"].dtype
    x, w, b = _f(s["x"]), _f(s["w"]), _f(s["b"])
    if s["way"] == "forward":
        y = _act(s["act"], _dense(x, w, b))[0] * s["scale"]
        return (y if s["r"] is None else y + _f(s["r"])).to(dt)
    dz = _f(s["dy"]) * s["scale"]
    if s["act"] != "identity":
        dz = dz * _act(s["act"], _dense(x, w, b))[1]
    out = [dz @ w, dz.t() @ x]
    if b is not None:
        out.append(dz.sum(0))
    return [t.to(dt) for t in out]


def _norm_rows(kind, x, w, b):
    """(normalised and scaled rows, normalised rows, 1 / sigma)."""
    if kind == "none":
        return x, None, None
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    inv = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    n = x * inv
    o = n if w is None else n * w
    return (o if b is None else o + b), n, inv


def _norm_rows_back(kind, do, n, inv, w):
    """(gradient of the rows, of the weight, of the bias)."""
    if kind == "none":
        return do, None, None
    dn = do if w is None else do * w
    dx = dn - n * (dn * n).mean(1, keepdim=True)
    if kind == "layer":
        dx = dx - dn.mean(1, keepdim=True)
    return dx * inv, (do * n).sum(0), do.sum(0)


def _plain_norm(s):
    dt = s["r"].dtype
    r, y, w, pw, gate = _f(s["r"]), _f(s["y"]), _f(s["weight"]), _f(s["post_weight"]), _f(s["gate"])
    u, pn, pinv = _norm_rows(s["post"], y, pw, _f(s["post_bias"]))
    stream = s["scale"] * r + (u if gate is None else gate * u)
    out, n, inv = _norm_rows(s["norm"], stream, w, _f(s["bias"]))
    if s["way"] == "forward":
        return [stream.to(dt), out.to(dt)]
    dx, dw, db = _norm_rows_back(s["norm"], _f(s["do"]), n, inv, w)
    dstream = _f(s["ds"]) + dx
    du = dstream if gate is None else dstream * gate
    dy, dpw, dpb = _norm_rows_back(s["post"], du, pn, pinv, pw)
    grads = {"residual": s["scale"] * dstream, "y": dy, "weight": dw}
    if s["bias"] is not None:
        grads["bias"] = db
    if pw is not None:
        grads["post_weight"] = dpw
    if s["post_bias"] is not None:
        grads["post_bias"] = dpb
    if gate is not None:
        dg = dstream * u
        grads["gate"] = dg if gate.dim() == 2 else dg.sum(0)
    return {k: t.to(dt) for k, t in grads.items()}


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        ops = _ops()
        if s["op"] == "gated_linear":
            args = (s["x"], s["w_gate"], s["w_value"], s["b_gate"], s["b_value"], s["act"])
            if s["way"] == "forward":
                return ops.gated_linear(*args)
            return [t for t in ops.gated_linear_backward(s["dh"], *args) if t is not None]
        if s["op"] == "linear":
            if s["way"] == "forward":
                return ops.linear(s["x"], s["w"], s["b"], s["act"], s["r"], s["scale"])
            return [t for t in ops.linear_backward(s["dy"], s["x"], s["w"], s["b"], s["act"], s["scale"])
                    if t is not None]
        args = (s["r"], s["y"], s["weight"], s["bias"], s["post_weight"], s["post_bias"], s["gate"], s["scale"],
                s["norm"], s["post"], EPS)
        if s["way"] == "forward":
            return list(ops.residual_norm(*args))
        return {k: t for k, t in ops.residual_norm_backward(s["ds"], s["do"], *args)._asdict().items()
                if t is not None}
    if s["op"] == "gated_linear":
        return _plain_gated(s)
    if s["op"] == "linear":
        return _plain_linear(s)
    return _plain_norm(s)


def work(case):
    """Each input read once, each output written once; the products of the definition."""
    size = 4 if case["dtype"] == "f32" else 2
    m, back = case["m"], case["way"] == "backward"
    if case["op"] == "gated_linear":
        k, f = case["k"], case["f"]
        weights = 2 * f * k + (2 * f if case["bias"] else 0)
        values = m * k + weights + m * f  # x, weights, h or dh
        if back:  # both projections again, then the gradients of x and of the weights
            return {"bytes": size * (values + m * k + weights), "flops": 12 * m * k * f}
        return {"bytes": size * values, "flops": 4 * m * k * f}
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        weights = n * k + (n if case["bias"] else 0)
        if back:
            flops = (4 if case["act"] == "identity" else 6) * m * k * n
            return {"bytes": size * (2 * m * k + m * n + 2 * weights), "flops": flops}
        rows = m * k + m * n * (2 if case["residual"] else 1)
        return {"bytes": size * (rows + weights), "flops": 2 * m * k * n}
    d = case["d"]
    gate = {"none": 0, "channel": d, "row": m * d}[case["gate"]]
    vectors = (1 + (case["post"] != "none")) * (1 + bool(case["bias"])) * d + gate
    if back:  # residual, y, dstream, dout in; dresidual, dy out
        return {"bytes": size * (6 * m * d + 2 * vectors), "flops": 30 * m * d}
    return {"bytes": size * (4 * m * d + vectors), "flops": 12 * m * d}


# --------------------------------------------------------------------------
# 64 bits, from the definitions
# --------------------------------------------------------------------------
_PHI = {
    "identity": lambda z: z,
    "sigmoid": torch.sigmoid,
    "silu": lambda z: z * torch.sigmoid(z),
    "gelu": lambda z: z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0)),
    "gelu_tanh": lambda z: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)),
    "relu": lambda z: torch.clamp(z, min=0),
}


def _exact_norm(kind, t, w, b):
    if kind == "none":
        return t
    mean = t.mean(1, keepdim=True) if kind == "layer" else 0.0
    t = (t - mean) * torch.rsqrt(((t - mean) ** 2).mean(1, keepdim=True) + EPS)
    t = t if w is None else t * w
    return t if b is None else t + b


def exact(case, seed):
    """The definitions in 64 bits; the gradients by differentiating them."""
    s = prepare(case, seed)
    back = case["way"] == "backward"
    leaf = {k: t.double().requires_grad_(back) for k, t in s.items() if isinstance(t, torch.Tensor)}
    at = leaf.get
    with torch.set_grad_enabled(back):
        if case["op"] == "gated_linear":
            names = ["x", "w_gate", "w_value"] + (["b_gate", "b_value"] if case["bias"] else [])
            bg, bv = (leaf["b_gate"], leaf["b_value"]) if case["bias"] else (0.0, 0.0)
            h = _PHI[case["act"]](leaf["x"] @ leaf["w_gate"].T + bg) * (leaf["x"] @ leaf["w_value"].T + bv)
            if not back:
                return h
            return list(torch.autograd.grad(h, [leaf[n] for n in names], leaf["dh"].detach()))
        if case["op"] == "linear":
            names = ["x", "w"] + (["b"] if case["bias"] else [])
            y = case["scale"] * _PHI[case["act"]](leaf["x"] @ leaf["w"].T + (leaf["b"] if case["bias"] else 0.0))
            if not back:
                return y + leaf["r"] if case["residual"] else y
            return list(torch.autograd.grad(y, [leaf[n] for n in names], leaf["dy"].detach()))
        u = _exact_norm(case["post"], leaf["y"], at("post_weight"), at("post_bias"))
        stream = case["scale"] * leaf["r"] + (u if at("gate") is None else leaf["gate"] * u)
        out = _exact_norm(case["norm"], stream, leaf["weight"], at("bias"))
        if not back:
            return [stream, out]
        names = {"residual": "r", "y": "y", "weight": "weight", "bias": "bias", "post_weight": "post_weight",
                 "post_bias": "post_bias", "gate": "gate"}
        names = {k: n for k, n in names.items() if n in leaf}
        grads = torch.autograd.grad([stream, out], [leaf[n] for n in names.values()],
                                    [leaf["ds"].detach(), leaf["do"].detach()])
        return dict(zip(names, grads))
