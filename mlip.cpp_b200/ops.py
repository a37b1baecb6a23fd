"""Transformer-block operators on CUDA tensors (torch), forward and backward.

    gated_linear   h = act(x Wg^T + bg) * (x Wv^T + bv)
    linear         y = residual + scale act(x W^T + b)
    residual_norm  stream = scale residual + gate post(y);  out = norm(stream)

They are the feed-forward half of a pre-norm block: ``residual_norm`` adds a
sublayer's output to the stream and normalises it for the next sublayer,
``gated_linear`` and ``linear`` are that sublayer.  The library's PET models
with gated feed-forward layers run on the same kernels; here they take any
tensors, e.g. to build and train a model around it.

Types: float32, float16 and bfloat16, one per call.  Leading dimensions are
flattened to rows (there may be none); a tensor whose rows are not contiguous
is copied first.  Everything runs on the tensors' device and its current
stream, without waiting; the working memory comes from torch's allocator.
Where an input requires grad, the forwards record themselves for autograd
(first derivatives); the ``*_backward`` functions are the same gradients
called directly.

The kernels are those of the C API (include/mlipcpp_b200.h), which states
precision and limits; a refused call raises MLIPError.
"""
from __future__ import annotations

import ctypes
from collections import namedtuple

import torch

from . import INVALID_PARAMETER, MLIPError, _check, lib

#: names of the activations and norms, in the order of the C enums
ACTIVATIONS = ("identity", "sigmoid", "silu", "gelu", "gelu_tanh", "relu")
NORMS = ("none", "rms", "layer")

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


def _fields(spec: str, kind):
    return [(name, kind) for name in spec.split()]


class _GatedLinear(ctypes.Structure):
    _fields_ = (_fields("dtype activation", _i32) + _fields("rows in_features hidden", _i64)
                + _fields("x w_gate w_value b_gate b_value", _vp) + _fields("ldx ldw_gate ldw_value", _i64)
                + [("h", _vp), ("ldh", _i64), ("dh", _vp), ("lddh", _i64)]
                + _fields("dx dw_gate dw_value db_gate db_value", _vp) + _fields("lddx lddw_gate lddw_value", _i64))


class _Linear(ctypes.Structure):
    _fields_ = (_fields("dtype activation", _i32) + _fields("rows in_features out_features", _i64)
                + [("scale", _f32)] + _fields("x w b residual", _vp) + _fields("ldx ldw ldresidual", _i64)
                + [("y", _vp), ("ldy", _i64), ("dy", _vp), ("lddy", _i64)]
                + _fields("dx dw db", _vp) + _fields("lddx lddw", _i64))


class _ResidualNorm(ctypes.Structure):
    _fields_ = (_fields("dtype norm post_norm", _i32) + _fields("rows features", _i64) + _fields("scale eps", _f32)
                + _fields("residual y weight bias post_weight post_bias gate", _vp)
                + _fields("ldresidual ldy ldgate", _i64) + _fields("stream out", _vp) + _fields("ldstream ldout", _i64)
                + _fields("dstream dout", _vp) + _fields("lddstream lddout", _i64)
                + _fields("dresidual dy dweight dbias dpost_weight dpost_bias dgate", _vp)
                + _fields("lddresidual lddy lddgate", _i64))


def _refuse(message: str):
    raise MLIPError(INVALID_PARAMETER, message)


def _index(name, names, what: str) -> int:
    name = names[0] if name is None else name
    if name not in names:
        _refuse(f"{what} must be one of {', '.join(names)} (got {name!r})")
    return names.index(name)


def _same(first: torch.Tensor, **others):
    """Refuses tensors of another type or device than `first`."""
    if first.dtype not in _DTYPES:
        _refuse(f"the type must be float32, float16 or bfloat16 (got {first.dtype})")
    if not first.is_cuda:
        _refuse("the tensors must be on a CUDA device (this backend has no CPU fallback)")
    for name, t in others.items():
        if t is not None and (t.dtype != first.dtype or t.device != first.device):
            _refuse(f"{name} is {t.dtype} on {t.device}, expected {first.dtype} on {first.device}")


def _shape(t, name: str, shape):
    if t is not None and tuple(t.shape) != tuple(shape):
        _refuse(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _rows(t: torch.Tensor | None, cols: int):
    """`t` as a [rows, cols] matrix with contiguous rows."""
    if t is None:
        return None
    t = t.detach().reshape(-1, cols) if t.dim() != 2 else t.detach()
    if t.shape[0] > 1 and t.stride(0) < cols or cols > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t


def _vec(t: torch.Tensor | None):
    return None if t is None else t.detach().contiguous()


def _p(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _ld(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.stride(0)


def _call(name: str, args, device: torch.device, backward: bool):
    """One operator on the device's current stream, with its workspace."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _call(name, args, device, backward)
    L, ref = lib(), ctypes.byref(args)
    need = getattr(L, name + "_workspace")(ref, backward)
    if need < 0:
        _check(-need)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _check(getattr(L, name + "_backward" if backward else name)(
        ref, _p(ws), need, torch.cuda.current_stream(device).cuda_stream))


def _recorded(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---------------------------------------------------------------------------
# gated_linear
# ---------------------------------------------------------------------------
def _gated_args(x, w_gate, w_value, b_gate, b_value, activation):
    act = _index(activation, ACTIVATIONS, "activation")
    if w_gate.dim() != 2 or x.dim() < 1:
        _refuse("w_gate must have two dimensions and x at least one")
    f, k = w_gate.shape
    _same(x, w_gate=w_gate, w_value=w_value, b_gate=b_gate, b_value=b_value)
    _shape(w_value, "w_value", (f, k))
    _shape(b_gate, "b_gate", (f,))
    _shape(b_value, "b_value", (f,))
    if x.shape[-1] != k:
        _refuse(f"x has {x.shape[-1]} features, expected {k}")
    keep = (_rows(x, k), _rows(w_gate, k), _rows(w_value, k), _vec(b_gate), _vec(b_value))
    a = _GatedLinear(dtype=_DTYPES[x.dtype], activation=act, rows=keep[0].shape[0], in_features=k, hidden=f,
                     x=_p(keep[0]), w_gate=_p(keep[1]), w_value=_p(keep[2]), b_gate=_p(keep[3]), b_value=_p(keep[4]),
                     ldx=_ld(keep[0]), ldw_gate=_ld(keep[1]), ldw_value=_ld(keep[2]))
    return a, keep


class _GatedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_value, b_gate, b_value, activation):
        ctx.save_for_backward(x, w_gate, w_value, b_gate, b_value)
        ctx.activation = activation
        return gated_linear(x, w_gate, w_value, b_gate, b_value, activation)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        return (*gated_linear_backward(dh, *ctx.saved_tensors, ctx.activation, ctx.needs_input_grad[:5]), None)


def gated_linear(x, w_gate, w_value, b_gate=None, b_value=None, activation="silu"):
    """act(x w_gate^T + b_gate) * (x w_value^T + b_value): x [..., K], weights
    [F, K], biases [F] -> [..., F].  Both projections, the activation and the
    product are one kernel."""
    if _recorded(x, w_gate, w_value, b_gate, b_value):
        return _GatedLinearFn.apply(x, w_gate, w_value, b_gate, b_value, activation)
    a, keep = _gated_args(x, w_gate, w_value, b_gate, b_value, activation)
    h = torch.empty(x.shape[:-1] + (a.hidden,), dtype=x.dtype, device=x.device)
    a.h, a.ldh = h.data_ptr(), a.hidden
    _call("mlipcpp_b200_gated_linear", a, x.device, False)
    return h


def gated_linear_backward(dh, x, w_gate, w_value, b_gate=None, b_value=None, activation="silu", needs=(True,) * 5):
    """(dx, dw_gate, dw_value, db_gate, db_value) for the gradient dh [..., F]
    of gated_linear's result; None for those not in `needs` and for biases
    that are not there."""
    a, keep = _gated_args(x, w_gate, w_value, b_gate, b_value, activation)
    _same(x, dh=dh)
    _shape(dh, "dh", x.shape[:-1] + (a.hidden,))
    m = _rows(dh, a.hidden)
    a.dh, a.lddh = _p(m), _ld(m)
    out = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None and need else None
           for t, need in zip((x, w_gate, w_value, b_gate, b_value), needs)]
    a.dx, a.dw_gate, a.dw_value, a.db_gate, a.db_value = (_p(t) for t in out)
    a.lddx = a.lddw_gate = a.lddw_value = a.in_features
    _call("mlipcpp_b200_gated_linear", a, x.device, True)
    return tuple(out)


# ---------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------
def _linear_args(x, w, bias, activation, scale):
    act = _index(activation, ACTIVATIONS, "activation")
    if w.dim() != 2 or x.dim() < 1:
        _refuse("w must have two dimensions and x at least one")
    n, k = w.shape
    _same(x, w=w, bias=bias)
    _shape(bias, "bias", (n,))
    if x.shape[-1] != k:
        _refuse(f"x has {x.shape[-1]} features, expected {k}")
    keep = (_rows(x, k), _rows(w, k), _vec(bias))
    a = _Linear(dtype=_DTYPES[x.dtype], activation=act, rows=keep[0].shape[0], in_features=k, out_features=n,
                scale=scale, x=_p(keep[0]), w=_p(keep[1]), b=_p(keep[2]), ldx=_ld(keep[0]), ldw=_ld(keep[1]))
    return a, keep


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, activation, residual, scale):
        ctx.save_for_backward(x, w, bias)
        ctx.activation, ctx.scale = activation, scale
        return linear(x, w, bias, activation, residual, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        dx, dw, db = linear_backward(dy, *ctx.saved_tensors, ctx.activation, ctx.scale, ctx.needs_input_grad[:3])
        return dx, dw, db, None, dy if ctx.needs_input_grad[4] else None, None


def linear(x, w, bias=None, activation="identity", residual=None, scale=1.0):
    """residual + scale act(x w^T + bias): x [..., K], w [N, K], bias [N],
    residual [..., N] -> [..., N], in one kernel."""
    if _recorded(x, w, bias, residual):
        return _LinearFn.apply(x, w, bias, activation, residual, scale)
    a, keep = _linear_args(x, w, bias, activation, scale)
    shape = x.shape[:-1] + (a.out_features,)
    _same(x, residual=residual)
    _shape(residual, "residual", shape)
    r = _rows(residual, a.out_features)
    a.residual, a.ldresidual = _p(r), _ld(r)
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    a.y, a.ldy = y.data_ptr(), a.out_features
    _call("mlipcpp_b200_linear", a, x.device, False)
    return y


def linear_backward(dy, x, w, bias=None, activation="identity", scale=1.0, needs=(True,) * 3):
    """(dx, dw, dbias) for the gradient dy [..., N] of linear's result (the
    residual's gradient is dy itself); None for those not in `needs` and for
    a bias that is not there."""
    a, keep = _linear_args(x, w, bias, activation, scale)
    _same(x, dy=dy)
    _shape(dy, "dy", x.shape[:-1] + (a.out_features,))
    m = _rows(dy, a.out_features)
    a.dy, a.lddy = _p(m), _ld(m)
    out = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None and need else None
           for t, need in zip((x, w, bias), needs)]
    a.dx, a.dw, a.db = (_p(t) for t in out)
    a.lddx = a.lddw = a.in_features
    _call("mlipcpp_b200_linear", a, x.device, True)
    return tuple(out)


# ---------------------------------------------------------------------------
# residual_norm
# ---------------------------------------------------------------------------
ResidualNormGrads = namedtuple("ResidualNormGrads", "residual y weight bias post_weight post_bias gate")


def _norm_args(residual, y, weight, bias, post_weight, post_bias, gate, scale, norm, post_norm, eps):
    kinds = _index(norm, NORMS, "norm"), _index(post_norm, NORMS, "post_norm")
    if residual.dim() < 1:
        _refuse("residual must have at least one dimension")
    d = residual.shape[-1]
    _same(residual, y=y, weight=weight, bias=bias, post_weight=post_weight, post_bias=post_bias, gate=gate)
    _shape(y, "y", residual.shape)
    for name, t in (("weight", weight), ("bias", bias), ("post_weight", post_weight), ("post_bias", post_bias)):
        _shape(t, name, (d,))
    if gate is not None and tuple(gate.shape) not in ((d,), tuple(residual.shape)):
        _refuse(f"gate has shape {tuple(gate.shape)}, expected {(d,)} or {tuple(residual.shape)}")
    channel = gate is not None and gate.dim() == 1
    keep = (_rows(residual, d), _rows(y, d), _vec(weight), _vec(bias), _vec(post_weight), _vec(post_bias),
            _vec(gate) if channel else _rows(gate, d))
    r, ym, g = keep[0], keep[1], keep[6]
    a = _ResidualNorm(dtype=_DTYPES[r.dtype], norm=kinds[0], post_norm=kinds[1], rows=r.shape[0], features=d,
                      scale=scale, eps=eps, residual=_p(r), y=_p(ym), weight=_p(keep[2]), bias=_p(keep[3]),
                      post_weight=_p(keep[4]), post_bias=_p(keep[5]), gate=_p(g), ldresidual=_ld(r), ldy=_ld(ym),
                      ldgate=0 if channel or g is None else max(g.stride(0), d))
    return a, keep


class _ResidualNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, y, weight, bias, post_weight, post_bias, gate, *how):
        ctx.save_for_backward(residual, y, weight, bias, post_weight, post_bias, gate)
        ctx.how = how
        ctx.set_materialize_grads(False)
        return residual_norm(residual, y, weight, bias, post_weight, post_bias, gate, *how)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dstream, dout):
        if dstream is None and dout is None:
            return (None,) * 11
        g = residual_norm_backward(dstream, dout, *ctx.saved_tensors, *ctx.how, needs=ctx.needs_input_grad[:7])
        return (*g, None, None, None, None)


def residual_norm(residual, y=None, weight=None, bias=None, post_weight=None, post_bias=None, gate=None, scale=1.0,
                  norm="rms", post_norm="none", eps=1e-5):
    """(stream, out) with stream = scale residual + gate post(y) and out =
    norm(stream), over the last dimension (at most 16384): norms "none", "rms"
    or "layer" with optional weight and bias, a gate [d] for all rows or one
    of the residual's shape.  y None: stream = scale residual."""
    if _recorded(residual, y, weight, bias, post_weight, post_bias, gate):
        return _ResidualNormFn.apply(residual, y, weight, bias, post_weight, post_bias, gate, scale, norm, post_norm,
                                     eps)
    a, keep = _norm_args(residual, y, weight, bias, post_weight, post_bias, gate, scale, norm, post_norm, eps)
    stream = torch.empty(residual.shape, dtype=residual.dtype, device=residual.device)
    out = torch.empty_like(stream)
    a.stream, a.out, a.ldstream, a.ldout = stream.data_ptr(), out.data_ptr(), a.features, a.features
    _call("mlipcpp_b200_residual_norm", a, residual.device, False)
    return stream, out


def residual_norm_backward(dstream, dout, residual, y=None, weight=None, bias=None, post_weight=None, post_bias=None,
                           gate=None, scale=1.0, norm="rms", post_norm="none", eps=1e-5, needs=(True,) * 7):
    """ResidualNormGrads for the gradients of residual_norm's two results
    (either may be None); None for inputs not in `needs` or not there."""
    a, keep = _norm_args(residual, y, weight, bias, post_weight, post_bias, gate, scale, norm, post_norm, eps)
    _same(residual, dstream=dstream, dout=dout)
    _shape(dstream, "dstream", residual.shape)
    _shape(dout, "dout", residual.shape)
    d = a.features
    ms, mo = _rows(dstream, d), _rows(dout, d)
    a.dstream, a.dout, a.lddstream, a.lddout = _p(ms), _p(mo), _ld(ms), _ld(mo)
    g = ResidualNormGrads(*(torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None and need else None
                            for t, need in zip((residual, y, weight, bias, post_weight, post_bias, gate), needs)))
    a.dresidual, a.dy, a.dweight, a.dbias, a.dpost_weight, a.dpost_bias, a.dgate = (_p(t) for t in g)
    a.lddresidual = a.lddy = a.lddgate = d
    _call("mlipcpp_b200_residual_norm", a, residual.device, True)
    return g


def check_status(device=None):
    """Waits for the current stream of `device` and raises if an operator's
    tensor-core pipeline has given up since the last check."""
    with torch.cuda.device(device):
        _check(lib().mlipcpp_b200_ops_status(torch.cuda.current_stream().cuda_stream))
