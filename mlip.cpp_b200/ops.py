"""Transformer-block operators on CUDA tensors (torch), forward and backward.

    gated_linear   h = act(x Wg^T + bg) * (x Wv^T + bv)
    linear         y = residual + scale act(x W^T + b)
    residual_norm  stream = scale residual + gate post(y);  out = norm(stream)

They are the feed-forward half of a pre-norm block: ``residual_norm`` adds a
sublayer's output to the stream and normalises it for the next sublayer,
``gated_linear`` and ``linear`` are that sublayer.  The library's PET models
with gated feed-forward layers run the first two of these on the same kernels
(in float32); here they take any tensors, e.g. to build and train a model
around it.

Types: float32, float16 and bfloat16, one per call.  Leading dimensions are
flattened to rows (there may be none); a tensor whose rows are not contiguous
is copied first.  Everything runs on the tensors' device and its current
stream, without waiting; the working memory comes from torch's allocator.
Where an input requires grad, the forwards record themselves for autograd
(first derivatives, reverse mode; forward-mode duals are refused); the
``*_backward`` functions are the same gradients called directly.  An autograd
backward is captured into a CUDA graph only when nothing recorded earlier with
the same parameters is still held (torch ties a parameter's accumulation to the
stream of its first use); the ``*_backward`` functions have no such condition.

The kernels are those of the C API (include/mlipcpp_b200.h), which states
precision and limits; a refused call raises MLIPError.
"""
from __future__ import annotations

import numbers
import struct
from collections import namedtuple

import torch
from torch.autograd import forward_ad

from . import INVALID_PARAMETER, MLIPError, _check, lib

#: names of the activations and norms, in the order of the C enums
ACTIVATIONS = ("identity", "sigmoid", "silu", "gelu", "gelu_tanh", "relu")
NORMS = ("none", "rms", "layer")

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
# the C structures' layouts (native alignment), filled in the order of their
# fields: int32 i, int64 and pointers q, float f.  A small call is mostly host
# time, and packing costs a third of what a ctypes.Structure does.
_GATED = struct.Struct("2i 3q 5q 3q 2q 2q 5q 3q")
_LINEAR = struct.Struct("2i 3q f 4q 3q 2q 2q 3q 2q")
_NORM = struct.Struct("3i 2q 2f 7q 3q 2q 2q 2q 2q 7q 3q")


def _refuse(message: str):
    raise MLIPError(INVALID_PARAMETER, message)


def _index(name, names, what: str) -> int:
    if name is None:
        return 0
    if name not in names:
        _refuse(f"{what} must be one of {', '.join(names)} (got {name!r})")
    return names.index(name)


def _number(v, what: str) -> float:
    """A number that float32 holds (a tensor would be read on the host, and
    its gradient lost)."""
    if (type(v) is float or isinstance(v, numbers.Real)) and abs(v) <= 3.4028234663852886e38:
        return float(v)
    _refuse(f"{what} must be a finite float32 number (got {v!r})")


def _dtype(t: torch.Tensor) -> int:
    """The C type of a call's first tensor."""
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        _refuse(f"the type must be float32, float16 or bfloat16 (got {t.dtype})")
    if not t.is_cuda:
        _refuse("the tensors must be on a CUDA device (this backend has no CPU fallback)")
    return dt


def _take(t, first, shape, cols: int, keep: list, name: str):
    """(address, row stride) of `t`, a tensor of `shape` with rows of `cols`
    elements and of the type and device of `first`; (0, cols) for None.  What
    had to be copied is appended to `keep`."""
    if t is None:
        return 0, cols
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        _refuse(f"{name} carries a forward-mode tangent, which the operators do not propagate")
    if t.dtype is not first.dtype or t.get_device() != first.get_device():
        _refuse(f"{name} is {t.dtype} on {t.device}, expected {first.dtype} on {first.device}")
    if t.shape != shape:
        _refuse(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    negated = t.is_neg()  # a view whose memory holds the values' opposites
    if t.is_contiguous() and not negated:
        return t.data_ptr(), cols
    t = t.detach()
    if negated:
        t = t.resolve_neg()
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    if t.shape[0] > 1 and t.stride(0) < cols or cols > 1 and t.stride(1) != 1:
        t = t.contiguous()
    keep.append(t)
    return t.data_ptr(), max(t.stride(0), cols)


def _call(name: str, args: bytes, index: int, backward: bool):
    """One operator on the device's current stream, with its workspace."""
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return _call(name, args, index, backward)
    forms = _FORMS.get(name)
    if forms is None:
        L = lib()
        forms = _FORMS[name] = tuple(getattr(L, f"mlipcpp_b200_{name}{end}") for end in
                                     ("_workspace", "", "_backward"))
    need = forms[0](args, backward)
    if need < 0:
        _check(-need)
    ws = torch.empty(need, dtype=torch.uint8, device=index) if need else None
    code = forms[2 if backward else 1](args, ws.data_ptr() if need else 0, need,
                                       torch._C._cuda_getCurrentRawStream(index))
    if code:
        _check(code)


_FORMS: dict = {}


def _wants(t) -> bool:
    return t is not None and t.requires_grad


def _result(x, m: int, n: int):
    """Uninitialised [..., n] of x's rows, type and device."""
    return x.new_empty((m, n) if x.dim() == 2 else x.shape[:-1] + (n,))


def _grads(inputs, needs):
    """Uninitialised gradients of the inputs that are there and needed, and
    their addresses."""
    if len(needs) != len(inputs):
        _refuse(f"needs must have {len(inputs)} entries (got {len(needs)})")
    out = tuple([t.new_empty(t.shape) if t is not None and need else None for t, need in zip(inputs, needs)])
    return out, [0 if t is None else t.data_ptr() for t in out]


# ---------------------------------------------------------------------------
# gated_linear
# ---------------------------------------------------------------------------
def _gated_inputs(x, w_gate, w_value, b_gate, b_value, activation, keep):
    """(rows, K, F, the leading fields of the C structure)."""
    act = _index(activation, ACTIVATIONS, "activation")
    dt = _dtype(x)
    if w_gate.dim() != 2 or x.dim() < 1 or x.shape[-1] != w_gate.shape[1]:
        _refuse(f"x {tuple(x.shape)} and w_gate {tuple(w_gate.shape)} do not fit: expected [..., K] and [F, K]")
    f, k = w_gate.shape
    if k < 1 or f < 1:
        _refuse("there must be at least one feature")
    px, lx = _take(x, x, x.shape, k, keep, "x")
    pg, lg = _take(w_gate, x, w_gate.shape, k, keep, "w_gate")
    pv, lv = _take(w_value, x, w_gate.shape, k, keep, "w_value")
    pbg = 0 if b_gate is None else _take(b_gate, x, (f,), f, keep, "b_gate")[0]
    pbv = 0 if b_value is None else _take(b_value, x, (f,), f, keep, "b_value")[0]
    m = x.numel() // k
    return m, k, f, (dt, act, m, k, f, px, pg, pv, pbg, pbv, lx, lg, lv)


class _GatedLinear(torch.autograd.Function):
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
    product are one kernel; operands that are split (float32) or packed (rows
    that are not 16-byte aligned) and a divided contraction take another each."""
    if ((x.requires_grad or w_gate.requires_grad or w_value.requires_grad or _wants(b_gate) or _wants(b_value))
            and torch.is_grad_enabled()):
        return _GatedLinear.apply(x, w_gate, w_value, b_gate, b_value, activation)
    keep: list = []
    m, k, f, fields = _gated_inputs(x, w_gate, w_value, b_gate, b_value, activation, keep)
    h = _result(x, m, f)
    _call("gated_linear", _GATED.pack(*fields, h.data_ptr(), f, 0, f, 0, 0, 0, 0, 0, k, k, k), x.get_device(), False)
    return h


def gated_linear_backward(dh, x, w_gate, w_value, b_gate=None, b_value=None, activation="silu", needs=(True,) * 5):
    """(dx, dw_gate, dw_value, db_gate, db_value) for the gradient dh [..., F]
    of gated_linear's result; None for those not in `needs` and for biases
    that are not there."""
    keep: list = []
    m, k, f, fields = _gated_inputs(x, w_gate, w_value, b_gate, b_value, activation, keep)
    pd, ld = _take(dh, x, x.shape[:-1] + (f,), f, keep, "dh")
    out, at = _grads((x, w_gate, w_value, b_gate, b_value), needs)
    _call("gated_linear", _GATED.pack(*fields, 0, f, pd, ld, *at, k, k, k), x.get_device(), True)
    return out


# ---------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------
def _linear_inputs(x, w, bias, activation, residual, scale, keep):
    act = _index(activation, ACTIVATIONS, "activation")
    dt = _dtype(x)
    if w.dim() != 2 or x.dim() < 1 or x.shape[-1] != w.shape[1]:
        _refuse(f"x {tuple(x.shape)} and w {tuple(w.shape)} do not fit: expected [..., K] and [N, K]")
    n, k = w.shape
    if k < 1 or n < 1:
        _refuse("there must be at least one feature")
    px, lx = _take(x, x, x.shape, k, keep, "x")
    pw, lw = _take(w, x, w.shape, k, keep, "w")
    pb = 0 if bias is None else _take(bias, x, (n,), n, keep, "bias")[0]
    pr, lr = (0, n) if residual is None else _take(residual, x, x.shape[:-1] + (n,), n, keep, "residual")
    m = x.numel() // k
    return m, k, n, (dt, act, m, k, n, _number(scale, "scale"), px, pw, pb, pr, lx, lw, lr)


class _Linear(torch.autograd.Function):
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
    residual [..., N] -> [..., N], in the kernels of gated_linear."""
    if ((x.requires_grad or w.requires_grad or _wants(bias) or _wants(residual)) and torch.is_grad_enabled()):
        return _Linear.apply(x, w, bias, activation, residual, scale)
    keep: list = []
    m, k, n, fields = _linear_inputs(x, w, bias, activation, residual, scale, keep)
    y = _result(x, m, n)
    _call("linear", _LINEAR.pack(*fields, y.data_ptr(), n, 0, n, 0, 0, 0, k, k), x.get_device(), False)
    return y


def linear_backward(dy, x, w, bias=None, activation="identity", scale=1.0, needs=(True,) * 3):
    """(dx, dw, dbias) for the gradient dy [..., N] of linear's result (the
    residual's gradient is dy itself); None for those not in `needs` and for
    a bias that is not there."""
    keep: list = []
    m, k, n, fields = _linear_inputs(x, w, bias, activation, None, scale, keep)
    pd, ld = _take(dy, x, x.shape[:-1] + (n,), n, keep, "dy")
    out, at = _grads((x, w, bias), needs)
    _call("linear", _LINEAR.pack(*fields, 0, n, pd, ld, *at, k, k), x.get_device(), True)
    return out


# ---------------------------------------------------------------------------
# residual_norm
# ---------------------------------------------------------------------------
ResidualNormGrads = namedtuple("ResidualNormGrads", "residual y weight bias post_weight post_bias gate")


def _norm_inputs(residual, y, weight, bias, post_weight, post_bias, gate, scale, norm, post_norm, eps, keep):
    kinds = _index(norm, NORMS, "norm"), _index(post_norm, NORMS, "post_norm")
    dt = _dtype(residual)
    if residual.dim() < 1 or residual.shape[-1] < 1:
        _refuse("residual must have at least one dimension and one feature")
    shape, d = residual.shape, residual.shape[-1]
    if y is None and (kinds[1] or gate is not None):
        _refuse("a post norm or a gate needs y")
    pr, lr = _take(residual, residual, shape, d, keep, "residual")
    py, ly = (0, d) if y is None else _take(y, residual, shape, d, keep, "y")
    pw = 0 if weight is None else _take(weight, residual, (d,), d, keep, "weight")[0]
    pb = 0 if bias is None else _take(bias, residual, (d,), d, keep, "bias")[0]
    ppw = 0 if post_weight is None else _take(post_weight, residual, (d,), d, keep, "post_weight")[0]
    ppb = 0 if post_bias is None else _take(post_bias, residual, (d,), d, keep, "post_bias")[0]
    pg = lg = 0
    if gate is not None:
        channel = gate.dim() == 1
        pg, lg = _take(gate, residual, (d,) if channel else shape, d, keep, "gate")
        if channel:
            lg = 0
    return d, (dt, *kinds, residual.numel() // d, d, _number(scale, "scale"), _number(eps, "eps"), pr, py, pw, pb,
               ppw, ppb, pg, lr, ly, lg)


class _ResidualNorm(torch.autograd.Function):
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
    if ((residual.requires_grad or _wants(y) or _wants(weight) or _wants(bias) or _wants(post_weight)
            or _wants(post_bias) or _wants(gate)) and torch.is_grad_enabled()):
        return _ResidualNorm.apply(residual, y, weight, bias, post_weight, post_bias, gate, scale, norm, post_norm,
                                   eps)
    keep: list = []
    d, fields = _norm_inputs(residual, y, weight, bias, post_weight, post_bias, gate, scale, norm, post_norm, eps, keep)
    stream, out = torch.empty_like(residual, memory_format=torch.contiguous_format), torch.empty_like(
        residual, memory_format=torch.contiguous_format)
    _call("residual_norm", _NORM.pack(*fields, stream.data_ptr(), out.data_ptr(), d, d, 0, 0, d, d,
                                      0, 0, 0, 0, 0, 0, 0, d, d, d), residual.get_device(), False)
    return stream, out


def residual_norm_backward(dstream, dout, residual, y=None, weight=None, bias=None, post_weight=None, post_bias=None,
                           gate=None, scale=1.0, norm="rms", post_norm="none", eps=1e-5, needs=(True,) * 7):
    """ResidualNormGrads for the gradients of residual_norm's two results
    (either may be None); None for inputs not in `needs` or not there."""
    keep: list = []
    d, fields = _norm_inputs(residual, y, weight, bias, post_weight, post_bias, gate, scale, norm, post_norm, eps, keep)
    ps, ls = _take(dstream, residual, residual.shape, d, keep, "dstream")
    po, lo = _take(dout, residual, residual.shape, d, keep, "dout")
    out, at = _grads((residual, y, weight, bias, post_weight, post_bias, gate), needs)
    _call("residual_norm", _NORM.pack(*fields, 0, 0, d, d, ps, po, ls, lo, *at, d, d, d), residual.get_device(), True)
    return ResidualNormGrads(*out)


def check_status(device=None):
    """Waits for the current stream of `device` and raises if an operator's
    tensor-core pipeline has given up since the last check."""
    with torch.cuda.device(device):
        _check(lib().mlipcpp_b200_ops_status(torch.cuda.current_stream().cuda_stream))
