"""The transformer-block operators' refusals, on the CPU: every argument check
comes before any device work, so invalid calls are turned down without a GPU."""
import ctypes
import struct

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mlipcpp_b200 as mb  # noqa: E402
from mlipcpp_b200 import ops  # noqa: E402

NULL, INVALID = mb.NULL_POINTER, mb.INVALID_PARAMETER
P = 1 << 20  # an aligned address that no refused call may touch


def gated(backward=False, workspace=0, size=0, **over):
    f = dict(dtype=0, activation=2, rows=4, k=8, f=16, x=P, w_gate=P, w_value=P, b_gate=0, b_value=0, ldx=8,
             ldw_gate=8, ldw_value=8, h=P, ldh=16, dh=P, lddh=16, dx=P, dw_gate=P, dw_value=P, db_gate=0, db_value=0,
             lddx=8, lddw_gate=8, lddw_value=8)
    f.update(over)
    fn = mb.lib().mlipcpp_b200_gated_linear_backward if backward else mb.lib().mlipcpp_b200_gated_linear
    return fn(ops._GATED.pack(*f.values()), workspace, size, None)


def linear(backward=False, **over):
    f = dict(dtype=0, activation=0, rows=4, k=8, n=16, scale=1.0, x=P, w=P, b=0, residual=0, ldx=8, ldw=8,
             ldresidual=16, y=P, ldy=16, dy=P, lddy=16, dx=P, dw=P, db=0, lddx=8, lddw=8)
    f.update(over)
    fn = mb.lib().mlipcpp_b200_linear_backward if backward else mb.lib().mlipcpp_b200_linear
    return fn(ops._LINEAR.pack(*f.values()), 0, 0, None)


def norm(backward=False, **over):
    f = dict(dtype=0, norm=1, post=0, rows=4, d=8, scale=1.0, eps=1e-5, residual=P, y=P, weight=P, bias=0,
             post_weight=0, post_bias=0, gate=0, ldresidual=8, ldy=8, ldgate=0, stream=P, out=P, ldstream=8, ldout=8,
             dstream=P, dout=P, lddstream=8, lddout=8, dresidual=P, dy=P, dweight=P, dbias=0, dpost_weight=0,
             dpost_bias=0, dgate=0, lddresidual=8, lddy=8, lddgate=8)
    f.update(over)
    fn = mb.lib().mlipcpp_b200_residual_norm_backward if backward else mb.lib().mlipcpp_b200_residual_norm
    return fn(ops._NORM.pack(*f.values()), 0, 0, None)


def test_layouts_match_the_header(tmp_path):
    """The packed structures have the C compiler's sizes and, by a field near
    the end of each, its layout."""
    import os
    import subprocess
    from conftest import ROOT
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdbool.h>\n#include <stddef.h>\n#include <stdio.h>\n#include "mlipcpp_b200.h"\n'
                   'int main(void) { printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(mlipcpp_b200_gated_linear_t), '
                   'offsetof(mlipcpp_b200_gated_linear_t, db_value), sizeof(mlipcpp_b200_linear_t), '
                   'offsetof(mlipcpp_b200_linear_t, db), sizeof(mlipcpp_b200_residual_norm_t), '
                   'offsetof(mlipcpp_b200_residual_norm_t, dgate)); return 0; }\n')
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    tail = struct.calcsize("3q")
    assert got == [ops._GATED.size, ops._GATED.size - tail - 8, ops._LINEAR.size, ops._LINEAR.size - 16 - 8,
                   ops._NORM.size, ops._NORM.size - tail - 8]


@pytest.mark.parametrize("call", [gated, linear, norm])
@pytest.mark.parametrize("backward", [False, True])
def test_common_refusals(call, backward):
    assert call(backward, dtype=3) == INVALID
    assert call(backward, dtype=-1) == INVALID
    assert call(backward, rows=-1) == INVALID
    assert call(backward, rows=1 << 31) == INVALID


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("over", [
    dict(activation=6), dict(activation=-1), dict(k=0), dict(f=0), dict(k=1 << 31), dict(ldx=7), dict(ldw_gate=7),
    dict(ldw_value=0), dict(x=P + 2), dict(w_gate=P + 1), dict(b_gate=P + 1), dict(dtype=2, b_value=P + 1)], ids=str)
def test_gated_refusals(backward, over):
    assert gated(backward, **over) == INVALID


def test_gated_null_and_output_refusals():
    for name in ("x", "w_gate", "w_value"):
        assert gated(**{name: 0}) == NULL and gated(True, **{name: 0}) == NULL
    assert gated(h=0) == NULL
    assert gated(ldh=15) == INVALID
    assert gated(True, dh=0) == NULL
    assert gated(True, lddh=15) == INVALID
    assert gated(True, lddx=7) == INVALID
    assert gated(True, lddw_gate=7) == INVALID
    assert gated(True, db_gate=P + 2) == INVALID
    assert mb.lib().mlipcpp_b200_gated_linear(None, None, 0, None) == NULL
    assert mb.lib().mlipcpp_b200_gated_linear_workspace(None, False) == -NULL


def test_workspace_refusals():
    assert gated(workspace=P + 128, size=1 << 20) == INVALID
    assert gated(workspace=0, size=256) == INVALID
    assert gated(workspace=P, size=-1) == INVALID


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("over", [
    dict(activation=9), dict(k=0), dict(n=0), dict(ldx=7), dict(ldw=7), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(x=P + 1), dict(w=P + 2), dict(b=P + 3)], ids=str)
def test_linear_refusals(backward, over):
    assert linear(backward, **over) == INVALID


def test_linear_null_and_output_refusals():
    assert linear(x=0) == NULL and linear(w=0) == NULL and linear(y=0) == NULL and linear(True, dy=0) == NULL
    assert linear(ldy=15) == INVALID
    assert linear(residual=P, ldresidual=15) == INVALID
    assert linear(True, lddw=7) == INVALID
    assert linear(True, lddx=7) == INVALID


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("over", [
    dict(norm=3), dict(post=-1), dict(d=0), dict(d=16385), dict(eps=0.0), dict(eps=float("nan")),
    dict(scale=float("inf")), dict(y=0, post=1, dy=0), dict(y=0, gate=P, dy=0), dict(y=0, post_weight=P, dy=0),
    dict(post_weight=P), dict(post_bias=P), dict(norm=0), dict(ldresidual=7), dict(ldy=7), dict(gate=P, ldgate=7),
    dict(residual=P + 2), dict(weight=P + 1)], ids=str)
def test_norm_refusals(backward, over):
    assert norm(backward, **over) == INVALID


def test_norm_gradient_refusals():
    """A gradient of an input that is not there."""
    assert norm(True, y=0) == INVALID
    assert norm(True, dgate=P) == INVALID
    assert norm(True, dbias=P) == INVALID
    assert norm(True, dpost_weight=P) == INVALID
    assert norm(True, residual=0) == NULL
    assert norm(True, lddresidual=7) == INVALID
    assert norm(True, lddout=7) == INVALID


def test_valid_calls_reach_the_device():
    """The same calls without a fault are turned down only for want of a GPU."""
    if torch.cuda.is_available():
        pytest.skip("this machine has a GPU")
    for call in (gated, linear, norm):
        for backward in (False, True):
            assert call(backward) == mb.BACKEND
    assert mb.lib().mlipcpp_b200_ops_status(None) == mb.BACKEND


def test_python_refusals():
    """Wrong devices, types, shapes and names raise before the library is
    called, with the reason."""
    x, w = torch.zeros(4, 8), torch.zeros(16, 8)
    for call in (lambda: ops.gated_linear(x, w, w), lambda: ops.linear(x, w), lambda: ops.residual_norm(x)):
        with pytest.raises(mb.MLIPError, match="CUDA"):
            call()
    with pytest.raises(mb.MLIPError, match="float32, float16 or bfloat16"):
        ops.linear(x.double(), w.double())
    with pytest.raises(mb.MLIPError, match="activation"):
        ops.linear(x, w, activation="tanh")
    with pytest.raises(mb.MLIPError, match="norm"):
        ops.residual_norm(x, norm="batch")


class _FakeCuda:
    """The checks of shapes and types see CPU tensors as if on one device."""
    def __enter__(self):
        self.dtype = ops._dtype
        ops._dtype = lambda t: ops._DTYPES[t.dtype]

    def __exit__(self, *_):
        ops._dtype = self.dtype


@pytest.mark.parametrize("call", [
    lambda x, w: ops.gated_linear(x, w, w[:, :4]),
    lambda x, w: ops.gated_linear(x[:, :4], w, w),
    lambda x, w: ops.gated_linear(x, w, w.half()),
    lambda x, w: ops.gated_linear(x, w, w, w[:, 0][:5]),
    lambda x, w: ops.gated_linear(x, w[0], w),
    lambda x, w: ops.gated_linear(x[:, :0], w[:, :0], w[:, :0]),
    lambda x, w: ops.gated_linear_backward(x, x, w, w),
    lambda x, w: ops.linear(x, w, residual=x),
    lambda x, w: ops.linear(x, w, w[:, 0].double()),
    lambda x, w: ops.linear_backward(x, x, w),
    lambda x, w: ops.residual_norm(x, x[:2]),
    lambda x, w: ops.residual_norm(x, x, weight=w[0][:3]),
    lambda x, w: ops.residual_norm(x, x, gate=x[:2]),
    lambda x, w: ops.residual_norm(x, None, gate=x),
    lambda x, w: ops.residual_norm(x, None, post_norm="rms"),
    lambda x, w: ops.residual_norm_backward(x[:2], None, x),
    lambda x, w: ops.residual_norm_backward(None, x.half(), x)])
def test_python_shape_refusals(call):
    with _FakeCuda(), pytest.raises(mb.MLIPError):
        call(torch.zeros(4, 8), torch.zeros(16, 8))


def test_forward_mode_is_refused(monkeypatch):
    """A dual tensor is turned down instead of losing its tangent, whichever
    argument it is; tensors without one are not."""
    from torch.autograd import forward_ad
    x, w = torch.zeros(4, 8), torch.zeros(8, 8)
    v = torch.zeros(8)

    def calls(x, w, v):
        return [lambda: ops.gated_linear(x, w, w, v), lambda: ops.linear(x, w, v, residual=x),
                lambda: ops.residual_norm(x, x, v, v, v, v, v, post_norm="rms"),
                lambda: ops.gated_linear_backward(x, x, w, w), lambda: ops.linear_backward(x, x, w, v),
                lambda: ops.residual_norm_backward(x, x, x, x, v, gate=v)]

    reached = []
    monkeypatch.setattr(ops, "_call", lambda name, *_: reached.append(name))
    with _FakeCuda(), forward_ad.dual_level():
        for call in calls(x, w, v):
            call()
        assert len(reached) == 6
        for i in range(3):
            t = [x, w, v]
            t[i] = forward_ad.make_dual(t[i], torch.ones_like(t[i]))
            for n, call in enumerate(calls(*t)):
                if (i == 1 and n in (2, 5)) or (i == 2 and n == 3):
                    continue  # (does not take it)
                with pytest.raises(mb.MLIPError, match="tangent"):
                    call()
    assert len(reached) == 6


@pytest.mark.parametrize("bad", [torch.tensor(2.0), torch.tensor(2.0, requires_grad=True), 1e39, -1e39, float("nan"),
                                 float("inf"), None, "1"], ids=str)
def test_scale_and_eps_are_numbers(bad, monkeypatch):
    """A tensor as a scale would be read on the host and lose its gradient;
    numbers that float32 does not hold have no place in a call either."""
    reached = []
    monkeypatch.setattr(ops, "_call", lambda name, *_: reached.append(name))
    x, w = torch.zeros(4, 8), torch.zeros(8, 8)

    def calls(scale, eps):
        return [lambda: ops.linear(x, w, scale=scale), lambda: ops.linear_backward(x, x, w, scale=scale),
                lambda: ops.residual_norm(x, scale=scale), lambda: ops.residual_norm_backward(x, x, x, scale=scale),
                lambda: ops.residual_norm(x, eps=eps), lambda: ops.residual_norm_backward(x, x, x, eps=eps)]

    with _FakeCuda():
        for call in calls(bad, bad):
            with pytest.raises(mb.MLIPError) as e:
                call()
            assert e.value.code == INVALID
        assert not reached
        for good in (2, 2.0, np.float32(2), np.float64(2)):
            for call in calls(good, good):
                call()
    assert len(reached) == 24


def test_lazily_negated_tensors():
    """The imaginary part of a conjugate is a view whose values torch negates
    on reading: what the library is given holds them."""
    import ctypes
    for z in (torch.complex(torch.zeros(6, 1), torch.arange(6.0)[:, None]), torch.complex(torch.zeros(3, 4), torch.ones(3, 4))):
        x, keep = z.conj().imag, []
        assert x.is_neg()
        at, ld = ops._take(x, x, x.shape, x.shape[1], keep, "x")
        got = [[ctypes.c_float.from_address(at + 4 * (i * ld + j)).value for j in range(x.shape[1])]
               for i in range(x.shape[0])]
        assert got == x.tolist()


@pytest.mark.parametrize("needs", [(), (True,) * 2, (True,) * 8], ids=len)
def test_needs_has_an_entry_for_each_input(needs, monkeypatch):
    monkeypatch.setattr(ops, "_call", lambda *_: None)
    x, w = torch.zeros(4, 8), torch.zeros(8, 8)
    with _FakeCuda():
        for call in (lambda: ops.gated_linear_backward(x, x, w, w, needs=needs),
                     lambda: ops.linear_backward(x, x, w, needs=needs),
                     lambda: ops.residual_norm_backward(x, x, x, needs=needs)):
            with pytest.raises(mb.MLIPError) as e:
                call()
            assert e.value.code == INVALID
