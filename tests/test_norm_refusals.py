"""Arguments that the norms and the values of INT8 rows refuse, before any CUDA call (no GPU needed)."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from llm_accelerator_b200 import _lib as L
from llm_accelerator_b200 import norm, ptq

P = C.c_void_p(4096)     # never dereferenced: the checks come first
Q = C.c_void_p(8192)
ODD, HALF = C.c_void_p(4097), C.c_void_p(4098)


def _norm(X=P, t=L.TYPE_F16, ldx=32, R=P, ldr=32, H=P, ldh=32, W=P, wt=L.TYPE_F16, eps=1e-6, Y=Q, M=4, K=32):
    return L.lib.tac_rms_norm(X, t, ldx, R, ldr, H, ldh, W, wt, eps, Y, M, K, None)


def _i8(X=P, t=L.TYPE_F16, ldx=32, R=P, ldr=32, H=P, ldh=32, W=P, wt=L.TYPE_F16, eps=1e-6, Q=Q, s=P, M=4, K=32):
    return L.lib.tac_rms_norm_i8(X, t, ldx, R, ldr, H, ldh, W, wt, eps, Q, s, M, K, None)


BAD = [dict(X=None), dict(W=None), dict(R=None), dict(H=None), dict(t=3), dict(wt=-1), dict(M=0), dict(K=0), dict(M=-1),
       dict(ldx=31), dict(ldr=31), dict(ldh=31), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
       dict(X=ODD), dict(R=ODD), dict(H=ODD), dict(W=ODD), dict(W=HALF, wt=L.TYPE_F32), dict(X=HALF, t=L.TYPE_F32)]


@pytest.mark.parametrize("bad", BAD + [dict(Y=None), dict(Y=ODD), dict(Y=P), dict(K=(1 << 30) + 1, ldx=1 << 31, ldr=1 << 31, ldh=1 << 31)])
def test_norm_refusals(bad):
    assert _norm(**bad) == L.E_ARGUMENT


@pytest.mark.parametrize("bad", BAD + [dict(Q=None), dict(s=None), dict(Q=C.c_void_p(4104)), dict(s=HALF)])
def test_norm_i8_refusals(bad):
    assert _i8(**bad) == L.E_ARGUMENT


@pytest.mark.parametrize("bad", [dict(Q=None), dict(s=None), dict(Y=None), dict(yt=5), dict(M=0), dict(K=0),
                                 dict(Q=C.c_void_p(4104)), dict(s=HALF), dict(Y=ODD), dict(Y=HALF, yt=L.TYPE_F32)])
def test_dequantize_refusals(bad):
    a = dict(Q=P, s=P, Y=P, yt=L.TYPE_F16, M=3, K=20) | bad
    assert L.lib.tac_dequantize_rows_i8(a["Q"], a["s"], a["Y"], a["yt"], a["M"], a["K"], None) == L.E_ARGUMENT


def test_python_checks():
    one = torch.ones
    with pytest.raises(TypeError):
        norm.rms_norm(one(2, 16).double(), one(16))
    with pytest.raises(ValueError):     # CPU tensors
        norm.rms_norm(one(2, 16), one(16))
    with pytest.raises(ValueError):
        norm.rms_norm(one(16), one(16))
    with pytest.raises(ValueError):
        norm.rms_norm_i8(one(2, 0), one(0))
    codes = torch.zeros((2, 16), dtype=torch.int8)
    with pytest.raises(TypeError):
        ptq.dequantize_rows(codes.int(), one(2))
    with pytest.raises(TypeError):
        ptq.dequantize_rows(codes, one(2), dtype=torch.int8)
    with pytest.raises(ValueError):
        ptq.dequantize_rows(codes[:, :15], one(2))
    with pytest.raises(ValueError):
        ptq.dequantize_rows(codes, one(3))
    with pytest.raises(ValueError):     # CPU tensors
        ptq.dequantize_rows(codes, one(2))


def test_the_documentation_says_that_no_gradient_flows():
    for text in (norm.__doc__, ptq.dequantize_rows.__doc__):
        assert "o gradient flows through" in " ".join(text.split())


@pytest.mark.gpu
def test_python_checks_on_a_device():
    x, w = torch.ones((4, 32), device="cuda"), torch.ones(32, device="cuda")
    for bad, error in [(dict(residual=x.half()), TypeError), (dict(residual=x[:3]), ValueError), (dict(residual=x.cpu()), ValueError),
                       (dict(residual_out=x), ValueError), (dict(residual=x, residual_out=x.half()), TypeError),
                       (dict(residual=x, residual_out=x.t()), ValueError), (dict(eps=-1.0), ValueError),
                       (dict(eps=float("nan")), ValueError), (dict(residual=x[:1].expand(4, 32)), ValueError)]:
        for f in (norm.rms_norm, norm.rms_norm_i8):
            with pytest.raises(error):
                f(x, w, **bad)
    for bad in (w[:31], w.cpu(), torch.ones((32, 2), device="cuda")[:, 0]):
        with pytest.raises(ValueError):
            norm.rms_norm(x, bad)
    with pytest.raises(TypeError):
        norm.rms_norm(x, w.int())
    with pytest.raises(ValueError):
        norm.rms_norm(x.t(), torch.ones(4, device="cuda"))
    with pytest.raises(ValueError):
        norm.rms_norm(x, w, residual=x, residual_out=(y := torch.empty_like(x)), out=y)
    with pytest.raises(ValueError):
        norm.rms_norm(x, w, out=x.half())
    with pytest.raises(ValueError):
        norm.rms_norm(x, w, out=x.new_empty((4, 64))[:, :32])
