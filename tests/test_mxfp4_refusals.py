"""Arguments that the 4-bit rows and products refuse, before any CUDA call (no GPU needed)."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from llm_accelerator_b200 import _lib as L
from llm_accelerator_b200 import mxfp4

P = C.c_void_p(4096)     # never dereferenced: the checks come first
ODD, HALF, EIGHT = C.c_void_p(4097), C.c_void_p(4098), C.c_void_p(4104)


def _quantize(X=P, t=L.TYPE_F16, ldx=64, c=P, s=P, M=4, K=64):
    return L.lib.tac_mxfp4_quantize(X, t, ldx, c, s, M, K, None)


def _values(c=P, s=P, Y=P, t=L.TYPE_F16, M=4, K=64):
    return L.lib.tac_mxfp4_values(c, s, Y, t, M, K, None)


def _gemm(ac=P, as_=P, bc=P, bs=P, bias=None, bt=0, Y=P, yt=L.TYPE_F16, M=4, N=8, K=64):
    return L.lib.tac_mxfp4_gemm(ac, as_, bc, bs, bias, bt, Y, yt, M, N, K, None)


def _linear(X=P, t=L.TYPE_F16, ldx=64, bc=P, bs=P, bias=None, bt=0, Y=P, yt=L.TYPE_F16, ws=P, wn=1 << 24, M=200, N=8, K=64):
    return L.lib.tac_linear_mxfp4(X, t, ldx, bc, bs, bias, bt, Y, yt, ws, wn, M, N, K, None)


@pytest.mark.parametrize("bad", [dict(X=None), dict(c=None), dict(s=None), dict(t=3), dict(ldx=63), dict(M=0), dict(K=0),
                                 dict(K=(1 << 24) + 1, ldx=1 << 25), dict(c=EIGHT), dict(s=EIGHT), dict(X=ODD),
                                 dict(X=HALF, t=L.TYPE_F32)])
def test_quantize_refusals(bad):
    assert _quantize(**bad) == L.E_ARGUMENT


@pytest.mark.parametrize("bad", [dict(c=None), dict(s=None), dict(Y=None), dict(t=-1), dict(M=0), dict(K=0), dict(c=EIGHT),
                                 dict(s=EIGHT), dict(Y=ODD), dict(Y=HALF, t=L.TYPE_F32), dict(K=(1 << 24) + 1)])
def test_values_refusals(bad):
    assert _values(**bad) == L.E_ARGUMENT


PRODUCT = [dict(bc=None), dict(bs=None), dict(Y=None), dict(yt=3), dict(bias=P, bt=7), dict(M=0), dict(N=0), dict(K=0),
           dict(M=(1 << 20) + 1), dict(N=(1 << 30) + 1), dict(bc=EIGHT), dict(bs=EIGHT), dict(Y=ODD),
           dict(Y=HALF, yt=L.TYPE_F32), dict(bias=ODD, bt=L.TYPE_F16)]


@pytest.mark.parametrize("bad", PRODUCT + [dict(ac=None), dict(as_=None), dict(ac=EIGHT), dict(as_=EIGHT), dict(K=(1 << 24) + 1)])
def test_gemm_refusals(bad):
    assert _gemm(**bad) == L.E_ARGUMENT


@pytest.mark.parametrize("bad", PRODUCT + [dict(X=None), dict(t=3), dict(ldx=63), dict(X=ODD), dict(ws=None),
                                           dict(ws=C.c_void_p(4096 + 16)), dict(wn=100)])
def test_linear_refusals(bad):
    assert _linear(**bad) == L.E_ARGUMENT


def test_sizes():
    code, scale = L.lib.tac_mxfp4_code_bytes, L.lib.tac_mxfp4_scale_bytes
    assert code(0, 5) == scale(5, 0) == 0
    assert code(3, 33) == 3 * 32 and code(1 << 20, 1 << 20) == 1 << 39
    assert scale(1, 1) == 1024 and scale(129, 257) == 2 * 4 * 512
    assert L.lib.tac_linear_mxfp4_workspace_bytes(200, 8, 64) >= code(200, 64) + scale(200, 64)
    assert L.lib.tac_linear_mxfp4_workspace_bytes(0, 8, 64) == 0


def test_python_checks():
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    for args, error in [((u8(3, 32).int(), u8(1, 2, 32, 4, 4), 64), TypeError), ((u8(3, 31), u8(1, 2, 32, 4, 4), 64), ValueError),
                        ((u8(3, 32), u8(1, 1, 32, 4, 4), 64), ValueError), ((u8(3, 32), u8(1, 2, 32, 4, 4), 64), ValueError),
                        ((u8(3, 0), u8(1, 0, 32, 4, 4), 0), ValueError)]:
        with pytest.raises(error):
            mxfp4.Mxfp4(*args)
    with pytest.raises(TypeError):
        mxfp4.Mxfp4.from_tensors(u8(3, 32), u8(3, 2).int(), 64)
    with pytest.raises(ValueError):
        mxfp4.Mxfp4.from_tensors(u8(3, 32), u8(3, 3), 64)
    with pytest.raises(ValueError):
        mxfp4.Mxfp4.from_tensors(u8(96), u8(3, 2), 64)
    for x, error in [(torch.ones((2, 8)).double(), TypeError), (torch.ones(8), ValueError), (torch.ones((2, 0)), ValueError),
                     (torch.ones((8, 2)).t(), ValueError), (torch.ones((1, 8)).expand(3, 8), ValueError),
                     (torch.ones((2, 8)), ValueError)]:
        with pytest.raises(error):
            mxfp4.quantize(x)
        with pytest.raises(error):
            mxfp4.linear(x, None)
    assert "o gradient flows through" in " ".join(mxfp4.__doc__.split())


@pytest.mark.gpu
def test_python_checks_on_a_device():
    w = mxfp4.quantize(torch.ones((8, 64), device="cuda"))
    x = torch.ones((3, 64), device="cuda")
    for args, error in [(dict(bias=torch.ones(7, device="cuda")), ValueError), (dict(bias=torch.ones(8)), ValueError),
                        (dict(bias=torch.ones(8, device="cuda").int()), TypeError),
                        (dict(out=torch.ones((3, 8), device="cuda").half()), ValueError),
                        (dict(out=torch.ones((3, 16), device="cuda")[:, :8]), ValueError),
                        (dict(ws=torch.ones(100000, device="cuda")), ValueError), (dict(ws=torch.ones(8).byte()), ValueError)]:
        with pytest.raises(error):
            mxfp4.linear(x, w, **args)
    with pytest.raises(ValueError):
        mxfp4.linear(x[:, :63], w)
    with pytest.raises(ValueError):
        mxfp4.gemm(mxfp4.quantize(x[:, :32].contiguous()), w)
    with pytest.raises(TypeError):
        mxfp4.gemm(w, w, out_dtype=torch.int8)
    with pytest.raises(ValueError):
        mxfp4.Mxfp4(w.codes.view(-1)[8:8 * 32 + 8 - 32].view(7, 32), w.scales, 64)
