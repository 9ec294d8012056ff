"""Arguments that the scaled INT8 products and the row quantiser refuse, before any CUDA call (no GPU needed)."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from llm_accelerator_b200 import _lib as L
from llm_accelerator_b200 import gemm, ptq

P = C.c_void_p(4096)     # never dereferenced: the checks come first
ODD = C.c_void_p(4104)


def _gemm(A=P, Bt=P, sa=P, sb=P, sbt=L.TYPE_F32, bias=None, bt=0, Y=P, yt=L.TYPE_F16, M=4, N=8, K=32):
    return L.lib.tac_gemm_i8_scaled(A, Bt, sa, sb, sbt, bias, bt, Y, yt, M, N, K, None)


def _linear(X=P, xt=L.TYPE_F16, ldx=32, Bt=P, sb=P, sbt=L.TYPE_F16, bias=None, bt=0, Y=P, yt=L.TYPE_F16, ws=P,
            wn=1 << 20, M=40, N=8, K=32):
    return L.lib.tac_linear_w8a8(X, xt, ldx, Bt, sb, sbt, bias, bt, Y, yt, ws, wn, M, N, K, None)


def _rows(X=P, xt=L.TYPE_F16, ldx=32, Q=P, s=P, M=4, K=32):
    return L.lib.tac_quantize_rows_i8(X, xt, ldx, Q, s, M, K, None)


@pytest.mark.parametrize("bad", [dict(A=None), dict(Bt=None), dict(sa=None), dict(sb=None), dict(Y=None), dict(M=0),
                                 dict(N=-1), dict(K=0), dict(K=40), dict(A=ODD), dict(Bt=ODD), dict(sbt=L.TYPE_BF16),
                                 dict(yt=3), dict(bias=P, bt=7), dict(K=1 << 17), dict(M=(1 << 20) + 1),
                                 dict(N=(1 << 30) + 1), dict(Y=C.c_void_p(4097)), dict(Y=C.c_void_p(4098), yt=L.TYPE_F32),
                                 dict(sb=C.c_void_p(4098)), dict(sb=C.c_void_p(4097), sbt=L.TYPE_F16), dict(sa=C.c_void_p(4098)),
                                 dict(bias=C.c_void_p(4097), bt=L.TYPE_BF16)])
def test_gemm_refusals(bad):
    assert _gemm(**bad) == L.E_ARGUMENT


@pytest.mark.parametrize("bad", [dict(X=None), dict(Bt=None), dict(sb=None), dict(Y=None), dict(ws=None),
                                 dict(ws=C.c_void_p(4096 + 16)), dict(wn=100), dict(ldx=31), dict(xt=3), dict(yt=-1),
                                 dict(M=0), dict(N=0), dict(K=-5), dict(Bt=ODD), dict(K=1 << 17), dict(X=C.c_void_p(4097))])
def test_linear_refusals(bad):
    assert _linear(**bad) == L.E_ARGUMENT


@pytest.mark.parametrize("bad", [dict(X=None), dict(Q=None), dict(s=None), dict(xt=3), dict(ldx=31), dict(Q=ODD),
                                 dict(M=0), dict(K=0), dict(X=C.c_void_p(4098), xt=L.TYPE_F32), dict(s=C.c_void_p(4098))])
def test_quantize_rows_refusals(bad):
    assert _rows(**bad) == L.E_ARGUMENT


def test_workspace_bytes():
    assert L.lib.tac_linear_w8a8_workspace_bytes(0, 5) == 0
    assert L.lib.tac_linear_w8a8_workspace_bytes(16, 8192) == 0          # few rows need none
    assert L.lib.tac_linear_w8a8_workspace_bytes(17, 17) >= 17 * 32 + 17 * 4
    assert L.lib.tac_linear_w8a8_workspace_bytes(16, 8193) >= 16 * 8208 + 64
    assert L.lib.tac_linear_w8a8_workspace_bytes(1 << 20, 131071) > 1 << 36


def _i8(*shape):
    return torch.zeros(shape, dtype=torch.int8)


def test_python_checks():
    one = torch.ones
    with pytest.raises(TypeError):
        gemm.gemm_i8_scaled(one(2, 16), _i8(4, 16), one(2), one(4))
    with pytest.raises(TypeError):
        gemm.gemm_i8_scaled(_i8(2, 16), _i8(4, 16), one(2), one(4).bfloat16())
    with pytest.raises(TypeError):
        gemm.gemm_i8_scaled(_i8(2, 16), _i8(4, 16), one(2), one(4), out_dtype=torch.int8)
    with pytest.raises(ValueError):
        gemm.gemm_i8_scaled(_i8(2, 16), _i8(4, 32), one(2), one(4))
    with pytest.raises(ValueError):
        gemm.gemm_i8_scaled(_i8(2, 16), _i8(4, 16), one(3), one(4))
    with pytest.raises(ValueError):
        gemm.gemm_i8_scaled(_i8(2, 16), _i8(4, 16), one(2), one(5))
    with pytest.raises(ValueError):     # CPU tensors
        gemm.gemm_i8_scaled(_i8(2, 16), _i8(4, 16), one(2), one(4))
    with pytest.raises(ValueError):     # K_pad of 20 columns is 32
        gemm.linear_w8a8(one(2, 20), _i8(4, 20), one(4))
    with pytest.raises(ValueError):     # columns that are not contiguous
        gemm.linear_w8a8(one(16, 2).t(), _i8(4, 16), one(4))
    with pytest.raises(ValueError):     # rows that overlap
        gemm.linear_w8a8(one(1, 16).expand(3, 16), _i8(4, 16), one(4))
    with pytest.raises(TypeError):
        gemm.linear_w8a8(one(2, 16).double(), _i8(4, 16), one(4))
    with pytest.raises(TypeError):
        ptq.quantize_rows(one(2, 16))
    assert gemm.pad_k16(_i8(3, 20)).shape == (3, 32) and gemm.pad_k16(_i8(3, 32)).shape == (3, 32)
