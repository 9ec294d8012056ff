"""A launch that fails is reported once and not made again."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from llm_accelerator_b200 import _lib as L
from llm_accelerator_b200.errors import EngineError

pytestmark = pytest.mark.gpu


def _addresses(ts):
    return [C.cast(getattr(L.lib, "tac_" + name), C.c_void_p).value for name in ts.ENTRIES]


def _calls():
    """Name of the entry, and a call that reaches it."""
    from llm_accelerator_b200 import logprobs, mxfp4, norm, ptq
    x, w = torch.ones((3, 64), device="cuda"), torch.ones(64, device="cuda")
    q, scale = norm.rms_norm_i8(x, w)
    a = mxfp4.quantize(x)
    many = torch.ones((200, 64), device="cuda")
    return {"rms_norm": lambda: norm.rms_norm(x, w), "rms_norm_i8": lambda: norm.rms_norm_i8(x, w, residual=x),
            "dequantize_rows_i8": lambda: ptq.dequantize_rows(q, scale), "mxfp4_quantize": lambda: mxfp4.quantize(x),
            "mxfp4_values": a.values, "mxfp4_gemm": lambda: mxfp4.gemm(a, a), "linear_mxfp4": lambda: mxfp4.linear(many, a),
            "token_logprobs": lambda: logprobs.token_logprobs(x, torch.zeros(3, dtype=torch.int64, device="cuda"), 3)}


@pytest.mark.parametrize("name", ["rms_norm", "rms_norm_i8", "dequantize_rows_i8", "mxfp4_quantize", "mxfp4_values", "mxfp4_gemm",
                                  "linear_mxfp4", "token_logprobs"])
def test_one_launch_and_one_error(name, monkeypatch):
    from llm_accelerator_b200 import _tensors as ts
    call, at = _calls()[name], ts.ENTRIES.index(name)
    restype, argtypes = L.SIGNATURES["tac_" + name]
    made = []

    def fails(*args):
        made.append(args)
        return L.E_CUDA

    fake = C.CFUNCTYPE(restype, *argtypes)(fails)
    good = _addresses(ts)
    want = call()
    try:
        ts.front.bind(*good[:at], C.cast(fake, C.c_void_p).value, *good[at + 1:], L.check)
        with pytest.raises(EngineError, match="tac_" + name):
            call()
    finally:
        ts.front.bind(*good, L.check)
    assert len(made) == 1
    again = call()
    for a, b in zip(*((t if isinstance(t, tuple) else (t,)) for t in (want, again))):
        if torch.is_tensor(a):
            assert torch.equal(a, b)


def test_a_function_that_does_not_raise():
    from llm_accelerator_b200 import _tensors as ts, norm
    x, w = torch.ones((3, 64), device="cuda"), torch.ones(64, device="cuda")
    restype, argtypes = L.SIGNATURES["tac_rms_norm"]
    fake = C.CFUNCTYPE(restype, *argtypes)(lambda *args: L.E_CUDA)
    good = _addresses(ts)
    try:
        ts.front.bind(C.cast(fake, C.c_void_p).value, *good[1:], lambda status, name: None)
        with pytest.raises(RuntimeError, match="tac_rms_norm"):
            norm.rms_norm(x, w)
    finally:
        ts.front.bind(*good, L.check)
    with pytest.raises(TypeError):
        ts.front.bind(*good)
