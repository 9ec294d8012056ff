"""Arguments that the log-probabilities refuse, before any CUDA call (no GPU needed)."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from llm_accelerator_b200 import _lib as L
from llm_accelerator_b200 import logprobs

P = C.c_void_p(4096)     # never dereferenced: the checks come first
ODD, HALF, FOUR = C.c_void_p(4097), C.c_void_p(4098), C.c_void_p(4100)


def _call(X=P, t=L.TYPE_F16, ld=100, tok=P, t64=1, M=4, V=100, top=5, lp=P, e=P, tl=P, ti=P):
    return L.lib.tac_token_logprobs(X, t, ld, tok, t64, M, V, top, lp, e, tl, ti, None)


@pytest.mark.parametrize("bad", [dict(X=None), dict(tok=None), dict(lp=None), dict(e=None), dict(tl=None), dict(ti=None), dict(t=3),
                                 dict(M=0), dict(V=0), dict(M=-2), dict(ld=99), dict(top=-1), dict(top=33), dict(V=4, top=5),
                                 dict(X=ODD), dict(X=HALF, t=L.TYPE_F32), dict(tok=FOUR), dict(tok=HALF, t64=0), dict(lp=HALF),
                                 dict(e=HALF), dict(tl=HALF), dict(ti=HALF)])
def test_refusals(bad):
    assert _call(**bad) == L.E_ARGUMENT


def test_python_checks():
    x, t = torch.zeros((3, 50)), torch.zeros(3, dtype=torch.int64)
    for args, error in [((x.double(), t), TypeError), ((x[0], t), ValueError), ((x.t(), t), ValueError),
                        ((x[:1].expand(3, 50), t), ValueError), ((x[:, :0], t), ValueError), ((x, t), ValueError)]:
        with pytest.raises(error):
            logprobs.token_logprobs(*args)
    assert "o gradient flows through" in " ".join(logprobs.__doc__.split())


@pytest.mark.gpu
def test_python_checks_on_a_device():
    x, t = torch.zeros((3, 50), device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for args, error in [((x, t.float()), TypeError), ((x, t[:2]), ValueError), ((x, t.cpu()), ValueError),
                        ((x, torch.zeros((3, 2), dtype=torch.int64, device="cuda")[:, 0]), ValueError), ((x, t, 33), ValueError),
                        ((x[:, :4], t, 5), ValueError), ((x, t, -1), ValueError)]:
        with pytest.raises(error):
            logprobs.token_logprobs(*args)
