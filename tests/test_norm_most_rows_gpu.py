"""As many rows as an int counts."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_most_rows():
    from llm_accelerator_b200 import norm
    M = 2 ** 31 - 1
    x = torch.full((M, 1), 2.0, dtype=torch.float16, device="cuda")
    x[1::3] = -4.0
    y = norm.rms_norm(x, torch.ones(1, device="cuda"), 0.0)
    x.sign_()
    assert torch.equal(x, y)
