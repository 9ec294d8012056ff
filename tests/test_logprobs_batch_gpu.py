"""A row's results are those of its own logits, whatever other rows are asked for with it."""
from __future__ import annotations

import pytest
import torch

from test_logprobs_gpu import BF16, F16, F32, _logits, _tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("V", [900, 9001, 50257])
def test_rows_alone_and_among_others(V, dtype):
    """Batches for which a row has one, two or eight CTAs, eight or four warps, or one: each result is within the tolerance
    of ln S of the definition, so two are within twice that; the likeliest tokens are exact."""
    from llm_accelerator_b200 import logprobs
    x, tokens = _logits(2000, V, dtype, V, 3)
    x[2, ::2] = -float("inf")
    x[3] = 1.0
    alone = [torch.cat(t) for t in zip(*(logprobs.token_logprobs(x[i:i + 1], tokens[i:i + 1], top=20) for i in range(8)))]
    tol = 2 * _tolerance(V)
    for M in (8, 40, 150, 300, 500, 800, 1000, 2000):
        for rows in (slice(0, 8), slice(M - 8, M)):      # the same eight rows first and last
            y, t = x[:M].clone(), tokens[:M].clone()
            y[rows], t[rows] = x[:8], tokens[:8]
            lp, entropy, top_lp, ids = (r[rows] for r in logprobs.token_logprobs(y, t, top=20))
            assert torch.equal(ids, alone[3])
            for a, b in ((lp, alone[0]), (top_lp, alone[2])):
                assert bool(((a == b) | ((a - b).abs() <= tol)).all())
            assert bool(((entropy - alone[1]).abs() <= tol * (2 + 2 * alone[1].abs())).all())
