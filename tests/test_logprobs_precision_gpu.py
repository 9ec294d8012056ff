"""How far entropies of rows with a few logits far above the rest are from the definition in 64 bits, over many rows."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


# rows of a CTA of eight and of four warps, of a warp each, of two and eight CTAs each
@pytest.mark.parametrize("M,V", [(512, 50257), (1000, 50257), (20000, 1000), (64, 50257), (16, 100003)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_entropy_over_many_rows(M, V, dtype):
    """H = ln S - T / S with H below 8 (a row whose H is above has last places twice as large, and counts half).  The last
    steps round three numbers below 8, by a root mean square of 2^-21 / sqrt(12) = 1.4e-7 each (ln S below 4 by a whole last
    place at most, which is the same): 2.4e-7.  A term's exponential has 2^-22 / sqrt(3) = 1.4e-7 and its argument, within a
    few units of 0, 1e-7; a sum T of a few units as much S, 0.7e-7 an addition of the few that matter, and the shift to the
    row's largest as much again: 2e-7, of terms whose shares add up to one.  Altogether 3.2e-7; 5e-7 leaves a half for the
    sums' lengths.  (Sums about a value 16 below the largest lose four bits of T and give 1e-6.)"""
    from llm_accelerator_b200 import logprobs
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn((M, V), generator=g, device="cuda") * 2.5
    for _ in range(12):
        x.scatter_add_(1, torch.randint(0, V, (M, 1), generator=g, device="cuda"), torch.rand((M, 1), generator=g, device="cuda") * 14)
    x = x.to(dtype)
    tokens = x.float().argmax(1)
    lp, entropy = logprobs.token_logprobs(x, tokens)
    off, off_lp = [], []
    for i in range(0, M, 500):
        z = x[i:i + 500].double()
        z = z - torch.logsumexp(z, 1, keepdim=True)
        p = z.exp()
        h = -torch.special.xlogy(p, p).sum(1)
        assert float(h.max()) < 16
        off.append((entropy[i:i + 500].double() - h) / torch.where(h < 8, 1, 2))
        off_lp.append(lp[i:i + 500].double() - z.gather(1, tokens[i:i + 500, None])[:, 0])
    for d in (off, off_lp):
        d = torch.cat(d)
        assert float(d.square().mean().sqrt()) <= 5e-7, (float(d.square().mean().sqrt()), float(d.abs().max()))
