"""Log-probabilities of finite logits of any magnitude: masks and rows of values from 10^6 to the ends of the types, in
every shape of the kernel."""
from __future__ import annotations

import pytest
import torch

from test_logprobs_gpu import BF16, F32, _check

pytestmark = pytest.mark.gpu

SIZES = [1e6, 1e7, 1e8, 1e9, 4e9, 1e10, 1e11, 1e12, 1e15, 1e18, 1e20, 1e25, 1e30, 1e38, 3.3e38]
KINDS = [(kind, size * sign) for kind in range(5) for size in SIZES for sign in (-1, 1)]


def _rows(kinds, V, dtype):
    """Rows of one value alone, of it around a few ordinary logits, beside a half of ordinary ones, alternating with a
    neighbour of its size, and of it and the three numbers of the type next to it."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn((len(kinds), V), generator=g)
    step = torch.finfo(dtype).eps
    for row, (kind, v) in zip(x, kinds):
        if kind == 0:
            row[:] = v
        elif kind == 1:
            few, at = row[:3].clone(), torch.randint(0, V, (3,), generator=g)
            row[:] = v
            row[at] = few
        elif kind == 2:
            row[V // 2:] = v
        elif kind == 3:
            row[::2] = v
            row[1::2] = v * (1 - step)
        else:
            row[:] = v * (1 - torch.randint(0, 4, (V,), generator=g) * step)
    return x.to(dtype).cuda(), torch.randint(0, V, (len(kinds),), generator=g).cuda()


# a warp, eight and four warps a row, two and eight CTAs a row
@pytest.mark.parametrize("M,V", [(150, 700), (300, 9000), (900, 9000), (150, 50257), (16, 100003)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_every_magnitude(M, V, dtype):
    for first in range(0, len(KINDS), M):
        x, tokens = _rows([KINDS[(first + r) % len(KINDS)] for r in range(M)], V, dtype)
        _check(x, tokens, 5)
    _check(x, tokens, 0)
