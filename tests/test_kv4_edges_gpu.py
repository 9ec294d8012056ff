"""Attention over the 4-bit cache where a softmax state begins late or sits at the ends of the types, on the GPU against
the definition in 64 bits (tests/kv4_helpers.py derives the tolerances)."""
from __future__ import annotations

import pytest
import torch

from kv4_helpers import Batch, check, check_lse, queries, reference

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _reload(b):
    """The cache after changes to b.host and b.table."""
    for t, h in zip((b.cache.k_codes, b.cache.k_params, b.cache.v_codes, b.cache.v_params), b.host):
        t.copy_(h)
    b.d_table = b.table.cuda()


@pytest.mark.parametrize("scores", [-173.0, -20.0, 100.0])
@pytest.mark.parametrize("zeros", [256, 512])
@pytest.mark.parametrize("D,group,new", [(64, 1, 1), (64, 1, 12), (128, 4, 1), (128, 4, 5), (64, 16, 600), (64, 16, 1000)])
def test_a_context_that_begins_with_missing_pages_and_zero_values(D, group, new, zeros, scores):
    """The first 256 positions have no page, the next `zeros` hold values of zero, and all scores are alike (in powers of
    two, far below 2^-126 in the first case): the keys of the zeros weigh as much as the others."""
    from llm_accelerator_b200 import kv4
    b = Batch([1024], 1, D, 16)
    b.table[0, :16] = -1
    b.host[0][:] = 0xFF                                   # keys: 15 in every channel
    b.host[1][:] = 0x3F800000
    for j in range(16, 16 + zeros // 16):
        b.host[2][int(b.table[0, j])] = 0
        b.host[3][int(b.table[0, j])] = 0
    _reload(b)
    q = torch.full((new, group, D), scores * 0.6931471805599453 / (15 * D ** 0.5), dtype=torch.float16, device="cuda")
    out, lse = kv4.attention(q, b.cache, b.d_table, b.d_lens, _i32([0, new]), return_lse=True, causal=new < 20)
    want, wlse, tol = reference(b, q, [0, new], causal=new < 20)
    check(out, want, tol)
    check_lse(lse, wlse)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("loud", [None, 3, 700, 1290])
@pytest.mark.parametrize("D,group,new,vmul", [(64, 1, 1, 2.0 ** 103), (64, 4, 9, 2.0 ** 103), (64, 16, 1100, 2.0 ** 103),
                                              (128, 16, 1300, 2.0 ** 103), (128, 16, 700, 2.0 ** 91)])
def test_the_largest_values(D, group, new, vmul, loud, dtype):
    """Scales of up to 2^105 (what is promised ends at 2^107), one token louder than the others by 2^3 or 2^12; both
    kernels, and a row's unit that starts low and ends high.  FP16 results beyond its range are infinities."""
    from llm_accelerator_b200 import kv4
    b = Batch([1300], 1, D, 32, vscale=vmul)
    if loud is not None:
        b.host[3][int(b.table[0, loud // 32]), 0, loud % 32] += (12 if vmul < 2.0 ** 100 else 3) << 23
        _reload(b)
    q = queries(new, group, D, dtype)
    out, lse = kv4.attention(q, b.cache, b.d_table, b.d_lens, _i32([0, new]), return_lse=True)
    want, wlse, tol = reference(b, q, [0, new])
    if dtype == torch.float16:
        sure = want.abs() > tol + 65536
        assert (out.cpu()[sure].double() == torch.copysign(torch.tensor(float("inf")).double(), want[sure])).all()
    else:
        check(out, want, tol)
    check_lse(lse, wlse)


def _sharp(b, q):
    """(out, tol) float64 of one sequence's last rows, causal, with the tolerance of tests/kv4_helpers.py but for the unit
    of the weights: FP16 weights below 2^-14 of it are off by 2^-25 of it, it is at most the largest scale among the keys
    that the ROW sees, and the sum that they are divided by is at least z = sum exp(score - top)."""
    q = q.cpu().double()
    c, group, D = q.shape
    n = b.lens[0]
    K, ok = b.rows(0, 0, 0, n)
    V, _ = b.rows(0, 1, 0, n)
    scales = torch.stack([(b.host[3][int(b.table[0, j // b.page]), 0, j % b.page] & -65536).view(torch.float32).double()
                          for j in range(n)])
    seen = torch.arange(n)[None, :] <= (n - c + torch.arange(c))[:, None]
    s = torch.einsum("cgd,nd->cgn", q, K) * D ** -0.5
    ds = (torch.einsum("cgd,nd->cgn", q.abs(), K.abs()) * (2 * D + 4) * 2.0 ** -24
          + q.abs().amax(-1, keepdim=True) * K.abs().sum(-1) * 2.0 ** -25) * D ** -0.5
    s = s.masked_fill(~seen[:, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    z = p.sum(-1, keepdim=True)
    p = p / z
    rel = 2.0 ** -11 + 2.0 ** -19 + 2 * ds.masked_fill(~seen[:, None], 0).amax(-1, keepdim=True) + n * 2.0 ** -24
    big = torch.where(seen, scales[None, :], 0.0).amax(-1)[:, None, None]
    out = p @ V
    tol = rel * (p @ V.abs()) + seen.sum(-1)[:, None, None] * 2.0 ** -25 * 15 * big / z
    return out, tol + 2.0 ** -8 * out.abs() * (1 + 2.0 ** -8) + 2.0 ** -134


@pytest.mark.parametrize("n,group,new", [(700, 1, 1), (700, 1, 130), (700, 4, 9), (1500, 16, 700), (1500, 16, 1400)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("back", [5, 90, 400])
def test_a_loud_token_coarsens_only_the_rows_that_see_it(back, D, n, group, new):
    """One token, `back` before the end, with values 2^20 times the others'.  Rows before it are held to the ordinary
    tolerance, of which a row of zeros would be far outside."""
    from llm_accelerator_b200 import kv4
    b = Batch([n], 1, D, 16)
    pos = n - back
    b.host[3][int(b.table[0, pos // 16]), 0, pos % 16] += 20 << 23
    _reload(b)
    q = queries(new, group, D, torch.bfloat16)
    got = kv4.attention(q, b.cache, b.d_table, b.d_lens, _i32([0, new])).cpu().double()
    want, tol = _sharp(b, q)
    over = (got - want).abs() / tol
    assert over.max() <= 1, f"worst {over.max():.3f} of the tolerance"
    quiet = torch.arange(n - new, n) < pos
    if quiet.any():
        assert (tol[quiet].mean() < 0.05 * want[quiet].abs().mean()) and want[quiet].abs().max() < 50
