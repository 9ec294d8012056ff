"""Sizes of the INT8 linear layer that take paths of their own: the row quantiser's four-warp form (K above 2048) and
its padding columns, the product's ring of weights when it goes round, on the GPU against the definition in 64 bits
(tests/test_w8a8_gpu.py derives the tolerances)."""
from __future__ import annotations

import pytest
import torch

from llm_accelerator_b200 import _lib as L
from test_w8a8_gpu import _check, _quant_rows_cpu

pytestmark = pytest.mark.gpu
HALF = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,K", [(40, 4096), (300, 8192), (20, 2056), (70, 776), (17, 2048), (33, 8184), (5, 4104)])
def test_rows_of_whole_chunks(M, K, dtype):
    """16-byte chunks; K of 8 more than a multiple of 16 leaves padding columns."""
    from llm_accelerator_b200 import gemm, ptq
    g = torch.Generator().manual_seed(M + K)
    x = (torch.randn((M, K), generator=g) * torch.logspace(-5, 3, M)[:, None]).to(dtype).cuda()
    x[M // 2] = 0
    q, s = ptq.quantize_rows(x)
    wq, ws = _quant_rows_cpu(x)
    assert q.shape == (M, -(-K // 16) * 16) and torch.equal(s.cpu(), ws)
    assert torch.equal(q.cpu()[:, :K], wq) and not q[:, K:].any()
    N = 300
    Bt = gemm.pad_k16(torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)).cuda()
    sb, bias = torch.rand(N, generator=g).cuda() * 1e-3, torch.randn(N, generator=g).to(dtype).cuda()
    x = torch.randn((M, K), generator=g).to(dtype).cuda()
    wq, ws = _quant_rows_cpu(x)
    _check(gemm.linear_w8a8(x, Bt, sb, bias=bias), wq, Bt, ws, sb, bias)
    bad = x.clone()
    bad[M // 3, K - 1] = float("nan")
    got = gemm.linear_w8a8(bad, Bt, sb, bias=bias)
    keep = torch.arange(M, device="cuda") != M // 3
    assert got[M // 3].isnan().all() and torch.equal(got[keep], gemm.linear_w8a8(x, Bt, sb, bias=bias)[keep])
    assert L.lib.tac_gemm_status(None) == L.OK


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,N,K", [(1, 5000, 8192), (16, 5000, 4096), (1, 12000, 4096), (7, 12000, 8192), (2, 30000, 4096),
                                   (16, 30000, 8192), (40, 9000, 4096), (100, 30000, 2048)])
def test_weights_in_more_stages_than_the_ring_has(M, N, K, dtype):
    """40 to 235 channel tiles, so that a CTA takes 16 to 64 K blocks through its 4 to 8 stages."""
    from llm_accelerator_b200 import gemm
    g = torch.Generator(device="cuda").manual_seed(N + K)
    x = torch.randn((M, K), generator=g, device="cuda").to(dtype)
    Bt = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8, device="cuda")
    sb = torch.rand(N, generator=g, device="cuda") * 1e-3
    y = gemm.linear_w8a8(x, Bt, sb)
    q, s = _quant_rows_cpu(x)
    for n in range(0, N, 4096):                       # in parts: the definition is in float64
        _check(y[:, n:n + 4096], q, Bt[n:n + 4096], s, sb[n:n + 4096], None)
    assert L.lib.tac_gemm_status(None) == L.OK
