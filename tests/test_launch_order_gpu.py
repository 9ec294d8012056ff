"""Kernels that start while the one before them ends: each still sees what all before it wrote, and writes nothing that they
still read.  Chains without a host wait against the same chains with one behind each call."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _chain(wait, M, N, K, rounds):
    from llm_accelerator_b200 import gemm, logprobs, mxfp4, norm, ptq
    g = torch.Generator(device="cuda").manual_seed(M)
    sync = torch.cuda.synchronize if wait else (lambda: None)
    weight = torch.ones(K, device="cuda").half()
    h = torch.randn((M, K), generator=g, device="cuda").half()
    tokens = torch.randint(0, N, (M,), generator=g, device="cuda")
    ws, out = mxfp4.linear_workspace(M, K), torch.empty((M, N), dtype=torch.float16, device="cuda")
    found = []
    for i in range(rounds):
        W = torch.randn((N, K), generator=g, device="cuda") * K ** -0.5
        x = torch.randn((M, K), generator=g, device="cuda").half()
        sync()
        w = mxfp4.quantize(W)                                     # read by the very next product
        sync()
        y, h = norm.rms_norm(x, weight, residual=h, residual_out=h)       # in place, call after call
        sync()
        mxfp4.linear(y, w, ws=ws, out=out)                        # one workspace and one result
        sync()
        lp = logprobs.token_logprobs(out, tokens, top=3)
        sync()
        q, s, h = norm.rms_norm_i8(y, weight, residual=h, residual_out=h)
        sync()
        v = ptq.dequantize_rows(q, s, K, torch.float16)
        sync()
        z = gemm.gemm_i8_scaled(q, gemm.pad_k16(q[:, :K].contiguous()), s, s)
        sync()
        back = mxfp4.quantize(v).values(torch.float16)
        sync()
        found += [h.clone(), *lp, s, z, back, mxfp4.gemm(mxfp4.quantize(back), w)]
        sync()
    return found


@pytest.mark.parametrize("M,N,K", [(1, 4096, 1024), (3, 301, 96), (40, 2048, 2048), (64, 5001, 512), (300, 3000, 768), (1100, 2500, 264)])
def test_chains(M, N, K):
    want = _chain(True, M, N, K, 6)
    for _ in range(3):
        got = _chain(False, M, N, K, 6)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # captured: the same kernels with programmatic edges
    from llm_accelerator_b200 import mxfp4, norm
    x = torch.randn((M, K), device="cuda").half()
    W = mxfp4.quantize(torch.randn((N, K), device="cuda"))
    D = mxfp4.quantize(torch.randn((K, N), device="cuda") * 0.01)
    one = torch.ones(K, device="cuda").half()

    def steps(a):
        for _ in range(4):
            y = mxfp4.linear(norm.rms_norm(a, one), W)
            a = norm.rms_norm(mxfp4.linear(y, D), one, residual=a)[1]
        return a
    want = steps(x)
    torch.cuda.synchronize()
    b = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = steps(b)
    for _ in range(3):
        b.copy_(x)
        graph.replay()
        assert torch.equal(got, want)
        b.zero_()
        graph.replay()
