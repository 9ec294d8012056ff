"""linear_w8a8 of up to 16 rows in one launch (rows quantised inside), which every such call without a workspace takes,
against the same layer in two calls.

Both quantise by the same float32 formula, sum integers and share their epilogue, so results are equal bit for bit;
tests/test_w8a8_gpu.py holds the two calls against the definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

from llm_accelerator_b200 import _lib as L

pytestmark = pytest.mark.gpu


def _two_calls(x, Bt, sb, bias=None):
    from llm_accelerator_b200 import gemm, ptq
    q, s = ptq.quantize_rows(x)
    return gemm.gemm_i8_scaled(q, Bt, s, sb, bias=bias, out_dtype=x.dtype)


def _one_launch(x, Bt, sb, bias=None):
    """A workspace too small to use: the rows are quantised in the product."""
    from llm_accelerator_b200 import gemm
    return gemm.linear_w8a8(x, Bt, sb, bias=bias, ws=torch.empty(0, dtype=torch.uint8, device="cuda"))


def _weights(N, K, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    Bt = torch.randint(-127, 128, (N, -(-K // 16) * 16), generator=g, dtype=torch.int8, device="cuda")
    return Bt, torch.rand(N, generator=g, device="cuda") * 1e-3 + 1e-4


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 100), (3, 100), (3, 250), (16, 17), (15, 255), (16, 128)])
def test_the_largest_value_at_every_column(M, K, dtype):
    """The row's maximum in each lane's chunk in turn: rows whose last chunks are ragged, warps with half their lanes."""
    Bt, sb = _weights(130, K)
    base = torch.randn((M, K + 1), device="cuda").to(dtype)
    for off in (0, 1):                                # rows with and without whole 16-byte chunks
        for c in range(K):
            x = base.clone()[:, off:off + K]
            x[torch.arange(M), (c + 37 * torch.arange(M)) % K] = -50.0
            assert torch.equal(_one_launch(x, Bt, sb), _two_calls(x, Bt, sb))
    assert L.lib.tac_gemm_status(None) == L.OK


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 130, 600), (1, 4096, 1024), (3, 300, 2000), (5, 129, 1025), (16, 1000, 4096),
                                   (16, 4700, 1500), (7, 256, 8192), (2, 9472, 1024)])
def test_rows_shared_by_a_cluster(M, N, K, dtype):
    """K split over 2, 4 and 8 CTAs, the largest value in each CTA's share in turn, call after call, beside a kernel that
    keeps other SMs busy (CTAs of a cluster then start at different times)."""
    Bt, sb = _weights(N, K, N + K)
    bias = torch.randn(N, device="cuda").to(dtype)
    x = torch.randn((M, K), device="cuda").to(dtype)
    side, load = torch.cuda.Stream(), torch.randn((2048, 2048), device="cuda")
    rows = torch.arange(M)
    want, got = [], []
    for i in range(24):
        y = x.clone()
        y[rows, (i * K // 24 + 131 * rows) % K] = 40.0 + i
        want.append((y, _two_calls(y, Bt, sb, bias)))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(8):
            load = (load @ load).clamp_(-1, 1)
    for y, _ in want:
        got.append(_one_launch(y, Bt, sb, bias))
    torch.cuda.synchronize()
    for g, (_, w) in zip(got, want):
        assert torch.equal(g, w)
    assert L.lib.tac_gemm_status(None) == L.OK


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("N", [9472, 9473, 10240, 18944, 18945])
@pytest.mark.parametrize("K", [6016, 6017, 6032, 7168, 8192])
def test_long_rows_over_every_number_of_channel_tiles(N, K, dtype):
    """74 to 149 channel tiles: CTAs that hold rows of up to 64 K blocks beside their ring of weights."""
    Bt, sb = _weights(N, K)
    for M in (1, 16):
        x = torch.randn((M, K), device="cuda").to(dtype)
        assert torch.equal(_one_launch(x, Bt, sb), _two_calls(x, Bt, sb))
    assert L.lib.tac_gemm_status(None) == L.OK


def test_a_workspace_is_used_where_two_launches_are_faster():
    best, least = L.lib.tac_linear_w8a8_best_workspace_bytes, L.lib.tac_linear_w8a8_workspace_bytes
    assert best(1, 4096, 1024) == 0 and best(2, 28672, 1024) == 0 and best(1, 4096, 8192) == 0
    for M, N, K in ((16, 28672, 8192), (16, 4096, 4096), (1, 10240, 8192), (1, 28672, 4096)):
        assert best(M, N, K) >= M * K + 4 * M and least(M, K) == 0
    assert best(40, 300, 1000) == least(40, 1000) > 0 and best(0, 5, 5) == best(5, 0, 5) == best(5, 5, 0) == 0


@pytest.mark.parametrize("M,N,K", [(1, 4096, 1024), (16, 4096, 1024), (7, 1000, 8192), (16, 10240, 4096), (3, 20000, 1000)])
def test_every_workspace_gives_the_same_result(M, N, K):
    """None, one of another call's sizes, too small, misplaced for all but one launch; captured and replayed."""
    from llm_accelerator_b200 import gemm
    Bt, sb = _weights(N, K)
    x = torch.randn((M, K), device="cuda").bfloat16()
    want = _two_calls(x, Bt, sb)
    big, small = gemm.linear_workspace(M, K), torch.empty(100, dtype=torch.uint8, device="cuda")
    for ws in (None, big, big[1:], small, gemm.linear_workspace(M + 9, K + 77)):
        assert torch.equal(gemm.linear_w8a8(x, Bt, sb, ws=ws), want)
    n = big.numel() - 256 - (-big.data_ptr() & 255)
    out = torch.empty_like(want)
    for p, size in ((None, 0), (big.data_ptr(), n), (big.data_ptr() + 16, n)):      # the last is not on a boundary
        out.zero_()
        torch.cuda.synchronize()
        assert L.lib.tac_linear_w8a8(x.data_ptr(), L.TYPE_BF16, K, Bt.data_ptr(), sb.data_ptr(), L.TYPE_F32, None, 0,
                                     out.data_ptr(), L.TYPE_BF16, p, size, M, N, K, None) == L.OK
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gemm.linear_w8a8(x, Bt, sb)
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, -want)
    assert L.lib.tac_gemm_status(None) == L.OK
