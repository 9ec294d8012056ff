"""INT8 linear layers with a scale for each token and output channel, on the
GPU against the definition in 64 bits.

Tolerance.  The integer sums are exact, so a result differs from the
definition by the float32 epilogue (int -> float32, two products and a sum,
each off by at most 2^-24 of its magnitude) and one rounding to the output's
type (half a step: eps / 2 of the value, or half the smallest subnormal):
|y - exact| <= eps/2 |exact| + 4 * 2^-24 * (1 + eps) * (|acc a b| + |bias|) + tiny / 2.
Row quantisation is IEEE float32 arithmetic, so its codes and scales are equal
bit for bit to the same formula on the CPU."""
from __future__ import annotations

import pytest

from llm_accelerator_b200 import _lib as L

pytestmark = pytest.mark.gpu
SMALLEST = {"float16": 2.0 ** -24, "bfloat16": 2.0 ** -133, "float32": 2.0 ** -149}


def _torch():
    import torch
    return torch


def _quant_rows_cpu(x):
    torch = _torch()
    x = x.cpu().float()
    t = x.abs().amax(1).clamp(min=1e-8)
    c = torch.full_like(t, 127.0)
    return torch.round(x * (c / t)[:, None]).to(torch.int8), t / c


def _check(y, A, Bt, a_scale, b_scale, bias):
    torch = _torch()
    K = A.shape[1]
    p = (A.cpu().double() @ Bt.cpu()[:, :K].double().t()) * a_scale.cpu().double()[:, None] * b_scale.cpu().double()
    b = torch.zeros(Bt.shape[0], dtype=torch.float64) if bias is None else bias.cpu().double()
    exact = p + b
    eps = torch.finfo(y.dtype).eps
    tol = eps / 2 * exact.abs() + 4 * 2.0 ** -24 * (1 + eps) * (p.abs() + b.abs()) + SMALLEST[str(y.dtype)[6:]] / 2
    got = y.cpu().double()
    assert torch.isfinite(got).all()
    assert (got - exact).abs().le(tol).all(), f"worst {((got - exact).abs() / tol).max():.3f} of the tolerance"


def _operands(M, N, K, seed, bdt="float32"):
    torch = _torch()
    g = torch.Generator().manual_seed(seed)
    A = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8)
    Bt = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    a_scale = torch.rand(M, generator=g) * 0.02 + 1e-3
    b_scale = (torch.rand(N, generator=g) * 1e-3 + 1e-5).to(getattr(torch, bdt))
    bias = torch.randn(N, generator=g)
    return A.cuda(), Bt.cuda(), a_scale.cuda(), b_scale.cuda(), bias.cuda()


# one token to several token tiles, one channel to several channel tiles, one K block to many, partial tiles of each
SHAPES = [(1, 1, 16), (1, 7, 48), (1, 4096, 1024), (2, 129, 128), (15, 1000, 144), (16, 128, 2048), (17, 64, 64),
          (33, 200, 4096), (64, 257, 400), (65, 384, 1040), (128, 128, 128), (129, 127, 272), (300, 515, 768),
          (513, 640, 256), (1000, 2051, 1024), (2304, 768, 96), (777, 50257, 64)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_i8_scaled(M, N, K, dtype):
    torch = _torch()
    from llm_accelerator_b200 import gemm
    dt = getattr(torch, dtype)
    A, Bt, sa, sb, bias = _operands(M, N, K, M + 3 * N + K, "float16" if N % 2 else "float32")
    for b in (None, bias.to(dt)):
        _check(gemm.gemm_i8_scaled(A, Bt, sa, sb, bias=b, out_dtype=dt), A, Bt, sa, sb, b)
    assert L.lib.tac_gemm_status(None) == L.OK


@pytest.mark.parametrize("M,N", [(1, 33), (40, 300), (400, 1025)])
def test_extreme_codes_and_one_hot_rows(M, N):
    """Sums of the largest codes (127 * 128 * K, beyond 2^24) and one-hot rows, whose sums are single products."""
    torch = _torch()
    from llm_accelerator_b200 import gemm
    K = 4096
    A = torch.full((M, K), -127, dtype=torch.int8, device="cuda")
    Bt = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    assert (gemm.gemm_i8_scaled(A, Bt, *one, out_dtype=torch.float32) == 127 * 128 * K).all()
    A = torch.zeros((M, K), dtype=torch.int8, device="cuda")
    hot = torch.arange(M, device="cuda") * 37 % K
    A[torch.arange(M, device="cuda"), hot] = 1
    Bt = torch.randint(-128, 128, (N, K), dtype=torch.int8, device="cuda")
    assert torch.equal(gemm.gemm_i8_scaled(A, Bt, *one, out_dtype=torch.float32), Bt.float().t()[hot])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 1024), (3, 17), (5, 100), (64, 768), (2, 8195), (7, 20000), (1000, 129)])
def test_quantize_rows_bit_exact(M, K, dtype):
    torch = _torch()
    from llm_accelerator_b200 import ptq
    g = torch.Generator().manual_seed(M * K)
    x = (torch.randn((M, K), generator=g) * torch.logspace(-6, 3, M)[:, None]).to(getattr(torch, dtype)).cuda()
    x[M // 2] = 0
    q, s = ptq.quantize_rows(x)
    wq, ws = _quant_rows_cpu(x)
    assert q.shape == (M, -(-K // 16) * 16) and torch.equal(s.cpu(), ws)
    assert torch.equal(q.cpu()[:, :K], wq) and not q[:, K:].any()


def test_quantize_rows_of_slices():
    """Rows at any stride and offset: columns of a wider tensor."""
    torch = _torch()
    from llm_accelerator_b200 import ptq
    wide = torch.randn((9, 1000), device="cuda").half()
    for o, k in ((0, 512), (8, 512), (1, 511), (3, 90), (999, 1)):
        x = wide[:, o:o + k]
        q, s = ptq.quantize_rows(x)
        wq, ws = _quant_rows_cpu(x)
        assert torch.equal(q.cpu()[:, :k], wq) and torch.equal(s.cpu(), ws)


# (M, K): decode rows, K past one 16-byte group, K that no vector load divides, prompts
LINEAR = [(1, 1024), (1, 33), (1, 1), (3, 8192), (5, 8208), (15, 1000), (4, 768), (16, 4096), (17, 100), (40, 2048), (64, 1023), (130, 768), (600, 1040)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("M,K", LINEAR)
def test_linear_w8a8(M, K, dtype):
    torch = _torch()
    from llm_accelerator_b200 import gemm
    dt = getattr(torch, dtype)
    N = 300 + M % 7
    g = torch.Generator().manual_seed(M + K)
    x = (torch.randn((M, K + 24), generator=g) * 2).to(dt).cuda()[:, 8:8 + K]
    Bt = gemm.pad_k16(torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)).cuda()
    sb = (torch.rand(N, generator=g) * 1e-3 + 1e-4).half().cuda()
    bias = torch.randn(N, generator=g).to(dt).cuda()
    q, s = _quant_rows_cpu(x)
    for b in (None, bias):
        y = gemm.linear_w8a8(x, Bt, sb, bias=b)
        assert y.dtype == dt
        _check(y, q, Bt, s, sb, b)
    # a reused workspace (of larger calls too) and a given output
    ws = gemm.linear_workspace(M + 3, K + 500)
    out = torch.full((M, N), 7.0, dtype=dt, device="cuda")
    assert gemm.linear_w8a8(x, Bt, sb, bias=bias, out=out, ws=ws) is out
    assert torch.equal(out, y)
    assert L.lib.tac_gemm_status(None) == L.OK


@pytest.mark.parametrize("M", [1, 5, 70, 300])
def test_rows_without_a_finite_scale_give_nan_rows_only(M):
    torch = _torch()
    from llm_accelerator_b200 import gemm
    K, N = 200, 130
    x = torch.randn((M, K), device="cuda").half()
    Bt = gemm.pad_k16(torch.randint(-127, 128, (N, K), dtype=torch.int8, device="cuda"))
    sb = torch.full((N,), 1e-3, device="cuda")
    clean = gemm.linear_w8a8(x, Bt, sb)
    for bad in (float("nan"), float("inf"), float("-inf")):
        y = x.clone()
        y[M // 2, K // 3] = bad
        got = gemm.linear_w8a8(y, Bt, sb)
        keep = torch.arange(M, device="cuda") != M // 2
        assert got[M // 2].isnan().all() and torch.equal(got[keep], clean[keep])
    x[M // 2] = 0                    # a row of zeros is a row of zeros
    assert not gemm.linear_w8a8(x, Bt, sb)[M // 2].any()


def test_weights_of_the_offline_quantiser():
    """ptq.quantize_tensor gives the weights and scales that linear_w8a8 takes."""
    torch = _torch()
    from llm_accelerator_b200 import gemm, ptq
    W = torch.randn((96, 300), device="cuda") * 0.05
    x = torch.randn((20, 300), device="cuda").bfloat16()
    Q, s = ptq.quantize_tensor(W)
    Q = gemm.pad_k16(Q)
    q, sx = _quant_rows_cpu(x)
    _check(gemm.linear_w8a8(x, Q, s), q, Q, sx, s, None)


def test_empty_results():
    torch = _torch()
    from llm_accelerator_b200 import gemm, ptq
    z = torch.zeros
    assert gemm.linear_w8a8(z((0, 32), device="cuda").half(), z((5, 32), dtype=torch.int8, device="cuda"),
                            torch.ones(5, device="cuda")).shape == (0, 5)
    assert gemm.gemm_i8_scaled(z((3, 32), dtype=torch.int8, device="cuda"), z((0, 32), dtype=torch.int8, device="cuda"),
                               torch.ones(3, device="cuda"), torch.ones(0, device="cuda")).shape == (3, 0)
    assert ptq.quantize_rows(z((0, 20), device="cuda"))[0].shape == (0, 32)


def test_graph_replay_and_side_streams():
    """Two captured graphs and an eager call, each with its own workspace, on two streams: replays follow the inputs."""
    torch = _torch()
    from llm_accelerator_b200 import gemm
    N, K = 500, 768
    Bt = torch.randint(-127, 128, (N, K), dtype=torch.int8, device="cuda")
    sb = torch.rand(N, device="cuda") * 1e-3
    xs = [torch.randn((m, K), device="cuda").half() for m in (1, 48, 300)]
    ref = [gemm.linear_w8a8(x, Bt, sb) for x in xs]
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(gemm.linear_w8a8(x, Bt, sb))
        graphs.append(g)
    for x in xs:
        x.mul_(-1)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            graphs[0].replay()
            graphs[2].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
            eager = gemm.linear_w8a8(xs[2], Bt, sb)
    torch.cuda.synchronize()
    for o, r in zip(outs, ref):
        assert torch.equal(o, -r)
    assert torch.equal(eager, -ref[2])
