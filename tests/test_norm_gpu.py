"""The root-mean-square norm, its INT8 form and the values of INT8 rows, against their formulas in 64 bits."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
SMALLEST = {F16: 2.0 ** -24, BF16: 2.0 ** -133, F32: 2.0 ** -149}    # steps of subnormal values
ULP = 2.0 ** -24                                                      # half a step of float32

# Roundings of float32 between h and y: the square sum (at most 128 terms one after the other, 5 exchanges, 32 warps; halved
# by the root), mean, eps, root, h itself and two products.
NORM = ((128 + 5 + 32) / 2 + 8) * ULP


def _inputs(M, K, dtype, wtype, seed, pad=0, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((M, K + pad), generator=g) * (torch.rand((M, 1), generator=g) + 0.2)
    r = torch.randn((M, K + pad), generator=g) * 3
    w = 1 + 0.3 * torch.randn(K, generator=g)
    x, r = x.to(dtype).cuda()[:, :K], r.to(dtype).cuda()[:, :K]
    return x, (r if residual else None), w.to(wtype).cuda()


def _exact(x, r, w, eps):
    h = x.double() + (0 if r is None else r.double())
    return h, h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * w.double()


def _near(got, want, rel, dtype):
    """Rounded once to dtype after relative errors `rel` in float32."""
    d = (got.double() - want).abs()
    room = want.abs() * (torch.finfo(dtype).eps / 2 * (1 + rel) + rel) + SMALLEST[dtype]
    assert bool((d <= room).all()), float((d / room).max())


# one warp to sixteen a row; rows that begin and end anywhere; too long for registers
SHAPES = [(1, 1, 0), (3, 7, 0), (5, 32, 0), (4, 512, 0), (7, 1024, 8), (9, 1032, 0), (33, 4096, 0), (6, 4096, 5),
          (3, 8192, 0), (2, 16384, 16), (5, 1000, 3), (4, 4097, 0), (2, 16383, 0), (2, 20001, 0), (300, 768, 0)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,K,pad", SHAPES)
def test_rms_norm(M, K, pad, dtype):
    from llm_accelerator_b200 import norm
    for residual in (False, True):
        x, r, w = _inputs(M, K, dtype, dtype, M + K, pad, residual)
        h, y = _exact(x, r, w, 1e-5)
        got = norm.rms_norm(x, w, 1e-5, residual=r)
        if residual:
            got, new = got
            _near(new, h, ULP, dtype)
        _near(got, y, NORM, dtype)


def _check_i8(q, scale, y, K, rel=NORM):
    top = y.abs().amax(1).clamp(min=1e-8)
    assert bool(((scale.double() - top / 127).abs() <= top / 127 * (rel + 2 * ULP)).all())
    want = y / (top / 127)[:, None]
    # half a step of rounding, and the relative errors of y and of 127 / t
    assert float((q[:, :K].double() - want).abs().max()) <= 0.5 + 127 * (2 * rel + 4 * ULP)
    assert q.shape[1] % 16 == 0 and not q[:, K:].any()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,K,pad", SHAPES)
def test_rms_norm_i8(M, K, pad, dtype):
    from llm_accelerator_b200 import norm
    for residual in (False, True):
        x, r, w = _inputs(M, K, dtype, dtype, M * 3 + K, pad, residual)
        h, y = _exact(x, r, w, 1e-6)
        q, scale, *new = norm.rms_norm_i8(x, w, residual=r)
        _check_i8(q, scale, y, K)
        if residual:
            _near(new[0], h, ULP, dtype)


@pytest.mark.parametrize("wtype", [F16, BF16, F32])
def test_weights_of_another_type_or_alignment(wtype):
    from llm_accelerator_b200 import norm
    x, r, _ = _inputs(6, 2048, F16, F16, 4)
    w = (1 + torch.arange(2049) / 4096).to(wtype).cuda()[1:]
    _, y = _exact(x, r, w, 1e-6)
    _near(norm.rms_norm(x, w, residual=r)[0], y, NORM, F16)
    q, s, _ = norm.rms_norm_i8(x, w, residual=r)
    _check_i8(q, s, y, 2048)


@pytest.mark.parametrize("K", [768, 1001, 20001])
@pytest.mark.parametrize("over", ["residual", "x"])
def test_the_new_residual_may_lie_over_an_input(K, over):
    from llm_accelerator_b200 import norm
    x, r, w = _inputs(40, K, BF16, BF16, 5, pad=7)
    want_h = norm.rms_norm(x, w, residual=r)[1]
    _, y = _exact(x, r, w, 1e-6)
    for f in (norm.rms_norm, norm.rms_norm_i8):
        # the copies are aligned otherwise than the slices: their sums may run in another order
        a, b = x.clone(), r.clone()
        *got, h = f(a, w, residual=b, residual_out=b if over == "residual" else a)
        assert h is (b if over == "residual" else a) and torch.equal(h, want_h)
        if f is norm.rms_norm:
            _near(got[0], y, NORM, BF16)
        else:
            _check_i8(*got, y, K)


@pytest.mark.parametrize("K", [1024, 1001, 20001])
def test_the_result_may_lie_over_an_input(K):
    from llm_accelerator_b200 import norm
    x, r, w = _inputs(30, K, F16, F16, 12)
    want, _ = norm.rms_norm(x, w, residual=r)
    for over in range(2):
        a, b = x.clone(), r.clone()
        y, _ = norm.rms_norm(a, w, residual=b, out=(a, b)[over])
        assert torch.equal(y, want)


def test_rows_without_finite_values_stay_among_themselves():
    from llm_accelerator_b200 import norm
    for K in (64, 777, 4096, 17000):
        x, _, w = _inputs(6, K, F16, F16, 6, residual=False)
        clean = norm.rms_norm(x, w)
        x[1, K // 2] = float("nan")
        x[3, 5] = float("inf")
        x[4] = 0
        y = norm.rms_norm(x, w)
        q, s = norm.rms_norm_i8(x, w)
        assert torch.equal(y[[0, 2, 5]], clean[[0, 2, 5]])
        assert y[1].isnan().all()
        assert y[3, 5].isnan() and (y[3, :5] == 0).all() and (y[3, 6:] == 0).all()
        assert not y[4].any() and not q[4].any() and float(s[4]) == pytest.approx(1e-8 / 127, rel=1e-6)
        assert s[[1, 3]].isnan().all() and not q[[1, 3]].any() and s[[0, 2, 4, 5]].isfinite().all()


def test_out_and_empty_batches():
    from llm_accelerator_b200 import norm
    x, r, w = _inputs(5, 256, F16, F16, 7)
    out = torch.full((5, 256), 9.0, dtype=F16, device="cuda")
    y, h = norm.rms_norm(x, w, residual=r, out=out)
    assert y is out and torch.equal(y, norm.rms_norm(x, w, residual=r)[0])
    y, h = norm.rms_norm(x[:0], w, residual=r[:0])
    assert y.shape == h.shape == (0, 256)
    q, s, h = norm.rms_norm_i8(x[:0], w, residual=r[:0])
    assert q.shape == (0, 256) and s.shape == (0,)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 16), (5, 40), (70, 4096), (9, 5001), (2, 20000)])
def test_dequantize_rows(M, K, dtype):
    from llm_accelerator_b200 import ptq
    g = torch.Generator().manual_seed(K)
    q = torch.randint(-128, 128, (M, -(-K // 16) * 16), generator=g).to(torch.int8).cuda()
    s = torch.rand(M, generator=g).cuda()
    assert torch.equal(ptq.dequantize_rows(q, s, K, dtype), (q[:, :K].float() * s[:, None]).to(dtype))
    assert ptq.dequantize_rows(q[:0], s[:0]).shape == (0, q.shape[1])


def test_codes_feed_the_int8_product():
    from llm_accelerator_b200 import gemm, norm, ptq
    x, r, w = _inputs(37, 1000, F16, F16, 8)
    q, s, _ = norm.rms_norm_i8(x, w, residual=r)
    W = torch.randn((256, 1000), generator=torch.Generator().manual_seed(3)).cuda()
    Bt, bs = ptq.quantize_tensor(W)
    y = gemm.gemm_i8_scaled(q, gemm.pad_k16(Bt), s, bs, out_dtype=F32)
    want = (ptq.dequantize_rows(q, s, 1000).double() @ (Bt.double() * bs.double()[:, None]).t())
    # int32 sums are exact; three roundings behind them
    scale = (q[:, :1000].double() @ Bt.double().t()).abs() * s.double()[:, None] * bs.double()[None, :]
    assert bool(((y.double() - want).abs() <= scale * 4 * ULP + 1000 * 127 * 127 * 1e-12).all())


def test_another_stream_and_a_captured_call():
    from llm_accelerator_b200 import norm
    x, r, w = _inputs(64, 1024, BF16, BF16, 9)
    want, want_h = norm.rms_norm(x, w, residual=r)
    a, b = torch.zeros_like(x), torch.zeros_like(r)
    norm.rms_norm(a, w, residual=b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = norm.rms_norm(a, w, residual=b)
        q, s, _ = norm.rms_norm_i8(a, w, residual=b)
    a.copy_(x)
    b.copy_(r)
    graph.replay()
    assert torch.equal(y, want) and torch.equal(h, want_h)
    q0, s0, _ = norm.rms_norm_i8(x, w, residual=r)
    assert torch.equal(q, q0) and torch.equal(s, s0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y2, _ = norm.rms_norm(x, w, residual=r)
    stream.synchronize()
    assert torch.equal(y2, want)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,K,pad", [(3, 8544, 128), (2, 8543, 0), (5, 13548, 5), (160, 4095, 1), (4, 2047, 0), (2, 16381, 7), (3, 40004, 4)])
def test_wide_rows_at_any_alignment(M, K, pad, dtype):
    """Shares of a row that end inside, at and behind its last 16 bytes, for weights of either size and alignment."""
    from llm_accelerator_b200 import norm
    for wtype, shift in ((dtype, 0), (F32, 1), (BF16, 1)):
        x, r, w = _inputs(M, K, dtype, wtype, M + K, pad, True)
        if shift:
            w = torch.cat([w[:1], w])[1:]
        h, y = _exact(x, r, w, 1e-5)
        got, new = norm.rms_norm(x, w, 1e-5, residual=r)
        _near(new, h, ULP, dtype)
        _near(got, y, NORM, dtype)
        q, scale, same = norm.rms_norm_i8(x, w, 1e-5, residual=r)
        assert torch.equal(same, new)
        _check_i8(q, scale, y, K)
