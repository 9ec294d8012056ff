"""The front ends' C++ side answers usual calls as the Python side does, and gives None for all others."""
from __future__ import annotations

import pytest
import torch

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def test_unusual_arguments_are_left_to_python():
    from llm_accelerator_b200._tensors import front
    x = torch.ones((2, 8), dtype=F16)
    for args in ((), (1,), (x,), (x, x[0], 1e-6, None), (None, None, 1e-6, None), (x, x[0], 1e-6, x, x)):
        assert front.rms_norm(*args) is None and front.rms_norm_i8(*args) is None
    for args in ((), (x, x[:, 0], None, F32), (x, x[:, 0], None, "float32"), (1, 2, 3, 4)):
        assert front.dequantize_rows(*args) is None
    for args in ((), (1,), (x,), ([x],)):
        assert front.quantize(*args) is None
    for args in ((), (x, x[:, 0], 1), (x, None, 1), (x, x[:, 0], 1.5)):
        assert front.token_logprobs(*args) is None
    for args in ((), (x, (16, 16), 2, 8, 0, None), (x, None, 2, 8, 0, None), (x, (16, 16), "2", 8, 0, None)):
        assert front.linear(*args) is None
    for args in ((), ((0, 16), 2, 8, 0, F16), ((16,), 2, 8, 0, F16), ((16, 16), 0, 8, 0, F16), ((16, 16), 2, 8, -1, F16),
                 ((16, 16), 2 ** 40, 8, 0, F16), ((16, 16), 2, 2 ** 70, 0, F16)):
        assert front.values(*args) is None
        assert front.gemm(*args[:4], *args[:4], None, F16) is None


def _same(a, b):
    a, b = (t if isinstance(t, tuple) else (t,) for t in (a, b))
    assert len(a) == len(b)
    for s, t in zip(a, b):
        assert s.dtype == t.dtype and s.shape == t.shape and s.stride() == t.stride() and torch.equal(s, t)


class _Silent:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,K,pad", [(1, 1024, 0), (3, 77, 5), (70, 256, 8)])
def test_usual_calls_are_answered_alike(M, K, pad, dtype, monkeypatch):
    from llm_accelerator_b200 import logprobs, mxfp4, norm, ptq
    from llm_accelerator_b200._tensors import front
    g = torch.Generator().manual_seed(M + K)
    x, r = ((torch.randn((M, K + pad), generator=g)).to(dtype).cuda()[:, :K] for _ in range(2))
    w, bias = torch.rand(K, generator=g).cuda(), torch.randn(40, generator=g).to(dtype).cuda()
    weights = mxfp4.quantize(torch.randn((40, K), generator=g).cuda())
    tokens = torch.randint(0, K, (M,), generator=g).cuda()
    assert front.rms_norm(x, w, 1e-6, None) is not None and front.quantize(x) is not None
    assert front.token_logprobs(x, tokens, 5) is not None
    assert front.linear(x, weights._pointers, weights.rows, weights.cols, weights._index, bias) is not None

    def calls():
        q = mxfp4.quantize(x)
        codes, scale, h = norm.rms_norm_i8(x, w, 1e-6, residual=r)
        return [norm.rms_norm(x, w, 1e-6), norm.rms_norm(x, w, 1e-6, residual=r), norm.rms_norm_i8(x, w, 1e-6), (codes, scale, h),
                ptq.dequantize_rows(codes, scale, K, dtype), ptq.dequantize_rows(codes, scale), (q.codes, q.values(dtype)),
                q.values(), mxfp4.linear(x, weights, bias=bias), mxfp4.linear(x, weights), mxfp4.gemm(q, weights, bias, dtype),
                mxfp4.gemm(q, weights), logprobs.token_logprobs(x, tokens), logprobs.token_logprobs(x, tokens.int(), 7),
                (q.scale_bytes(), torch.tensor([q.rows, q.cols, q._index, *(p % 16 for p in q._pointers)]))]

    fast = calls()
    for module in (norm, ptq, mxfp4, logprobs):
        monkeypatch.setattr(module, "front", _Silent())
    for a, b in zip(fast, calls()):
        _same(a, b)


@pytest.mark.gpu
def test_tensors_without_memory_and_threads():
    from concurrent.futures import ThreadPoolExecutor

    from llm_accelerator_b200 import norm
    from llm_accelerator_b200.errors import EngineError
    w, freed = torch.ones(64, device="cuda"), torch.ones((4, 64), device="cuda")
    freed.untyped_storage().resize_(0)                 # a null address, which the library refuses
    with pytest.raises(EngineError):
        norm.rms_norm(freed, w)
    x = torch.randn((4, 64), generator=torch.Generator().manual_seed(1)).cuda()
    want = norm.rms_norm(x, w)
    with ThreadPoolExecutor(4) as pool:                # the interpreter's lock has been taken back
        assert all(torch.equal(y, want) for y in pool.map(lambda _: norm.rms_norm(x, w), range(200)))


@pytest.mark.gpu
def test_refusals_are_those_of_python():
    from llm_accelerator_b200 import logprobs, mxfp4, norm, ptq
    x, w = torch.ones((4, 64), dtype=F16, device="cuda"), torch.ones(64, device="cuda")
    weights = mxfp4.quantize(x)
    with pytest.raises(TypeError):
        norm.rms_norm(x.double(), w)
    with pytest.raises(ValueError):
        norm.rms_norm(x, w[:32])
    with pytest.raises(ValueError):
        norm.rms_norm_i8(x, w, -1.0)
    with pytest.raises(ValueError):
        norm.rms_norm(x.t(), torch.ones(4, device="cuda"))
    with pytest.raises(ValueError):
        norm.rms_norm(x, w, residual=x[:2])
    with pytest.raises(TypeError):
        norm.rms_norm(x, w, residual=x.float())
    with pytest.raises(ValueError):
        mxfp4.linear(x[:, :32], weights)
    with pytest.raises(ValueError):
        mxfp4.linear(x, weights, bias=w[:3])
    with pytest.raises(ValueError):
        mxfp4.gemm(mxfp4.quantize(x[:, :32].contiguous()), weights)
    with pytest.raises(TypeError):
        mxfp4.gemm(weights, weights, out_dtype=torch.int8)
    with pytest.raises(ValueError):
        logprobs.token_logprobs(x, torch.zeros(4, dtype=torch.int64, device="cuda"), top=33)
    with pytest.raises(TypeError):
        logprobs.token_logprobs(x, torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError):
        ptq.dequantize_rows(torch.zeros((2, 32), dtype=torch.int8, device="cuda"), torch.ones(2, device="cuda"), 8)
    for empty in (x[:0], x[:0, :32]):
        assert norm.rms_norm(empty, w[: empty.shape[1]]).shape == empty.shape
