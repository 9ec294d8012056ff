"""Log-probabilities, entropy and the likeliest tokens against the softmax in 64 bits."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
ULP = 2.0 ** -24
INF = float("inf")


def _tolerance(V):
    """Absolute error of ln S: V / 256 terms one after the other in a thread at most (one CTA a row), 40 joins of sums, each
    term's exponential (2^-22) and the rounding of its argument (relative, of magnitudes whose weighted mean is below 2^5)."""
    return (V / 256 + 16 + 40 * 3 + 4 + 64) * ULP


def _want(x, tokens, top):
    x = x.double().cpu()
    x = x - x.amax(1, keepdim=True)     # next to values of 10^38, ln S is below even a step of float64
    tokens = tokens.long().cpu()
    logp = x - torch.logsumexp(x, 1, keepdim=True)
    p = logp.exp()
    entropy = -torch.special.xlogy(p, p).sum(1)
    inside = (tokens >= 0) & (tokens < x.shape[1])
    lp = logp.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    lp[~inside] = float("nan")
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return lp, entropy, logp.gather(1, ids), ids


def _check(x, tokens, top):
    from llm_accelerator_b200 import logprobs
    got = logprobs.token_logprobs(x, tokens, top=top)
    assert len(got) == (4 if top else 2)
    lp, entropy, top_lp, ids = _want(x, tokens, top)
    tol = _tolerance(x.shape[1])

    def near(a, b):
        a, b = a.double().cpu(), b.float().double()    # past float32's range, as the difference of its ends, it is -inf
        same = (a == b) | (a.isnan() & b.isnan())
        fine = a.isfinite() & b.isfinite() & ((a - b).abs() <= tol + b.abs() * 4 * ULP)
        assert bool((same | fine).all()), (a[~(same | fine)][:4], b[~(same | fine)][:4])

    near(got[0], lp)
    e = got[1].double().cpu()
    # ln S as above; T / S has the relative error of both sums
    ok = (e.isnan() & entropy.isnan()) | ((e - entropy).abs() <= tol * (2 + 2 * entropy.abs()))
    assert bool(ok.all()), (e[~ok][:4], entropy[~ok][:4])
    if top:
        near(got[2], top_lp)
        assert got[3].dtype == torch.int32 and torch.equal(got[3].cpu().long(), ids)
    return got


def _logits(M, V, dtype, seed, pad=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((M, V + pad), generator=g) * spread).to(dtype).cuda()[:, :V], \
        torch.randint(0, V, (M,), generator=g).cuda()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,V,pad,top", [(1, 1, 0, 1), (2, 2, 1, 2), (3, 7, 0, 5), (1, 31, 0, 31), (5, 100, 3, 20), (2, 257, 0, 32),
                                         (3, 2054, 1, 32), (4, 4099, 0, 8), (1, 8192, 0, 20), (2, 16391, 6, 20), (1, 50257, 0, 5),
                                         (7, 50257, 0, 20), (64, 50257, 47, 32), (160, 33000, 0, 3), (700, 1500, 0, 5), (250, 50257, 1, 20), (460, 9001, 3, 7),
                                         (1200, 9001, 0, 32), (1250, 3001, 5, 32),
                                         (1, 262144, 0, 32), (2, 131073, 0, 0)])
def test_against_64_bits(M, V, pad, top, dtype):
    x, tokens = _logits(M, V, dtype, M * 7 + V, pad)
    _check(x, tokens, top)
    _check(x, tokens.int(), min(top, 1))


@pytest.mark.parametrize("start", range(1, 8))
def test_rows_at_every_offset(start):
    """A slice of a buffer that begins anywhere, and an odd stride: ends of a row that no whole 16 bytes cover."""
    for dtype in (F16, F32):
        buf = torch.randn((9, 5003), generator=torch.Generator().manual_seed(start)).to(dtype).cuda()
        x = buf[:, start:start + 4990]
        _check(x, torch.full((9,), 4989, device="cuda"), 20)
        _check(buf[:, start:start + 5], torch.full((9,), 4, device="cuda"), 5)


@pytest.mark.parametrize("M", [2, 600])
@pytest.mark.parametrize("V", [50, 3000, 50257])
def test_masks(M, V):
    """Few unmasked tokens, one, none; masks of the type's lowest value; a masked token asked for."""
    g = torch.Generator().manual_seed(V)
    for dtype in (F16, BF16, F32):
        for keep in (1, 3, 40):
            x = torch.full((M, V), -INF)
            at = torch.randint(0, V, (M, keep), generator=g)
            x.scatter_(1, at, torch.randn((M, keep), generator=g))
            x = x.to(dtype).cuda()
            _check(x, at[:, 0].cuda(), 20)
            _check(x, torch.randint(0, V, (M,), generator=g).cuda(), 5)
    x, tokens = _logits(M, V, F16, 3)
    x[0] = -INF                                    # masked whole
    x[1, : V // 2] = torch.finfo(F16).min
    got = _check(x, tokens, 20)
    assert got[0][0].isnan() and got[1][0].isnan() and got[3][0].tolist() == list(range(20))
    low = torch.full((M, V), torch.finfo(F16).min, dtype=F16, device="cuda")
    _check(low, tokens, 20)                        # a uniform distribution
    low[:, 1::2] = -INF
    _check(low, tokens, 20)


@pytest.mark.parametrize("M,V", [(1, 50257), (5, 300), (700, 9000)])
def test_equal_logits_go_to_the_lowest_index(M, V):
    x = torch.zeros((M, V), dtype=F16, device="cuda")
    tokens = torch.zeros(M, dtype=torch.int64, device="cuda")
    _check(x, tokens, 32)
    x[:, 1::3] = -0.0                              # equal to 0
    _check(x, tokens, 32)
    x[:, ::2] = 1.0
    _check(x, tokens, 32)
    x[:, V - 5:] = 2.0                             # the first five come last
    _check(x, tokens, 32)


@pytest.mark.parametrize("order", ["up", "down"])
@pytest.mark.parametrize("M,V", [(1, 200000), (300, 30000), (2, 5000)])
def test_sorted_rows(M, V, order):
    x = torch.arange(V, dtype=F32).expand(M, V) / V * 8
    x = (x if order == "up" else x.flip(1)).contiguous().cuda()
    _check(x, torch.full((M,), V // 2, device="cuda"), 32)


@pytest.mark.parametrize("M,V", [(1, 1000000), (600, 200000)])
def test_the_largest_values_of_few_threads(M, V):
    """More entries above every bound than are collected at once: 16-byte pieces 0, 32, 64 .. of each 256 are larger, which
    fall to eight threads."""
    M = min(M, 600)
    x = torch.rand((1, V), generator=torch.Generator().manual_seed(1)).cuda()
    piece = torch.arange(V, device="cuda") // 4
    ctas = 8 if M == 1 else 1
    pieces = V // 4
    for r in range(ctas):
        a, b = pieces * r // ctas, pieces * (r + 1) // ctas
        here = (piece >= a) & (piece < b) & ((piece - a) % 32 == 0)
        x[0, here] += 4
    x = x.expand(M, V).contiguous()
    rows = torch.arange(M, device="cuda")
    x[rows, rows] += 1
    from llm_accelerator_b200 import logprobs
    if M == 1:
        _check(x, torch.zeros(M, dtype=torch.int64, device="cuda"), 20)
    else:
        got = logprobs.token_logprobs(x, rows, top=20)
        want = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :20]
        assert torch.equal(got[3].long(), want)
        _check(x[:3].contiguous(), rows[:3], 20)


def test_values_that_are_not_numbers():
    x, tokens = _logits(6, 5000, BF16, 11)
    clean = _check(x, tokens, 8)
    x[1, 100] = float("nan")
    x[3, 4999] = INF
    x[4, 0] = -INF
    from llm_accelerator_b200 import logprobs
    lp, entropy, top_lp, ids = logprobs.token_logprobs(x, tokens, top=8)
    for r in (1, 3):
        assert lp[r].isnan() and entropy[r].isnan() and top_lp[r].isnan().all()
    assert ids[1, 0] == 100 and ids[3, 0] == 4999
    for r in (0, 2, 5):
        assert lp[r] == clean[0][r] and entropy[r] == clean[1][r] and torch.equal(ids[r], clean[3][r])
    x[:] = float("nan")
    assert logprobs.token_logprobs(x, tokens, top=8)[3].tolist() == [list(range(8))] * 6


def test_the_ends_of_float32():
    x = torch.full((2, 3000), -3.4e38, dtype=F32, device="cuda")
    x[:, 7] = 3.4e38
    x[1, 9] = 3.4e38
    got = _check(x, torch.tensor([7, 8], device="cuda"), 3)
    assert got[0].tolist()[0] == 0 and got[1].tolist()[0] == 0
    sure = torch.zeros((1, 50257), dtype=F32, device="cuda")
    sure[0, 5] = 30.0
    _check(sure, torch.tensor([5], device="cuda"), 5)


def test_tokens_outside_the_vocabulary_and_empty_batches():
    from llm_accelerator_b200 import logprobs
    x, _ = _logits(4, 100, F16, 1)
    for t in (torch.int32, torch.int64):
        lp, entropy = logprobs.token_logprobs(x, torch.tensor([-1, 100, 5, -100], dtype=t, device="cuda"))
        assert lp.isnan().tolist() == [True, True, False, True] and entropy.isfinite().all()
    big = torch.tensor([1 << 40, 2, -(1 << 40), 3], device="cuda")
    assert logprobs.token_logprobs(x, big)[0].isnan().tolist() == [True, False, True, False]
    out = logprobs.token_logprobs(x[:0], big[:0], top=3)
    assert [tuple(t.shape) for t in out] == [(0,), (0,), (0, 3), (0, 3)]


def test_results_do_not_depend_on_the_batch_or_the_call():
    from llm_accelerator_b200 import logprobs
    x, tokens = _logits(40, 30011, F16, 5)
    a = logprobs.token_logprobs(x, tokens, top=10)
    b = logprobs.token_logprobs(x, tokens, top=10)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_another_stream_and_a_captured_call():
    from llm_accelerator_b200 import logprobs
    x, tokens = _logits(8, 50257, F16, 6)
    want = logprobs.token_logprobs(x, tokens, top=5)
    a, t = torch.zeros_like(x), torch.zeros_like(tokens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = logprobs.token_logprobs(a, t, top=5)
    a.copy_(x)
    t.copy_(tokens)
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = logprobs.token_logprobs(x, tokens, top=5)
    stream.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_the_batched_runner_gives_them_for_its_step():
    import numpy as np
    from helpers import load_bundle
    from llm_accelerator_b200.runner import BatchedRunner
    r = BatchedRunner(load_bundle("tiny_l2_d128"), 5)
    r.step("prefill", [1, 2, 3, 4, 5], [0] * 5)
    for name in ("prefill", "decode"):
        if name == "decode":
            r.step("decode", [6, 7, 8, 9, 10], [1] * 5)
        vocab = r.logits_count - 3
        logits = torch.from_numpy(np.stack([r.logits(name, s)[:vocab] for s in range(5)]))
        tokens = [0, 1, vocab - 1, 7, 2]
        got = r.token_logprobs(name, tokens, vocab, top=4)
        lp, entropy, top_lp, ids = _want(logits, torch.tensor(tokens), 4)
        tol = _tolerance(vocab)
        assert float((got[0].double().cpu() - lp).abs().max()) <= tol + float(lp.abs().max()) * 4 * ULP
        assert torch.equal(got[3].cpu().long(), ids)
        greedy = torch.zeros(5, dtype=torch.int32, device="cuda")
        r.argmax_async(name, greedy.data_ptr(), vocab, torch.cuda.current_stream().cuda_stream)
        assert torch.equal(greedy, got[3][:, 0])
        again = r.token_logprobs(name, torch.tensor(tokens, dtype=torch.int32, device="cuda"), vocab)
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
    with pytest.raises(ValueError):
        r.token_logprobs("decode", [0] * 5, r.logits_count + 1)
    with pytest.raises(ValueError):
        r.token_logprobs("decode", [0] * 4, 10)


@pytest.mark.parametrize("top", [8, 20, 21, 32])
@pytest.mark.parametrize("V", [33, 100, 255, 500, 776, 900, 1024, 1027, 2048, 3001])
def test_many_of_short_rows(V, top):
    """Rows of a warp each: with fewer of its threads' values than are picked, equal ones, masked ones, all or none."""
    for dtype in (F16, F32):
        x, tokens = _logits(50, V, dtype, V + top, V % 3)
        x = x.clone()
        x[::3] = torch.where(torch.rand((17, V), generator=torch.Generator().manual_seed(V)).cuda() < 1 / 64, x[::3], -INF)
        x[1::6] = x[1::6].round()                  # a few dozen values, many times each
        x[4] = 0.0
        x[7] = torch.arange(V, device="cuda").to(dtype) / 8
        x[10] = -x[7]
        _check(x, tokens, top)


@pytest.mark.parametrize("V", [200, 1000, 5000])
def test_equal_logits_below_zero(V):
    """More of them than a share's list has places for; some rows with a few above and below."""
    for dtype in (F16, BF16, F32):
        x = torch.full((1800, V), -1.5, dtype=dtype, device="cuda")
        x[1::2, 3:V:7] = -2.5
        x[::5, 11:V:97] = -0.5
        _check(x, torch.arange(1800, device="cuda") % V, 32)


def test_rows_of_two_ctas_each():
    """More rows than SMs, long ones."""
    x, tokens = _logits(500, 100003, F16, 5, 1)
    x[::3, ::2] = -INF
    _check(x, tokens, 20)
