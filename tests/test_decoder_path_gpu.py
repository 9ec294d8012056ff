"""From the residual stream to tokens' probabilities, as a decoder's end runs it: norm to INT8 rows and an INT8 layer, the
residual's addition and norm, a rotated 4-bit layer, a 4-bit vocabulary layer, log-probabilities.  Eager and captured."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F16 = torch.float16
HIDDEN, FFN, VOCAB = 512, 1024, 5003


class Model:
    def __init__(self):
        from llm_accelerator_b200 import gemm, mxfp4, ptq, quarot
        g = torch.Generator().manual_seed(0)

        def weight(n, k):
            return torch.randn((n, k), generator=g).cuda() * k ** -0.5
        self.w1 = (1 + 0.1 * torch.randn(HIDDEN, generator=g)).half().cuda()
        self.w2 = (1 + 0.1 * torch.randn(HIDDEN, generator=g)).half().cuda()
        q, s = ptq.quantize_tensor(weight(HIDDEN, HIDDEN))
        self.proj = gemm.pad_k16(q), s
        self.up = mxfp4.quantize(weight(FFN, HIDDEN))
        self.down_f = quarot.fwht_f16(weight(HIDDEN, FFN).half(), 256)          # input columns rotated
        self.down = mxfp4.quantize(self.down_f)
        self.head = mxfp4.quantize(weight(VOCAB, HIDDEN))

    def run(self, x, residual, tokens, top=5):
        from llm_accelerator_b200 import gemm, logprobs, mxfp4, norm, quarot
        q, s, h = norm.rms_norm_i8(x, self.w1, 1e-5, residual=residual)
        y = gemm.gemm_i8_scaled(q, self.proj[0], s, self.proj[1])
        y, h = norm.rms_norm(y, self.w2, 1e-5, residual=h, residual_out=h)
        a = torch.relu(mxfp4.linear(y, self.up))
        y = mxfp4.linear(quarot.fwht_f16(a, 256), self.down)
        logits = mxfp4.linear(norm.rms_norm(y, self.w2, 1e-5, residual=h)[0], self.head)
        return (q, s, h, a, y, logits, *logprobs.token_logprobs(logits, tokens, top))


def _inputs(M, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((M, HIDDEN), generator=g).half().cuda(), torch.randn((M, HIDDEN), generator=g).half().cuda(), \
        torch.randint(0, VOCAB, (M,), generator=g).cuda()


@pytest.mark.parametrize("M", [1, 7, 64, 333])
def test_the_whole_path_against_its_formulas(M):
    """Each step from what the one before it gave, in 64 bits: errors do not add up along the path."""
    from llm_accelerator_b200 import quarot
    from mxfp4_helpers import quantise, values
    model = Model()
    x, r, tokens = _inputs(M, M)
    q, s, h, a, y, logits, lp, entropy, top_lp, ids = model.run(x, r, tokens)

    def through(t):
        return values(*quantise(t), t.shape[1]).cuda()
    first = q.double() * s.double()[:, None]
    t = first @ (model.proj[0].double() * model.proj[1].double()[:, None]).t()
    # INT8 sums are exact; the result is rounded to FP16 and added to h1 = x + r, which is rounded too
    y1 = t.half()
    h1 = (x.double() + r.double()).half()
    want_h = y1.double() + h1.double()
    # t's float32 epilogue may round to the other neighbour: a step of FP16 and half a step of h
    assert float(((h.double() - want_h).abs() - 2.0 ** -10 * t.abs() - 2.0 ** -11 * want_h.abs()).max()) <= 2.0 ** -24
    rotated = quarot.fwht_f16(a, 256)
    want = through(rotated) @ model.down.values().double().t()
    room = (FFN / 32 + 4) * 2.0 ** -23 * (through(rotated).abs() @ model.down.values().double().abs().t())
    assert bool(((y.double() - want).abs() <= room + 2.0 ** -11 * (want.abs() + room) + 2.0 ** -25).all())
    z = logits.double()
    logp = z - torch.logsumexp(z, 1, keepdim=True)
    assert float((lp.double() - logp.gather(1, tokens[:, None])[:, 0]).abs().max()) < 1e-4
    assert float((entropy.double() + (logp.exp() * logp).sum(1)).abs().max()) < 1e-3
    assert torch.equal(ids.long(), torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :5])


def test_a_captured_step_follows_its_inputs_and_two_streams_do_not_meet():
    model = Model()
    x, r, tokens = _inputs(24, 5)
    want = model.run(x, r.clone(), tokens)
    a, b, t = torch.zeros_like(x), torch.zeros_like(r), torch.zeros_like(tokens)
    model.run(a, b, t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = model.run(a, b, t)
    for _ in range(2):
        a.copy_(x)
        b.copy_(r)
        t.copy_(tokens)
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(12):
        st = streams[i % 3]
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append(model.run(x, r, tokens))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, want))
