"""Operators between the residual stream and a token's probability, as cases that can be timed and checked.

Three groups that a quantised decoder runs one after the other:

  norm       h = x + r, y = h / sqrt(mean(h^2) + eps) * w: as floating-point rows, or quantised to int8 with a scale for
             each row (t = max(max |y|, 1e-8), scale = t / 127, code = rint(y * (127 / t))), returned as the values that
             the codes stand for
  mxfp4      blocks of 32 values along K with one power of two each: e = floor(log2 max |x|) - 2, codes the nearest of
             0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (ties to the even code, at most 6), values code * 2^e.  quant: rows
             to that form and back; linear: floating-point rows times weights of that form; gemm: both of that form
  logprobs   of rows of logits: the log-probability of a given token, the entropy, and the k likeliest tokens with their
             log-probabilities (ties to the lowest index)

`run` computes the plain form where `own` is false and calls llm_accelerator_b200 where it is true.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-5


# ---- cases --------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding sequence at GPT-2 medium's width, codes for the INT8 projection that follows: the smallest call
        dict(name="norm_token", op="norm", M=1, K=1024, dtype="f16", residual=True, i8=True, pad=0),
        # a decode step of 64 sequences, rows for a 16-bit or 4-bit layer
        dict(name="norm_decode", op="norm", M=64, K=4096, dtype="bf16", residual=True, i8=False, pad=0),
        # eight prompts of 1024 tokens, codes for an INT8 layer
        dict(name="norm_prompt", op="norm", M=8192, K=4096, dtype="bf16", residual=True, i8=True, pad=0),
        # rows of ragged prompts at GPT-2 XL's width, a slice of a wider buffer
        dict(name="quant_ragged", op="quant", M=777, K=1600, dtype="f16", pad=64),
        # the hidden rows of eight prompts before fc2 of GPT-2 medium
        dict(name="quant_prompt", op="quant", M=8192, K=4096, dtype="bf16", pad=0),
        # fc1 of GPT-2 medium for one decoding sequence
        dict(name="linear_token", op="linear", M=1, N=4096, K=1024, dtype="f16", bias=True),
        # a square projection for 64 decoding sequences
        dict(name="linear_decode", op="linear", M=64, N=4096, K=4096, dtype="bf16", bias=False),
        # lm_head of GPT-2 small over the rows of ragged prompts; odd rows and an odd vocabulary
        dict(name="linear_vocab", op="linear", M=333, N=50257, K=768, dtype="f16", bias=False),
        # the large square product of the INT8 GEMM benchmark
        dict(name="gemm_4096", op="gemm", M=4096, N=4096, K=4096, dtype="bf16", bias=False),
        # one sequence's step: its token's log-probability and five alternatives
        dict(name="logprobs_token", op="logprobs", M=1, V=50257, top=5, dtype="f16", masked=False, pad=0),
        # a decode step of 64 sequences, some under a grammar that masks most of the vocabulary
        dict(name="logprobs_decode", op="logprobs", M=64, V=50257, top=20, dtype="f16", masked=True, pad=47),
        # every position of four prompts of 1024 tokens
        dict(name="logprobs_prompt", op="logprobs", M=4096, V=50257, top=5, dtype="bf16", masked=False, pad=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "quant", "linear", "linear", "gemm", "logprobs"])
    if op in ("norm", "quant"):
        K = _log(rng, 32, 16384)
        if rng.random() < 0.7:
            K = max(32, K // 32 * 32)
        M = _log(rng, 1, max(1, min(8192, 2 ** 25 // K)))
        dtype, pad = rng.choice(["f16", "bf16"]), rng.choice([0, 0, 8, 128, 5])
        if op == "quant":
            return dict(op=op, M=M, K=K, dtype=dtype, pad=pad)
        i8 = rng.random() < 0.6
        return dict(op=op, M=M, K=K, dtype=dtype if i8 else rng.choice(["f16", "bf16", "f32"]),
                    residual=rng.random() < 0.7, i8=i8, pad=pad)
    if op in ("linear", "gemm"):
        K = 32 * _log(rng, 1, 256)
        if rng.random() < 0.3:
            K -= rng.randrange(32)
        N = _log(rng, 17, 50257)
        M = _log(rng, 1, max(1, min(8192, 2 ** 35 // (N * K), 2 ** 27 // N)))
        return dict(op=op, M=M, N=N, K=K, dtype=rng.choice(["f16", "bf16"] if op == "linear" else ["f16", "bf16", "f32"]),
                    bias=rng.random() < 0.5)
    V = _log(rng, 100, 262144)
    M = _log(rng, 1, max(1, min(4096, 3 * 2 ** 25 // V)))
    return dict(op=op, M=M, V=V, top=rng.choice([0, 1, 5, 8, 20, 32]), dtype=rng.choice(["f16", "bf16", "f32"]),
                masked=rng.random() < 0.4, pad=rng.choice([0, 0, 1, 64]))


# ---- work that a pass cannot do without ---------------------------------------------------------------------------
def work(case):
    op, M, e = case["op"], case["M"], 4 if case["dtype"] == "f32" else 2
    if op == "norm":
        K = case["K"]
        # rows (and the residual, in and out), the weight, and the normalised values; int8 codes are written and read
        # again by what gives their values
        b = M * K * e * (3 if case["residual"] else 1) + K * e + M * K * e + ((2 * M * K + 8 * M) if case["i8"] else 0)
        return {"bytes": b, "flops": M * K * (10 if case["i8"] else 6)}
    if op == "quant":
        K = case["K"]
        return {"bytes": M * K * 2 * e + 2 * M * (-(-K // 32)) * 17, "flops": 4 * M * K}
    if op == "logprobs":
        return {"bytes": M * (case["V"] * e + 16 + 8 * case["top"]), "flops": 5 * M * case["V"]}
    N, K = case["N"], case["K"]
    blocks = -(-K // 32)
    a = M * blocks * 17 if op == "gemm" else M * K * e
    return {"bytes": a + N * blocks * 17 + M * N * e + (N * e if case["bias"] else 0), "flops": 2 * M * N * K}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(M, K, pad, dtype, g, loud=6.0):
    """Rows of a residual stream: each token with a size of its own, a few channels louder; `pad` more columns a row."""
    x = torch.randn((M, K + pad), generator=g, device="cuda")
    x *= torch.rand((M, 1), generator=g, device="cuda") + 0.5
    x[:, torch.randperm(K + pad, generator=g, device="cuda")[:max(1, K // 100)]] *= loud
    return x.to(dtype)[:, :K]


def _weights(N, K, g):
    """Rows in 4-bit form: (codes uint8 [N, 16 * blocks], scale bytes uint8 [N, blocks]), the missing columns zero."""
    blocks = -(-K // 32)
    w = torch.zeros((N, 32 * blocks), device="cuda")
    w[:, :K] = torch.randn((N, K), generator=g, device="cuda") * (torch.rand((N, 1), generator=g, device="cuda") + 0.5) * 0.03
    w = w.view(N, blocks, 32)
    e = _exponent(w)
    a = _e2m1(w.abs() / torch.exp2(e)[..., None])
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | ((w < 0).to(torch.uint8) << 3)
    code = code.view(N, 32 * blocks)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), (e + 127).to(torch.uint8)


def prepare(case, seed):
    g = _gen(seed)
    op, M, dt = case["op"], case["M"], _DT[case["dtype"]]
    st = dict(case=case)
    if op in ("norm", "quant"):
        K = case["K"]
        st["x"] = _rows(M, K, case["pad"], dt, g)
        if op == "norm":
            st["r"] = _rows(M, K, 0, dt, g) if case["residual"] else None
            st["w"] = (1.0 + 0.2 * torch.randn(K, generator=g, device="cuda")).to(dt)
    elif op in ("linear", "gemm"):
        N, K = case["N"], case["K"]
        st["w"] = _weights(N, K, g)
        st["bias"] = (torch.randn(N, generator=g, device="cuda") * 0.5).to(dt) if case["bias"] else None
        if op == "linear":
            st["x"] = _rows(M, K, 0, dt, g)
        else:
            st["a"] = _weights(M, K, g)
        if own:
            from llm_accelerator_b200 import mxfp4
            st["weights"] = mxfp4.Mxfp4.from_tensors(*st["w"], K)
            if op == "gemm":
                st["rows"] = mxfp4.Mxfp4.from_tensors(*st["a"], K)
    else:
        V = case["V"]
        z = torch.randn((M, V + case["pad"]), generator=g, device="cuda", dtype=torch.float32 if M * V < 2 ** 24 else dt)
        z *= 2.5
        # a few tokens of each row stand out
        for _ in range(12):              # one at a time: two of a row may meet
            z.scatter_add_(1, torch.randint(0, V, (M, 1), generator=g, device="cuda"),
                           (torch.rand((M, 1), generator=g, device="cuda") * 14).to(z.dtype))
        if case["masked"]:               # every third row keeps one token in 64
            keep = torch.rand((-(-M // 3), V + case["pad"]), generator=g, device="cuda") < 1 / 64
            z[::3] = torch.where(keep, z[::3], torch.full((), float("-inf"), dtype=z.dtype, device="cuda"))
        st["logits"] = z.to(dt)[:, :V]
        # tokens as they come out of sampling: the best of eight
        pick = torch.randint(0, V, (M, 8), generator=g, device="cuda")
        pick[:, 0] = st["logits"].float().argmax(1)
        best = st["logits"].gather(1, pick).float() + 4 * torch.rand((M, 8), generator=g, device="cuda")
        st["tokens"] = pick.gather(1, best.argmax(1, keepdim=True))[:, 0].contiguous()
    return st


# ---- the operators ------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    return (_own if own else _plain)[op](state)


def _own_norm(st):
    from llm_accelerator_b200 import norm, ptq
    x, w, r = st["x"], st["w"], st["r"]
    if not st["case"]["i8"]:
        return norm.rms_norm(x, w, _EPS, residual=r)
    q, scale, *h = norm.rms_norm_i8(x, w, _EPS, residual=r)
    return (ptq.dequantize_rows(q, scale, x.shape[1], x.dtype), scale, *h)


def _own_quant(st):
    from llm_accelerator_b200 import mxfp4
    return mxfp4.quantize(st["x"]).values(st["x"].dtype)


def _own_linear(st):
    from llm_accelerator_b200 import mxfp4
    return mxfp4.linear(st["x"], st["weights"], bias=st["bias"])


def _own_gemm(st):
    from llm_accelerator_b200 import mxfp4
    return mxfp4.gemm(st["rows"], st["weights"], bias=st["bias"], out_dtype=_DT[st["case"]["dtype"]])


def _own_logprobs(st):
    from llm_accelerator_b200 import logprobs
    return logprobs.token_logprobs(st["logits"], st["tokens"], top=st["case"]["top"])


_own = {"norm": _own_norm, "quant": _own_quant, "linear": _own_linear, "gemm": _own_gemm, "logprobs": _own_logprobs}


def _plain_norm(st):
    x = st["x"]
    h = x.float() if st["r"] is None else x.float() + st["r"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + _EPS) * st["w"].float()
    if not st["case"]["i8"]:
        y = y.to(x.dtype)
        return y if st["r"] is None else (y, h.to(x.dtype))
    t = y.abs().amax(1).clamp(min=1e-8)
    scale = t / 127.0
    q = torch.round(y * (127.0 / t)[:, None])
    v = (q * scale[:, None]).to(x.dtype)
    return (v, scale) if st["r"] is None else (v, scale, h.to(x.dtype))


def _exponent(blocks):
    """floor(log2 max |x|) - 2 of blocks [..., 32], at least -127."""
    return (torch.frexp(blocks.abs().amax(-1)).exponent - 3).clamp(min=-127).float()


def _e2m1(a):
    """The nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 to magnitudes a; a tie goes to the even code."""
    return torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2)).clamp(max=6.0)


def _through(x):
    """float32 [M, K]: the values that rows x stand for in 4-bit form."""
    M, K = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -K % 32)).view(M, -1, 32)
    s = torch.exp2(_exponent(b))[..., None]
    return (torch.sign(b) * _e2m1(b.abs() / s) * s).view(M, -1)[:, :K]


def _values(codes, scales, K):
    """float32 [N, K] that codes and scale bytes stand for."""
    c = torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1, 32)
    v = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)[c.int()]
    return (v * torch.exp2(scales.float() - 127)[..., None]).view(codes.shape[0], -1)[:, :K]


def _plain_quant(st):
    return _through(st["x"]).to(st["x"].dtype)


def _product(a, st):
    y = a @ _values(*st["w"], st["case"]["K"]).t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return y.to(_DT[st["case"]["dtype"]])


def _plain_linear(st):
    return _product(_through(st["x"]), st)


def _plain_gemm(st):
    return _product(_values(*st["a"], st["case"]["K"]), st)


def _plain_logprobs(st):
    x, k = st["logits"].float(), st["case"]["top"]
    top = x.amax(1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    entropy = (torch.log(s) - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / s)[:, 0]
    lse = top + torch.log(s)
    lp = (x.gather(1, st["tokens"][:, None].long()) - lse)[:, 0]
    if k == 0:
        return lp, entropy
    # one whole number an entry that orders by value, then by index
    i = (x + 0.0).view(torch.int32)
    key = torch.where(i < 0, i ^ 0x7FFFFFFF, i).long() * 2 ** 32 + (2 ** 32 - 1 - torch.arange(x.shape[1], device=x.device))
    ids = 2 ** 32 - 1 - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)
    return lp, entropy, x.gather(1, ids) - lse, ids.int()


_plain = {"norm": _plain_norm, "quant": _plain_quant, "linear": _plain_linear, "gemm": _plain_gemm,
          "logprobs": _plain_logprobs}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "quant": _exact_quant, "linear": _exact_product, "gemm": _exact_product,
            "logprobs": _exact_logprobs}[case["op"]](st)


def _exact_norm(st):
    h = st["x"].double()
    if st["r"] is not None:
        h = h + st["r"].double()
    K = h.shape[1]
    y = h / torch.sqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True).square() / K + _EPS) * st["w"].double()
    if not st["case"]["i8"]:
        return y if st["r"] is None else (y, h)
    scale = torch.maximum(y.max(1).values, -y.min(1).values).clamp(min=1e-8) / 127
    v = torch.round(y / scale[:, None]) * scale[:, None]
    return (v, scale) if st["r"] is None else (v, scale, h)


def _exact_rows(x):
    """float64 [M, K]: what rows stand for, by a table of the borders between codes."""
    M, K = x.shape
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5], dtype=torch.float64, device=x.device)
    out = torch.empty((M, K), dtype=torch.float64, device=x.device)
    for k in range(0, K, 32):
        b = x[:, k:k + 32].double()
        big = b.abs().max(1).values
        # the exponent bits of a float64 are the whole part of its logarithm
        step = torch.exp2(((big.clamp(min=2.0 ** -120).view(torch.int64) >> 52) - 1025).double())[:, None]
        a = (b / step).abs()
        low, high = torch.bucketize(a, border), torch.bucketize(a, border, right=True)      # differ on a border
        out[:, k:k + 32] = torch.copysign(grid[torch.where(low % 2 == 0, low, high)] * step, b)
    return out


def _exact_quant(st):
    return _exact_rows(st["x"])


def _exact_parts(parts, K):
    codes, scales = parts
    v = torch.empty((codes.shape[0], 2 * codes.shape[1]), dtype=torch.float64, device=codes.device)
    for j in range(2):
        c = codes // 16 if j else codes % 16
        m = (c % 8).double()
        # exponent bits e and one fraction bit f: f / 2, then (1 + f / 2) 2^(e - 1)
        e, f = torch.floor(m / 2), m % 2
        m = torch.where(e == 0, f / 2, (1 + f / 2) * torch.exp2(e - 1))
        v[:, j::2] = torch.where(c >= 8, -m, m)
    v *= torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    return v[:, :K]


def _exact_product(st):
    K = st["case"]["K"]
    a = _exact_rows(st["x"]) if "x" in st else _exact_parts(st["a"], K)
    y = torch.mm(a, _exact_parts(st["w"], K).t())
    return y if st["bias"] is None else y.add_(st["bias"].double())


def _exact_logprobs(st):
    logits, k, parts = st["logits"], st["case"]["top"], []
    for i in range(0, logits.shape[0], 512):
        x = logits[i:i + 512].double()
        log_p = x - torch.logsumexp(x, 1, keepdim=True)
        p = torch.exp(log_p)
        row = [log_p[torch.arange(x.shape[0], device=x.device), st["tokens"][i:i + 512]], -torch.special.xlogy(p, p).sum(1)]
        if k:
            ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
            row += [torch.take_along_dim(log_p, ids, 1), ids.int()]
        parts.append(row)
    return tuple(torch.cat(col) for col in zip(*parts))
