"""Stand-alone operators of quantised serving, as cases that can be timed and checked.

Four operators in two groups that a quantised decoder layer runs together:

  gemm_i8_scaled   y = (A @ Bt^T) * a_scale[m] * b_scale[n] (+ bias[n]), A and Bt int8, a scale for each token
                   (row of A) and each output channel (row of Bt)
  linear_w8a8      the same product of floating-point rows: each row quantised to int8 by its own maximum first
  kv4_append       keys and values of new tokens quantised to 4 bits into a paged cache (read back as the values
                   that the codes stand for)
  kv4_attention    attention of new tokens over such a cache

4-bit form of a row x[0..D) (one token, one head): lo = min(0, min x), hi = max(0, max x),
s = bf16((hi - lo) / 15), z = rint(-lo / s), code = clip(rint(x / s) + z, 0, 15); it stands for s * (code - z).
A page holds page_size tokens: codes [pages, heads, page_size, D / 2] with code 2j in the low and 2j + 1 in the high
half of byte j, and one 32-bit word a row, the bits of s in its upper and z in its lower half.

`run` computes the plain form where `own` is false and calls llm_accelerator_b200 where it is true.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases --------------------------------------------------------------------------------------------------------
def listed():
    return [
        # fc1 of GPT-2 medium for 64 decoding sequences, rows quantised once for several products
        dict(name="gemm_decode64", op="gemm", M=64, N=4096, K=1024, dtype="f16", bias=True, wscale="f16"),
        # the large square product of the INT8 GEMM benchmark
        dict(name="gemm_4096", op="gemm", M=4096, N=4096, K=4096, dtype="bf16", bias=False, wscale="f32"),
        # fc1 of GPT-2 medium for one decoding sequence: the smallest call
        dict(name="linear_token", op="linear", M=1, N=4096, K=1024, dtype="f16", bias=True, wscale="f16"),
        # lm_head of GPT-2 small over the rows of ragged prompts; odd rows and an odd vocabulary
        dict(name="linear_vocab", op="linear", M=333, N=50257, K=768, dtype="f16", bias=False, wscale="f16"),
        # fc2 of GPT-2 medium over eight prompts of 1024 tokens
        dict(name="linear_prompt", op="linear", M=8192, N=1024, K=4096, dtype="bf16", bias=True, wscale="f32"),
        # one decode step of 64 GPT-2 medium sequences, 16 heads of 64
        dict(name="append_decode", op="append", B=64, Hkv=16, D=64, page=32, lo=5, hi=1024, new=1, dtype="f16",
             fused=True),
        # eight ragged prompts, 8 key-value heads of 128
        dict(name="append_prompt", op="append", B=8, Hkv=8, D=128, page=64, lo=700, hi=4096, new=-1, dtype="bf16",
             fused=False),
        # one GPT-2 medium sequence near its context limit: the smallest call
        dict(name="attn_token", op="attn", B=1, Hq=16, Hkv=16, D=64, page=32, lo=1003, hi=1003, new=1, empty=0,
             dtype="f16", fused=False),
        # a serving batch with grouped heads, ragged contexts, two of its slots idle
        dict(name="attn_batch", op="attn", B=64, Hq=32, Hkv=8, D=128, page=64, lo=1000, hi=8192, new=1, empty=2,
             dtype="bf16", fused=True),
        # two sequences with a long context
        dict(name="attn_long", op="attn", B=2, Hq=32, Hkv=4, D=128, page=128, lo=100001, hi=131072, new=1, empty=0,
             dtype="f16", fused=False),
        # five drafted tokens for each of 16 sequences, checked in one pass
        dict(name="attn_draft", op="attn", B=16, Hq=16, Hkv=16, D=64, page=16, lo=77, hi=1024, new=5, empty=0,
             dtype="f16", fused=True),
        # ragged prompt chunks behind earlier context
        dict(name="attn_chunk", op="attn", B=4, Hq=32, Hkv=8, D=128, page=64, lo=1500, hi=4096, new=-2, empty=0,
             dtype="bf16", fused=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gemm", "linear", "append", "attn", "attn"])
    if op in ("gemm", "linear"):
        K = 16 * _log(rng, 3, 512)
        if op == "linear" and rng.random() < 0.5:
            K -= rng.randrange(16)
        N = _log(rng, 17, 50257)
        M = _log(rng, 1, max(1, min(8192, 2 ** 35 // (N * K), 2 ** 27 // N)))
        return dict(op=op, M=M, N=N, K=K, dtype=rng.choice(["f16", "bf16", "f32"] if op == "gemm" else ["f16", "bf16"]),
                    bias=rng.random() < 0.5, wscale=rng.choice(["f16", "f32"]))
    D, page, dtype = rng.choice([64, 128]), rng.choice([16, 32, 64, 128]), rng.choice(["f16", "bf16"])
    Hkv = rng.choice([1, 2, 3, 4, 8, 12, 16])
    if op == "append":
        B = _log(rng, 1, 128)
        hi = _log(rng, 2, max(2, min(4096, 2 ** 25 // (B * Hkv * D))))
        return dict(op=op, B=B, Hkv=Hkv, D=D, page=page, lo=rng.randint(1, hi), hi=hi, new=rng.choice([1, 3, -1, -2]),
                    dtype=dtype, fused=rng.random() < 0.5)
    G = rng.choice([1, 2, 4, 5, 7, 8, 16])
    new = rng.choice([1, 1, rng.randint(2, 9), -2])
    B = _log(rng, 1, 64 if new > 0 else 4)
    hi = _log(rng, 20, max(20, min(65536 if new > 0 else 4096, 2 ** 28 // (B * Hkv * D))))
    if new < 0:                      # scores of a plain form grow with the square of the length
        Hkv = min(Hkv, 8)
        G = min(G, 32 // Hkv)
    return dict(op=op, B=B, Hq=Hkv * G, Hkv=Hkv, D=D, page=page, lo=rng.randint(max(1, hi // 16), hi), hi=hi, new=new,
                empty=rng.choice([0, 0, 1]), dtype=dtype, fused=rng.random() < 0.5)


def _lens(case):
    """(length of each sequence with its new tokens, number of new tokens of each)."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    lens = [lo + (hi - lo) * ((i * 37 + 11) % B) // max(B - 1, 1) if B > 1 else hi for i in range(B)]
    for i in range(min(case.get("empty", 0), B)):
        lens[(i * 29 + B // 2) % B] = 0
    new = case["new"]
    # n > 0: n each; -1: the whole sequence; -2: its last half
    cnt = [min(n, new) if new > 0 else n if new == -1 else (n + 1) // 2 for n in lens]
    if new == 1:
        cnt = [1] * B                # a decode step has one row for every slot, idle ones too
    return lens, cnt


# ---- work that a pass cannot do without ---------------------------------------------------------------------------
def work(case):
    if case["op"] in ("gemm", "linear"):
        M, N, K = case["M"], case["N"], case["K"]
        e = 4 if case["dtype"] == "f32" else 2
        x = M * K * 2 if case["op"] == "linear" else M * K + 4 * M
        b = x + N * K + N * (2 if case["wscale"] == "f16" else 4) + M * N * e + (N * e if case["bias"] else 0)
        return {"bytes": b, "flops": 2 * M * N * K}
    lens, cnt = _lens(case)
    D, Hkv, T = case["D"], case["Hkv"], sum(cnt)
    row = D // 2 + 4                                    # a stored row: codes and parameter word
    if case["op"] == "append":
        # new keys and values in, stored rows out, and the values they stand for (float32)
        return {"bytes": 2 * T * Hkv * (2 * D + row + 4 * D), "flops": 6 * T * Hkv * D}
    pairs = sum(sum(max(0, n - c + i + 1) for i in range(c)) for n, c in zip(lens, cnt))
    return {"bytes": 2 * sum(lens) * Hkv * row + 2 * T * case["Hq"] * D * 2, "flops": 4 * pairs * case["Hq"] * D}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _quant4(x):
    """(codes uint8 [..., D / 2], words int32 [...]) of float32 rows x [..., D]."""
    lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    s = ((hi - lo) / torch.full_like(hi, 15.0)).to(torch.bfloat16)
    sf = torch.where(s == 0, torch.ones_like(hi), s.float())
    z = torch.round(-lo / sf).clamp(0, 15)
    c = (torch.round(x / sf[..., None]) + z[..., None]).clamp(0, 15).to(torch.uint8)
    word = (s.view(torch.int16).to(torch.int32) << 16) | z.to(torch.int32)
    return c[..., 0::2] | (c[..., 1::2] << 4), word


def _pages(case, lens, g):
    """(page_table int32 [B, width], number of pages): every page in use once, in a shuffled order."""
    page, B = case["page"], case["B"]
    need = [-(-n // page) for n in lens]
    width, total = max(1, max(need)), max(1, sum(need))
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    o = 0
    for b in range(B):
        table[b, :need[b]] = perm[o:o + need[b]]
        o += need[b]
    return table, total


def _activations(T, heads, D, dtype, g):
    """Rows of a projection's output: normal, each token with a size of its own."""
    x = torch.randn((T, heads * D), generator=g, device="cuda")
    x *= torch.rand((T, 1), generator=g, device="cuda") + 0.5
    return x.to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    st = dict(case=case)
    if case["op"] in ("gemm", "linear"):
        M, N, K = case["M"], case["N"], case["K"]
        Kp = -(-K // 16) * 16

        def codes(rows):
            return torch.randn((rows, Kp), generator=g, device="cuda").mul_(34.0).round_().clamp_(-127, 127).to(torch.int8)

        st["Bt"] = codes(N)
        st["Bt"][:, K:] = 0
        st["b_scale"] = (torch.rand(N, generator=g, device="cuda") * 4e-4 + 4e-4).to(_DT[case["wscale"]])
        st["bias"] = (torch.randn(N, generator=g, device="cuda") * 0.5).to(dt) if case["bias"] else None
        if case["op"] == "gemm":
            st["A"] = codes(M)
            st["a_scale"] = torch.rand(M, generator=g, device="cuda") * 0.03 + 0.01
        else:
            x = torch.randn((M, K), generator=g, device="cuda")
            ch = torch.randperm(K, generator=g, device="cuda")[:max(1, K // 100)]
            x[:, ch] *= 6.0          # a few channels are louder, as in a residual stream
            st["x"] = x.to(dt)
        return st
    lens, cnt = _lens(case)
    D, Hkv, page, T = case["D"], case["Hkv"], case["page"], sum(cnt)
    table, total = _pages(case, lens, g)
    st["table"] = table
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ptr = [0]
    for c in cnt:
        ptr.append(ptr[-1] + c)
    # one token for each sequence needs no offsets
    st["indptr"] = None if case["new"] == 1 else torch.tensor(ptr, dtype=torch.int32, device="cuda")
    st["host"] = (lens, cnt)
    # idle slots of a decode step have no position for their row
    st["nrows"] = T
    cache = []
    for _ in range(2):               # keys, values
        cc = torch.empty((total, Hkv, page, D // 2), dtype=torch.uint8, device="cuda")
        pp = torch.empty((total, Hkv, page), dtype=torch.int32, device="cuda")
        if case["op"] == "append":
            cc.zero_()
            pp.zero_()
        else:
            step = max(1, 2 ** 24 // (Hkv * page * D))
            for i in range(0, total, step):
                n = min(step, total - i)
                x = torch.randn((n, Hkv, page, D), generator=g, device="cuda")
                x *= torch.rand((n, Hkv, page, 1), generator=g, device="cuda") + 0.5
                cc[i:i + n], pp[i:i + n] = _quant4(x)
        cache += [cc, pp]
    st["cache"] = tuple(cache)
    Hq = case.get("Hq", Hkv)
    if case["op"] == "append":
        if case["fused"]:            # slices of one fused projection's output
            qkv = _activations(T, 3 * Hkv, D, dt, g).view(T, 3 * Hkv, D)
            st["k"], st["v"] = qkv[:, Hkv:2 * Hkv], qkv[:, 2 * Hkv:]
        else:
            st["k"] = _activations(T, Hkv, D, dt, g).view(T, Hkv, D)
            st["v"] = _activations(T, Hkv, D, dt, g).view(T, Hkv, D)
    elif case["fused"]:
        st["q"] = _activations(T, Hq + 2 * Hkv, D, dt, g).view(T, Hq + 2 * Hkv, D)[:, :Hq]
    else:
        st["q"] = _activations(T, Hq, D, dt, g).view(T, Hq, D)
    if own:
        from llm_accelerator_b200 import kv4
        st["kv"] = kv4.Kv4Cache.from_tensors(*st["cache"])
    return st


# ---- the operators ------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    return (_own if own else _plain)[op](state)


def _own_gemm(st):
    from llm_accelerator_b200 import gemm
    return gemm.gemm_i8_scaled(st["A"], st["Bt"], st["a_scale"], st["b_scale"], bias=st["bias"],
                               out_dtype=_DT[st["case"]["dtype"]])


def _own_linear(st):
    from llm_accelerator_b200 import gemm
    return gemm.linear_w8a8(st["x"], st["Bt"], st["b_scale"], bias=st["bias"])


def _own_append(st):
    from llm_accelerator_b200 import kv4
    kv4.append(st["kv"], st["k"], st["v"], st["table"], st["lens"], indptr=st["indptr"])
    return kv4.read(st["kv"], st["table"], st["lens"], indptr=st["indptr"], total=st["nrows"])


def _own_attn(st):
    from llm_accelerator_b200 import kv4
    return kv4.attention(st["q"], st["kv"], st["table"], st["lens"], indptr=st["indptr"])


_own = {"gemm": _own_gemm, "linear": _own_linear, "append": _own_append, "attn": _own_attn}


def _int_product(A, Bt):
    """A @ Bt^T of whole numbers up to 127: sums over 1024 of them are exact in float32, and those sums are added in
    float64."""
    K = A.shape[1]
    if K <= 1024:
        return A.float() @ Bt.float().t()
    acc = torch.zeros((A.shape[0], Bt.shape[0]), dtype=torch.float64, device=A.device)
    for k in range(0, K, 1024):
        acc += A[:, k:k + 1024].float() @ Bt[:, k:k + 1024].float().t()
    return acc.float()


def _scaled(acc, a_scale, b_scale, bias, dt):
    y = acc * a_scale[:, None] * b_scale.float()[None, :]
    if bias is not None:
        y = y + bias.float()
    return y.to(dt)


def _plain_gemm(st):
    return _scaled(_int_product(st["A"], st["Bt"]), st["a_scale"], st["b_scale"], st["bias"], _DT[st["case"]["dtype"]])


def _plain_linear(st):
    x = st["x"].float()
    a = x.abs().amax(1).clamp(min=1e-8)
    c127 = torch.full_like(a, 127.0)
    q = torch.round(x * (c127 / a)[:, None]).clamp(-127, 127)
    return _scaled(_int_product(q, st["Bt"][:, :x.shape[1]]), a / c127, st["b_scale"], st["bias"], st["x"].dtype)


def _plain_append(st):
    case = st["case"]
    page = case["page"]
    lens, indptr, table = st["lens"].long(), st["indptr"], st["table"].long()
    T, B = st["nrows"], case["B"]
    rows = torch.arange(T, device=table.device)
    if indptr is None:
        seq, pos = rows, lens - 1
    else:
        ends = indptr[1:].long()
        seq = torch.searchsorted(ends, rows, right=True)
        pos = lens[seq] - (ends[seq] - rows)
    p, slot = table[seq, pos // page], pos % page
    out = []
    for x, cc, pp in ((st["k"], *st["cache"][:2]), (st["v"], *st["cache"][2:])):
        codes, words = _quant4(x.float())
        cc[p, :, slot] = codes
        pp[p, :, slot] = words
        out.append(_values(cc[p, :, slot], pp[p, :, slot]))
    return tuple(out)


def _values(codes, words):
    """float32 rows that codes [..., D / 2] with words [...] stand for."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    s = (words & -65536).view(torch.float32)
    return (c - (words & 65535).float()[..., None]) * s[..., None]


def _plain_attn(st):
    case = st["case"]
    q, table, (kc, kp, vc, vp) = st["q"], st["table"], st["cache"]
    Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    lens, cnt = st["host"]
    out = torch.zeros((st["nrows"], Hq, D), dtype=q.dtype, device=q.device)
    o = 0
    for b, (n, c) in enumerate(zip(lens, cnt)):
        if n and c:
            ids = table[b, :-(-n // page)].long()
            k = _values(kc[ids], kp[ids]).transpose(1, 2).reshape(-1, Hkv, D)[:n]      # [n, Hkv, D]
            v = _values(vc[ids], vp[ids]).transpose(1, 2).reshape(-1, Hkv, D)[:n]
            qb = q[o:o + c].float().view(c, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3).reshape(Hkv, -1, D)
            s = (qb @ k.permute(1, 2, 0)) * (D ** -0.5)                                # [Hkv, G * c, n]
            if c > 1:
                i = torch.arange(c, device=q.device)[:, None] + (n - c)
                hidden = torch.arange(n, device=q.device)[None, :] > i
                s = s.view(Hkv, -1, c, n).masked_fill_(hidden, float("-inf")).view(Hkv, -1, n)
            s = torch.exp(s - s.amax(-1, keepdim=True))
            y = (s @ v.transpose(0, 1)) / s.sum(-1, keepdim=True)
            out[o:o + c] = y.view(Hkv, Hq // Hkv, c, D).permute(2, 0, 1, 3).reshape(c, Hq, D).to(q.dtype)
        o += c
    return out


_plain = {"gemm": _plain_gemm, "linear": _plain_linear, "append": _plain_append, "attn": _plain_attn}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"gemm": _exact_product, "linear": _exact_product, "append": _exact_append, "attn": _exact_attn}[case["op"]](st)


def _exact_product(st):
    w = st["Bt"].double()
    if "A" in st:
        a, row = st["A"].double(), st["a_scale"].double()
    else:
        x = st["x"].double()
        top = torch.maximum(x.max(1).values, -x.min(1).values).clamp(min=1e-8)
        row = top / 127
        a = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float64, device=x.device)
        a[:, :x.shape[1]] = torch.round(x / row[:, None])
    y = torch.mm(a, w.t()).mul_(row.unsqueeze(1)).mul_(st["b_scale"].double())
    return y if st["bias"] is None else y.add_(st["bias"].double())


def _exact_append(st):
    res = []
    for x in (st["k"].double(), st["v"].double()):
        low = torch.minimum(x.min(-1, keepdim=True).values, torch.zeros((), dtype=x.dtype, device=x.device))
        high = torch.maximum(x.max(-1, keepdim=True).values, torch.zeros((), dtype=x.dtype, device=x.device))
        step = ((high - low) / 15).to(torch.bfloat16).double()      # the step is held in 16 bits
        step = torch.where(step == 0, torch.ones_like(step), step)
        zero = torch.round(-low / step)
        res.append(step * ((torch.round(x / step) + zero).clamp(0, 15) - zero))
    return tuple(res)


def _exact_attn(st):
    case, q, (kc, kp, vc, vp) = st["case"], st["q"], st["cache"]
    Hkv, G, D, page = case["Hkv"], case["Hq"] // case["Hkv"], case["D"], case["page"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)

    def rows(codes, words, ids, h, n):
        c, w = codes[ids, h].reshape(-1, D // 2)[:n], words[ids, h].reshape(-1)[:n]
        x = torch.empty((n, D), dtype=torch.float64, device=q.device)
        x[:, 0::2], x[:, 1::2] = (c % 16).double(), (c // 16).double()
        scale = (w >> 16).to(torch.int16).view(torch.bfloat16).double()
        return x.sub_((w % 16).double()[:, None]).mul_(scale[:, None])

    first = 0
    for b, (n, c) in enumerate(zip(*st["host"])):
        for h in range(Hkv if n and c else 0):
            ids = st["table"][b, :-(-n // page)].long()
            K, V = rows(kc, kp, ids, h, n), rows(vc, vp, ids, h, n)
            for j in range(G):
                head = h * G + j
                s = torch.mm(q[first:first + c, head].double(), K.t()) / math.sqrt(D)
                if c > 1:
                    s = s + torch.full((c, n), float("-inf"), dtype=s.dtype, device=s.device).triu(n - c + 1)
                out[first:first + c, head] = torch.mm(torch.exp(s - torch.logsumexp(s, 1, keepdim=True)), V)
        first += c
    return out
