"""Batches of a 4-bit paged cache for tests, and its definition in 64 bits on the CPU."""
from __future__ import annotations

import torch


def quantise(x):
    """(codes [..., D], s [...], z [...]) of rows x, in float32 as the cache's definition has it; s float32."""
    x = x.cpu().float()
    lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    s = ((hi - lo) / torch.full_like(hi, 15.0)).to(torch.bfloat16).float()
    d = torch.where(s == 0, torch.ones_like(s), s)
    z = torch.round(-lo / d).clamp(0, 15)
    c = (torch.round(x / d[..., None]) + z[..., None]).clamp(0, 15)
    c = torch.where(s[..., None] == 0, torch.zeros_like(c), c)
    return c, s, torch.where(s == 0, torch.zeros_like(z), z)


def pack(c, s, z):
    c = c.to(torch.uint8)
    word = (s.to(torch.bfloat16).view(torch.int16).to(torch.int32) << 16) | z.to(torch.int32)
    return c[..., 0::2] | (c[..., 1::2] << 4), word


def values(codes, words):
    """float64 rows [..., D] that codes [..., D / 2] with words [...] stand for."""
    codes, words = codes.cpu(), words.cpu()
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
    s = (words & -65536).view(torch.float32).double()
    return (c - (words & 65535).double()[..., None]) * s[..., None]


class Batch:
    """Sequences of the given lengths on shuffled pages of a cache filled with random rows; slots that hold no token
    are filled with `junk` (codes, word)."""

    def __init__(self, lens, heads, D, page, seed=0, spare=2, junk=(0xFF, 0x7FC0000F), spread=1.0, vscale=1.0):
        from llm_accelerator_b200 import kv4
        g = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.D, self.page = list(lens), heads, D, page
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g)
        width = max(1, max(need)) + 1
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        o = 0
        for b, n in enumerate(need):
            table[b, :n] = order[o:o + n].to(torch.int32)
            o += n
        live = torch.zeros((self.pages, page), dtype=torch.bool)
        for b, n in enumerate(lens):
            for j in range(need[b]):
                live[table[b, j], :min(page, n - j * page)] = True
        parts = []
        for mul in (1.0, vscale):
            x = torch.randn((self.pages, heads, page, D), generator=g) * mul
            x *= torch.exp(torch.randn((self.pages, heads, page, 1), generator=g) * 0.3 * spread)
            codes, words = pack(*quantise(x))
            dead = ~live[:, None, :].expand(self.pages, heads, page)
            codes[dead] = junk[0]
            words[dead] = junk[1]
            parts += [codes, words]
        self.host = parts
        self.table = table
        self.cache = kv4.Kv4Cache.from_tensors(*(p.cuda() for p in parts))
        self.d_table = table.cuda()
        self.d_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def rows(self, b, which, head, n):
        """(float64 [n, D], bool [n]) of sequence b's first n tokens; False where its page holds no tokens."""
        codes, words = self.host[2 * which], self.host[2 * which + 1]
        x = torch.zeros((n, self.D), dtype=torch.float64)
        ok = torch.zeros(n, dtype=torch.bool)
        for j in range(-(-n // self.page)):
            p = int(self.table[b, j])
            m = min(self.page, n - j * self.page)
            if 0 <= p < self.pages:
                x[j * self.page:j * self.page + m] = values(codes[p, head, :m], words[p, head, :m])
                ok[j * self.page:j * self.page + m] = True
        return x, ok


def reference(batch, q, indptr=None, causal=True, scale=None):
    """(out, lse, tol) float64: the definition, and how far a kernel may be from it before the last rounding.

    A score is an FP16 product sum: q is exact in FP16 up to 2^-25 of its row's largest magnitude, codes are whole
    numbers, and D products are added in float32 (at most 2 D 2^-24 of their magnitudes' sum, were each addition cut
    off); two float32 factors follow.  exp2 is good to 2^-21.  A weight p s' is rounded once to FP16: 2^-11 of it, or
    2^-25 of the unit that brings the largest s' into [1, 2).  Output sums run in float32 over n tokens."""
    lens, D = batch.lens, batch.D
    q = q.cpu()
    total, hq, _ = q.shape
    group = hq // batch.heads
    scale = D ** -0.5 if scale is None else scale
    if indptr is None:
        indptr = list(range(len(lens) + 1))
    out = torch.full((total, hq, D), float("nan"), dtype=torch.float64)
    lse = torch.full((total, hq), float("nan"), dtype=torch.float64)
    tol = torch.full((total, hq, D), float("nan"), dtype=torch.float64)
    step = torch.finfo(q.dtype).eps / 2
    for b, n in enumerate(lens):
        a, e = indptr[b], indptr[b + 1]
        for h in range(batch.heads if e > a else 0):
            K, ok = batch.rows(b, 0, h, n)
            V, _ = batch.rows(b, 1, h, n)
            vs = (batch.host[3][:, h] & -65536).view(torch.float32).double()
            qq = q[a:e, h * group:(h + 1) * group].double()              # [c, group, D]
            s = (qq @ K.t()) * scale if n else torch.zeros((e - a, group, 0), dtype=torch.float64)
            ds = ((qq.abs() @ K.abs().t()) * (2 * D + 4) * 2.0 ** -24
                  + qq.abs().amax(-1, keepdim=True) * K.abs().sum(-1) * 2.0 ** -25) * abs(scale)
            seen = ok[None, :].expand(e - a, n).clone()
            if causal:
                seen &= torch.arange(n)[None, :] <= (n - (e - a) + torch.arange(e - a))[:, None]
            s = s.masked_fill(~seen[:, None, :], float("-inf"))
            top = s.amax(-1, keepdim=True) if n else torch.full((e - a, group, 1), float("-inf"), dtype=torch.float64)
            some = torch.isfinite(top) | torch.isnan(top)
            p = torch.exp(s - torch.where(some, top, torch.zeros_like(top)))
            p = torch.where(seen[:, None, :], p, torch.zeros_like(p))
            z = p.sum(-1, keepdim=True)
            p = torch.where(z > 0, p / z, p)
            dmax = torch.where(seen[:, None, :], ds, torch.zeros_like(ds)).amax(-1, keepdim=True) if n else 0 * top
            rel = 2.0 ** -11 + 2.0 ** -19 + 2 * dmax + max(n, 1) * 2.0 ** -24
            Vc = torch.where(ok[:, None], V, torch.zeros_like(V))
            out[a:e, h * group:(h + 1) * group] = torch.where(z > 0, p @ Vc, torch.zeros(()).double()) if n else 0.0
            lse[a:e, h * group:(h + 1) * group] = (top + torch.log(z))[..., 0]
            ids = batch.table[b][(batch.table[b] >= 0) & (batch.table[b] < batch.pages)].long()
            big = torch.nan_to_num(vs[ids], nan=0.0).max() if n and ok.any() else 0.0
            tol[a:e, h * group:(h + 1) * group] = rel * (p @ Vc.abs() if n else 0.0) + n * 2.0 ** -24 * 15 * float(big)
    tiny = 2.0 ** (-25 if q.dtype == torch.float16 else -134)       # half a subnormal step
    tol = tol + step * out.abs() * (1 + step) + tiny
    return out, lse, tol


def check(got, want, tol):
    """Rows of no sequence (NaN in `tol`) are not looked at."""
    got = got.cpu().double()
    row = ~torch.isnan(tol)
    assert torch.isfinite(got[row]).all()
    over = ((got - want).abs() / tol)[row]
    assert over.numel() == 0 or over.max() <= 1, f"worst {over.max():.3f} of the tolerance"


def check_lse(got, want, ds=2.0 ** -9):
    """Scores up to 2^7 in float32 products of 128 terms: off by less than 2^-9; log2 and the sum add 2^-20."""
    got = got.cpu().double()
    row = ~torch.isnan(want)
    inf = row & torch.isinf(want)
    assert (got[inf] == float("-inf")).all()
    fin = row & ~inf
    assert ((got - want).abs()[fin] <= ds * (1 + want.abs()[fin] / 128)).all()


def queries(total, hq, D, dtype, seed=0, mul=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((total, hq, D), generator=g) * mul).to(dtype).cuda()

