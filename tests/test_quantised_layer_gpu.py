"""The INT8 products and the 4-bit cache together, as a quantised decoder layer uses them: QKV projection, rotation of
queries and keys, append, attention, output projection; a prompt chunk, then single tokens, then drafted tokens.

Each stage is held against its definition in 64 bits on the inputs that it got, so a tolerance never covers more than
one stage (tests/kv4_helpers.py and tests/test_w8a8_gpu.py derive them)."""
from __future__ import annotations

import pytest
import torch

from kv4_helpers import check, pack, quantise, reference, values
from test_w8a8_gpu import _check as check_product
from test_w8a8_gpu import _quant_rows_cpu

pytestmark = pytest.mark.gpu


class _Layer:
    def __init__(self, d, hq, hkv, D, pages, page, seed=0):
        from llm_accelerator_b200 import gemm, kv4, ptq
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.hq, self.hkv, self.D = hq, hkv, D
        n = (hq + 2 * hkv) * D
        self.wqkv, self.sqkv = ptq.quantize_tensor(torch.randn((n, d), generator=g, device="cuda") * d ** -0.5)
        self.wo, self.so = ptq.quantize_tensor(torch.randn((d, hq * D), generator=g, device="cuda") * (hq * D) ** -0.5)
        self.wqkv, self.wo = gemm.pad_k16(self.wqkv), gemm.pad_k16(self.wo)
        self.bias = (torch.randn(n, generator=g, device="cuda") * 0.1).half()
        self.cache = kv4.Kv4Cache(pages, page, hkv, D)

    def __call__(self, x, table, lens, indptr=None):
        """The layer on rows x of the sequences' new tokens, and every stage's result."""
        from llm_accelerator_b200 import gemm, kv4, quarot
        hq, hkv, D, T = self.hq, self.hkv, self.D, x.shape[0]
        qkv = gemm.linear_w8a8(x, self.wqkv, self.sqkv, bias=self.bias)
        qk = quarot.fwht_f16(qkv[:, :(hq + hkv) * D].contiguous(), D).view(T, hq + hkv, D)   # cancels in q . k
        v = qkv.view(T, -1, D)[:, hq + hkv:]
        kv4.append(self.cache, qk[:, hq:], v, table, lens, indptr)
        a = kv4.attention(qk[:, :hq], self.cache, table, lens, indptr)
        return qkv, qk, v, a, gemm.linear_w8a8(a.view(T, hq * D), self.wo, self.so)


@pytest.mark.parametrize("d,hq,hkv,D,page", [(256, 4, 4, 64, 16), (384, 6, 2, 64, 32), (512, 8, 1, 128, 64)])
def test_prompt_decode_and_draft(d, hq, hkv, D, page):
    lens = [150, 3, 41]
    layer = _Layer(d, hq, hkv, D, pages=40, page=page, seed=d)
    order = torch.randperm(40, generator=torch.Generator().manual_seed(1))[:36].view(3, 12).to(torch.int32)
    table = order.cuda()
    held = [[[], []] for _ in lens]              # the values that each sequence's cache stands for
    done = [0, 0, 0]
    g = torch.Generator(device="cuda").manual_seed(7)
    for new in (lens, [1, 1, 1], [1, 1, 1], [5, 5, 5], [1, 1, 1]):
        T = sum(new)
        done = [a + b for a, b in zip(done, new)]
        ptr = [0]
        for n in new:
            ptr.append(ptr[-1] + n)
        decode = new == [1, 1, 1]
        x = torch.randn((T, d), generator=g, device="cuda").half()
        d_lens = torch.tensor(done, dtype=torch.int32, device="cuda")
        d_ptr = None if decode else torch.tensor(ptr, dtype=torch.int32, device="cuda")
        qkv, qk, v, a, y = layer(x, table, d_lens, d_ptr)
        # the projections
        q8, s8 = _quant_rows_cpu(x)
        check_product(qkv, q8, layer.wqkv, s8, layer.sqkv, layer.bias)
        q8, s8 = _quant_rows_cpu(a.view(T, hq * D))
        check_product(y, q8, layer.wo, s8, layer.so, None)
        # the cache: what every token of a sequence stands for, those of earlier calls unchanged
        for s in range(3):
            for w, rows in enumerate((qk[ptr[s]:ptr[s + 1], hq:], v[ptr[s]:ptr[s + 1]])):
                held[s][w].append(values(*pack(*quantise(rows))))
        from llm_accelerator_b200 import kv4
        full = [0]
        for n in done:
            full.append(full[-1] + n)
        rk, rv = kv4.read(layer.cache, table, d_lens, torch.tensor(full, dtype=torch.int32, device="cuda"), total=full[-1])
        for w, r in enumerate((rk, rv)):
            assert torch.equal(r.cpu().double(), torch.cat([torch.cat(held[s][w]) for s in range(3)]))
        # attention over it
        batch = _Held(layer.cache, order, done)
        want, _, tol = reference(batch, qk[:, :hq], ptr)
        check(a, want, tol)


class _Held:
    """A cache's contents in the form that kv4_helpers.reference reads."""

    def __init__(self, cache, table, lens):
        self.lens, self.heads, self.D, self.page, self.pages = lens, cache.heads, cache.head_dim, cache.page_size, cache.num_pages
        self.table = table
        self.host = [t.cpu() for t in (cache.k_codes, cache.k_params, cache.v_codes, cache.v_params)]

    from kv4_helpers import Batch as _B
    rows = _B.rows


def test_rotated_keys_attend_alike():
    """The rotation of queries and keys changes what the cache holds, not what attention computes: with and without it
    the outputs differ by the keys' quantisation only."""
    from llm_accelerator_b200 import kv4, quarot
    T, H, D = 300, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn((T, H, D), generator=g, device="cuda").half() for _ in range(3))
    k[:, :, 5] *= 20                              # a loud channel, which 4 bits a row resolve badly
    table = torch.arange(10, dtype=torch.int32, device="cuda").view(1, 10)
    lens, ptr = torch.tensor([T], dtype=torch.int32, device="cuda"), torch.tensor([0, T], dtype=torch.int32, device="cuda")
    errs = []
    for rotate in (False, True):
        a, b = q, k
        if rotate:
            a, b = (quarot.fwht_f16(t.reshape(T, H * D), D).view(T, H, D) for t in (q, k))
        cache = kv4.Kv4Cache(10, 32, H, D)
        kv4.append(cache, b, v, table, lens, ptr)
        rk, _ = kv4.read(cache, table, lens, ptr, total=T)
        errs.append((rk - b.float()).square().mean().item())
        s = torch.einsum("thd,shd->hts", a.double(), rk.double()) * D ** -0.5
        t = torch.einsum("thd,shd->hts", q.double(), k.double()) * D ** -0.5
        errs.append((s - t).square().mean().item())
    assert errs[2] < errs[0] and errs[3] < errs[1]   # the rotated cache is nearer, in its rows and in the scores
