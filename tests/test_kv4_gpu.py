"""The 4-bit paged cache and attention over it, on the GPU against their definitions in 64 bits
(tests/kv4_helpers.py derives the tolerances)."""
from __future__ import annotations

import subprocess
import sys
import textwrap
from pathlib import Path

import pytest
import torch

from kv4_helpers import Batch, check, check_lse, pack, quantise, queries, reference, values

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- append and read ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D,heads,page,lens,new", [
    (64, 1, 16, [1], [1]), (64, 16, 32, [5, 33, 64, 1024], [1, 1, 1, 1]), (128, 8, 64, [70, 64, 1, 0], [70, 3, 1, 0]),
    (128, 3, 128, [300, 129], [299, 128]), (64, 5, 16, [17, 500, 31], [17, 0, 9]), (128, 1, 16, [2000], [1777])])
def test_append_and_read_bit_exact(D, heads, page, lens, new, dtype):
    """Codes and words as the definition gives them, in their places, and not a byte elsewhere."""
    from llm_accelerator_b200 import kv4
    b = Batch(lens, heads, D, page, seed=D + page)
    before = [t.clone() for t in b.host]
    T = sum(new)
    g = torch.Generator().manual_seed(T)
    wide = (torch.randn((T, 3 * heads, D), generator=g) * 2).to(DT[dtype])
    wide[0, :, 1] = 0
    wide[T // 2, heads:] = 0                          # a row of zeros
    wide[T - 1, heads:] = wide[T - 1, heads:].abs()   # no negative value
    d = wide.cuda()
    k, v = d[:, heads:2 * heads], d[:, 2 * heads:]    # slices of a fused projection
    ptr = [0]
    for n in new:
        ptr.append(ptr[-1] + n)
    decode = new == [1] * len(lens)
    indptr = None if decode else _i32(ptr)
    kv4.append(b.cache, k, v, b.d_table, b.d_lens, indptr)
    rk, rv = kv4.read(b.cache, b.d_table, b.d_lens, indptr, total=T)
    for which, (x, back) in enumerate(((k, rk), (v, rv))):
        codes, words = pack(*quantise(x))
        for s, (n, c) in enumerate(zip(lens, new)):
            for i in range(c):
                pos = n - c + i
                p, slot = int(b.table[s, pos // page]), pos % page
                before[2 * which][p, :, slot] = codes[ptr[s] + i]
                before[2 * which + 1][p, :, slot] = words[ptr[s] + i]
        assert torch.equal(back.cpu().double(), values(codes, words))
    got = (b.cache.k_codes, b.cache.k_params, b.cache.v_codes, b.cache.v_params)
    for w, x in zip(before, got):
        assert torch.equal(x.cpu(), w)


def test_append_any_stride_and_alignment():
    from llm_accelerator_b200 import kv4
    T, H, D = 7, 3, 64
    for dtype in DT.values():
        flat = torch.randn(20000, device="cuda").to(dtype)
        for off, st in ((0, (H * D, D)), (1, (H * D + 1, D + 1)), (3, (D + 5, T * (D + 5))), (8, (0, D)), (0, (D, 0))):
            x = flat.as_strided((T, H, D), (*st, 1), off)
            cache = kv4.Kv4Cache(2, 16, H, D)
            table, lens = _i32([[1]]), _i32([T])
            kv4.append(cache, x, x, table, lens, _i32([0, T]))
            rk, rv = kv4.read(cache, table, lens, _i32([0, T]), total=T)
            want = values(*pack(*quantise(x)))
            assert torch.equal(rk.cpu().double(), want) and torch.equal(rv.cpu().double(), want)


def test_values_that_are_not_finite_and_extreme_ranges():
    """A row with an infinity or a NaN reads as NaN and leaves its neighbours alone; the smallest and largest values."""
    from llm_accelerator_b200 import kv4
    H, D = 4, 64
    x = torch.randn((6, H, D), device="cuda")
    x[0, 1, 5], x[1, 2, 0], x[2, 3, 63] = float("nan"), float("inf"), float("-inf")
    x[3] *= 1e-38
    x[4] *= 2.0 ** 120
    x[5] = 2.0 ** -149
    cache = kv4.Kv4Cache(1, 16, H, D)
    kv4.append(cache, x, x, _i32([[0]]), _i32([6]), _i32([0, 6]))
    rk, rv = kv4.read(cache, _i32([[0]]), _i32([6]), _i32([0, 6]), total=6)
    bad = torch.zeros((6, H), dtype=torch.bool)
    bad[0, 1] = bad[1, 2] = bad[2, 3] = True
    want = values(*pack(*quantise(torch.where(bad[..., None].cuda(), 0.0, x))))
    for r in (rk.cpu(), rv.cpu()):
        assert r[bad].isnan().all() and torch.equal(r[~bad].double(), want[~bad])


def test_rows_without_a_place_are_skipped():
    """Before position 0, past the table, on a page outside the cache, and of no sequence."""
    from llm_accelerator_b200 import kv4
    H, D = 2, 64
    cache = kv4.Kv4Cache(3, 16, H, D)
    x = torch.randn((60, H, D), device="cuda")
    #        before 0      past the table   pages -1 and 7      unused rows 50..59
    table = _i32([[0, -1], [1, 2], [-1, 7]])
    lens, ptr = _i32([4, 40, 20]), _i32([0, 6, 30, 50])
    kv4.append(cache, x, x, table, lens, ptr)
    rk, _ = kv4.read(cache, table, lens, ptr, total=60)
    want = values(*pack(*quantise(x)))
    place = torch.zeros(60, dtype=torch.bool)
    place[2:6] = True                     # positions 0..3 of sequence 0
    place[6:22] = True                    # positions 16..31 of sequence 1 (32..39 are past its two pages)
    assert torch.equal(rk.cpu().double()[place], want[place])
    assert not rk.cpu()[~place].any()
    used = cache.k_params.cpu()[0, 0] != 0
    assert used.tolist() == [True] * 4 + [False] * 12
    assert not cache.k_params.cpu()[1].any() and (cache.k_params.cpu()[2] != 0).all()


# ---- attention ------------------------------------------------------------------------------------------------------
DECODE = [
    # D, heads, group, page, lens
    (64, 16, 1, 32, [1003]), (64, 1, 1, 16, [1]), (128, 1, 1, 128, [2, 1, 0]), (64, 2, 3, 16, [15, 16, 17, 31, 32, 33]),
    (128, 8, 4, 64, [127, 128, 129, 1000, 0, 64]), (128, 4, 8, 128, [5000, 1]), (128, 2, 7, 16, [300, 77]),
    (64, 1, 16, 32, [500, 1, 0]), (128, 1, 32, 64, [513, 40]), (64, 3, 9, 64, [256, 255]), (64, 12, 1, 16, [64] * 9),
    (128, 1, 1, 16, [20011]), (64, 2, 2, 16, list(range(0, 150))),
    # more sequences than threads of a CTA, with and without a context that is shared out
    (64, 1, 2, 16, [i * 7 % 60 for i in range(600)]), (64, 1, 1, 16, [i * 7 % 60 for i in range(599)] + [5000]),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,heads,group,page,lens", DECODE)
def test_single_tokens(D, heads, group, page, lens, dtype):
    from llm_accelerator_b200 import kv4
    b = Batch(lens, heads, D, page, seed=len(lens) + D)
    q = queries(len(lens), heads * group, D, DT[dtype])
    out, lse = kv4.attention(q, b.cache, b.d_table, b.d_lens, return_lse=True)
    want, wlse, tol = reference(b, q)
    check(out, want, tol)
    check_lse(lse, wlse)
    assert torch.equal(out, kv4.attention(q, b.cache, b.d_table, b.d_lens))     # the same from run to run


SEVERAL = [
    # D, heads, group, page, lens, new
    (64, 16, 1, 16, [77, 1024, 300], [5, 5, 5]), (128, 2, 4, 64, [129, 64, 9], [3, 1, 9]), (64, 1, 1, 32, [40], [40]),
    (128, 1, 5, 16, [500, 0, 20], [17, 0, 20]), (64, 2, 8, 128, [300, 10], [2, 7]), (64, 4, 2, 16, [33, 1], [33, 1]),
    (128, 8, 4, 64, [700, 333], [260, 333]), (64, 3, 1, 32, [1030], [513]), (128, 1, 16, 128, [260], [130]),
    (64, 2, 3, 64, [5, 9, 200], [8, 9, 130]),       # more rows than positions: the first rows see nothing
    # enough rows for the prompt kernel: partial row blocks and tiles, one and two row groups, many sequences
    (128, 8, 4, 64, [300, 333], [300, 200]), (64, 8, 2, 16, [700, 129, 64], [700, 100, 64]), (64, 16, 1, 128, [1030], [900]),
    (128, 2, 5, 32, [900], [850]), (64, 2, 3, 64, [500, 9, 1100], [600, 11, 1101]), (128, 1, 16, 16, [640, 0], [640, 0]),
    (64, 2, 8, 16, list(range(20, 90)), [20] * 70),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,heads,group,page,lens,new", SEVERAL)
def test_several_tokens(D, heads, group, page, lens, new, dtype, causal):
    from llm_accelerator_b200 import kv4
    b = Batch(lens, heads, D, page, seed=sum(new) + D)
    ptr = [0]
    for n in new:
        ptr.append(ptr[-1] + n)
    total = ptr[-1] + 3                               # rows behind the last sequence
    wide = queries(total, heads * group + 2, D, DT[dtype])
    q = wide[:, 1:-1]
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    got, lse = kv4.attention(q, b.cache, b.d_table, b.d_lens, _i32(ptr), causal=causal, return_lse=True, out=out)
    assert got is out and (out[ptr[-1]:] == 7).all()
    want, wlse, tol = reference(b, q, ptr, causal)
    check(out, want, tol)
    check_lse(lse, wlse)


@pytest.mark.parametrize("new", [1, 3, 200, 1500])
def test_what_unused_slots_hold_does_not_matter(new):
    """Slots past a sequence's end and pages of no sequence: zeros, NaN words and infinities give the same bits."""
    from llm_accelerator_b200 import kv4
    lens = [230, 201, 300] if new <= 200 else [1530, 1501, 1600]
    ptr = [0, new, 2 * new, 3 * new]
    q = queries(3 * new, 6, 64, torch.float16)
    outs = []
    for junk in ((0, 0), (0xFF, 0x7FC0000F), (0xA5, 0x7F800003), (0x13, 0x7F7F000F), (0x77, -1), (0x77, 0x7FFFFFFF)):
        b = Batch(lens, 2, 64, 16, junk=junk)
        outs.append(kv4.attention(q, b.cache, b.d_table, b.d_lens, _i32(ptr), return_lse=True))
    for o, l in outs[1:]:
        assert torch.equal(o, outs[0][0]) and torch.equal(l, outs[0][1])


@pytest.mark.parametrize("new", [1, 4, 150, 2300])
def test_a_nan_token_reaches_only_the_rows_that_see_it(new):
    from llm_accelerator_b200 import kv4
    n = 400 if new < 400 else 2500
    for which in (0, 1):
        b = Batch([n], 2, 128, 32)
        pos = n - (new + 1) // 2                       # among the new tokens, seen by the rows from there on
        p, slot = int(b.table[0, pos // 32]), pos % 32
        clean = kv4.attention(queries(new, 4, 128, torch.bfloat16), b.cache, b.d_table, b.d_lens, _i32([0, new]))
        (b.cache.k_params, b.cache.v_params)[which][p, 1, slot] = 0x7FC00000
        got = kv4.attention(queries(new, 4, 128, torch.bfloat16), b.cache, b.d_table, b.d_lens, _i32([0, new]))
        first = pos - (n - new)
        assert got[first:, 2:].isnan().all()
        assert torch.equal(got[:first], clean[:first]) and torch.equal(got[:, :2], clean[:, :2])


@pytest.mark.parametrize("new", [1, 200, 5400])
def test_pages_without_tokens(new):
    """Page numbers outside the cache, inside and at the ends of a sequence, hold no keys; a sequence of none of them
    gives zeros."""
    from llm_accelerator_b200 import kv4
    b = Batch([400 if new < 400 else 6000, 400, 300, 33], 2, 64, 16)
    b.table[0, 0] = -1
    b.table[0, 7:11] = b.pages
    b.table[1, 12:] = 2 ** 31 - 1
    b.table[2, :] = -7
    b.d_table = b.table.cuda()
    ptr = [0, new, new + 1, new + 2, new + 3]
    q = queries(new + 3, 2, 64, torch.float16)
    out, lse = kv4.attention(q, b.cache, b.d_table, b.d_lens, _i32(ptr), return_lse=True)
    want, wlse, tol = reference(b, q, ptr)
    check(out, want, tol)
    check_lse(lse, wlse)
    assert not out[new + 1].any()


@pytest.mark.parametrize("new", [1, 140, 1500])
@pytest.mark.parametrize("dtype,qmul,vmul", [("f16", 1.0, 1e-6), ("f16", 60.0, 1.0), ("bf16", 1.0, 1e30),
                                             ("bf16", 1e-20, 1e-30), ("f16", 1e-6, 4000.0), ("bf16", 40.0, 1e-3)])
def test_magnitudes(dtype, qmul, vmul, new):
    """Values near the ends of the types' ranges, and scores of some hundreds (one key takes it all)."""
    from llm_accelerator_b200 import kv4
    b = Batch([500, 333] if new < 300 else [1600, 1520], 2, 64, 32, vscale=vmul)
    q = queries(2 * new, 4, 64, DT[dtype], mul=qmul)
    out = kv4.attention(q, b.cache, b.d_table, b.d_lens, _i32([0, new, 2 * new]))
    want, _, tol = reference(b, q, [0, new, 2 * new])
    check(out, want, tol)


@pytest.mark.parametrize("new", [1, 130, 10600])
def test_a_loud_token_among_quiet_ones(new):
    """One token with values 2^20 times the others', early and late: no weight is lost on either side of it."""
    from llm_accelerator_b200 import kv4
    for pos in (3, 250, 580) if new < 700 else (3, 5000, 10690):
        b = Batch([700 if new < 700 else 10700], 1, 64, 16)
        p, slot = int(b.table[0, pos // 16]), pos % 16
        for t in (b.host[3], b.cache.v_params):
            t[p, 0, slot] += 20 << 23
        q = queries(new, 1, 64, torch.bfloat16)
        out = kv4.attention(q, b.cache, b.d_table, b.d_lens, _i32([0, new]))
        want, _, tol = reference(b, q, [0, new])
        check(out, want, tol)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_scale(scale):
    from llm_accelerator_b200 import kv4
    b = Batch([200, 90], 2, 64, 16)
    for ptr in ([0, 1, 2], [0, 150, 152], [0, 3000, 3002]):
        q = queries(ptr[-1], 4, 64, torch.float16)
        out = kv4.attention(q, b.cache, b.d_table, b.d_lens, _i32(ptr), scale=scale)
        want, _, tol = reference(b, q, ptr, scale=scale)
        check(out, want, tol)


def test_parts_join_by_their_lse():
    """Attention over two halves of a context, joined by lse, is attention over the whole."""
    from llm_accelerator_b200 import kv4
    b = Batch([512], 4, 128, 64)
    q = queries(1, 8, 128, torch.bfloat16)
    whole, lse = kv4.attention(q, b.cache, b.d_table, b.d_lens, return_lse=True)
    a, la = kv4.attention(q, b.cache, b.d_table[:, :4].contiguous(), _i32([256]), return_lse=True)
    c, lc = kv4.attention(q, b.cache, b.d_table[:, 4:].contiguous(), _i32([256]), return_lse=True)
    top = torch.logaddexp(la, lc)
    joined = a.float() * torch.exp(la - top)[..., None] + c.float() * torch.exp(lc - top)[..., None]
    assert (top - lse).abs().max() <= 2.0 ** -8
    _, _, tol = reference(b, q)
    # three kernel results, each within its tolerance of the definition
    assert ((joined - whole.float()).cpu().double().abs() <= 3 * tol + 2.0 ** -9 * joined.cpu().double().abs()).all()


def test_a_cache_beyond_32_bit_offsets():
    """Pages past 2^31 bytes of codes and rows."""
    from llm_accelerator_b200 import kv4
    pages, H, P, D = 4200, 32, 128, 128              # 1.1e9 bytes of codes for keys; rows at offsets past 2^31 / D
    big = 2 * pages
    codes = torch.zeros((big, H, P, D // 2), dtype=torch.uint8, device="cuda")      # 2.2e9 bytes
    words = torch.zeros((big, H, P), dtype=torch.int32, device="cuda")
    cache = kv4.Kv4Cache.from_tensors(codes, words, codes, words)                   # keys and values the same rows
    table, lens = _i32([[big - 1, big - 3]]), _i32([200])
    x = torch.randn((200, H, D), device="cuda").half()
    kv4.append(cache, x, x, table, lens, _i32([0, 200]))
    rk, rv = kv4.read(cache, table, lens, _i32([0, 200]), total=200)
    want = values(*pack(*quantise(x)))
    assert torch.equal(rk.cpu().double(), want) and torch.equal(rv.cpu().double(), want)
    q = queries(1, H, D, torch.float16)
    out = kv4.attention(q, cache, table, lens)
    s = torch.einsum("hd,nhd->hn", q[0].cpu().double(), want) * D ** -0.5
    ref = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), want)
    # weights rounded to FP16 once, scores good to 2^-10: a relative 2^-11 + 2^-9 of sum p |v|, and the output's rounding
    tol = (2.0 ** -11 + 2.0 ** -9) * torch.einsum("hn,nhd->hd", torch.softmax(s, -1), want.abs()) + 2.0 ** -11 * ref.abs()
    assert ((out[0].cpu().double() - ref).abs() <= tol).all()


def test_captured_calls_follow_their_inputs():
    """A decode step captured once, replayed while the sequences grow past a page's end; a second graph of another
    batch and eager calls in between, on another stream."""
    from llm_accelerator_b200 import kv4
    H, G, D, P = 2, 4, 64, 16
    cache = kv4.Kv4Cache(12, P, H, D)
    table, lens = _i32([[3, 0, 5], [8, 1, 9]]), _i32([14, 15])
    k = torch.randn((2, H, D), device="cuda").half()
    v, q = torch.randn_like(k), torch.randn((2, H * G, D), device="cuda").half()
    other = Batch([300, 40], H, D, P)
    oq = queries(2, H * G, D, torch.bfloat16)
    first = kv4.attention(oq, other.cache, other.d_table, other.d_lens)
    hist = torch.randn((29, H, D), device="cuda").half()
    kv4.append(cache, hist, hist, table, lens, _i32([0, 14, 29]))
    lens += 1
    torch.cuda.synchronize()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv4.append(cache, k, v, table, lens)
        out = kv4.attention(q, cache, table, lens)
    with torch.cuda.graph(graph2):
        out2 = kv4.attention(oq, other.cache, other.d_table, other.d_lens)
    side = torch.cuda.Stream()
    for step in range(4):
        k.copy_(torch.randn_like(k))
        v.copy_(torch.randn_like(v))
        q.copy_(torch.randn_like(q))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            graph2.replay()
            eager = kv4.attention(oq, other.cache, other.d_table, other.d_lens)
        torch.cuda.synchronize()
        assert torch.equal(out2, first) and torch.equal(eager, first)
        assert torch.equal(out, kv4.attention(q, cache, table, lens))
        ns = lens.tolist()
        rk, rv = kv4.read(cache, table, lens, _i32([0, ns[0], sum(ns)]), total=sum(ns))
        want = values(*pack(*quantise(k)))
        assert torch.equal(rk.cpu().double()[[ns[0] - 1, sum(ns) - 1]], want)
        for s, (a, e) in enumerate(((0, ns[0]), (ns[0], sum(ns)))):
            kk, vv = rk[a:e].double(), rv[a:e].double()
            for h in range(H * G):
                p = torch.softmax(q[s, h].double() @ kk[:, h // G].t() * D ** -0.5, -1)
                # weights rounded to FP16, scores good to 2^-12, the output's rounding
                tol = (2.0 ** -11 + 2.0 ** -11) * (p @ vv[:, h // G].abs()) + 2.0 ** -11 * (p @ vv[:, h // G]).abs()
                assert ((out[s, h].double() - p @ vv[:, h // G]).abs() <= tol).all()
        lens += 1


def test_malformed_offsets_stay_inside():
    """Offsets and lengths that no batch should have lead nowhere outside the tensors."""
    from llm_accelerator_b200 import kv4
    b = Batch([100, 50], 2, 64, 16)
    q = queries(10, 2, 64, torch.float16)
    x = torch.randn((10, 2, 64), device="cuda").half()
    for ptr, lens in (([5, 3, 50], [100, 50]), ([-4, 2, 10], [2 ** 31 - 1, -5]), ([0, 2 ** 31 - 1, 3], [100, 2 ** 30])):
        kv4.attention(q, b.cache, b.d_table, _i32(lens), _i32(ptr))
        kv4.append(b.cache, x, x, b.d_table, _i32(lens), _i32(ptr))
        kv4.read(b.cache, b.d_table, _i32(lens), _i32(ptr), total=10)
    # many sequences that all claim the same rows, contexts whole and shared out, by both kernels
    for hist, T, heads in (([40] * 300, 300, 2), ([40] * 299 + [3000], 300, 2), ([700] * 8, 9000, 6)):
        b = Batch(hist, heads, 64, 16)
        ptr = _i32([0, T] * (len(hist) // 2) + [0])
        assert kv4.attention(queries(T, heads, 64, torch.float16), b.cache, b.d_table, b.d_lens, ptr).shape == (T, heads, 64)
    torch.cuda.synchronize()


def test_first_calls_inside_a_capture():
    """In a fresh process the first append, attention (both kernels) and products are captured, then replayed."""
    code = textwrap.dedent(f"""
        import sys
        sys.path[:0] = [{str(ROOT)!r}, {str(ROOT / 'tests')!r}]
        import torch
        from llm_accelerator_b200 import gemm, kv4
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        g = torch.Generator(device="cuda").manual_seed(0)
        cache = kv4.Kv4Cache(80, 16, 4, 64)
        table = torch.arange(80, dtype=torch.int32, device="cuda").view(1, 80)
        k = torch.randn((1200, 4, 64), generator=g, device="cuda").half()
        q = torch.randn((1200, 16, 64), generator=g, device="cuda").half()
        lens, ptr = i32([1200]), i32([0, 1200])
        xs = [torch.randn((m, 256), generator=g, device="cuda").half() for m in (1, 40, 1024)]
        w, s = torch.randint(-127, 128, (5000, 256), dtype=torch.int8, device="cuda", generator=g), torch.rand(5000, generator=g, device="cuda")
        def calls():
            kv4.append(cache, k, k, table, lens, ptr)
            a = kv4.attention(q, cache, table, lens, ptr)
            return [a, kv4.attention(q[-1:], cache, table, lens), *(gemm.linear_w8a8(x, w, s) for x in xs)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = calls()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(got, calls()))
        assert all(t.isfinite().all() for t in got)
        print("ok")
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr


def test_nothing_to_do():
    from llm_accelerator_b200 import kv4
    b = Batch([0, 0], 2, 64, 16)
    q = queries(2, 4, 64, torch.float16)
    out, lse = kv4.attention(q, b.cache, b.d_table, b.d_lens, return_lse=True)
    assert not out.any() and (lse == float("-inf")).all()
    e = torch.empty((0, 4, 64), dtype=torch.float16, device="cuda")
    assert kv4.attention(e, b.cache, b.d_table, b.d_lens, _i32([0, 0, 0])).shape == (0, 4, 64)
    kv4.append(b.cache, e[:, :2], e[:, :2], b.d_table, b.d_lens, _i32([0, 0, 0]))
    k, _ = kv4.read(b.cache, b.d_table, b.d_lens, _i32([0, 0, 0]), total=3)
    assert not k.any()
