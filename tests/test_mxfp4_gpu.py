"""4-bit microscaled rows: quantiser, values, products and linear layers, against their definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

from mxfp4_helpers import GRID, on_device, pack, quantise, random_rows, values

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


# ---- rows -----------------------------------------------------------------------------------------------------------
def _check_rows(x):
    from llm_accelerator_b200 import mxfp4
    q = mxfp4.quantize(x)
    codes, scales = quantise(x)
    assert torch.equal(q.scale_bytes().cpu().long(), scales)
    assert torch.equal(q.codes.cpu(), pack(codes))
    want = values(codes, scales, x.shape[1])
    for dtype in (F32, x.dtype):
        got = q.values(dtype)
        assert torch.equal(got.cpu().isnan(), want.isnan())
        assert torch.equal(got.cpu().nan_to_num(nan=7.0), want.to(dtype).nan_to_num(nan=7.0))
    return q


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,K,pad", [(1, 1, 0), (3, 31, 0), (2, 32, 0), (5, 33, 0), (129, 64, 8), (31, 255, 1), (4, 256, 0),
                                     (200, 257, 0), (33, 1600, 64), (130, 1000, 5), (1, 8192, 0), (300, 768, 0)])
def test_quantize(M, K, pad, dtype):
    g = torch.Generator().manual_seed(M + K)
    x = torch.randn((M, K + pad), generator=g) * torch.exp(2 * torch.randn((M, 1), generator=g))
    x[:, ::7] *= 30
    _check_rows(x.to(dtype).cuda()[:, :K])


def test_every_tie_and_every_float16():
    # next to the borders between codes, at every power of two that the block's largest value can bring
    steps = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.0, 7.999])
    rows = []
    for e in (-20, -3, 0, 5, 12):
        for up in (1.0, 1.0 - 2.0 ** -11, 1.0 + 2.0 ** -10):
            row = torch.zeros(32)
            row[:10], row[10:20], row[31] = steps * up, -steps * up, 4.0
            rows.append(row * 2.0 ** e)
    for dtype in (F16, BF16, F32):
        _check_rows(torch.stack(rows).to(dtype).cuda())
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(F16).view(-1, 32)
    _check_rows(every.cuda())
    _check_rows(every.t().contiguous().cuda())
    _check_rows(torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(BF16).view(64, -1).cuda())


def test_blocks_of_zeros_and_of_the_smallest_and_largest_values():
    x = torch.zeros((9, 96))
    x[1, 5] = 2.0 ** -149                          # float32's smallest
    x[2, 40] = 2.0 ** -126
    x[3, 64:] = 3.4e38
    x[4, 3] = float("inf")
    x[5, 70] = float("nan")
    x[6, 33] = -float("inf")
    x[7, :32] = 2.0 ** -125
    x[8, 32:64] = -1.5 * 2.0 ** -124
    q = _check_rows(x.cuda())
    assert q.scale_bytes()[4].tolist() == [255, 0, 0] and q.scale_bytes()[5].tolist() == [0, 0, 255]


def test_scale_bytes_go_in_and_out():
    from llm_accelerator_b200 import mxfp4
    for M, K in ((1, 5), (130, 300), (256, 512)):
        codes, scales = random_rows(M, K, M)
        q = on_device(codes, scales, K)
        assert torch.equal(q.scale_bytes().cpu().long(), scales)
        again = mxfp4.Mxfp4(q.codes, q.scales, K)
        assert torch.equal(again.values().cpu().double(), values(codes, scales, K))
    x = torch.randn((70, 200), device="cuda")
    q = mxfp4.quantize(x)
    assert torch.equal(mxfp4.Mxfp4.from_tensors(q.codes, q.scale_bytes(), 200).values(), q.values())
    assert mxfp4.quantize(x[:0]).values().shape == (0, 200)


# ---- products -------------------------------------------------------------------------------------------------------
def _sum_room(a, b, K):
    """Room of a float32 sum of K exact products, a rounding (of a whole step: the tensor cores may cut off) for each block
    of 32 and four more."""
    return (K / 32 + 4) * 2.0 ** -23 * (a.abs() @ b.abs().t())


def _near(got, want, room, dtype):
    top = torch.finfo(dtype).max
    small = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -150}[dtype]
    assert torch.equal(got.cpu().isnan(), want.isnan())
    fine = ~want.isnan() & (want.abs() + room < top)
    d = (got.cpu().double() - want).abs()[fine]
    room = (room + torch.finfo(dtype).eps / 2 * (want.abs() + room))[fine] + small
    assert bool((d <= room).all()), float((d / room).max())


# (M, N, K): every number of tokens a tile can have and one more, ragged channels and columns, split and unsplit sums,
# one tile and several for each CTA
SIZES = [(1, 1, 1), (1, 17, 32), (3, 128, 33), (16, 129, 64), (5, 300, 96), (17, 64, 256), (32, 257, 255), (33, 100, 257),
         (1, 4096, 1024), (16, 512, 4096), (2, 1000, 8192), (64, 384, 2048), (65, 130, 300), (100, 1111, 513), (128, 128, 128),
         (129, 50, 40), (200, 1025, 777), (256, 2048, 512), (333, 5001, 768), (600, 640, 1000), (1000, 999, 256),
         (1, 50257, 768), (40, 20000, 96), (2500, 300, 64), (1025, 4097, 320), (4097, 257, 1280)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_products_that_are_exact(M, N, K):
    """Scales of 2^-1 to 2^1: every partial sum is a multiple of 2^-4 below 2^20 and so exact in float32, whatever the order:
    codes, scales and places are right or the results are not equal."""
    from llm_accelerator_b200 import mxfp4
    a, sa = random_rows(M, K, 1, 126, 128)
    b, sb = random_rows(N, K, 2, 126, 128)
    want = values(a, sa, K).cuda() @ values(b, sb, K).t().cuda()
    got = mxfp4.gemm(on_device(a, sa, K), on_device(b, sb, K), out_dtype=F32)
    assert torch.equal(got.double(), want)


# Tiles of 64, 128, 192 and 256 tokens on pairs of CTAs, in one round and (the last three) in more than two, with token tiles
# that begin inside a piece of scales, ragged last tiles, and 16-bit rows that begin between two words
PAIRS = [(200, 4000, 320), (100, 4096, 512), (128, 3001, 96), (195, 19035, 96), (513, 15225, 288), (386, 19018, 544), (700, 13001, 1030),
         (1537, 6000, 200), (4100, 2050, 64)]


@pytest.mark.parametrize("M,N,K", PAIRS)
def test_products_on_pairs(M, N, K):
    from llm_accelerator_b200 import mxfp4
    a, sa = random_rows(M, K, 11, 126, 128)
    b, sb = random_rows(N, K, 12, 126, 128)
    want = values(a, sa, K).cuda() @ values(b, sb, K).t().cuda()
    qa, qb = on_device(a, sa, K), on_device(b, sb, K)
    assert torch.equal(mxfp4.gemm(qa, qb, out_dtype=F32).double(), want)
    bias = torch.arange(N, device="cuda").remainder(64).float()
    # exact before the one rounding
    assert torch.equal(mxfp4.gemm(qa, qb, bias=bias, out_dtype=BF16), (want + bias.double()).to(BF16))
    out = torch.full((M + 1, N), -3.0, dtype=F16, device="cuda")
    mxfp4.gemm(qa, qb, out=out[:M])
    assert torch.equal(out[:M], want.to(F16)) and (out[M] == -3).all()


@pytest.mark.parametrize("M,N,K", SIZES)
def test_products(M, N, K):
    from llm_accelerator_b200 import mxfp4
    a, sa = random_rows(M, K, 3)
    b, sb = random_rows(N, K, 4, 100, 127)
    A, B = values(a, sa, K), values(b, sb, K)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(5))
    qa, qb = on_device(a, sa, K), on_device(b, sb, K)
    room, want = _sum_room(A.cuda(), B.cuda(), K).cpu(), (A.cuda() @ B.cuda().t()).cpu()
    for dtype in (F32, F16, BF16):
        _near(mxfp4.gemm(qa, qb, out_dtype=dtype), want, room, dtype)
        added = bias.to(dtype)
        _near(mxfp4.gemm(qa, qb, bias=added.cuda(), out_dtype=dtype), want + added.double(),
              room + 2.0 ** -24 * (want.abs() + added.double().abs()), dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,N,K", [s for s in SIZES if s[0] * s[1] * s[2] < 2 ** 30])
def test_linear(M, N, K, dtype):
    from llm_accelerator_b200 import mxfp4
    g = torch.Generator().manual_seed(M)
    x = (torch.randn((M, K + 8), generator=g) * 3).to(dtype).cuda()[:, :K]
    b, sb = random_rows(N, K, 6, 115, 120)
    bias = torch.randn(N, generator=g)
    A, B = values(*quantise(x), K), values(b, sb, K)
    room, want = _sum_room(A, B, K), A @ B.t()
    w = on_device(b, sb, K)
    _near(mxfp4.linear(x, w), want, room, dtype)
    got = mxfp4.linear(x, w, bias=bias.cuda())
    _near(got, want + bias.double(), room + 2.0 ** -24 * (want.abs() + bias.double().abs()), dtype)
    ws = mxfp4.linear_workspace(M, K)
    out = torch.empty_like(got)
    assert mxfp4.linear(x, w, bias=bias.cuda(), ws=ws, out=out) is out and torch.equal(out, got)
    # rows that are not aligned to 16 bytes
    y = torch.empty((M, K + 3), dtype=dtype, device="cuda")[:, 1:K + 1]
    y.copy_(x)
    assert torch.equal(mxfp4.linear(y, w, bias=bias.cuda()), got)


@pytest.mark.parametrize("M", [1, 20, 200, 600])
def test_blocks_without_numbers_reach_their_rows_and_channels_only(M):
    from llm_accelerator_b200 import mxfp4
    K, N = 300, 260
    g = torch.Generator().manual_seed(9)
    x = torch.randn((M, K), generator=g).half().cuda()
    b, sb = random_rows(N, K, 7, 115, 120)
    clean = mxfp4.linear(x, on_device(b, sb, K))
    x[M // 2, 290] = float("inf")
    sb[5, 3] = 255
    y = mxfp4.linear(x, on_device(b, sb, K))
    bad = torch.zeros((M, N), dtype=torch.bool, device="cuda")
    bad[M // 2], bad[:, 5] = True, True
    assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], clean[~bad])


@pytest.mark.parametrize("M,N,K", [(1, 333, 512), (48, 256, 2048), (700, 513, 160)])
def test_outputs_at_any_alignment(M, N, K):
    import ctypes as C
    from llm_accelerator_b200 import _lib as L
    from llm_accelerator_b200 import mxfp4
    a, sa = random_rows(M, K, 1, 126, 128)
    b, sb = random_rows(N, K, 2, 126, 128)
    qa, qb = on_device(a, sa, K), on_device(b, sb, K)
    want = mxfp4.gemm(qa, qb, out_dtype=BF16)
    for off in (1, 2, 3, 7):
        buf = torch.full((M * N + 16,), -5.0, dtype=BF16, device="cuda")
        s = L.lib.tac_mxfp4_gemm(*(C.c_void_p(p) for p in (*qa._pointers, *qb._pointers)), None, 0,
                                 C.c_void_p(buf.data_ptr() + 2 * off), L.TYPE_BF16, M, N, K, None)
        torch.cuda.synchronize()
        assert s == L.OK
        assert torch.equal(buf[off:off + M * N].view(M, N), want)
        assert (buf[:off] == -5).all() and (buf[off + M * N:] == -5).all()


def test_results_do_not_depend_on_the_call():
    from llm_accelerator_b200 import mxfp4
    for M, N, K in ((1, 4096, 4096), (40, 512, 4096), (300, 1024, 1024)):
        x = torch.randn((M, K), device="cuda").half()
        w = mxfp4.quantize(torch.randn((N, K), device="cuda"))
        first = mxfp4.linear(x, w)
        assert all(torch.equal(mxfp4.linear(x, w), first) for _ in range(5))
        assert torch.equal(mxfp4.gemm(mxfp4.quantize(x), w), first)


def test_another_stream_and_a_captured_call():
    from llm_accelerator_b200 import mxfp4
    for M in (4, 150):
        x = torch.randn((M, 1024), device="cuda").half()
        w = mxfp4.quantize(torch.randn((768, 1024), device="cuda"))
        want = mxfp4.linear(x, w)
        a = torch.zeros_like(x)
        mxfp4.linear(a, w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = mxfp4.linear(a, w)
            z = mxfp4.gemm(mxfp4.quantize(a), w)
        a.copy_(x)
        graph.replay()
        assert torch.equal(y, want) and torch.equal(z, want)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            y = mxfp4.linear(x, w)
        stream.synchronize()
        assert torch.equal(y, want)


def test_empty_operands_and_no_device_faults():
    from llm_accelerator_b200 import _lib as L
    from llm_accelerator_b200 import mxfp4
    w = mxfp4.quantize(torch.randn((40, 64), device="cuda"))
    x = torch.randn((3, 64), device="cuda").half()
    assert mxfp4.linear(x[:0], w).shape == (0, 40)
    assert mxfp4.linear(x, mxfp4.quantize(torch.randn((0, 64), device="cuda"))).shape == (3, 0)
    assert mxfp4.gemm(mxfp4.quantize(x[:0]), w).shape == (0, 40)
    assert L.lib.tac_gemm_status(None) == L.OK


def test_grid_of_values():
    """Every code at every scale byte."""
    codes = torch.arange(16).repeat(255, 2)
    scales = torch.arange(255)[:, None]
    got = on_device(codes, scales, 32).values().cpu().double()
    want = (GRID * torch.exp2(scales.double() - 127)).float().double()    # 2^128 and more is infinite in float32
    assert torch.equal(got[:, :8], want) and torch.equal(got[:, 8:16], -want)


@pytest.mark.parametrize("M", [1, 100, 300])
@pytest.mark.parametrize("one,other", [(0, 254), (254, 0), (1, 253), (20, 234), (127, 0), (0, 127), (200, 30)])
def test_products_at_the_ends_of_the_scales(M, one, other):
    """2^-127 is half of float32's smallest normal number as a scale, and no less a scale for it."""
    from llm_accelerator_b200 import mxfp4
    K, N = 96, 300
    a, _ = random_rows(M, K, 21)
    b, _ = random_rows(N, K, 22)
    sa, sb = torch.full((M, 3), one), torch.full((N, 3), other)
    want = (values(a, sa, K) @ values(b, sb, K).t()).float()
    got = mxfp4.gemm(on_device(a, sa, K), on_device(b, sb, K), out_dtype=F32).cpu()
    # sums of a few multiples of one step are exact; below float32's normal numbers they may be taken for zero
    tiny = want.abs() < 2.0 ** -126
    assert torch.equal(got[~tiny], want[~tiny]) and bool((got[tiny].abs() < 2.0 ** -126).all())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,N,K", [(133, 22, 512), (4700, 60, 100), (300, 9000, 768), (66, 31, 6144), (67, 33, 6400), (200, 60, 8192),
                                   (85, 301, 7000), (40, 260, 2048), (64, 100, 4096), (50, 129, 1500), (33, 600, 3000)])
def test_linear_calls_behind_each_other(M, N, K, dtype):
    """Few channels, K shared by CTAs or by none, tiles of 16 to 256 tokens, pairs with and without a tile; each call starts
    while the one before it ends."""
    from llm_accelerator_b200 import mxfp4
    g = torch.Generator().manual_seed(M + N)
    x = torch.randn((M, K), generator=g).to(dtype)
    b, sb = random_rows(N, K, 3, 115, 120)
    bias = torch.randn(N, generator=g)
    A, B = values(*quantise(x), K), values(b, sb, K)
    room, want = _sum_room(A, B, K), A @ B.t() + bias.double()
    room = room + 2.0 ** -23 * (want.abs() + bias.double().abs())
    w, x, bias = on_device(b, sb, K), x.cuda(), bias.cuda()
    flipped = x.flip(0).contiguous()
    got = [mxfp4.linear(x if i % 2 == 0 else flipped, w, bias=bias) for i in range(6)]
    _near(got[0], want, room, dtype)
    for i, y in enumerate(got):
        assert torch.equal(y if i % 2 == 0 else y.flip(0), got[0])
