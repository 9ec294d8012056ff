"""4-bit rows that are copied, pickled, given other tensors or moved: what they stand for and what is multiplied is in
their own tensors."""
from __future__ import annotations

import copy
import io
import pickle

import pytest
import torch

from llm_accelerator_b200 import mxfp4
from llm_accelerator_b200.errors import EngineError


def _on_host(rows, cols):
    """As an object that was loaded without a device."""
    w = mxfp4.Mxfp4.__new__(mxfp4.Mxfp4)
    w.codes = torch.randint(0, 256, (rows, (cols + 31) // 32 * 16), dtype=torch.uint8)
    w.scales = torch.full(mxfp4._scale_shape(rows, cols), 127, dtype=torch.uint8)
    w.cols = cols
    return w


def _through_a_file(w):
    f = io.BytesIO()
    torch.save(w, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


COPIES = [copy.deepcopy, copy.copy, lambda w: pickle.loads(pickle.dumps(w)), _through_a_file]


@pytest.mark.parametrize("copied", COPIES)
def test_addresses_are_the_copys_own(copied):
    w = _on_host(5, 40)
    c = copied(w)
    assert c._pointers == (c.codes.data_ptr(), c.scales.data_ptr())
    assert (c.rows, c.cols, c.device) == (5, 40, torch.device("cpu"))
    if copied is not copy.copy:
        assert c.codes.data_ptr() != w.codes.data_ptr() and torch.equal(c.codes, w.codes) and torch.equal(c.scales, w.scales)


def test_other_tensors_are_taken_at_the_next_call():
    w = _on_host(5, 40)
    w.codes = w.codes.clone()
    w.scales = w.scales.clone()
    assert w._pointers == (w.codes.data_ptr(), w.scales.data_ptr())
    w.codes = torch.zeros((7, 32), dtype=torch.uint8)
    assert w.rows == 7


def test_what_a_file_of_an_earlier_version_held():
    """Addresses, rows and a device index beside the tensors."""
    w = mxfp4.Mxfp4.__new__(mxfp4.Mxfp4)
    w.__dict__.update(_on_host(5, 40).__dict__, rows=6, _index=3, _pointers=(16, 32))
    assert w._pointers == (w.codes.data_ptr(), w.scales.data_ptr()) and w.rows == 5 and w._index == -1


def test_rows_on_the_host_are_refused():
    """Their addresses are not the device's."""
    w = _on_host(5, 40)
    with pytest.raises(ValueError):
        w.values()
    with pytest.raises(ValueError):
        mxfp4.gemm(w, w)


@pytest.mark.gpu
@pytest.mark.parametrize("copied", COPIES)
def test_products_of_copies(copied):
    g = torch.Generator().manual_seed(3)
    x = torch.randn((3, 96), generator=g).cuda()
    w = mxfp4.quantize(torch.randn((50, 96), generator=g).cuda())
    a = mxfp4.quantize(x)
    want = w.values().clone(), mxfp4.linear(x, w), mxfp4.gemm(a, w), mxfp4.gemm(w, a)
    c = copied(w)
    if copied is not copy.copy:
        w.codes.zero_()
        w.scales.zero_()
    del w
    torch.cuda.synchronize()
    other = [torch.full((50 * 48,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]   # where the first one's were
    for got, y in zip((c.values(), mxfp4.linear(x, c), mxfp4.gemm(a, c), mxfp4.gemm(c, a)), want):
        assert torch.equal(got, y)
    del other


@pytest.mark.gpu
def test_products_after_an_assignment():
    g = torch.Generator().manual_seed(4)
    x = torch.randn((200, 96), generator=g).cuda()
    one, two = (mxfp4.quantize(torch.randn((50, 96), generator=g).cuda()) for _ in range(2))
    want = two.values(), mxfp4.linear(x, two), mxfp4.linear(x[:1], two)
    one.codes, one.scales = two.codes, two.scales
    for got, y in zip((one.values(), mxfp4.linear(x, one), mxfp4.linear(x[:1], one)), want):
        assert torch.equal(got, y)
    one.codes = two.codes[:30].clone()               # of the same tiles of scales
    assert mxfp4.linear(x, one).shape == (200, 30) and torch.equal(mxfp4.linear(x, one), want[1][:, :30])
    for bad in (two.codes[:, :32], two.codes.cpu(), two.codes.int(), two.codes.t(), torch.zeros((129, 48), dtype=torch.uint8, device="cuda")):
        one.codes = bad
        for call in (one.values, lambda: mxfp4.linear(x, one), lambda: mxfp4.gemm(one, two), lambda: mxfp4.gemm(two, one)):
            with pytest.raises((TypeError, ValueError)):
                call()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 200])
def test_out_and_workspace(M):
    """The same tensor comes back, with what a call without it gives; those that do not fit are refused."""
    g = torch.Generator().manual_seed(M)
    x, w = torch.randn((M, 96), generator=g).cuda(), mxfp4.quantize(torch.randn((50, 96), generator=g).cuda())
    a, want = mxfp4.quantize(x), mxfp4.linear(x, w)
    y, ws = torch.full((M, 50), 7.0, device="cuda"), mxfp4.linear_workspace(M, 96)
    assert mxfp4.linear(x, w, out=y) is y and torch.equal(y, want)
    for space in (ws, ws[1:], None):
        y.fill_(7.0)
        assert mxfp4.linear(x, w, out=y, ws=space) is y and torch.equal(y, want)
        assert torch.equal(mxfp4.linear(x, w, ws=space), want)
    half = torch.empty((M, 50), dtype=torch.float16, device="cuda")
    assert mxfp4.gemm(a, w, out=half) is half and torch.equal(half, mxfp4.gemm(a, w))
    assert mxfp4.gemm(a, w, out=y, out_dtype=torch.float32) is y and torch.equal(y, want)
    for bad in (half, y[:, :40], torch.empty((M + 1, 50), device="cuda"), y.cpu(), torch.empty((50, M + 1), device="cuda").t()):
        with pytest.raises(ValueError):
            mxfp4.linear(x, w, out=bad)
    with pytest.raises(ValueError):
        mxfp4.gemm(a, w, out=half, out_dtype=torch.float32)
    for bad in (ws.cpu(), ws.int(), ws[::2]):
        with pytest.raises(ValueError):
            mxfp4.linear(x, w, ws=bad)
    if M > 64:
        with pytest.raises(EngineError):
            mxfp4.linear(x, w, ws=ws[:300])


@pytest.mark.gpu
@pytest.mark.parametrize("M,K", [(1, 1024), (40, 512), (64, 4096), (300, 768)])
def test_results_over_the_rows(M, K):
    g = torch.Generator().manual_seed(K)
    w = mxfp4.quantize(torch.randn((K, K), generator=g).cuda())
    for dtype in (torch.bfloat16, torch.float32):
        for at in (0, 8):
            space = torch.randn(M * K + 64, generator=g).to(dtype).cuda()
            x, y = space[:M * K].view(M, K), space[at:at + M * K].view(M, K)
            want = mxfp4.gemm(mxfp4.quantize(x), w, out_dtype=dtype)
            assert mxfp4.linear(x, w, out=y) is y and torch.equal(y, want)
