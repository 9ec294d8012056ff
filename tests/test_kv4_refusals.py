"""Arguments that the 4-bit cache's calls refuse, before any CUDA call (no GPU needed)."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from llm_accelerator_b200 import _lib as L
from llm_accelerator_b200 import kv4

P = 4096     # never dereferenced: the checks come first


def _cache(**bad):
    f = dict(k_codes=P, v_codes=P, k_params=P, v_params=P, num_pages=4, page_size=16, heads=2, head_dim=64)
    f.update(bad)
    return L.Kv4CacheRecord(*(f[n] for n, _ in L.Kv4CacheRecord._fields_))


def _seqs(table=P, lens=P, indptr=P, batch=2, width=300, total=5):
    return table, lens, indptr, batch, width, total


def _append(cache=None, seqs=None, K=P, ks=(128, 64), V=P, vs=(128, 64), t=L.TYPE_F16):
    return L.lib.tac_kv4_append(C.byref(cache or _cache()), *(seqs or _seqs()), K, *ks, V, *vs, t, None)


def _read(cache=None, seqs=None, K=P, V=P):
    return L.lib.tac_kv4_read(C.byref(cache or _cache()), *(seqs or _seqs()), K, V, None)


def _attn(cache=None, seqs=None, Q=P, qs=(256, 64), hq=4, t=L.TYPE_F16, O=P, lse=None, ws=P, wn=1 << 40):
    return L.lib.tac_kv4_attention(C.byref(cache or _cache()), *(seqs or _seqs()), Q, *qs, hq, t, 0.1, 1, O, lse, ws, wn,
                                   None)


BAD_CACHE = [dict(k_codes=None), dict(v_codes=None), dict(k_params=None), dict(v_params=None), dict(num_pages=0),
             dict(page_size=8), dict(page_size=48), dict(page_size=256), dict(heads=0), dict(head_dim=96),
             dict(k_codes=P + 8), dict(v_params=P + 4)]
BAD_SEQS = [dict(table=None), dict(lens=None), dict(batch=0), dict(width=0), dict(total=0), dict(indptr=None),
            dict(width=(1 << 26) + 1)]


@pytest.mark.parametrize("call", [_append, _read, _attn])
def test_cache_and_batch(call):
    for bad in BAD_CACHE:
        assert call(cache=_cache(**bad)) == L.E_ARGUMENT, bad
    for bad in BAD_SEQS:
        assert call(seqs=_seqs(**bad)) == L.E_ARGUMENT, bad


@pytest.mark.parametrize("bad", [dict(K=None), dict(V=None), dict(t=3), dict(ks=(-1, 64)), dict(vs=(128, -64)),
                                 dict(K=C.c_void_p(4097)), dict(V=C.c_void_p(4098), t=L.TYPE_F32)])
def test_append(bad):
    assert _append(**bad) == L.E_ARGUMENT


@pytest.mark.parametrize("bad", [dict(K=None), dict(V=None), dict(K=P + 4)])
def test_read(bad):
    assert _read(**bad) == L.E_ARGUMENT


@pytest.mark.parametrize("bad", [dict(Q=None), dict(O=None), dict(t=L.TYPE_F32), dict(hq=0), dict(hq=3), dict(qs=(-8, 64)),
                                 dict(ws=None), dict(ws=P + 16), dict(wn=0), dict(Q=P + 1), dict(lse=P + 2)])
def test_attention(bad):
    assert _attn(**bad) == L.E_ARGUMENT


def test_workspace_query():
    f = L.lib.tac_kv4_attention_workspace_bytes
    assert f(0, 99, 64, 1, 4, 2, 64) == 0 and f(1, 99, 64, 0, 4, 2, 64) == 0 and f(1, 99, 64, 1, 3, 2, 64) == 0
    assert f(1, 99, 64, 1, 4, 2, 80) == 0
    assert f(1, 16, 64, 1, 4, 2, 64) == 0            # short contexts are not split
    assert f(1, 99, 64, 4000, 32, 8, 64) == 0        # nor are prompts
    assert f(1, 99, 64, 1, 4, 2, 64) > 0 and f(1, 99, 64, 99, 4, 2, 64) > 0


def test_record_matches_the_header():
    assert C.sizeof(L.Kv4CacheRecord) == 48


class _Fake:
    """What the checks read of a cache, without a GPU."""
    heads, head_dim, page_size, device, _index = 2, 64, 16, torch.device("cpu"), -1


def test_python_checks():
    i32 = torch.int32
    table, lens = torch.zeros((2, 3), dtype=i32), torch.zeros(2, dtype=i32)
    q = torch.zeros((2, 4, 64), dtype=torch.float16)
    c = _Fake()
    with pytest.raises(ValueError):
        kv4.Kv4Cache(4, 24, 2, 64, device="cpu")
    with pytest.raises(ValueError):
        kv4.Kv4Cache(4, 16, 2, 80, device="cpu")
    with pytest.raises(ValueError):
        kv4.Kv4Cache(0, 16, 2, 64, device="cpu")
    with pytest.raises(ValueError):     # a cache lives on a GPU
        kv4.Kv4Cache(4, 16, 2, 64, device="cpu")
    with pytest.raises(TypeError):
        kv4.attention(q.float(), c, table, lens)
    with pytest.raises(ValueError):
        kv4.attention(q[:, :3], c, table, lens)
    with pytest.raises(ValueError):
        kv4.attention(q[..., :32], c, table, lens)
    with pytest.raises(ValueError):
        kv4.attention(q.transpose(1, 2).contiguous().transpose(1, 2), c, table, lens)
    with pytest.raises(TypeError):
        kv4.attention(q, c, table.long(), lens)
    with pytest.raises(ValueError):
        kv4.attention(q, c, table[:1], lens)
    with pytest.raises(ValueError):     # three rows, two sequences, no indptr
        kv4.attention(torch.zeros((3, 4, 64), dtype=torch.float16), c, table, lens)
    with pytest.raises(ValueError):
        kv4.attention(q, c, table, lens, torch.zeros(2, dtype=i32))
    with pytest.raises(ValueError):
        kv4.attention(q, c, table, lens, out=q.float())
    with pytest.raises(TypeError):
        kv4.append(c, q[:, :2], q[:, :2].bfloat16(), table, lens)
    with pytest.raises(ValueError):
        kv4.append(c, q, q, table, lens)
    with pytest.raises(ValueError):
        kv4.read(c, table, lens, torch.zeros(3, dtype=i32))
