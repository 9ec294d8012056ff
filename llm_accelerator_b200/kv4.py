"""4-bit paged key / value cache and attention over it (torch tensors as device-memory plumbing).

``Kv4Cache(pages, page_size, heads, head_dim)``  one layer's cache
``append(cache, k, v, page_table, lens)``        new tokens' keys and values quantised into it
``attention(q, cache, page_table, lens)``        attention of the new tokens over their sequences
``read(cache, page_table, lens)``                the values that the new tokens' rows stand for

A row x (one token, one head) stands for s (c - z) with lo = min(0, min x), hi = max(0, max x), s = bf16((hi - lo) / 15),
z = rint(-lo / s) and 4-bit codes c = clip(rint(x / s) + z, 0, 15).  Rows are quantised as they come: rotate queries and
keys by ``quarot.fwht_f16`` with block = head_dim first (the rotation cancels in their products) where a few channels
are much larger than the rest.

The three calls share their description of the batch.  page_table int32 [batch, width]: the page of each page_size
positions of a sequence; numbers outside [0, pages) stand for pages without tokens (never used, or given up).  lens
int32 [batch]: tokens of each sequence, the new ones included.  indptr int32 [batch + 1]: new tokens of sequence b are
rows indptr[b] .. indptr[b + 1) of k, v and q, the last of its positions; None: one new token a sequence, row b.  All
are device tensors that are read when the call runs, so a captured call follows them.

The calls are for inference: no gradient flows through them, also from tensors that require one.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib as L
from ._tensors import TYPES, call, type_code

_I32, _F32 = torch.int32, torch.float32
_append, _read, _attention = L.lib.tac_kv4_append, L.lib.tac_kv4_read, L.lib.tac_kv4_attention
_workspace_bytes = lru_cache(maxsize=1024)(L.lib.tac_kv4_attention_workspace_bytes)   # sizes alone decide

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


class Kv4Cache:
    """The cache of one layer: `num_pages` pages of `page_size` tokens, `heads` key-value heads of `head_dim` values.

    k_codes, v_codes uint8 [pages, heads, page_size, head_dim / 2] (code 2j in the low, 2j + 1 in the high half of
    byte j), k_params, v_params int32 [pages, heads, page_size] (the bits of s above those of z)."""

    def __init__(self, num_pages: int, page_size: int, heads: int, head_dim: int, device="cuda"):
        if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} and head_dim of {HEAD_DIMS}, got {page_size} "
                             f"and {head_dim}")
        if num_pages <= 0 or heads <= 0:
            raise ValueError("num_pages and heads must be positive")
        codes, words = (num_pages, heads, page_size, head_dim // 2), (num_pages, heads, page_size)
        self._set(torch.zeros(codes, dtype=torch.uint8, device=device),
                  torch.zeros(words, dtype=torch.int32, device=device),
                  torch.zeros(codes, dtype=torch.uint8, device=device),
                  torch.zeros(words, dtype=torch.int32, device=device))

    @classmethod
    def from_tensors(cls, k_codes, k_params, v_codes, v_params) -> "Kv4Cache":
        """A cache over tensors that the caller holds (a layer's slice of a larger allocation, a loaded prefix), each of
        which begins on a 16-byte boundary."""
        self = cls.__new__(cls)
        self._set(k_codes, k_params, v_codes, v_params)
        return self

    def _set(self, k_codes, k_params, v_codes, v_params):
        if any(t.data_ptr() & 15 for t in (k_codes, k_params, v_codes, v_params)):
            raise ValueError("the cache's tensors must begin on 16-byte boundaries")
        for c, p in ((k_codes, k_params), (v_codes, v_params)):
            if c.dtype != torch.uint8 or p.dtype != torch.int32:
                raise TypeError("codes must be uint8 and parameter words int32")
            if c.dim() != 4 or c.shape != k_codes.shape or p.shape != c.shape[:3] or not c.is_contiguous() \
                    or not p.is_contiguous():
                raise ValueError("codes must be contiguous [pages, heads, page_size, head_dim / 2] tensors with "
                                 "parameter words [pages, heads, page_size]")
            if c.device != k_codes.device or p.device != k_codes.device or c.device.type != "cuda":
                raise ValueError("the cache's tensors must be on one CUDA device")
        pages, heads, page_size, half = k_codes.shape
        if page_size not in PAGE_SIZES or 2 * half not in HEAD_DIMS or pages == 0 or heads == 0:
            raise ValueError(f"unsupported cache shape {tuple(k_codes.shape)}: page_size {PAGE_SIZES}, head_dim "
                             f"{HEAD_DIMS}")
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        self.num_pages, self.heads, self.page_size, self.head_dim = pages, heads, page_size, 2 * half
        self.device, self._index = k_codes.device, k_codes.get_device()
        self._record = L.Kv4CacheRecord(k_codes.data_ptr(), v_codes.data_ptr(), k_params.data_ptr(),
                                        v_params.data_ptr(), pages, page_size, heads, 2 * half)
        self._ref = L.C.addressof(self._record)


def _batch(cache, page_table, lens, indptr, total):
    """Checks of the batch's description; (page_table, lens, indptr, batch, width, total) as the C calls take them."""
    if page_table.dtype is not _I32 or lens.dtype is not _I32 or (indptr is not None and indptr.dtype is not _I32):
        raise TypeError("page_table, lens and indptr must be int32")
    shape = page_table.shape
    if len(shape) != 2 or lens.shape != shape[:1]:
        raise ValueError(f"page_table must be [batch, width] and lens [batch], got {tuple(shape)} and "
                         f"{tuple(lens.shape)}")
    batch, width = shape
    if width == 0:
        raise ValueError("page_table must have a column")
    if not (page_table.is_contiguous() and lens.is_contiguous()):
        raise ValueError("page_table and lens must be contiguous")
    dev = cache._index
    if page_table.get_device() != dev or lens.get_device() != dev:
        raise ValueError("page_table and lens must be on the cache's device")
    if indptr is None:
        if total != batch:
            raise ValueError(f"without indptr there is one row a sequence: {batch} sequences, {total} rows")
        return page_table.data_ptr(), lens.data_ptr(), None, batch, width, total
    if indptr.shape != (batch + 1,) or not indptr.is_contiguous() or indptr.get_device() != dev:
        raise ValueError(f"indptr must be a contiguous [{batch + 1}] tensor on the cache's device")
    return page_table.data_ptr(), lens.data_ptr(), indptr.data_ptr(), batch, width, total


def _rows(x, shape, heads, cache, what):
    """Checks of rows [rows, heads, head_dim]; their strides."""
    if len(shape) != 3 or shape[2] != cache.head_dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what} must be [rows, {heads or 'heads'}, {cache.head_dim}], got {tuple(shape)}")
    stride = x.stride()
    if stride[2] != 1:
        raise ValueError(f"the values of a head must be contiguous in {what}, got strides {stride}")
    if x.get_device() != cache._index:
        raise ValueError(f"{what} must be on the cache's device")
    return stride


def append(cache: Kv4Cache, k, v, page_table, lens, indptr=None) -> None:
    """Quantises the new tokens' k and v [rows, heads, head_dim] (float32, float16 or bfloat16, any row and head
    strides: slices of a fused projection will do) into the cache.  Rows without a place (before position 0, past
    the table, on a page number outside the cache, or of no sequence) are skipped.  No two rows of a call may have
    the same place, which only sequences that share a page could bring about."""
    t = type_code(k.dtype, "k")
    if v.dtype is not k.dtype:
        raise TypeError(f"k and v must have one type, got {k.dtype} and {v.dtype}")
    shape = k.shape
    if v.shape != shape:
        raise ValueError(f"k and v must have one shape, got {tuple(shape)} and {tuple(v.shape)}")
    ks = _rows(k, shape, cache.heads, cache, "k")
    vs = _rows(v, shape, cache.heads, cache, "v")
    total = shape[0]
    args = _batch(cache, page_table, lens, indptr, total)
    if total and args[3]:
        call("tac_kv4_append", _append, cache._index, cache._ref, *args, k.data_ptr(), ks[0], ks[1], v.data_ptr(),
             vs[0], vs[1], t)


def read(cache: Kv4Cache, page_table, lens, indptr=None, total=None):
    """(k, v) float32 [rows, heads, head_dim] that the new tokens' rows of the cache stand for; zeros for rows without
    a place.  total: the number of rows with indptr (a captured call cannot ask the device for it).  A whole prefix
    is read with indptr = 0, lens[0], lens[0] + lens[1], ..."""
    if total is None:
        if indptr is not None:
            raise ValueError("total is needed with indptr")
        total = lens.shape[0]
    args = _batch(cache, page_table, lens, indptr, total)
    k = torch.empty((total, cache.heads, cache.head_dim), dtype=_F32, device=cache.device)
    v = torch.empty_like(k)
    if total:
        if args[3]:
            call("tac_kv4_read", _read, cache._index, cache._ref, *args, k.data_ptr(), v.data_ptr())
        else:
            k.zero_()
            v.zero_()
    return k, v


def attention(q, cache: Kv4Cache, page_table, lens, indptr=None, *, scale=None, causal: bool = True,
              return_lse: bool = False, out=None):
    """Attention of the new tokens over the cached tokens of their sequences (append them first):
    out[i] = sum_j p_j v_j with p = softmax_j(scale q[i] . k_j), over the tokens up to the row's own position, or all
    tokens of the sequence with causal=False.

    q [rows, q_heads, head_dim] float16 or bfloat16, any row and head strides; query head h reads key-value head
    h // (q_heads // heads).  scale defaults to head_dim ** -0.5.  The result has q's type; with return_lse also
    float32 [rows, q_heads] log sum_j exp(scale q . k_j), by which parts of one attention can be joined.  A row that
    sees no token is zero (lse -inf); rows of no sequence are left as they are in `out`.  Weights times the values'
    scales are rounded to FP16, by at most 2^-11 of each (float16 results are 18 to 38 % further from exact ones than with
    float32 weights, bfloat16 ones as near); with scales above 2^107 (values of 10^33) they can overflow in calls of many
    rows."""
    dt = q.dtype
    if dt is not torch.float16 and dt is not torch.bfloat16:
        raise TypeError(f"q must be float16 or bfloat16, got {dt}")
    shape = q.shape
    qs = _rows(q, shape, None, cache, "q")
    total, hq, D = shape
    if hq == 0 or hq % cache.heads:
        raise ValueError(f"{hq} query heads over {cache.heads} key-value heads")
    args = _batch(cache, page_table, lens, indptr, total)
    if out is None:
        out = q.new_empty(shape)
    elif out.dtype is not dt or out.shape != shape or not out.is_contiguous() or out.get_device() != cache._index:
        raise ValueError(f"out must be a contiguous {dt} {tuple(shape)} tensor on q's device")
    lse = torch.empty((total, hq), dtype=_F32, device=cache.device) if return_lse else None
    if total and args[3]:
        need = _workspace_bytes(args[3], args[4], cache.page_size, total, hq, cache.heads, D)
        ws = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
        call("tac_kv4_attention", _attention, cache._index, cache._ref, *args, q.data_ptr(), qs[0], qs[1], hq,
             TYPES[dt], D ** -0.5 if scale is None else scale, causal, out.data_ptr(),
             None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), need)
    return (out, lse) if return_lse else out
