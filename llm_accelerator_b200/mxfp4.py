"""4-bit microscaled rows (MXFP4) and linear layers of them.

``Mxfp4``                    rows held as E2M1 codes with a power of two for each 32 columns
``quantize(X)``              floating-point rows to that form
``gemm(a, b)``               Y = A @ B^T (+ bias) of two operands in that form
``linear(X, w)``             the same product of floating-point rows, quantised in the call
``linear_workspace(M, K)``   workspace of linear calls

A block of 32 values along K (the last one may have fewer) has e = max(floor(log2 max |x|) - 2, -127) and stands for 2^e
times the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign: ties go to the even code, magnitudes above 6 to 6.  A block
that holds an infinity or a NaN stands for NaN.  Products are summed in float32 and rounded once.  A few channels much
larger than the rest take the steps of their whole block: rotate rows and weights by ``quarot.fwht_f16`` first where there
are such.

The calls are for inference: no gradient flows through them, also from tensors that require one.
"""
from __future__ import annotations

import torch

from . import _lib as L
from ._tensors import TYPES, call, empty, front, of_device, type_code

_U8, _F16, _F32 = torch.uint8, torch.float16, torch.float32
_quantize, _values, _gemm, _linear = (L.lib.tac_mxfp4_quantize, L.lib.tac_mxfp4_values, L.lib.tac_mxfp4_gemm,
                                      L.lib.tac_linear_mxfp4)
_ws_bytes = of_device(L.lib.tac_linear_mxfp4_workspace_bytes)


def _scale_shape(rows: int, cols: int):
    """[128 rows][128 columns][row % 32][row / 32 % 4][block]; an even number of column groups."""
    return -(-rows // 128), -(-cols // 256) * 2, 32, 4, 4


def _check_tensors(codes, scales, cols: int):
    if codes.dtype is not _U8 or scales.dtype is not _U8:
        raise TypeError("codes and scales must be uint8")
    shape = codes.shape
    if len(shape) != 2 or cols <= 0 or shape[1] != (cols + 31) // 32 * 16:
        raise ValueError(f"codes of {cols} columns must be [rows, {(cols + 31) // 32 * 16}], got {tuple(shape)}")
    if scales.shape != _scale_shape(shape[0], cols):
        raise ValueError(f"scales must be {_scale_shape(shape[0], cols)}, got {tuple(scales.shape)}")
    if not (codes.is_contiguous() and scales.is_contiguous()):
        raise ValueError("codes and scales must be contiguous")
    dev = codes.get_device()
    if dev < 0 or scales.get_device() != dev:
        raise ValueError("codes and scales must be on one CUDA device")
    if (codes.data_ptr() | scales.data_ptr()) & 15:
        raise ValueError("codes and scales must begin on 16-byte boundaries")


class Mxfp4:
    """`rows` rows of `cols` values: codes uint8 [rows, 16 blocks] (value 2j in the low, 2j + 1 in the high half of byte j),
    scales uint8 (the bytes e + 127, 255 for NaN) as the tensor cores take them.  ``from_tensors`` takes scale bytes
    [rows, blocks] and ``scale_bytes`` gives them back; blocks = cols / 32 rounded up.  Every call takes the tensors that
    codes and scales are then, so that a copy, a loaded one or one that was given other tensors works on its own."""

    def __init__(self, codes, scales, cols: int):
        _check_tensors(codes, scales, cols)
        self.codes, self.scales, self.cols = codes, scales, cols

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    @property
    def device(self):
        return self.codes.device

    @property
    def _index(self) -> int:
        return self.codes.get_device()

    @property
    def _pointers(self):
        return self.codes.data_ptr(), self.scales.data_ptr()

    def _now(self):
        """(rows, columns, device, addresses), checked."""
        _check_tensors(self.codes, self.scales, self.cols)
        return self.rows, self.cols, self._index, self._pointers

    @classmethod
    def from_tensors(cls, codes, scale_bytes, cols: int) -> "Mxfp4":
        """Of codes [rows, 16 blocks] and scale bytes [rows, blocks]; the scales are laid out once, here.  Columns from
        `cols` on of the last block must have the code 0."""
        if scale_bytes.dtype is not _U8:
            raise TypeError("scale_bytes must be uint8")
        rows, blocks = codes.shape[0] if codes.dim() == 2 else -1, (cols + 31) // 32
        if rows < 0 or scale_bytes.shape != (rows, blocks):
            raise ValueError(f"codes and scale_bytes must be [rows, {16 * blocks}] and [rows, {blocks}], got "
                             f"{tuple(codes.shape)} and {tuple(scale_bytes.shape)}")
        r, c = _scale_shape(rows, cols)[:2]
        laid = torch.zeros((r * 128, c * 4), dtype=_U8, device=scale_bytes.device)
        laid[:rows, :blocks] = scale_bytes
        return cls(codes, laid.view(r, 4, 32, c, 4).permute(0, 3, 2, 1, 4).contiguous(), cols)

    def scale_bytes(self):
        """uint8 [rows, blocks]."""
        r, c = self.scales.shape[:2]
        return self.scales.permute(0, 3, 2, 1, 4).reshape(r * 128, c * 4)[:self.rows, :(self.cols + 31) // 32]

    def values(self, dtype=_F32):
        """[rows, cols] that the codes stand for, rounded to `dtype`."""
        y = front.values((self.codes, self.scales), None, self.cols, None, dtype)
        if y is not None:
            return y
        M, K, dev, pointers = self._now()
        yt = TYPES.get(dtype)
        if yt is None:
            type_code(dtype, "dtype")
        y = empty((M, K), dtype, dev)
        if M:
            call("tac_mxfp4_values", _values, dev, *pointers, y.data_ptr(), yt, M, K)
        return y


def _rows(X):
    """(type, row stride, M, K, device) of floating-point rows X."""
    xt, shape, dev = TYPES.get(X.dtype), X.shape, X.get_device()
    if xt is None:
        type_code(X.dtype, "X")
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError(f"X must be [M, K], got {tuple(shape)}")
    M, K = shape
    ldx, step = X.stride()
    if step != 1 or ldx < K:
        if step != 1 and K > 1:
            raise ValueError(f"the rows of X must be contiguous, got strides {(ldx, step)}")
        if M > 1 and ldx < K:
            raise ValueError(f"rows of X overlap (stride {ldx}, {K} columns)")
        ldx = max(ldx, K)
    if dev < 0:
        raise ValueError("X must be on a CUDA device")
    return xt, ldx, M, K, dev


def quantize(X) -> Mxfp4:
    """X [M, K] (float32, float16 or bfloat16, contiguous rows at any row stride) in 4-bit form."""
    q = Mxfp4.__new__(Mxfp4)
    done = front.quantize(X)
    if done is not None:
        q.codes, q.scales, q.cols = done
        return q
    xt, ldx, M, K, dev = _rows(X)
    tiles, groups = (M + 127) // 128, (K + 255) // 256 * 2
    q.codes = empty((M, (K + 31) // 32 * 16), _U8, dev)
    q.scales = empty((tiles, groups, 32, 4, 4), _U8, dev, (groups * 512, 512, 16, 4, 1))
    q.cols = K
    if M:
        call("tac_mxfp4_quantize", _quantize, dev, X.data_ptr(), xt, ldx, *q._pointers, M, K)
    return q


def _result(w, M, K, dev, bias, out, dtype):
    """Checks of what both products share; (out, its type, N, w's addresses, bias pointer, bias type)."""
    N, cols, index, pointers = w._now()
    if cols != K or index != dev:
        raise ValueError(f"the operands must have one number of columns and one device, got {K} and {cols} columns")
    bp, bt = None, 0
    if bias is not None:
        bt = type_code(bias.dtype, "bias")
        if bias.shape != (N,) or not bias.is_contiguous() or bias.get_device() != dev:
            raise ValueError(f"bias must be a contiguous [{N}] tensor on the operands' device")
        bp = bias.data_ptr()
    yt = type_code(dtype, "out_dtype")
    if out is None:
        out = empty((M, N), dtype, dev)
    elif out.dtype is not dtype or out.shape != (M, N) or not out.is_contiguous() or out.get_device() != dev:
        raise ValueError(f"out must be a contiguous {dtype} [{M}, {N}] tensor on the operands' device")
    return out, yt, N, pointers, bp, bt


def gemm(a: Mxfp4, b: Mxfp4, bias=None, out_dtype=None, out=None):
    """Y [a.rows, b.rows] = A @ B^T (+ bias[n]); bias and output float32, float16 or bfloat16 (default: out's type, else
    float16)."""
    if out_dtype is None:
        out_dtype = _F16 if out is None else out.dtype
    if type(b) is Mxfp4:
        y = front.gemm((a.codes, a.scales), None, a.cols, None, (b.codes, b.scales), None, b.cols, None, bias, out_dtype, out)
        if y is not None:
            return y
    M, K, dev, rows = a._now()
    out, yt, N, channels, bp, bt = _result(b, M, K, dev, bias, out, out_dtype)
    if M and N:
        call("tac_mxfp4_gemm", _gemm, dev, *rows, *channels, bp, bt, out.data_ptr(), yt, M, N, K)
    return out


def linear(X, w: Mxfp4, bias=None, out=None, ws=None):
    """Y [M, N] in X's type = X [M, K] @ w^T (+ bias[n]), X quantised as ``quantize`` does.

    X float32, float16 or bfloat16 with contiguous rows at any row stride; out may be X's memory.  ws: a ``linear_workspace`` to reuse across
    calls on one stream; by default a call allocates its own where it needs one.  A block of X with an infinity or a NaN
    gives a row of NaN."""
    if type(w) is Mxfp4:
        y = front.linear(X, (w.codes, w.scales), None, w.cols, None, bias, out, ws)
        if y is not None:
            return y
    xt, ldx, M, K, dev = _rows(X)
    given = out
    out, yt, N, channels, bp, bt = _result(w, M, K, dev, bias, out, X.dtype)
    if M and N:
        if given is not None:
            x, y, e = X.data_ptr(), out.data_ptr(), X.element_size()
            if x < y + M * N * e and y < x + ((M - 1) * ldx + K) * e:   # one launch would read rows beside their results
                return gemm(quantize(X), w, bias, out.dtype, out)
        wp, wn = None, 0
        if ws is not None:
            if ws.get_device() != dev or ws.dtype is not _U8 or not ws.is_contiguous():
                raise ValueError("ws must be a linear_workspace on X's device")
        else:
            need = _ws_bytes(dev, M, N, K)
            ws = empty((need,), _U8, dev) if need else None
        if ws is not None:
            p = ws.data_ptr()
            wp = (p + 255) & ~255
            wn = max(ws.numel() - (wp - p), 0)
        call("tac_linear_mxfp4", _linear, dev, X.data_ptr(), xt, ldx, *channels, bp, bt, out.data_ptr(), yt, wp, wn, M, N, K)
    return out


def linear_workspace(M: int, K: int, device="cuda"):
    """A workspace for linear calls of at most M rows of K columns (calls that share one must not overlap)."""
    codes, scales = L.lib.tac_mxfp4_code_bytes(M, K), L.lib.tac_mxfp4_scale_bytes(M, K)
    return torch.empty((codes + 255) // 256 * 256 + (scales + 255) // 256 * 256 + 256, dtype=_U8, device=device)
