"""INT8 linear layers with a scale for each token and output channel (also reached as ``gemm.*``).

``gemm_i8_scaled``    y = (A @ Bt^T) * a_scale[m] * b_scale[n] (+ bias[n]) of INT8 operands
``linear_w8a8``       the same product of floating-point rows, each quantised to INT8 in the call
``linear_workspace``  workspace of linear_w8a8 calls
``pad_k16``           INT8 weights padded to whole groups of 16 columns

The products are for inference: no gradient flows through them, also from rows, scales or a bias that require one.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib as L
from ._tensors import TYPES, call, type_code

_I8, _F32, _F16 = torch.int8, torch.float32, torch.float16
_gemm, _linear = L.lib.tac_gemm_i8_scaled, L.lib.tac_linear_w8a8
_ws_bytes = lru_cache(maxsize=1024)(L.lib.tac_linear_w8a8_best_workspace_bytes)   # sizes alone decide


def _check(rows, Bt, b_scale, bias, out, out_dtype, M, K):
    """Checks of what both products share; (N, out, bias pointer, bias type)."""
    if Bt.dtype is not _I8 or (b_scale.dtype is not _F16 and b_scale.dtype is not _F32):
        raise TypeError("Bt must be int8 and b_scale float32 or float16")
    shape = Bt.shape
    if len(shape) != 2 or shape[1] != K:
        raise ValueError(f"Bt must be [N, {K}], got {tuple(shape)}")
    N = shape[0]
    if b_scale.shape != (N,):
        raise ValueError(f"b_scale must be [{N}], got {tuple(b_scale.shape)}")
    if not (Bt.is_contiguous() and b_scale.is_contiguous()):
        raise ValueError("Bt and b_scale must be contiguous")
    dev = rows.get_device()                       # -1 on the CPU
    if dev < 0 or Bt.get_device() != dev or b_scale.get_device() != dev:
        raise ValueError("the operands must be on one CUDA device")
    bp, bt = None, 0
    if bias is not None:
        bt = type_code(bias.dtype, "bias")
        if bias.shape != (N,) or not bias.is_contiguous() or bias.get_device() != dev:
            raise ValueError(f"bias must be a contiguous [{N}] tensor on the operands' device")
        bp = bias.data_ptr()
    if out is None:
        out = rows.new_empty((M, N), dtype=out_dtype)
    elif out.dtype is not out_dtype or out.shape != (M, N) or not out.is_contiguous() or out.get_device() != dev:
        raise ValueError(f"out must be a contiguous {out_dtype} [{M}, {N}] tensor on the operands' device")
    return N, out, bp, bt


def gemm_i8_scaled(A, Bt, a_scale, b_scale, bias=None, out_dtype=None, out=None):
    """Y [M, N] = (A int8 [M, K] @ Bt int8 [N, K]^T) * a_scale[m] * b_scale[n] (+ bias[n]).

    a_scale float32 [M], b_scale float32 or float16 [N] (``ptq.quantize_tensor`` gives Bt and b_scale,
    ``ptq.quantize_rows`` A and a_scale), bias and output float32, float16 or bfloat16 (default: out's type, else
    float16).  K a multiple of 16 (pad both operands with zero columns: ``pad_k16``), any M and N.  M or N of zero
    gives an empty result."""
    if A.dtype is not _I8 or a_scale.dtype is not _F32:
        raise TypeError("A must be int8 and a_scale float32")
    shape = A.shape
    if len(shape) != 2 or a_scale.shape != shape[:1]:
        raise ValueError(f"A must be [M, K] with a_scale [M], got {tuple(shape)} and {tuple(a_scale.shape)}")
    if not (A.is_contiguous() and a_scale.is_contiguous()):
        raise ValueError("A and a_scale must be contiguous")
    M, K = shape
    if out_dtype is None:
        out_dtype = _F16 if out is None else out.dtype
    yt = type_code(out_dtype, "out_dtype")
    if a_scale.get_device() != A.get_device():
        raise ValueError("the operands must be on one CUDA device")
    N, out, bp, bt = _check(A, Bt, b_scale, bias, out, out_dtype, M, K)
    if K == 0 or K % 16:
        raise ValueError(f"K must be a positive multiple of 16, got {K} (pad_k16 pads with zero columns)")
    if M and N:
        call("tac_gemm_i8_scaled", _gemm, A.get_device(), A.data_ptr(), Bt.data_ptr(), a_scale.data_ptr(),
             b_scale.data_ptr(), TYPES[b_scale.dtype], bp, bt, out.data_ptr(), yt, M, N, K)
    return out


def pad_k16(Q):
    """Q int8 [N, K] with zero columns appended up to a multiple of 16 (Q itself when there is nothing to add)."""
    pad = -Q.shape[1] % 16
    return torch.nn.functional.pad(Q, (0, pad)).contiguous() if pad else Q


def linear_w8a8(X, Bt, b_scale, bias=None, out=None, ws=None):
    """Y [M, N] in X's type = X [M, K] @ (Bt [N, K] * b_scale[n])^T (+ bias[n]) with INT8 products: each row of X is
    quantised by its own maximum (``ptq.quantize_rows``) in the call.

    X float32, float16 or bfloat16 with contiguous rows at any row stride; Bt int8 [N, K_pad], K_pad = K rounded up
    to 16 (``pad_k16``); b_scale and bias as in ``gemm_i8_scaled``.  Rotate X first (``quarot.fwht_f16``) where the
    weights are rotated.  ws: a ``linear_workspace`` to reuse across calls on one stream; by default a call
    allocates its own where it needs one.  A row with an infinity or a NaN gives a row of NaN."""
    xt = type_code(X.dtype, "X")
    shape, stride = X.shape, X.stride()
    if len(shape) != 2 or (shape[1] > 1 and stride[1] != 1):
        raise ValueError(f"X must be [M, K] with contiguous rows, got shape {tuple(shape)}, stride {stride}")
    M, K = shape
    if K == 0:
        raise ValueError("K must be positive")
    ldx = stride[0] if M > 1 else K
    if ldx < K:
        raise ValueError(f"rows of X overlap (stride {ldx}, {K} columns)")
    N, out, bp, bt = _check(X, Bt, b_scale, bias, out, X.dtype, M, (K + 15) // 16 * 16)
    if M and N:
        wp, wn = None, 0
        if ws is not None:
            if ws.get_device() != X.get_device() or ws.dtype is not torch.uint8 or not ws.is_contiguous():
                raise ValueError("ws must be a linear_workspace on X's device")
        else:
            need = _ws_bytes(M, N, K)
            ws = torch.empty(need + 256, dtype=torch.uint8, device=X.device) if need else None
        if ws is not None:
            p = ws.data_ptr()
            wp = (p + 255) & ~255
            wn = max(ws.numel() - (wp - p), 0)
        call("tac_linear_w8a8", _linear, X.get_device(), X.data_ptr(), xt, ldx, Bt.data_ptr(), b_scale.data_ptr(),
             TYPES[b_scale.dtype], bp, bt, out.data_ptr(), xt, wp, wn, M, N, K)
    return out


def linear_workspace(M: int, K: int, device="cuda"):
    """A workspace for linear_w8a8 calls of at most M rows of K columns (calls that share one must not overlap)."""
    codes, scales = M * ((K + 15) // 16 * 16), 4 * M
    return torch.empty((codes + 255) // 256 * 256 + (scales + 255) // 256 * 256 + 256, dtype=torch.uint8, device=device)
