"""Root-mean-square norm of rows, with the residual's addition before it and INT8 rows after it.

``rms_norm(x, weight, eps)``      y = h / sqrt(mean(h^2) + eps) * weight with h = x (+ residual), in x's type
``rms_norm_i8(x, weight, eps)``   the same as INT8 codes with a scale for each row: the A operand and a_scale of
                                  ``gemm.gemm_i8_scaled``

Sums and the norm are float32, of the unrounded h; y is rounded once.  Where the residual stream is rotated
(``ptq.rotate_residual_stream_state_dict``), a norm without a channel's own weight commutes with the rotation.

The calls are for inference: no gradient flows through them, also from tensors that require one.
"""
from __future__ import annotations

import torch

from . import _lib as L
from ._tensors import TYPES, call, empty, front, type_code

_norm, _norm_i8 = L.lib.tac_rms_norm, L.lib.tac_rms_norm_i8
_I8, _F32 = torch.int8, torch.float32


def _row_stride(x, dtype, shape, dev, what):
    """Row stride of x, which is to be a [M, K] tensor of this type with contiguous rows on device `dev`."""
    if x.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype} as x, got {x.dtype}")
    if x.shape != shape or x.get_device() != dev:
        raise ValueError(f"{what} must be {tuple(shape)} on x's device, got {tuple(x.shape)} on {x.device}")
    M, K = shape
    row, step = x.stride()
    if step == 1 and row >= K:
        return row
    if step != 1 and K > 1:
        raise ValueError(f"the rows of {what} must be contiguous, got strides {(row, step)}")
    if M > 1 and row < K:
        raise ValueError(f"rows of {what} overlap (stride {row}, {K} columns)")
    return max(row, K)


def _args(x, weight, eps, residual, residual_out):
    """Checks of what both norms share; (device, M, K, arguments of the C call up to eps, the new residual)."""
    dtype, shape, dev, wt = x.dtype, x.shape, x.get_device(), TYPES.get(weight.dtype)
    xt = TYPES.get(dtype)
    if xt is None or wt is None:
        type_code(dtype, "x"), type_code(weight.dtype, "weight")
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError(f"x must be [M, K], got {tuple(shape)}")
    if dev < 0:
        raise ValueError("x must be on a CUDA device")
    M, K = shape
    if weight.shape != shape[1:] or weight.get_device() != dev or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous [{K}] tensor on x's device")
    if not 0 <= eps <= 1e30:
        raise ValueError(f"eps must not be negative, got {eps}")
    ldx = _row_stride(x, dtype, shape, dev, "x")
    if residual is None:
        if residual_out is not None:
            raise ValueError("residual_out without a residual")
        return dev, M, K, (x.data_ptr(), xt, ldx, None, 0, None, 0, weight.data_ptr(), wt, eps), None
    ldr, ldh = _row_stride(residual, dtype, shape, dev, "residual"), K
    if residual_out is None:
        residual_out = empty((M, K), dtype, dev)
    else:
        ldh = _row_stride(residual_out, dtype, shape, dev, "residual_out")
    return dev, M, K, (x.data_ptr(), xt, ldx, residual.data_ptr(), ldr, residual_out.data_ptr(), ldh, weight.data_ptr(), wt,
                       eps), residual_out


def rms_norm(x, weight, eps: float = 1e-6, residual=None, residual_out=None, out=None):
    """y [M, K] in x's type; with a residual (y, h), h = x + residual rounded to that type.

    x, residual and residual_out [M, K] float32, float16 or bfloat16 with contiguous rows at any row stride; weight [K]
    of any of these types.  residual_out: where h goes, by default a new tensor; it may be `residual` or x itself, but
    may not overlap them otherwise.  out: y's tensor, which may be x or the residual (of one row stride, K).  A row whose h^2
    add up to more than float32 holds (values of 10^18) is zero; with an eps of 0 one whose h^2 are too small for it (values
    below 10^-19) loses places, and below 10^-23 is infinite.  An infinity makes NaN of its own place, a NaN of its whole
    row."""
    if residual_out is None and out is None:
        result = front.rms_norm(x, weight, eps, residual)
        if result is not None:
            return result
    dev, M, K, args, h = _args(x, weight, eps, residual, residual_out)
    if out is None:
        out = empty((M, K), x.dtype, dev)
    elif out.dtype is not x.dtype or out.shape != x.shape or not out.is_contiguous() or out.get_device() != dev:
        raise ValueError(f"out must be a contiguous {x.dtype} [{M}, {K}] tensor on x's device")
    elif h is not None and out.data_ptr() == h.data_ptr() and M:
        raise ValueError("out and residual_out must not be one tensor")
    if M:
        call("tac_rms_norm", _norm, dev, *args, out.data_ptr(), M, K)
    return out if h is None else (out, h)


def rms_norm_i8(x, weight, eps: float = 1e-6, residual=None, residual_out=None):
    """(codes int8 [M, K_pad], scale float32 [M]) of y as ``rms_norm`` defines it, unrounded; with a residual (codes,
    scale, h).  t = max(max |y|, 1e-8), scale = t / 127, code = rint(y * (127 / t)) as in ``ptq.quantize_rows``; K_pad = K
    rounded up to 16, padding columns zero.  A row of y that holds an infinity or a NaN gets the scale NaN.
    ``ptq.dequantize_rows`` gives the values back."""
    if residual_out is None:
        result = front.rms_norm_i8(x, weight, eps, residual)
        if result is not None:
            return result
    dev, M, K, args, h = _args(x, weight, eps, residual, residual_out)
    q, scale = empty((M, (K + 15) // 16 * 16), _I8, dev), empty((M,), _F32, dev)
    if M:
        call("tac_rms_norm_i8", _norm_i8, dev, *args, q.data_ptr(), scale.data_ptr(), M, K)
    return (q, scale) if h is None else (q, scale, h)
