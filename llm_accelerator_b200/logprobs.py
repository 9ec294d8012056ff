"""Log-probabilities of given tokens, entropy and the likeliest tokens of rows of logits.

``token_logprobs(logits, tokens, top)``  all of these in one read of the logits

``runner.BatchedRunner.token_logprobs`` gives them for the logits of its last step.  The call is for inference: no
gradient flows through it, also from logits that require one.
"""
from __future__ import annotations

import torch

from . import _lib as L
from ._tensors import TYPES, call, empty, front, type_code

_logprobs = L.lib.tac_token_logprobs
_F32, _I32, _I64 = torch.float32, torch.int32, torch.int64

MOST_TOP = 32


def token_logprobs(logits, tokens, top: int = 0):
    """(logprob float32 [M], entropy float32 [M]), and with top > 0 also (top_logprobs float32 [M, top], top_ids int32
    [M, top]), of the softmax of each row of logits.

    logits [M, V] float32, float16 or bfloat16 with contiguous rows at any row stride; tokens [M] int32 or int64.
    logprob[i] = log softmax(logits[i])[tokens[i]], in nats as the entropy -sum p log p.  The top tokens (at most 32) are
    in order, equal logits by the lowest index first.  A masked token (logit -inf) has the log-probability -inf and no
    part in the entropy; where fewer than `top` are unmasked, masked ones follow with -inf.  A token outside [0, V) (the
    padding of a batch) has the log-probability NaN.  A row that is masked whole, or holds a NaN or +inf, gives NaN; its
    top tokens are still ordered, NaN before all numbers."""
    result = front.token_logprobs(logits, tokens, top)
    if result is not None:
        return result
    xt, shape = TYPES.get(logits.dtype), logits.shape
    if xt is None:
        type_code(logits.dtype, "logits")
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError(f"logits must be [M, V], got {tuple(shape)}")
    M, V = shape
    ld, step = logits.stride()
    if step != 1 or ld < V:
        if step != 1 and V > 1:
            raise ValueError(f"the rows of logits must be contiguous, got strides {(ld, step)}")
        if M > 1 and ld < V:
            raise ValueError(f"rows of logits overlap (stride {ld}, {V} columns)")
        ld = max(ld, V)
    dev = logits.get_device()
    if dev < 0 or tokens.get_device() != dev:
        raise ValueError("logits and tokens must be on one CUDA device")
    return of_rows(logits.data_ptr(), xt, ld, M, V, tokens, top)


def of_rows(address: int, xt: int, ld: int, M: int, V: int, tokens, top: int):
    """``token_logprobs`` of rows that no tensor holds: M rows of V logits of type xt from `address` on, ld elements from
    one to the next, on the device of `tokens`."""
    wide = tokens.dtype is _I64
    if not wide and tokens.dtype is not _I32:
        raise TypeError(f"tokens must be int32 or int64, got {tokens.dtype}")
    if tokens.shape != (M,) or not tokens.is_contiguous():
        raise ValueError(f"tokens must be a contiguous [{M}] tensor, got {tuple(tokens.shape)}")
    if not 0 <= top <= min(MOST_TOP, V):
        raise ValueError(f"top must be 0 to {min(MOST_TOP, V)}, got {top}")
    dev = tokens.get_device()
    lp, entropy = empty((M,), _F32, dev), empty((M,), _F32, dev)
    if not top:
        if M:
            call("tac_token_logprobs", _logprobs, dev, address, xt, ld, tokens.data_ptr(), wide, M, V, 0,
                 lp.data_ptr(), entropy.data_ptr(), None, None)
        return lp, entropy
    top_lp, ids = empty((M, top), _F32, dev), empty((M, top), _I32, dev)
    if M:
        call("tac_token_logprobs", _logprobs, dev, address, xt, ld, tokens.data_ptr(), wide, M, V, top,
             lp.data_ptr(), entropy.data_ptr(), top_lp.data_ptr(), ids.data_ptr())
    return lp, entropy, top_lp, ids
