"""What the torch front ends of the stand-alone kernels share: type codes and calls on a tensor's device."""
from __future__ import annotations

import torch

from . import _lib as L

TYPES = {torch.float32: L.TYPE_F32, torch.float16: L.TYPE_F16, torch.bfloat16: L.TYPE_BF16}
_current = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream


def type_code(dtype, what: str) -> int:
    """enum tac_type of a torch dtype."""
    code = TYPES.get(dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, got {dtype}")
    return code


def call(name: str, fn, index: int, *args) -> None:
    """fn(*args, stream) with CUDA device `index` current and its current stream, whichever device was current."""
    if _current() == index:
        status = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _stream(index))
    if status:
        L.check(status, name)
