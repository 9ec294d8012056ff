"""What the torch front ends of the stand-alone kernels share: type codes and calls on a tensor's device."""
from __future__ import annotations

import torch

from . import _lib as L

TYPES = {torch.float32: L.TYPE_F32, torch.float16: L.TYPE_F16, torch.bfloat16: L.TYPE_BF16}
_current = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream
_quick = getattr(torch._C._dynamo.guards, "_empty_strided_cuda", None)


def empty(shape, dtype, index: int, stride=None):
    """A contiguous tensor (of one or two dimensions where `stride` is left out) on CUDA device `index`.  torch.empty
    spends twice as long on its arguments as on the memory (2.3 us a call, 0.8 without them), which is what a call of a
    few microseconds waits for."""
    if _quick is not None and _current() == index:
        return _quick(shape, stride or ((shape[1] or 1, 1) if len(shape) == 2 else (1,)), dtype)
    return torch.empty(shape, dtype=dtype, device=torch.device("cuda", index))


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
