"""What the torch front ends of the stand-alone kernels share: type codes, calls on a tensor's device, and ``front``, the
C++ side of the usual calls of some, each of which gives None where Python has to look at the arguments."""
from __future__ import annotations

import ctypes as C
from functools import lru_cache

import torch

from . import _lib as L

ENTRIES = ("rms_norm", "rms_norm_i8", "dequantize_rows_i8", "mxfp4_quantize", "mxfp4_values", "mxfp4_gemm", "linear_mxfp4",
           "linear_mxfp4_workspace_bytes", "token_logprobs")


class _PythonOnly:
    """In place of a ``front`` that is not built: leaves every call to Python."""

    def __getattr__(self, name):
        return lambda *args: None


def _load_front():
    import importlib.util
    import warnings

    from .build import front_path
    spec = importlib.util.spec_from_file_location(f"{__package__}._front", front_path())
    try:
        module = importlib.util.module_from_spec(spec)
    except ImportError as e:
        warnings.warn(f"the torch front ends' C++ side is not built for this torch and Python, and their calls take longer: "
                      f"run `python -m llm_accelerator_b200.build` ({e})", RuntimeWarning, stacklevel=3)
        return _PythonOnly()
    spec.loader.exec_module(module)
    module.bind(*(C.cast(getattr(L.lib, "tac_" + name), C.c_void_p).value for name in ENTRIES), L.check)
    return module


def __getattr__(name):
    if name != "front":                # loaded for the modules that have calls in it
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    globals()["front"] = found = _load_front()
    return found


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


def of_device(query):
    """The workspace query f(index, *sizes) of CUDA device `index`, by whose SMs `query` goes; asked once."""
    @lru_cache(maxsize=1024)
    def f(index: int, *sizes) -> int:
        if _current() == index:
            return query(*sizes)
        with torch.cuda.device(index):
            return query(*sizes)
    return f
