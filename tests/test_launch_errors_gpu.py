"""A call that fails leaves no error behind for the next one.

The failure is the host's: a stream whose capture has been invalidated refuses every launch."""
from __future__ import annotations

import ctypes as C
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest
import torch

from llm_accelerator_b200 import _lib as L

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


class _Refusing:
    """A stream on which a capture has begun and been invalidated."""

    def __enter__(self):
        self.cu, self.stream = C.CDLL("libcuda.so.1"), torch.cuda.Stream()
        self.handle = C.c_void_p(self.stream.cuda_stream)
        assert self.cu.cuStreamBeginCapture_v2(self.handle, 2) == 0          # relaxed
        assert self.cu.cuStreamQuery(self.handle) == 900                     # not allowed during a capture, and ends it
        return self.handle

    def __exit__(self, *exc):
        graph = C.c_void_p()
        assert self.cu.cuStreamEndCapture(self.handle, C.byref(graph)) == 901


def _calls():
    """name -> call(stream) of each entry point and each of its launchers."""
    from llm_accelerator_b200 import kv4
    z = lambda *s, dt=torch.float16: torch.zeros(s, dtype=dt, device="cuda")
    x, q, s = z(1024, 64), z(1024, 64, dt=torch.int8), z(1024, dt=torch.float32)
    w, sb, y = z(4096, 64, dt=torch.int8), z(4096, dt=torch.float32), z(1024, 4096)
    ws = z(1 << 20, dt=torch.uint8)
    cache = kv4.Kv4Cache(160, 16, 2, 64)
    table, lens, ptr = z(1, 160, dt=torch.int32), z(1, dt=torch.int32), z(2, dt=torch.int32)
    k, o = z(1024, 2, 64), z(1024, 16, 64)
    f = z(1024, 2, 64, dt=torch.float32)
    aws = z(1 << 24, dt=torch.uint8)
    p = lambda t: t.data_ptr()
    seqs = lambda total: (p(table), p(lens), p(ptr), 1, 160, total)
    keep = [x, q, s, w, sb, y, ws, cache, table, lens, ptr, k, o, f, aws]
    calls = {f"product of {m} rows": lambda st, m=m: L.lib.tac_gemm_i8_scaled(
        p(q), p(w), p(s), p(sb), L.TYPE_F32, None, 0, p(y), L.TYPE_F16, m, 4096, 64, st) for m in (1, 64, 1024)}
    calls |= {f"linear of {m} rows": lambda st, m=m: L.lib.tac_linear_w8a8(
        p(x), L.TYPE_F16, 64, p(w), p(sb), L.TYPE_F32, None, 0, p(y), L.TYPE_F16, p(ws), ws.numel(), m, 4096, 64, st)
        for m in (1, 64, 1024)}
    calls["quantiser"] = lambda st: L.lib.tac_quantize_rows_i8(p(x), L.TYPE_F16, 64, p(q), p(s), 1024, 64, st)
    calls["append"] = lambda st: L.lib.tac_kv4_append(cache._ref, *seqs(1024), p(k), 128, 64, p(k), 128, 64, L.TYPE_F16, st)
    calls["read"] = lambda st: L.lib.tac_kv4_read(cache._ref, *seqs(1024), p(f), p(f), st)
    calls |= {f"attention of {m} rows": lambda st, m=m: L.lib.tac_kv4_attention(
        cache._ref, *seqs(m), p(o), 1024, 64, 16, L.TYPE_F16, 0.1, 1, p(o), None, p(aws), aws.numel(), st)
        for m in (1, 1024)}
    return calls, keep


def test_failed_launches_fail_alone():
    calls, keep = _calls()
    for name, call in calls.items():                  # the first calls set kernels up
        assert call(None) == L.OK, name
    torch.cuda.synchronize()
    for name, call in calls.items():
        with _Refusing() as stream:
            assert call(stream) == L.E_CUDA, name
        for other, healthy in calls.items():
            assert healthy(None) == L.OK, f"{other} after {name}"
    torch.cuda.synchronize()
    assert L.lib.tac_gemm_status(None) == L.OK
    del keep


def test_calls_do_not_report_what_an_earlier_call_left():
    """An entry point that leaves the runtime's last error behind does not fail the calls after it.  In a process of its
    own, which the error ends with."""
    code = textwrap.dedent(f"""
        import ctypes as C, sys
        sys.path[:0] = [{str(ROOT)!r}, {str(ROOT / 'tests')!r}]
        import torch
        from llm_accelerator_b200 import _lib as L
        from test_launch_errors_gpu import _calls
        calls, keep = _calls()
        for name, call in calls.items():
            engine = C.c_void_p()
            assert L.lib.tac_engine_create(999, 1, 1 << 16, 0, C.byref(engine)) == L.E_CUDA     # there is no such device
            assert call(None) == L.OK, name
        torch.cuda.synchronize()
        print("ok")
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr
