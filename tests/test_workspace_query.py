"""Workspace queries of linear layers go by the device of the call (devices may have different numbers of SMs)."""
from __future__ import annotations

import pytest
import torch

from llm_accelerator_b200 import _tensors, mxfp4, w8a8


def test_each_device_is_asked_itself(monkeypatch):
    now, asked = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *e):
            now[0] = self.before

    def query(*sizes):
        asked.append(sizes)
        return 0 if now[0] == 0 else sum(sizes)        # device 1 has fewer SMs

    monkeypatch.setattr(_tensors, "_current", lambda: now[0])
    monkeypatch.setattr(_tensors.torch.cuda, "device", Device)
    f = _tensors.of_device(query)
    assert f(0, 64, 4096) == 0 and f(1, 64, 4096) == 4160 and now[0] == 0
    now[0] = 1
    assert f(0, 64, 4096) == 0 and f(1, 64, 4096) == 4160 and len(asked) == 2
    assert f(0, 3, 4) == 0 and f(1, 3, 4) == 7 and len(asked) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("module", [mxfp4, w8a8])
def test_linear_asks_for_its_rows_device(module, monkeypatch):
    x = torch.ones((200, 64), device="cuda")
    real, asked = module._ws_bytes, []
    monkeypatch.setattr(module, "_ws_bytes", lambda *a: asked.append(a) or real(*a))
    if module is mxfp4:
        w = mxfp4.quantize(x[:32])
        monkeypatch.setattr(mxfp4, "front", _tensors._PythonOnly())
        mxfp4.linear(x, w)
    else:
        w8a8.linear_w8a8(x, torch.ones((32, 64), dtype=torch.int8, device="cuda"), torch.ones(32, device="cuda"))
    assert asked == [(x.get_device(), 200, 32, 64)]
