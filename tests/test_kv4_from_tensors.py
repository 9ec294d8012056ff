"""Tensors that a cache is not built over, with what is wrong in the message (no GPU needed)."""
from __future__ import annotations

import pytest
import torch

from llm_accelerator_b200 import kv4


@pytest.mark.parametrize("which", range(4))
def test_tensors_that_do_not_begin_on_16_bytes(which):
    """A layer's slice of a larger allocation may begin anywhere: refused when the cache is made, not by each call."""
    shapes = [((3, 2, 16, 32), torch.uint8), ((3, 2, 16), torch.int32)] * 2
    parts = []
    for i, (shape, dt) in enumerate(shapes):
        n = torch.Size(shape).numel()
        flat = torch.zeros(n + 16, dtype=dt)
        off = -(flat.data_ptr() // dt.itemsize) % (16 // dt.itemsize) + (1 if i == which else 0)
        parts.append(flat[off:off + n].view(shape))
    with pytest.raises(ValueError, match="16-byte"):
        kv4.Kv4Cache.from_tensors(*parts)
