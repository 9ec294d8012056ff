"""The quantised operators say that no gradient flows through them (no GPU needed)."""
from __future__ import annotations

from pathlib import Path

from llm_accelerator_b200 import kv4, ptq, w8a8


def test_the_documentation_says_so():
    for text in (kv4.__doc__, w8a8.__doc__, ptq.quantize_rows.__doc__):
        assert "o gradient flows through" in " ".join(text.split())
    assert "No gradient flows through" in (Path(__file__).resolve().parent.parent / "INTEGRATION.md").read_text()
