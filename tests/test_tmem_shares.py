"""CTAs that hold TMEM while they wait for others of their cluster: whatever mix of them fits an SM's shared memory finds
its columns there, so that none waits for columns that another one's cluster holds."""
from __future__ import annotations

import re
import subprocess
from functools import lru_cache
from pathlib import Path

from llm_accelerator_b200 import build

CSRC = build.CSRC
SMEM, RESERVED, COLUMNS = 228 * 1024, 1024, 512      # of an SM; of each CTA for the system


@lru_cache(maxsize=None)
def _shares(folder):
    """({columns: least shared memory}, the least of a CTA of 512 columns) of the header."""
    src = Path(folder) / "shares.cu"
    src.write_text("""
        #include <cstdio>
        #include "tac_sm100.cuh"
        int main() {
          for (int c : {32, 64, 128, 256}) printf("%d ", tac::sm100::tmem_least_smem(c));
          int s = 0;
          while (!tac::sm100::tmem_alone(s)) ++s;
          printf("%d\\n", s);
        }""")
    out = Path(folder) / "shares"
    subprocess.run([build.NVCC, *build.ARCH, "-std=c++17", f"-I{CSRC}", str(src), "-o", str(out)], check=True)
    *least, alone = map(int, subprocess.run([str(out)], check=True, capture_output=True, text=True).stdout.split())
    return dict(zip((32, 64, 128, 256), least)), alone


def _most_columns(kinds, room):
    """Columns that the CTAs of any mix hold which fits `room`."""
    best = 0
    for i, (columns, smem) in enumerate(kinds):
        if smem + RESERVED <= room:
            best = max(best, columns + _most_columns(kinds[i:], room - smem - RESERVED))
    return best


def test_every_mix_has_its_columns(tmp_path):
    least, alone = _shares(str(tmp_path))
    small = sorted(least.items())
    assert _most_columns(small, SMEM) == 384 <= COLUMNS
    assert _most_columns([*small, (512, alone)], SMEM) <= COLUMNS
    assert alone <= 227 * 1024


def test_every_kernel_of_clusters_keeps_to_them():
    """Launches of clusters whose kernels hold TMEM go by the least shared memory; fixed sizes are asserted."""
    for name, launches in (("tac_w8a8.cu", 2), ("tac_mxfp4.cu", 2)):
        text = (CSRC / name).read_text()
        for f in re.split(r"\n}\n", text):
            if "ClusterDimension" in f:
                assert "sm100::tmem_least_smem(" in f, f[:200]
                launches -= 1
        assert launches == 0
    held = [p.name for p in sorted(CSRC.glob("*.cuh")) if re.search(r"__cluster_dims__", p.read_text()) and "tmem_alloc" in p.read_text()]
    assert held == ["tac_gemm_tc2.cuh", "tac_mxfp4.cuh", "tac_w8a8.cuh"]
    for name in held:
        assert "static_assert(sm100::tmem_alone(" in (CSRC / name).read_text()
    assert "tmem_least_smem(256)" in (CSRC / "tac_exec.cuh").read_text()
