"""The kernels whose warps issue whole, with one elected lane (tac_w8a8.cuh, tac_kv4_tc.cuh), read as text: a wait that
runs out cannot be caused without breaking a kernel, so what is checked is that no lane acts on a verdict of its own."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "llm_accelerator_b200" / "csrc"
FILES = sorted(p.name for p in CSRC.glob("*.cuh") if "elect_one()" in p.read_text() and p.name != "tac_sm100.cuh")


def test_the_files_are_found():
    assert {"tac_w8a8.cuh", "tac_kv4_tc.cuh"} <= set(FILES)


@pytest.mark.parametrize("name", FILES)
def test_no_lane_leaves_a_loop_by_itself(name):
    """elect.sync, __syncwarp and tcgen05 accesses wait for every lane.  Per-lane waits are those whose verdict nothing
    but the abort flag takes; what an elected lane does depends on no lane's own read of that flag."""
    for line in (CSRC / name).read_text().splitlines():
        if "mbar_wait(" in line or "mbar_try_wait(" in line:
            verdict_unused = re.match(r"\s*sm100::mbar_wait\(.*_DRAIN\);$", line)
            flag_only = re.match(r"\s*if \(!\*abort_v && !sm100::mbar_wait\(.*\)\) \*abort_v = 1;$", line) or \
                re.match(r"\s*if \(sm100::mbar_try_wait\(bar, parity\)\) return;$", line)
            assert verdict_unused or flag_only, line
        if "elect_one()" in line or "for (" in line or "while (" in line:
            assert "abort_v" not in line, line


def test_no_mask_is_read_off_the_converged_lanes():
    """__activemask says which lanes happen to be converged, not which take part: a collective that goes by it can lose
    lanes."""
    for p in sorted(CSRC.iterdir()):
        assert "__activemask" not in p.read_text(), p.name


def test_other_ctas_are_written_to_only_once_they_run():
    """A store into another CTA's shared memory lies behind a cluster barrier of the same kernel: before one, that CTA may
    not have started."""
    kernels = re.split(r"__global__", (CSRC / "tac_w8a8.cuh").read_text())[1:]
    writers = [k for k in kernels if "st.shared::cluster" in k]
    assert writers
    for k in writers:
        before = k[:k.index("st.shared::cluster")]
        assert before.count("cluster_arrive()") == 1 and before.count("cluster_wait()") == 1 or "cluster_sync()" in before
