"""Order of the programmatic launch instructions in the kernels' source, which no run can show reliably: on a
full GPU a dependent kernel rarely finds room early, whatever the source allows."""

import re
from pathlib import Path

CSRC = (Path(__file__).resolve().parent.parent /
        "bridge-aware-kv-cache-eviction-for-efficient-long-context-transformers_b200" / "csrc")


def kernels(name):
    """{kernel: body} of a source file, comments left out."""
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    parts = re.split(r"__global__\s+void\s+__launch_bounds__\([^)]*\)\s*(\w+)\(", text)
    return dict(zip(parts[1::2], parts[2::2]))


def test_the_join_reads_nothing_that_may_still_be_written():
    """join_kernel reads the lengths before it waits for tc_kernel; so tc_kernel must have waited for the
    kernel before it when it lets the join start."""
    bodies = kernels("tree_attn.cu")
    join, tc = bodies["join_kernel"], bodies["tc_kernel"]
    early = join.index("load_seq(") < join.rindex("griddepcontrol.wait")
    after_wait = tc.index("griddepcontrol.wait") < tc.index("griddepcontrol.launch_dependents")
    assert after_wait or not early


def test_every_kernel_launched_behind_another_waits_for_it():
    for name in ("tree_attn.cu", "paged_cache.cu"):
        for kernel, body in kernels(name).items():
            assert "griddepcontrol.wait" in body or "grid_dependency_wait()" in body, kernel


def test_warps_are_whole_at_instructions_that_want_them_whole():
    """TMEM loads and the cluster barrier are `.aligned`: behind waits, masks and an early `continue`, which lanes
    leave one by one, a __syncwarp() comes first."""
    tc = kernels("tree_attn.cu")["tc_kernel"]
    for start in ("if (masked) {", "take_over(quad", "for (int c = 0; c < D / 2; c += 32) {"):
        part = tc[tc.index(start):]
        first = min(part.find(x) for x in ("tmem_ld32(", "weights<") if x in part)
        assert "__syncwarp()" in part[:first], start
    update = re.sub(r"//[^\n]*", "", (CSRC / "paged_cache.cu").read_text())
    sync = update[update.index("void cluster_sync("):]
    assert "__syncwarp()" in sync[:sync.index(".aligned")]
