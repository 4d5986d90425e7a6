"""What the launches of the experts' tiles in 8-bit integers count on, from the compiler's figures of the last build."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "c0ven_amd", "csrc")


def tiles():
    """(kernel, runs of 32 rows a wave, waves a SIMD) of every kernel of the experts' tiles."""
    path = os.path.join(ROOT, "c0ven_amd", "_build", "kernel_resources.txt")
    if not os.path.exists(path):
        pytest.skip("no build in this tree (run __graft_entry__.build())")
    found = []
    for line in open(path):
        m = re.match(r"_ZN5c0ven\d+i8_(gate_up|down)_tilesILi(\d+)E", line)
        if m:
            found.append((m.group(1), int(m.group(2)), int(re.search(r"occupancy=(\d+)", line).group(1))))
    return found


def test_a_launch_is_what_the_device_holds_at_once():
    """The work-groups go from item to item, so that a launch has as many as fit at once: three a CU for tiles of 64 positions, two
    for tiles of 128 (a work-group's four waves are one a SIMD). Gate/up's kernel is there with a limit and without."""
    found = tiles()
    assert sorted(f[:2] for f in found) == [("down", 1), ("down", 2), ("gate_up", 1), ("gate_up", 1), ("gate_up", 2), ("gate_up", 2)]
    with open(os.path.join(CSRC, "i8_experts.hip")) as f:
        launched = {int(rows) // 64: int(n) for rows, n in re.findall(r"at\.rows == (\d+)\) run\([^;]*, (\d) \* kCus\);", f.read())}
    assert launched == {1: 3, 2: 2}
    for kernel, runs, waves in found:
        assert waves >= launched[runs], (kernel, runs, waves)
