"""What the sources of the 8-bit rows, their product and the verdict have to keep to, and no run shows.

Waits that may give up, in kernels whose warps work as wholes behind them:

A lane learns by itself whether a wait on an mbarrier gave up, and a phase may end between two lanes' last looks.  In
rf_i8_matmul.cu every wait is followed by something that the whole warp has to reach (shuffles of results, tcgen05.ld,
elect.sync, cluster barriers), so its warps take one answer for all lanes: wait_bar_warp.  Read from the sources, since no
test lets a wait run out."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ramforge_b200", "csrc")


def code(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def test_every_wait_of_the_product_is_the_warps():
    text = code("rf_i8_matmul.cu")
    assert not re.search(r"\bwait_bar\s*\(", text)
    assert len(re.findall(r"\bwait_bar_warp\s*\(", text)) == 8
    assert re.search(r"bool wait_bar_warp\([^)]*\) \{\s*return __all_sync\(0xffffffffu, wait_bar\(", code("rf_ring.cuh"))


@pytest.mark.parametrize("name", ["rf_i8.cu", "rf_i8_matmul.cu", "rf_accept.cu", "rf_act.cuh"])
def test_nothing_goes_through_the_read_only_path(name):
    """These kernels begin while the one before them still writes, and any of their inputs may be its output; the
    read-only path (.nc, __ldg) is for memory that nobody writes while a kernel runs."""
    assert not re.search(r"__ldg\b|\.nc\b|__restrict__", code(name))
