"""Waits in the product's kernels: what a warp does together behind a wait that
may give up is decided by all of its lanes. A wait that runs out cannot be made
on a GPU without holding it up, so this reads the source."""
import os
import re

from tests.conftest import ROOT


def test_warps_that_issue_or_read_decide_together():
    """Waits for full stages, free accumulators and finished products are made by
    whole warps. One lane that gives up alone would leave the others in the next
    instruction that wants all of them."""
    with open(os.path.join(ROOT, "snn_b200", "csrc", "b200_mx4_mma.cu")) as f:
        text = f.read()
    waits = list(re.finditer(r"\bok = [^;]*bar_wait\(&(s_full|s_free|s_ready)\b[^;]*;", text))
    assert len(waits) >= 4  # this reads what it means to
    for m in waits:
        behind = text[m.end():].lstrip().split(";")[0]
        assert "__all_sync(" in m.group(0) or behind.startswith("ok = __all_sync("), m.group(0)
