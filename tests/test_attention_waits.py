"""Waits of the soft reads' kernels, by reading their source: a wait that runs out cannot be shown on a GPU without making one hang."""
import os
import re

import pytest


def warp_branches(text):
    """The bodies of branches that only warp 1 runs, comments out."""
    text = re.sub(r"//[^\n]*", "", text)
    out = []
    for m in re.finditer(r"if \(warp == 1\) \{", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        out.append(text[m.end():i])
    return out


@pytest.mark.parametrize("name", ["attend.cu", "attend_backward.cu", "attention_mass.cu"])
def test_waits_that_steer_a_warp_are_voted_on(name):
    """A bounded wait may run out for some lanes of a warp and not for others.  Where a lane's own result decided whether it takes part in the next full-mask
    vote, the way out of a failure would hang: in a warp that issues products, every wait is the argument of a vote."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "faiss-metal_b200", "csrc", name)
    text = open(path).read()
    issuing = [b for b in warp_branches(text) if "tc_commit_by" in b]
    assert issuing
    for body in issuing:
        left = re.sub(r"__all_sync\(0xffffffffu, wait\([^;]*?\)\)", "", body)
        assert not re.search(r"(?<![a-z_])wait\(", left), re.search(r"[^\n]*(?<![a-z_])wait\([^\n]*", left).group(0)
