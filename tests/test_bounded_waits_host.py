"""Kernels some of whose warps may give up (a wait ran out) must not be waited for without
a bound: every wait looks at the CTA's abort flag, and behind a named barrier no warp that
it counts may have left."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "moe_overlap_b200" / "csrc"


def code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


@pytest.mark.parametrize("name", ["few_tokens.cu", "lora_few.cu"])
def test_waits_are_bounded_and_end_with_another_roles(name):
    text = code(name)
    waits = re.findall(r"mbar_wait\((.*?)\)\)?[;\s)]", text)
    assert waits and not [w for w in waits if "nullptr" in w]
    # giving up also waits for the copies under way
    assert not re.search(r"record_status\([\w.]*status, MOE_ERR_TIMEOUT\)", text)


def test_no_warp_leaves_before_a_barrier_that_counts_it():
    assert "bar.sync" not in code("few_tokens.cu")  # its warps may leave: mbarriers instead
    kernel = code("lora_few.cu").split("project_kernel(")[1].split("\nint project(")[0]
    consumers = kernel.split("const int cw = warp - 1")[1]
    assert "bar.sync" in consumers and "return" not in consumers
