"""Kernels whose warps may leave early (a wait ran out) must not be waited for without a
bound: no named barrier, and every wait looks at the CTA's abort flag."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "moe_overlap_b200" / "csrc"


@pytest.mark.parametrize("name", ["few_tokens.cu", "lora_few.cu"])
def test_waits_of_warps_that_may_leave_are_bounded(name):
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    assert "bar.sync" not in text
    waits = re.findall(r"mbar_wait\((.*?)\)\)?[;\s)]", text)
    assert waits and not [w for w in waits if "nullptr" in w]
    # a wait that gave up also waits for the copies under way (give_up) before it leaves
    assert "record_status(status, MOE_ERR_TIMEOUT)" not in text
    assert "record_status(p.status, MOE_ERR_TIMEOUT)" not in text
