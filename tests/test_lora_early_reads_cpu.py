"""The adapter kernels read what the launch before their predecessor wrote without waiting for their predecessor.  That is sound
because none of them lets its successor start before it has itself waited: in the sources every pdl_trigger() follows a
pdl_wait() at once, under the same condition.  (A race could not be seen reliably by running; the text can.)"""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "prismyra_b200" / "csrc"


@pytest.mark.parametrize("name", ["moe_lora.cu", "moe_lora_grad.cu", "moe_lora_tiles.cu"])
def test_no_launch_lets_its_successor_start_before_it_has_waited(name):
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    lines = [line.strip() for line in text.splitlines() if line.strip()]
    at = [i for i, line in enumerate(lines) if "pdl_trigger()" in line]
    assert at
    for i in at:
        assert lines[i] == "pdl_trigger();" and lines[i - 1] == "pdl_wait();", lines[i - 1:i + 1]
        assert not lines[i - 2].endswith(")") or lines[i - 2].startswith("asm"), lines[i - 2]  # no condition without braces
