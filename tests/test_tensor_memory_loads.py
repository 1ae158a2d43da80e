"""Loads from tensor memory are asynchronous, and their wait names no registers: unless the loaded
registers are marked as written behind it, the compiler may use them before it.  Such a
reordering need not show in a result, so the sources are looked at instead."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "nitrorag_b200" / "csrc"
FILES = sorted(p for p in CSRC.iterdir() if p.suffix in (".cu", ".cuh") and re.search("tcgen05|tmem_", p.read_text()))


@pytest.mark.parametrize("path", FILES, ids=lambda p: p.name)
def test_a_wait_for_loads_is_followed_by_their_registers(path):
    lines = path.read_text().splitlines()
    for i, line in enumerate(lines):
        if "tmem_wait_ld() {" in line:  # the wait itself
            continue
        if re.search(r"tcgen05\.wait::ld|tmem_wait_ld\(\)", line.split("//")[0]):
            after = [x for x in lines[i + 1:i + 4] if not x.lstrip().startswith("#")]
            assert any("tmem_regs_" in x for x in after[:2]), f"{path.name}:{i + 1}"


def test_files_were_found():
    assert {"tc_common.cuh", "prompt_attention.cu"} <= {p.name for p in FILES}
