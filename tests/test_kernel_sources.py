"""Rules that the kernels' sources keep and no run shows."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "parrotserve_b200" / "csrc"
EARLY = sorted(p.name for p in CSRC.glob("*.cu*") if "pdl_wait()" in p.read_text())


def code_of(name):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", (CSRC / name).read_text(), flags=re.S)


@pytest.mark.parametrize("name", EARLY)
def test_kernels_that_begin_early_read_with_ordinary_loads(name):
    """A kernel that begins while the one before it still writes may not read its inputs by the read-only path."""
    assert not re.search(r"__ldg\s*\(|\bld\.global\.nc\b", code_of(name))
