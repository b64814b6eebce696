"""What the sources of the serving kernels keep to, where no run can show it."""

from __future__ import annotations

from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "flux_b200" / "csrc"
SOURCES = sorted(p.name for pattern in ("paged*", "logits.cu") for p in CSRC.glob(pattern))


@pytest.mark.parametrize("name", SOURCES)
def test_no_loads_that_need_constant_memory(name):
    """These kernels are launched before the one in front of them has ended, and read what it wrote (page tables,
    lists): a non-coherent load is defined only for memory that nobody writes while the kernel is there."""
    text = (CSRC / name).read_text()
    assert "__ldg" not in text and "global.nc" not in text and "__restrict__" not in text
