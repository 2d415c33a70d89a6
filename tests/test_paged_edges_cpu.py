"""Rotary and paged-cache operators on the CPU: calls at the edge of what they take."""
import pathlib
import re

import pytest

from homebrewnlp_mtf_amd.ops import _lib as L

KERNELS = pathlib.Path(__file__).resolve().parent.parent / "csrc" / "kernels"


@pytest.mark.parametrize("source,name,packed", [("rotary.hip", "RotDesc", L.ROT_DESC), ("paged.hip", "PlanDesc", L.PLAN_DESC),
                                                ("paged.hip", "PagedDesc", L.PAGED_DESC)])
def test_packed_descriptors_are_as_long_as_the_structs(source, name, packed):
    """the launch reads the whole struct: its padded size, which the source asserts"""
    size = int(re.search(rf"static_assert\(sizeof\({name}\) == (\d+)\)", (KERNELS / source).read_text()).group(1))
    assert packed.size == size and size % 8 == 0
