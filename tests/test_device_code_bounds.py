"""Bounds of the loads to LDS that rely on their buffer resource's end (no GPU:
the sources are compiled for gfx950 here)."""

import os
import re

import pytest

from tests.test_device_code import HIPCC, _assembly


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
@pytest.mark.parametrize("source", ["packed.hip", "shared_prefix.hip"])
def test_rows_past_the_last_are_told_by_the_lanes_offsets(source, tmp_path):
    """Tiles of K/V rows are loaded whole, and the resource, which ends with the
    last row, makes zeros of the rest. The hardware compares a lane's offset with
    the resource's size less the scalar offset, so a scalar offset past that size
    by itself need not be refused: there must be none."""
    code = _assembly(source, str(tmp_path / "out.asm"))
    loads = [ins for ins in code if re.match(r"buffer_load_\w+ .*\blds$", ins)]
    assert loads
    for ins in loads:
        assert re.match(r"buffer_load_\w+ v\d+, s\[\d+:\d+\], 0 offen lds$", ins), ins
