"""Wait states in front of the loads to LDS of csrc/shared_prefix.hip, which are
inline assembly that the compiler adds none for (no GPU: the source is
compiled for gfx950 here)."""

import os
import re

import pytest

from tests.test_device_code import HIPCC, _assembly


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_loads_to_lds_wait_for_their_scalar_operands(tmp_path):
    """One wait state after a write of m0; five after a vector instruction's
    write of a scalar register that the load reads (resource or m0)."""
    code = _assembly("shared_prefix.hip", str(tmp_path / "out.asm"))
    loads = [i for i, ins in enumerate(code) if re.match(r"buffer_load_\w+ .*\blds$", ins)]
    assert loads
    for i in loads:
        read = {"m0"}
        for lo, hi in re.findall(r"\bs\[(\d+):(\d+)\]", code[i]):
            read |= {f"s{n}" for n in range(int(lo), int(hi) + 1)}
        read |= {f"s{n}" for n in re.findall(r"\bs(\d+)\b", code[i])}
        states = 0
        for ins in code[i - 1::-1]:
            if states >= 5:
                break
            wrote = re.match(r"v_read(?:first)?lane_b32 (s\d+|m0),", ins)
            assert not (wrote and wrote.group(1) in read), (ins, code[i])
            assert states >= 1 or not re.match(r"[sv]_\w+ m0,", ins), (ins, code[i])
            nop = re.match(r"s_nop (\d+)", ins)
            states += int(nop.group(1)) + 1 if nop else 1
