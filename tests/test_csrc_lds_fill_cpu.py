"""Copies into LDS written as asm statements: what the compiler does not check of them."""
import re

from test_csrc_source_cpu import _statements, _template


def test_lds_copies_wait_for_their_base():
    """Five wait states between a VALU write of an SGPR (m0 or the base address, which a
    readfirstlane may have written last) and the copy that reads it."""
    seen = 0
    for name, stmt in _statements():
        waits = 0
        for ins in _template(stmt):
            if ins.startswith("global_load_lds"):
                seen += 1
                assert waits >= 5, (name, stmt)
                assert '"m0"' in stmt.rsplit(":", 1)[1], (name, stmt)
            nop = re.match(r"s_nop\s+(\d+)", ins)
            waits += int(nop.group(1)) + 1 if nop else 1
    assert seen >= 2

