"""Who writes and reads the register m0 in the built library: loads to LDS take their address there from inline assembly, which cannot tell the
compiler so."""
import os
import re
import subprocess

import pytest

from hetuctr_amd import build
from tests.test_kernel_resources import OBJDUMP, code_objects, kernel_code

# what reads m0 without naming it, besides loads to LDS
IMPLICIT = re.compile(r"^(s_movrel|v_movrel|v_interp|ds_gws|ds_ordered|s_sendmsg|s_ttracedata|ds_.*_(gs_reg|addtid)|buffer_.*_addtid|global_load_lds|scratch_load_lds)")


def strange(body):
    """Instructions that use m0 otherwise than: set it, wait a cycle, load to LDS by it"""
    found, at = [], 0
    while at < len(body):
        address, op, operands, _ = body[at]
        if op == "s_mov_b32" and operands.startswith("m0,"):
            rest = [(o, a) for _, o, a, _ in body[at + 1:at + 3]]
            if len(rest) == 2 and rest[0][0] == "s_nop" and rest[1][0].startswith("buffer_load_dwordx4") and rest[1][1].split()[-1] == "lds":
                at += 3
                continue
            found.append(hex(address))
        elif re.search(r"\bm0\b", operands) or IMPLICIT.match(op) or (op.startswith("buffer_") and operands.split()[-1:] == ["lds"]):
            found.append(hex(address))
        at += 1
    return found


def test_the_search_finds_them():
    ours = [(0, "s_mov_b32", "m0, s3", ""), (4, "s_nop", "0", ""), (8, "buffer_load_dwordx4", "v1, s[4:7], 0 offen lds", "")]
    assert not strange(ours) and not strange(ours * 3)
    assert strange(ours[1:]) == ["0x8"] and strange(ours[:1] + ours[2:] + ours) == ["0x0", "0x8"]
    for op, operands in (("s_mov_b32", "m0, s1"), ("v_readlane_b32", "m0, v1, 3"), ("s_movrels_b32", "s1, s2"), ("s_add_u32", "s1, m0, s2"), ("s_sendmsg", "sendmsg(MSG_INTERRUPT)")):
        assert strange(ours + [(12, op, operands, "")] + ours) == ["0xc"]


@pytest.mark.skipif(not os.path.exists(OBJDUMP) or not os.path.exists(build.LIB), reason="needs the built library and llvm-objdump")
def test_nothing_else_uses_m0(tmp_path):
    others, loads = {}, 0
    for i, obj in enumerate(code_objects(build.LIB)):
        f = tmp_path / ("%d.o" % i)
        f.write_bytes(obj)
        listing = subprocess.run([OBJDUMP, "-d", str(f)], stdout=subprocess.PIPE, text=True, check=True).stdout
        for name, _, body in kernel_code(listing):
            here = sum(op.startswith("buffer_") and operands.split()[-1:] == ["lds"] for _, op, operands, _ in body)
            loads += here
            if here and (found := strange(body)):
                others[name] = found
    assert loads > 1000
    assert not others
