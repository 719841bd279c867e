"""The direct loads of the 8-bit cache's attention take their LDS address from m0, which their asm writes. The compiler reserves m0 (it
keeps no value of its own there, and warns at a clobber that names it), but instructions of its own may set and use it; the device
code holds none that do, so nothing can come between."""
import re

from tests.test_build_flags import device_asm, makefile_flags


def test_only_the_direct_loads_use_m0(tmp_path):
    text = device_asm("attn_kv8.hip", makefile_flags(), str(tmp_path / "attn_kv8.s"))
    inside, outside = 0, []
    for part in re.split(r"(;APP\b.*?;NO_APP\b|;;#ASMSTART.*?;;#ASMEND)", text, flags=re.S):
        mine = part.startswith((";APP", ";;#ASMSTART"))
        for line in part.split("\n"):
            if re.search(r"\bm0\b", line.split(";")[0]):
                inside += mine
                outside += [] if mine else [line]
    assert inside and not outside, outside[:5]
