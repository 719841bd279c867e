"""What the 8-bit cache's attention takes for granted of its device code.

Its direct loads take their LDS address from m0, which their asm writes. The compiler reserves m0 (it keeps no value of its own there,
and warns at a clobber that names it), but instructions of its own may set and use it; the code holds none that do, so nothing can come
between. And both of its kernels find the pages per split by themselves, in f32: the same operations, fused alike."""
import re
from collections import Counter

import pytest

from tests.test_build_flags import device_asm, makefile_flags


@pytest.fixture(scope="module")
def text(tmp_path_factory):
    return device_asm("attn_kv8.hip", makefile_flags(), str(tmp_path_factory.mktemp("asm") / "attn_kv8.s"))


def test_only_the_direct_loads_use_m0(text):
    inside, outside = 0, []
    for part in re.split(r"(;APP\b.*?;NO_APP\b|;;#ASMSTART.*?;;#ASMEND)", text, flags=re.S):
        mine = part.startswith((";APP", ";;#ASMSTART"))
        for line in part.split("\n"):
            if re.search(r"\bm0\b", line.split(";")[0]):
                inside += mine
                outside += [] if mine else [line]
    assert inside and not outside, outside[:5]


def test_both_kernels_split_alike(text):
    """The f32 operations up to the last count of splits (a ceil each), whatever their order: those of a sum over the lanes are
    scheduled among those of others."""
    by_rows = {}
    for name, body in re.findall(r"^(_ZN2it\S*attn_kv8\S*):[^\n]*\n(.*?)\.end_amdhsa_kernel", text, re.S | re.M):
        lines = [line.strip() for line in body.split("\n")]
        end = max(i for i, line in enumerate(lines) if line.startswith("v_ceil_f32")) + 8
        ops = [re.match(r"(v_(?:add|sub|subrev|mul|fma|fmac|fmaak|fmamk|mac|rcp|ceil|max|min|cmp_?\w*?)_f32)(\S*)", line) for line in lines[:end]]
        merge, n = "merge" in name, int(re.search(r"ILi\d+ELi(\d+)E", name)[1])
        by_rows.setdefault(n if merge else 16 * n, []).append((merge, Counter((m[1], "dpp" in m[2]) for m in ops if m)))
    assert sorted(by_rows) == [16, 32, 48, 64]
    for rows, found in by_rows.items():
        assert {merge for merge, _ in found} == {True, False}
        assert all(ops == found[0][1] for _, ops in found), rows
