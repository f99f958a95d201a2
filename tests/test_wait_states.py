"""CPU: wait states of the built kernels around instructions written as inline asm, where the compiler puts none."""

from __future__ import annotations

from collections import defaultdict

import pytest

from tests._listing import OBJDUMP, Function, check_library, registers


def _resource(fn: Function, i: int):
    """A resource word that the vector unit wrote is read by a memory instruction 5 wait states later or more."""
    load = fn[i]
    words = {r for r in registers(" ".join(load.operands)) if r[0] == "s"}
    for other, between in fn.before(i, 5):
        if other.op.startswith("v_") and other.writes() & words:
            yield "resource", f"{other.text} | {between} | {load.text}"


def _m0(fn: Function, i: int):
    """A load to LDS begins a wait state behind the write of its address into M0, or later."""
    for other, _ in fn.before(i, 1):
        if "m0" in other.writes():
            yield "m0", f"{other.text} | {fn[i].text}"


def check(fn: Function) -> list:
    found = []
    for i in fn.find(" lds"):
        found += _resource(fn, i)
        found += _m0(fn, i)
    return [(kind, fn.name, text) for kind, text in found]


@pytest.fixture(scope="module")
def found(tmp_path_factory):
    from convrot_mlx_amd import _native

    if not OBJDUMP.exists():
        pytest.skip("no disassembler")
    out = defaultdict(list)
    for kind, name, text in check_library(_native.LIB_PATH, tmp_path_factory.mktemp("code"), (" lds",), check):
        out[kind].append((name, text))
    return out


def function(*lines: str) -> Function:
    """Instructions of 4 bytes, the first at 0."""
    return Function("<f>:", [f"\t{line.split(' -> ')[0]}  // {4 * i:012X}: 00000000"
                             + (f" <f+0x{4 * int(line.split(' -> ')[1]):x}>" if " -> " in line else "")
                             for i, line in enumerate(lines)])


LOAD = "buffer_load_dword v1, s[8:11], 0 offen lds"


def test_the_check_of_resources():
    write, five = "v_readfirstlane_b32 s9, v3", ["s_nop 4"]
    assert [k for k, _, _ in check(function(write, "s_nop 3", LOAD))] == ["resource"]
    assert check(function(write, *five, LOAD)) == [] and check(function("v_readfirstlane_b32 s12, v3", LOAD)) == []
    assert check(function(write, "v_mov_b32_e32 v1, 0", "s_mov_b32 s1, 0", LOAD)) and check(function("s_mov_b32 s9, 0", LOAD)) == []
    # over a branch: from the end of a loop to its start, and past what it jumps over
    loop = ["s_nop 7", LOAD, "s_nop 0", write, "s_cbranch_scc1 65533 -> 1", "s_endpgm"]
    assert len(check(function(*loop))) == 1
    assert check(function(write, "s_cbranch_scc1 1 -> 3", "s_nop 7", LOAD))
    assert check(function(write, "s_branch 1 -> 3", "s_nop 7", "s_nop 3", LOAD)) == []


def test_the_check_of_m0():
    for write in ("s_mov_b32 m0, s3", "s_add_i32 m0, s3, s4"):
        assert [k for k, _, _ in check(function(write, LOAD))] == ["m0"]
        assert check(function(write, "s_nop 0", LOAD)) == []
    assert check(function("s_mov_b32 s3, m0", LOAD)) == []


def test_resources(found):
    assert found["resource"] == []


def test_m0(found):
    assert found["m0"] == []
