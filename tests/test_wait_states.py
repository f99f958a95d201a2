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


def _operands(fn: Function, i: int):
    """A matrix instruction reads what the vector unit wrote 2 wait states later or more."""
    mfma = fn[i]
    read = registers(" ".join(mfma.operands[1:]))
    for other, between in fn.before(i, 2):
        if other.op.startswith("v_") and not other.op.startswith("v_mfma") and other.writes() & read:
            yield "operand", f"{other.text} | {between} | {mfma.text}"


# wait states behind a matrix instruction before anything but one of its kind, on the same sums, may touch its results
RESULT = {"v_mfma_i32_16x16x64_i8": 8, "v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_i32_32x32x32_i8": 12,
          "v_mfma_f32_16x16x128_f8f6f4": 12, "v_mfma_scale_f32_16x16x128_f8f6f4": 12, "v_mfma_f32_4x4x4_16b_bf16": 5}


def _result(fn: Function, i: int):
    """The results of a matrix instruction are read and written over after its passes."""
    mfma = fn[i]
    out = registers(mfma.operands[0])
    for other, between in fn.after(i, RESULT[mfma.op]):
        if other is mfma or not other.op.startswith(("v_", "buffer_", "global_", "ds_")):
            continue
        touched = registers(" ".join(other.operands[1:3] if other.op.startswith("v_mfma") else other.operands))
        if touched & out:
            yield "result", f"{mfma.text} | {between} | {other.text}"


def check(fn: Function) -> list:
    found = []
    for i in fn.find(" lds"):
        found += _resource(fn, i)
        found += _m0(fn, i)
    for i in fn.find("v_mfma"):
        found += _operands(fn, i)
        found += _result(fn, i)
    return [(kind, fn.name, text) for kind, text in found]


@pytest.fixture(scope="module")
def found(tmp_path_factory):
    from convrot_mlx_amd import _native

    if not OBJDUMP.exists():
        pytest.skip("no disassembler")
    out = defaultdict(list)
    for kind, name, text in check_library(_native.LIB_PATH, tmp_path_factory.mktemp("code"), (" lds", "v_mfma"), check):
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


MFMA = "v_mfma_i32_16x16x64_i8 a[0:3], v[4:7], v[8:11], a[0:3]"
SCALED = "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[4:9], v[12:17], a[0:3], v20, v20 op_sel_hi:[0,0,0] cbsz:2 blgp:2"


def test_the_check_of_operands():
    for write, mfma in (("v_mov_b32_e32 v11, 0", MFMA), ("v_mov_b32_e32 v20, 0x82", SCALED), ("v_accvgpr_write_b32 a2, 0", MFMA)):
        assert [k for k, _, _ in check(function(write, "s_mov_b32 s1, 0", mfma))] == ["operand"]
        assert check(function(write, "s_nop 1", mfma)) == []
    assert check(function("v_mov_b32_e32 v3, 0", MFMA)) == [] and check(function(MFMA, MFMA)) == []


def test_the_check_of_results():
    for read in ("v_accvgpr_read_b32 v1, a2", "v_accvgpr_write_b32 a2, 0", "buffer_store_dword a2, v1, s[0:3], 0 offen"):
        assert [k for k, _, _ in check(function(MFMA, "s_nop 6", read))] == ["result"]
        assert check(function(MFMA, "s_nop 7", read)) == []
    assert check(function(MFMA, MFMA, "v_accvgpr_read_b32 v1, a4")) == []
    # at the end of a loop, and in its next turn
    assert check(function("v_accvgpr_read_b32 v1, a2", "s_nop 7", MFMA, "s_cbranch_scc1 65532 -> 0", "s_nop 7"))
    assert check(function(MFMA, "s_cbranch_scc1 65534 -> 0", "v_accvgpr_read_b32 v1, a2"))


def test_resources(found):
    assert found["resource"] == []


def test_m0(found):
    assert found["m0"] == []


def test_operands(found):
    assert found["operand"] == []


def test_results(found):
    assert found["result"] == []
