"""The machine code of the built library, as the disassembler lists it, for checks of its wait states."""

from __future__ import annotations

import re
import shutil
import subprocess
from collections import defaultdict
from concurrent.futures import ProcessPoolExecutor
from pathlib import Path

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
_REGISTER = re.compile(r"\b([sva])(?:(\d+)\b|\[(\d+):(\d+)\])|\b(vcc|m0|exec)\b")
_TARGET = re.compile(r"\+0x([0-9a-f]+)>")


def registers(text: str) -> set:
    """Registers that an operand (or several) names: ("v", 3), "m0", .."""
    out = set()
    for m in _REGISTER.finditer(text):
        if m[5]:
            out.add(m[5])
        elif m[2]:
            out.add((m[1], int(m[2])))
        else:
            out.update((m[1], i) for i in range(int(m[3]), int(m[4]) + 1))
    return out


class Instruction:
    __slots__ = ("op", "operands", "address", "text")

    def __init__(self, line: str):
        text, _, code = line.partition("//")
        self.text = text.strip()
        self.op, _, rest = self.text.partition(" ")
        self.operands = [t.strip() for t in rest.split(",")] if rest else []
        self.address = int(code.split(":", 1)[0], 16)

    def writes(self) -> set:
        """Registers a vector or scalar instruction writes (carries and the like among them)."""
        if not self.operands or self.op.startswith(("s_cmp", "s_bitcmp", "s_waitcnt", "s_nop", "s_cbranch", "s_branch")):
            return set()
        out = registers(self.operands[0])
        if self.op.startswith("v_") and len(self.operands) > 1 and (
                "_co_" in self.op or "swap" in self.op or self.op.startswith(("v_div_scale", "v_mad_u64", "v_mad_i64"))):
            out |= registers(self.operands[1])
        return out

    def states(self) -> int:
        return int(self.operands[0], 0) + 1 if self.op == "s_nop" else 1


class Function:
    """A kernel's instructions and the ways between them."""

    def __init__(self, name: str, lines: list[str]):
        self.name = name
        self._lines = lines
        self._parsed: dict[int, Instruction] = {}
        base = self[0].address
        places = {}
        branches = []
        for i, line in enumerate(lines):
            if "s_cbranch" in line or "s_branch" in line:
                m = _TARGET.search(line)
                branches.append((i, base + (int(m[1], 16) if m else 0)))
        if branches:
            places = {int(line.partition("//")[2].split(":", 1)[0], 16): i for i, line in enumerate(lines)}
        self._into = defaultdict(list)
        self._out = {}
        for i, target in branches:
            if target in places:
                self._into[places[target]].append(i)
                self._out[i] = places[target]

    def __len__(self) -> int:
        return len(self._lines)

    def __getitem__(self, i: int) -> Instruction:
        if i not in self._parsed:
            self._parsed[i] = Instruction(self._lines[i])
        return self._parsed[i]

    def find(self, text: str) -> list[int]:
        return [i for i, line in enumerate(self._lines) if text in line]

    def _near(self, i: int, states: int, steps):
        """(instruction, wait states between) for what lies within `states` of instruction i along any way."""
        best, todo = {}, [(i, 0)]
        while todo:
            j, between = todo.pop()
            for k in steps(j):
                if between < states and best.get(k, states) > between:
                    best[k] = between
                    todo.append((k, between + self[k].states()))
        return [(self[k], between) for k, between in best.items()]

    def before(self, i: int, states: int):
        def steps(j):
            back = list(self._into.get(j, ()))
            if j and not self[j - 1].op.startswith(("s_branch", "s_endpgm", "s_setpc")):
                back.append(j - 1)
            return back

        return self._near(i, states, steps)

    def after(self, i: int, states: int):
        def steps(j):
            on = [self._out[j]] if j in self._out else []
            if j + 1 < len(self) and not self[j].op.startswith(("s_branch", "s_endpgm", "s_setpc")):
                on.append(j + 1)
            return on

        return self._near(i, states, steps)


def _check(args) -> list:
    """What check(function) finds, over the functions of one code object whose lines hold one of `texts`."""
    path, texts, check = args
    found = []
    run = subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], stdout=subprocess.PIPE,
                           text=True)
    name, lines, wanted = "", [], False

    def done():
        if wanted and lines:
            found.extend(check(Function(name, lines)))

    for line in run.stdout:
        if line.startswith("\t"):
            if "//" in line:
                lines.append(line)
                wanted = wanted or any(t in line for t in texts)
        elif line.startswith("<"):
            done()
            name, lines, wanted = line.strip(), [], False
    done()
    assert run.wait() == 0
    return found


def check_library(library: Path, folder: Path, texts: tuple, check) -> list:
    """check(function) over the library's kernels (those with a line that holds one of `texts`), all it finds."""
    copy = folder / library.name
    shutil.copy(library, copy)
    subprocess.run([OBJDUMP, "--offloading", str(copy)], check=True, stdout=subprocess.DEVNULL)
    objects = sorted(folder.glob(f"{library.name}.*gfx950"), key=lambda p: -p.stat().st_size)
    assert objects
    with ProcessPoolExecutor(min(4, len(objects))) as pool:
        return [f for part in pool.map(_check, [(p, texts, check) for p in objects]) for f in part]
