"""The built kernels' matrix instructions: nothing takes a product's result before it is written.

The hardware does not wait by itself: between a matrix instruction and another use of its result (or another write of the same
registers) a number of wait states has to pass, 8 after the 16-row and 12 after the 32-row instructions of the bf16 and fp16
products here (4 and 8 passes). The compiler counts them, but behind the join of two paths it may count the longer one's.
Every path from every matrix instruction of the library is followed here, in the disassembly of this repository's own code.
"""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

from foldforge_amd import build

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
WAITS = {"16x16x16": 8, "16x16x32": 8, "32x32x16": 12}
FUNCTION = re.compile(r"^([0-9a-f]+) <(\S+)>:$")
LINE = re.compile(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]{12}): [0-9A-F ]+(?:<(\S+?)(?:\+0x([0-9a-f]+))?>)?$")
REGISTER = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def registers(operands: str) -> set[tuple[str, int]]:
    found = set()
    for kind, first, last, one in REGISTER.findall(operands):
        found |= {(kind, r) for r in range(int(first or one), int(last or one) + 1)}
    return found


def early_uses(name: str, start: int, code: list[tuple[int, str, str, int | None]]) -> list[str]:
    """Of one kernel (address, operation, operands, branch target): uses of a result that come too early."""
    at = {address: i for i, (address, *_) in enumerate(code)}
    found = []
    for i, (address, op, operands, _) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        need = WAITS[op.split("_")[3]]
        result = registers(re.match(r"[va]\[\d+:\d+\]", operands)[0])
        paths, best = [(i + 1, 0)], {}
        while paths:
            j, passed = paths.pop()
            if j >= len(code) or passed >= need or best.get(j, need) <= passed:
                continue
            best[j] = passed
            _, other, used, target = code[j]
            if other == "s_endpgm":
                continue
            if other == "s_nop":
                paths.append((j + 1, passed + int(used, 0) + 1))
                continue
            if other.startswith("v_mfma"):
                used = ", ".join(re.findall(r"[va]\[\d+:\d+\]", used)[1:3])  # (its sum may be the next one's)
            if other.startswith(("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")) and registers(used) & result:
                found.append(f"{name}: {op} at {address:x}, {other} {used} {passed} of {need} wait states on")
                continue
            if target is not None:
                paths.append((at[target], passed + 1))
            if other != "s_branch":
                paths.append((j + 1, passed + 1))
    return found


def test_registers():
    assert registers("v[2:4], a7, v10, s[0:3], 0x7f") == {("v", 2), ("v", 3), ("v", 4), ("a", 7), ("v", 10)}


def test_early_uses():
    """A join that a short path reaches, on code that is made up."""
    product = (0, "v_mfma_f32_32x32x16_bf16", "v[0:15], v[16:19], v[20:23], v[0:15]", None)
    code = [product, (8, "s_cbranch_vccz", "4", 24), (12, "s_nop", "11", None), (16, "s_nop", "0", None),
            (24, "s_nop", "5", None), (28, "v_mul_f32_e32", "v0, 2.0, v0", None), (32, "s_endpgm", "", None)]
    assert len(early_uses("kernel", 0, code)) == 1
    code[4] = (24, "s_nop", "10", None)
    assert early_uses("kernel", 0, code) == []


def test_no_result_is_used_before_it_is_written(tmp_path: Path):
    if not Path(OBJDUMP).exists():
        pytest.skip("no llvm-objdump")
    library = tmp_path / build.LIBRARY.name
    shutil.copy(build.LIBRARY, library)
    subprocess.run([OBJDUMP, "--offloading", library.name], cwd=tmp_path, check=True, capture_output=True)
    products, found = 0, []
    for code_object in sorted(tmp_path.glob(f"*{build.ARCH}")):
        listing = subprocess.run([OBJDUMP, "-d", str(code_object)], check=True, capture_output=True, text=True).stdout
        starts, kernels, current = {}, {}, None
        for line in listing.splitlines():
            head = FUNCTION.match(line)
            if head:
                current = kernels.setdefault(head[2], [])
                starts[head[2]] = int(head[1], 16)
                continue
            m = LINE.match(line)
            if m and current is not None:
                target = starts[m[4]] + int(m[5] or "0", 16) if m[4] and "branch" in m[1] else None
                current.append((int(m[3], 16), m[1], m[2], target))
                products += m[1].startswith("v_mfma")
        for name, code in kernels.items():
            found += early_uses(name, starts[name], code)
    assert products > 1000
    assert not found, "\n".join(found)
