"""Instruction-level check of the built gfx950 code of the products of 16-bit operands (CPU
only): their matrix instructions are inline asm, so the compiler pads nothing around them.
No accumulator of a v_mfma is read or written by another kind of instruction in the wait
states after it (16 x 16 x 32: eight passes, 11 wait states before a VALU or memory
instruction reads it), and no operand of one is written by a VALU instruction in the two wait
states before it, along the code as it lies."""
import os
import re
import shutil
import subprocess

import pytest

from test_isa_hazards import LIB, OBJDUMP, code_objects

NEED = 16
AGPR = re.compile(r"\ba(?:\[(\d+):(\d+)\]|(\d+)\b)")


def agprs(text):
    out = set()
    for m in AGPR.finditer(text):
        out |= set(range(int(m[1]), int(m[2]) + 1)) if m[1] else {int(m[3])}
    return out


def instructions(lines):
    for line in lines:
        s = line.split("//")[0].strip()
        if s and not s.endswith(">:") and not s.startswith((";", ".", "/", "Disassembly")):
            yield s


def early_uses(lines):
    """Uses of an accumulator fewer than NEED wait states after its v_mfma."""
    busy, hits, now = {}, [], 0
    for s in instructions(lines):
        op = s.split()[0]
        if op.startswith("v_mfma"):
            for r in agprs(s.split(",")[0]):
                busy[r] = now
            # a matrix instruction holds the next one back for its passes
            now += 4
            continue
        if op == "s_nop":
            now += int(s.split()[1], 0) + 1
            continue
        used = agprs(s)
        for r in used:
            if r in busy and now - busy[r] < NEED:
                hits.append(s)
                break
        now += 1
    return hits


VGPR = re.compile(r"\bv(?:\[(\d+):(\d+)\]|(\d+)\b)")


def registers(text):
    out = {("a", r) for r in agprs(text)}
    for m in VGPR.finditer(text):
        out |= {("v", r) for r in
                (range(int(m[1]), int(m[2]) + 1) if m[1] else (int(m[3]),))}
    return out


def late_writes(lines):
    """Operands of a v_mfma that a VALU instruction wrote fewer than two wait states before."""
    recent, hits = [], []  # (wait states since, registers)
    for s in instructions(lines):
        op = s.split()[0]
        if op == "s_nop":
            n = int(s.split()[1], 0) + 1
            recent = [(w + n, r) for w, r in recent if w + n < 2]
            continue
        if op.startswith("v_mfma"):
            used = registers(s)
            if any(r & used for _, r in recent):
                hits.append(s)
            recent = [(w + 1, r) for w, r in recent if w + 1 < 2]
            continue
        recent = [(w + 1, r) for w, r in recent if w + 1 < 2]
        if op.startswith("v_") and not op.startswith("v_cmp"):
            recent.append((0, registers(s.split(None, 1)[1].split(",")[0])))
    return hits


def kernels(asm):
    """{name: lines} of the tile kernels of one code object."""
    out, name = {}, None
    for line in asm.splitlines():
        m = re.match(r"^[0-9a-f]+ <(.+)>:$", line)
        if m:
            name = m[1] if "k_dense_tile" in m[1] else None
            if name:
                out[name] = []
        elif name:
            out[name].append(line)
    return out


@pytest.mark.skipif(not os.path.exists(LIB), reason="library not built")
@pytest.mark.skipif(not os.path.exists(OBJDUMP) or not shutil.which("objcopy"),
                    reason="llvm-objdump / objcopy not available")
def test_sums_are_waited_for(tmp_path):
    seen = 0
    for k, co in enumerate(code_objects(LIB)):
        if b"k_dense_tile" not in co:
            continue
        f = tmp_path / f"co{k}.o"
        f.write_bytes(co)
        asm = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(f)], check=True,
                             capture_output=True, text=True).stdout
        for name, lines in kernels(asm).items():
            assert any("v_mfma" in s for s in lines), name
            hits = early_uses(lines)
            assert not hits, (name, hits[:4])
            hits = late_writes(lines)
            assert not hits, (name, hits[:4])
            seen += 1
    assert seen > 0, "no tile kernels found: scan is broken"


def test_scanner_flags_the_measured_case():
    bad = ["\tv_mfma_f32_16x16x32_bf16 a[60:63], v[54:57], v[74:77], a[60:63]",
           "\ts_add_i32 s10, s10, 1", "\tv_accvgpr_read_b32 v54, a60"]
    assert len(early_uses(bad)) == 1
    assert early_uses([bad[0], "\ts_nop 15", "\ts_nop 15", bad[2]]) == []
    assert early_uses([bad[0], "\tv_accvgpr_read_b32 v54, a59"]) == []
    write = "\tv_accvgpr_write_b32 a60, 0"
    assert len(late_writes([write, bad[0]])) == 1
    assert len(late_writes([write, "\ts_nop 0", bad[0]])) == 1
    assert late_writes([write, "\ts_nop 1", bad[0]]) == []
    assert len(late_writes(["\tv_mov_b32_e32 v57, v1", bad[1], bad[0]])) == 1
    assert late_writes(["\tv_mov_b32_e32 v58, v1", bad[0]]) == []


@pytest.mark.skipif(not os.path.exists(LIB), reason="library not built")
@pytest.mark.skipif(not os.path.exists(OBJDUMP) or not shutil.which("objcopy"),
                    reason="llvm-objdump / objcopy not available")
def test_tiles_use_no_scratch(tmp_path):
    """Accumulators that the epilogue picks by an index that the compiler cannot see through go
    to scratch memory, all of them (4096 x 16384 x 4096: 425 us became 645)."""
    seen = 0
    for k, co in enumerate(code_objects(LIB)):
        if b"k_dense_tile" not in co:
            continue
        f = tmp_path / f"co{k}.o"
        f.write_bytes(co)
        asm = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(f)], check=True,
                             capture_output=True, text=True).stdout
        for name, lines in kernels(asm).items():
            hits = [s for s in instructions(lines) if s.startswith("scratch_")]
            assert not hits, (name, len(hits))
            seen += 1
    assert seen > 0, "no tile kernels found: scan is broken"
