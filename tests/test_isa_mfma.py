"""The built gfx950 code keeps the wait states between a matrix instruction and what touches its result (CPU: the library's own
kernels, disassembled). The hardware leaves them to software: a result of an instruction of P passes may be read or written by a
vector, memory or LDS instruction, or read as another matrix instruction's A or B, P + 4 wait states later at the earliest. The
compiler counts them, but where two ways lead from the matrix instruction to its reader it may count along the longer one only, so
every way is walked here. An instruction is one wait state, s_nop n is n + 1, and the next matrix instruction begins when the one
before has left the matrix core, its P passes later."""
import os
import re
import shutil
import subprocess

import pytest

from rustingstrata_amd import build

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
#: passes (4 cycles each) of the matrix instructions that the library uses
PASSES = {"16x16x32_i8": 4, "16x16x32_f16": 4, "16x16x16_f16": 4, "32x32x16_f16": 8, "16x16x64_i8": 4, "32x32x32_i8": 8, "16x16x32_bf16": 4, "32x32x16_bf16": 8}


def regs(text):
    """The vector and accumulation registers that an operand list names."""
    out = set()
    for kind, a, b, kind1, c in re.findall(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b", text):
        out.update((kind, i) for i in range(int(a), int(b) + 1)) if a else out.add((kind1, int(c)))
    return out


def operands(args):
    """Top-level operands of an instruction."""
    return [a.strip() for a in re.split(r",\s*(?![^\[]*\])", args)]


def parse(lines):
    """{kernel: [(address, op, args, target address or None)]}"""
    kernels, code = {}, None
    for line in lines:
        head = re.match(r"^([0-9a-f]+) <(.*)>:", line)
        if head:
            code = kernels.setdefault(head.group(2), [])
            continue
        body, _, note = line.partition("//")
        m = re.match(r"^\s+([a-z]\w+)\s*(.*?)\s*$", body)
        if code is None or not m:
            continue
        at = int(re.match(r"\s*([0-9A-Fa-f]+)", note).group(1), 16)
        target = None
        if m.group(1).startswith(("s_cbranch", "s_branch")):
            hit = re.search(r"<[^>]*\+0x([0-9a-f]+)>", note) or re.search(r"<[^>+]*>", note)
            target = hit.group(1) if hit and hit.groups() else "0"
        code.append((at, m.group(1), m.group(2), target))
    return kernels


def short_waits(kernels):
    """[(kernel, address, matrix instruction, address, reader, wait states)] of the ways that wait too little; how many were walked."""
    bad, n = [], 0
    for name, code in kernels.items():
        if not code:
            continue
        base = code[0][0]
        index = {at: i for i, (at, *_) in enumerate(code)}
        for i, (at, op, args, _) in enumerate(code):
            m = re.match(r"v_mfma_\w+?_(\d+x\d+x\d+_\w+)$", op)
            if not m:
                continue
            n += 1
            need = PASSES[m.group(1)] + 4
            dst = regs(operands(args)[0])
            todo, seen = [(i + 1, 0, need - 4)], {}  # next instruction, wait states so far, when the matrix core is free
            while todo:
                j, waited, free = todo.pop()
                if j >= len(code) or waited >= need or (waited, free) in seen.setdefault(j, set()):
                    continue
                seen[j].add((waited, free))
                a, o, g, target = code[j]
                if o.startswith("v_mfma"):
                    ops = operands(g)
                    passes = PASSES[re.match(r"v_mfma_\w+?_(\d+x\d+x\d+_\w+)$", o).group(1)]
                    before, waited = waited, max(waited, free)
                    free = waited + passes
                    if waited >= need:
                        continue
                    if (regs(ops[1]) | regs(ops[2])) & dst:
                        bad.append((name, hex(at), op, hex(a), o, before))
                    if regs(ops[0]) == dst:  # (it goes on with the sum, or replaces it: its own readers count from there)
                        continue
                elif o.startswith(("v_", "global_", "flat_", "buffer_", "scratch_", "ds_")) and regs(g) & dst:
                    bad.append((name, hex(at), op, hex(a), o + " " + g, waited))
                    continue
                waits = int(g, 0) + 1 if o == "s_nop" else 1
                if o == "s_endpgm":
                    continue
                if target is not None:
                    to = index.get(base + int(target, 16))
                    assert to is not None, (name, hex(a), o, target)
                    todo.append((to, waited + waits, free))
                if o != "s_branch":
                    todo.append((j + 1, waited + waits, free))
    return bad, n


def test_the_scan_sees_short_waits():
    code = """0000000000000000 <k>:
\tv_mfma_f32_32x32x16_f16 a[0:15], v[0:3], v[4:7], a[0:15]  // 000000000000: 0
\ts_cbranch_scc0 2  // 000000000008: 0 <k+0x14>
\ts_nop 7  // 00000000000C: 0
\ts_nop 7  // 000000000010: 0
\tv_accvgpr_read_b32 v8, a3  // 000000000014: 0
\tv_mfma_f32_16x16x32_f16 v[0:3], v[4:7], v[8:11], v[0:3]  // 000000000018: 0
\ts_nop 6  // 000000000020: 0
\tv_mfma_f32_16x16x32_f16 v[12:15], v[0:3], v[8:11], 0  // 000000000024: 0
\ts_endpgm  // 00000000002C: 0
""".splitlines()
    bad, n = short_waits(parse(code))
    assert n == 3 and [(b[1], b[3], b[5]) for b in bad] == [("0x0", "0x14", 1), ("0x18", "0x24", 7)]


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")
def test_matrix_results_keep_their_wait_states(tmp_path):
    if not os.path.exists(build.OUT):
        build.build()
    lib = shutil.copy(build.OUT, tmp_path)  # (the code objects are extracted beside the file)
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, capture_output=True)
    total = 0
    for f in sorted(f for f in os.listdir(tmp_path) if f.endswith("gfx950")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", os.path.join(tmp_path, f)], check=True, capture_output=True, text=True).stdout
        bad, n = short_waits(parse(text.splitlines()))
        total += n
        assert not bad, (f, len(bad), bad[:4])
    assert total > 0
