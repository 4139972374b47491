"""CPU: what the compiled kernels' assembly has to hold where no run would show its absence reliably.

No VALU instruction written as inline asm reads the result of a 32x32 16-bit MFMA before it stands. The compiler
puts the wait states that gfx950 asks for (12 behind an MFMA of eight passes) only in front of instructions of its
own, so a kernel's inline asm has to stay clear of fresh accumulators. Read from the assembly that the Makefile's
flags give, along every path of every kernel."""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from conftest import ROOT

WAIT = 12
CSRC = os.path.join(ROOT, "aria_amd", "csrc")


def registers(operand):
    m = re.match(r"[-|]*v(?:(\d+)|\[(\d+):(\d+)\])\|?$", operand)
    if not m:
        return []
    return [int(m[1])] if m[1] else range(int(m[2]), int(m[3]) + 1)


def parse(text):
    """kernel -> basic blocks [(label or None, [(line, mnemonic, operands, whether inline asm)])]"""
    out, cur, inline = {}, None, False
    for n, line in enumerate(text.splitlines(), 1):
        s = line.strip()
        if s.startswith(";;#ASM"):
            inline = "START" in s
            continue
        label = re.match(r"([\w.$]+):", line)
        if label:
            if label[1].startswith(".LBB"):
                cur.append((label[1], []))
            elif not label[1].startswith("."):
                cur = out.setdefault(label[1], [(label[1], [])])
            continue
        s = s.split(";")[0].strip()
        if cur is None or not s or s.startswith("."):
            continue
        op, rest = (s.split(None, 1) + [""])[:2]
        cur[-1][1].append((n, op, [o.strip() for o in rest.split(",")], inline))
        if op.startswith("s_cbranch") or op in ("s_branch", "s_endpgm"):
            cur.append((None, []))
    return out


def early_reads(blocks):
    """(line, mnemonic, register, wait states) of inline asm that reads an MFMA's result within WAIT of it, on any path"""
    at = {label: i for i, (label, _) in enumerate(blocks) if label}
    came = [None] * len(blocks)          # register -> least wait states since its MFMA, where a block begins
    came[0] = {}
    todo, found = [0], set()
    while todo:
        i = todo.pop()
        since, after = dict(came[i]), [i + 1]
        for n, op, ops, inline in blocks[i][1]:
            if inline and op.startswith("v_"):
                found.update((n, op, r, since[r]) for o in ops[1:] for r in registers(o) if r in since)
            states = int(ops[0], 0) + 1 if op == "s_nop" else 1
            since = {r: d + states for r, d in since.items() if d + states < WAIT}
            if op.startswith("v_mfma"):
                since.update((r, 0) for r in registers(ops[0]))
            elif op.startswith("v_"):
                for r in registers(ops[0]):
                    since.pop(r, None)
            elif op.startswith("s_cbranch"):
                after = [i + 1, at[ops[0]]]
            elif op in ("s_branch", "s_endpgm"):
                after = [at[ops[0]]] if op == "s_branch" else []
        for j in after:
            if j < len(blocks):
                new = dict(came[j] or {})
                for r, d in since.items():
                    new[r] = min(new.get(r, WAIT), d)
                if new != came[j]:
                    came[j] = new
                    todo.append(j)
    return sorted(found)


def test_the_reader():
    """A read behind a branch, one far enough away, and one of a register written since."""
    text = """k:
\tv_mfma_f32_32x32x16_f16 v[0:15], v[20:23], v[24:27], 0
\ts_cbranch_scc1 .LBB0_2
\ts_nop 11
\t;;#ASMSTART
\tv_max3_f32 v30, v0, v1, v2
\t;;#ASMEND
.LBB0_2:
\tv_mov_b32_e32 v3, 0
\t;;#ASMSTART
\tv_max3_f32 v31, v3, v4, v30
\t;;#ASMEND
\ts_endpgm
"""
    assert [(r, d) for _, _, r, d in early_reads(parse(text)["k"])] == [(4, 2)]


hipcc = pytest.mark.skipif(not shutil.which(os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")), reason="no hipcc")


def assembly(tmp_path, kernel):
    subprocess.run(["make", "-C", CSRC, f"OBJDIR={tmp_path}", f"{tmp_path}/{kernel}.s"], check=True, capture_output=True)
    with open(tmp_path / f"{kernel}.s") as f:
        return f.read()


@hipcc
@pytest.mark.parametrize("kernel", ["k_xattn", "k_attn"])
def test_inline_asm_behind_mfma(tmp_path, kernel):
    kernels = parse(assembly(tmp_path, kernel))
    assert any(op.startswith("v_mfma") for b in kernels.values() for _, ins in b for _, op, _, _ in ins)
    bad = {name: r[:3] for name, b in kernels.items() if (r := early_reads(b))}
    assert not bad, bad


@hipcc
def test_order_within_a_wave(tmp_path):
    """The MXFP4 products of one K group stage their output in LDS wave by wave, without a workgroup's barrier: around each
    of the FM blocks of rows the compiler is told of the order (its wave barrier, no instruction)."""
    text = assembly(tmp_path, "k_mx4_gemm")
    seen = 0
    for body in re.split(r"(?m)^(?=_Z\w+:)", text)[1:]:
        m = re.match(r"_Z10k_mx4_gemmILi(\d+)ELi\d+ELi\d+ELi\d+ELi(\d+)E", body)
        if m and int(m[2]) == 1:
            seen += 1
            assert body.split(".end_amdhsa_kernel")[0].count("; wave barrier") >= 2 * int(m[1]), body[:60]
    assert seen >= 6
