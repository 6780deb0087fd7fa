"""The windowed attention's kernels as they were compiled: no calls (a tile step that is not inlined goes through scratch memory), and every
result of a matrix instruction is left alone for as many wait states as the hardware asks for, on every path.  (Where a branch stands between
the instruction and the first read the compiler has counted along the longer path only; the source writes the wait states out.)"""
import glob
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/lib/llvm/bin/llvm-objdump"
OPERAND = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def _registers(text):
    return [(m.group(1), i) for m in OPERAND.finditer(text) for i in range(int(m.group(2) or m.group(4)), int(m.group(3) or m.group(4)) + 1)]


def _wait_states(op):
    """Between a matrix instruction and another unit's access to its result: 18 behind 16 passes (fp32), 12 behind 8 (16-bit)."""
    return 18 if "32x32x2_f32" in op else 12 if "32x32x16" in op else 20


def _kernels(isa):
    for name, body in re.findall(r"\n[0-9a-f]+ <(\S+)>:\n(.*?)(?=\n\n|\Z)", isa, flags=re.S):
        code = []
        for line in body.split("\n"):
            text, _, rest = line.partition("//")
            m = re.match(r"\s*([0-9A-F]+):[^<]*(?:<[^>]*?(?:\+0x([0-9a-f]+))?>)?", rest)
            if text.strip() and m:
                code.append((int(m.group(1), 16), text.strip(), int(m.group(2) or "0", 16)))
        yield name, code


def _early_accesses(code):
    first = code[0][0]
    at = {addr - first: i for i, (addr, _, _) in enumerate(code)}
    starts = {0} | {i + 1 for i, (_, t, _) in enumerate(code) if t.startswith(("s_cbranch", "s_branch", "s_endpgm"))}
    starts |= {at[target] for _, t, target in code if t.startswith(("s_cbranch", "s_branch"))}
    starts = sorted(s for s in starts if s < len(code))
    block_of = {s: b for b, s in enumerate(starts)}
    pending = [dict() for _ in starts]      # registers not ready yet at the block's start -> wait states still to pass
    todo, early = set(range(len(starts))), set()
    while todo:
        b = min(todo)
        todo.discard(b)
        wait, end = dict(pending[b]), starts[b + 1] if b + 1 < len(starts) else len(code)
        for i in range(starts[b], end):
            op, _, args = code[i][1].partition(" ")
            passed = int(args, 0) + 1 if op == "s_nop" else 1
            matrix = "mfma" in op
            if not matrix and op.startswith(("v_", "ds_", "global_", "buffer_", "scratch_", "flat_")):
                early |= {(code[i][1], r) for r in _registers(args) if r in wait}
            wait = {r: n - passed for r, n in wait.items() if n > passed}
            if matrix:
                wait.update((r, _wait_states(op)) for r in _registers(args.split(",")[0]))
        last, target = code[end - 1][1], code[end - 1][2]
        nxt = [] if last.startswith(("s_branch", "s_endpgm")) or end >= len(code) else [block_of[end]]
        if last.startswith(("s_branch", "s_cbranch")):
            nxt.append(block_of[at[target]])
        for n in nxt:
            more = {r: v for r, v in wait.items() if pending[n].get(r, 0) < v}
            if more:
                pending[n].update(more)
                todo.add(n)
    return early


def test_the_check_itself():
    mfma = "v_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], 0"
    for nops, left_out in ((11, False), (10, True)):
        code = [(0, mfma, 0), (8, f"s_nop {nops - 1}", 0), (12, "s_cbranch_scc1 1", 20), (16, "s_nop 0", 0), (20, "v_mov_b32_e32 v30, v3", 0),
                (24, "s_endpgm", 0)]
        assert bool(_early_accesses(code)) == left_out      # (taken: the branch and the no-operations alone stand between)


def test_window_kernels_in_the_library(tmp_path):
    from dose_prediction_amd import _lib
    if not os.path.exists(OBJDUMP):
        pytest.skip("llvm-objdump not available")
    so = shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", str(so)], check=True, capture_output=True, cwd=tmp_path)
    found = 0
    for co in sorted(glob.glob(str(tmp_path / "lib.so.*gfx950"))):
        if "k_win_dkv" not in subprocess.run([OBJDUMP, "-t", co], capture_output=True, text=True).stdout:
            continue
        isa = subprocess.run([OBJDUMP, "-d", co], capture_output=True, text=True, check=True).stdout
        assert "s_swappc" not in isa and "s_setpc" not in isa
        for name, code in _kernels(isa):
            if any("mfma" in t for _, t, _ in code):
                found += 1
                assert not _early_accesses(code), name
    assert found == 3 * 3 * 4 * 2      # forward, dQ, dK / dV of three types, four head dims, wide and narrow
