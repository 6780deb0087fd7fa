"""The windowed attention's kernels as they were compiled: what a matrix instruction multiplies is ready.  (tests/test_window_isa_cpu.py follows the
results to every other unit; a result that is the first or second operand of another matrix instruction has to wait as long.  An accumulator that is
handed on as the third operand does not.)"""
import glob
import os
import shutil
import subprocess

import pytest

from test_window_isa_cpu import OBJDUMP, _kernels, _registers, _wait_states


def _operands(args):
    """The operands of an instruction as register lists (commas inside brackets do not occur in this assembly)."""
    return [_registers(a) for a in args.split(",")]


def _early_products(code):
    """Matrix instructions that multiply a result before it is ready, over every path: for each instruction the states still to pass for every
    pending register when it is reached, the longest over all ways to it."""
    first = code[0][0]
    at = {addr - first: i for i, (addr, _, _) in enumerate(code)}
    todo, seen, early = [(0, {})], [None] * len(code), set()
    while todo:
        i, wait = todo.pop()
        while i < len(code):
            have = seen[i]
            if have is not None:
                if all(have.get(r, 0) >= n for r, n in wait.items()):
                    break
                wait = {r: max(have.get(r, 0), wait.get(r, 0)) for r in {*have, *wait}}
            seen[i] = wait
            text, target = code[i][1], code[i][2]
            op, _, args = text.partition(" ")
            passed = int(args, 0) + 1 if op == "s_nop" else 1
            matrix = _operands(args) if "mfma" in op else None
            if matrix:
                early |= {(text, r) for operand in matrix[1:3] for r in operand if r in wait}
            wait = {r: n - passed for r, n in wait.items() if n > passed}
            if matrix:
                wait.update((r, _wait_states(op)) for r in matrix[0])
            if op.startswith(("s_branch", "s_cbranch")):
                todo.append((at[target], wait))
            if op in ("s_branch", "s_endpgm"):
                break
            i += 1
    return early


def test_the_check_itself():
    mfma = "v_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], "
    for operands, waits, found in (("v[32:47], v[4:7], v[20:23], 0", 10, True), ("v[32:47], v[20:23], v[12:15], 0", 10, True),
                                   ("v[32:47], v[4:7], v[20:23], 0", 12, False), ("v[0:15], v[24:27], v[28:31], v[0:15]", 1, False)):
        use = "v_mfma_f32_32x32x16_bf16 " + operands
        straight = [(0, mfma + "0", 0), (8, f"s_nop {waits - 1}", 0), (12, use, 0), (20, "s_endpgm", 0)]
        assert bool(_early_products(straight)) == found, operands
        # (the same behind a loop's back edge, where the way around is the short one)
        loop = [(0, "s_branch 2", 20), (4, "s_nop 15", 0), (8, "s_nop 15", 0), (12, use, 0), (20, mfma + "0", 0), (28, f"s_nop {waits - 2}" if waits > 1 else "s_nop 0", 0),
                (32, "s_cbranch_scc1 1", 12), (36, "s_endpgm", 0)]
        assert bool(_early_products(loop)) == found, operands


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
        for name, code in _kernels(isa):
            if any("mfma" in t for _, t, _ in code):
                found += 1
                assert not _early_products(code), name
    assert found == 3 * 3 * 4 * 2      # forward, dQ, dK / dV of three types, four head dims, wide and narrow
