"""The fragment reads of csrc/class_loss.hip that are written in inline asm are waited for behind other instructions. The compiler takes their registers as written
at once, so nothing but its good will keeps a copy or a spill of one from coming before the wait. This looks through the assembly of the build: between such a
read and the next s_waitcnt lgkmcnt(0), on every path, no instruction names a register that is in flight."""
import re
import shlex
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "cerberusdet_amd" / "csrc"


def registers(text):
    out = set()
    for kind, lo, hi, one_kind, one in re.findall(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b", text):
        out |= {(one_kind, int(one))} if one else {(kind, r) for r in range(int(lo), int(hi) + 1)}
    return out


def touched_in_flight(assembly):
    """(reads in asm blocks, what touches their registers too early, waits that found some in flight)."""
    flying, at_label, in_asm, reads, bad, waits, seen = {}, {}, False, 0, [], 0, set()
    for number, line in enumerate(assembly.splitlines(), 1):
        label = re.match(r"([.\w$]+):", line)
        if label:
            if not label.group(1).startswith(".L"):
                if flying:
                    bad.append(f"{number}: a function ends with reads in flight")
                flying, at_label, seen = {}, {}, set()
            else:
                flying = {**at_label.pop(label.group(1), {}), **flying}
                seen.add(label.group(1))
            continue
        if "#ASMSTART" in line or "#ASMEND" in line:
            in_asm = "#ASMSTART" in line
            continue
        code = line.split(";")[0].strip()
        if not code or code.startswith("."):
            continue
        op, _, args = code.partition(" ")
        if op == "s_waitcnt" and "lgkmcnt(0)" in args:
            waits += bool(flying)
            flying = {}
            continue
        if op.startswith("s_cbranch") or op == "s_branch":
            target = args.strip()
            if flying and target in seen:
                bad.append(f"{number}: a loop is closed with reads in flight")
            at_label[target] = {**at_label.get(target, {}), **flying}
            continue
        early = registers(args) & set(flying)
        if early or (op == "s_endpgm" and flying):
            bad.append(f"{number}: {code} before the wait for {sorted(early)[:4]}")
        if in_asm and op.startswith("ds_read"):
            reads += 1
            flying.update((r, number) for r in registers(args.split(",")[0]))
    return reads, bad, waits


def test_the_check_sees_what_it_looks_for():
    read = ";;#ASMSTART\n\tds_read_b128 v[4:7], v1\n\t;;#ASMEND\n"
    assert touched_in_flight("f:\n" + read + "\tv_add_f32 v8, v9, v10\n\ts_waitcnt vmcnt(0) lgkmcnt(0)\n\tv_mov_b32_e32 v8, v4\n") == (1, [], 1)
    for early in ("\tv_mov_b32_e32 v8, v7\n", "\tscratch_store_dwordx2 off, v[6:7], off\n", "\tv_mov_b32_e32 v5, 0\n", read.replace("v1", "v2"), "\ts_waitcnt lgkmcnt(1)\n\tv_mov_b32_e32 v8, v4\n",
                  "\ts_endpgm\n"):
        assert touched_in_flight("f:\n" + read + early)[1]
    assert touched_in_flight("f:\n.LBB0_1:\n" + read + "\ts_cbranch_scc1 .LBB0_1\n\ts_waitcnt lgkmcnt(0)\n")[1]
    assert touched_in_flight("f:\n" + read + "\ts_cbranch_scc1 .LBB0_2\n\ts_waitcnt lgkmcnt(0)\n.LBB0_2:\n\tv_mov_b32_e32 v8, v4\n")[1]


@pytest.mark.skipif(not Path("/opt/rocm/bin/hipcc").exists() or not shutil.which("make"), reason="needs hipcc and make")
def test_no_register_of_a_read_in_flight_is_touched(tmp_path):
    lines = subprocess.run(["make", "-n", "-B", "build/class_loss.o"], cwd=CSRC, check=True, capture_output=True, text=True).stdout.splitlines()
    command = shlex.split(next(l for l in lines if "class_loss.hip" in l))
    out = tmp_path / "class_loss.s"
    i = command.index("-c")
    command = command[:i] + ["-S", "--cuda-device-only"] + command[i + 1:]
    command[command.index("-o") + 1] = str(out)
    subprocess.run(command, cwd=CSRC, check=True, capture_output=True)
    reads, bad, waits = touched_in_flight(out.read_text())
    assert reads >= 100 and waits >= 12  # both tiles' products are there
    assert not bad, bad[:10]
