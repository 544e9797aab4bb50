"""Loads straight into LDS are issued as inline assembly, whose inside the
compiler's hazard recognizer does not look at.  Two waits are then the source's
own: one wait state between a scalar write of M0, the load's LDS address, and
the load; five between a vector instruction's write of a scalar register
(v_readlane of a spilled one, say) and a memory instruction that reads it.
Checked in the assembly that the sources compile to, along every way to each
load.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
M0_STATES, SGPR_STATES = 1, 5


def registers(text):
    """The scalar registers that an operand list names."""
    found = set()
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        found |= set(range(int(a), int(b) + 1))
    found |= {int(a) for a in re.findall(r"\bs(\d+)\b", text)}
    if re.search(r"\bm0\b", text):
        found.add("m0")
    return found


def functions(text):
    """(name, instructions, predecessors of each) of every function."""
    for m in re.finditer(r"^(_Z\w+):[^\n]*\n(.*?)^\.Lfunc_end", text, re.S | re.M):
        code, labels, open_labels = [], {}, []
        for line in m.group(2).splitlines():
            line = line.split(";")[0].strip()
            if not line:
                continue
            if label := re.match(r"(\.L\w+):", line):
                open_labels.append(label.group(1))
            elif not line.startswith("."):
                for name in open_labels:
                    labels[name] = len(code)
                open_labels = []
                code.append(line)
        before = [[] for _ in code]
        for i, line in enumerate(code):
            if i + 1 < len(code) and not line.startswith(("s_branch", "s_endpgm", "s_setpc")):
                before[i + 1].append(i)
            if line.startswith(("s_branch", "s_cbranch")):
                target = line.split()[-1]
                if target in labels:
                    before[labels[target]].append(i)
        yield m.group(1), code, before


def written(line):
    """(scalar registers written, whether by a vector instruction)."""
    op, _, rest = line.partition(" ")
    first = rest.split(",")[0]
    if op.startswith("v_"):
        if op.startswith(("v_cmp", "v_readlane", "v_readfirstlane")):
            return registers(first), True
        if "_co_" in op or op.startswith("v_div_scale"):
            return registers(rest.split(",")[1] if "," in rest else ""), True
        return set(), True
    if op.startswith("s_") and not op.startswith(("s_nop", "s_waitcnt", "s_cbranch", "s_branch", "s_barrier", "s_setprio",
                                                  "s_cmp", "s_bitcmp", "s_endpgm")):
        return registers(first), False
    return set(), False


def states(line):
    m = re.match(r"s_nop (\w+)", line)
    return int(m.group(1), 0) + 1 if m else 1


def violations(text):
    """(loads into LDS, those that may come too early)."""
    loads, bad = 0, []
    for name, code, before in functions(text):
        for i, line in enumerate(code):
            if not (line.startswith("buffer_load") and line.endswith(" lds")):
                continue
            loads += 1
            reads = registers(line)
            ways, seen = [(j, 0) for j in before[i]], set()
            while ways:
                j, passed = ways.pop()
                if passed >= SGPR_STATES or (j, passed) in seen:
                    continue
                seen.add((j, passed))
                regs, vector = written(code[j])
                if "m0" in regs and passed < M0_STATES:
                    bad.append((name, "m0", code[j], line))
                if vector and regs & reads:
                    bad.append((name, "sgpr", code[j], line))
                ways += [(k, passed + states(code[j])) for k in before[j]]
    return loads, bad


def test_the_check_sees_what_it_looks_for():
    body = "_Zk:\n\ts_mov_b32 m0, s4\n%s\tbuffer_load_dwordx4 v1, s[8:11], 0 offen lds\n\ts_endpgm\n.Lfunc_end0:\n"
    assert [b[1] for b in violations(body % "")[1]] == ["m0"]
    assert violations(body % "\ts_nop 0\n") == (1, [])
    assert violations(body % "\tv_add_u32_e32 v2, v3, v4\n") == (1, [])
    assert [b[1] for b in violations(body % "\tv_readlane_b32 s9, v1, 3\n\ts_nop 3\n")[1]] == ["sgpr"]
    assert violations(body % "\tv_readlane_b32 s9, v1, 3\n\ts_nop 4\n") == (1, [])
    assert violations(body % "\tv_readlane_b32 s12, v1, 3\n\ts_nop 0\n") == (1, [])
    loop = "_Zk:\n.LBB0_1:\n\tbuffer_load_dwordx4 v1, s[8:11], 0 offen lds\n\ts_mov_b32 m0, s4\n%s.LBB0_2:\n" \
           "\ts_cbranch_scc1 .LBB0_1\n\ts_endpgm\n.Lfunc_end0:\n"
    assert violations(loop % "") == (1, [])  # the branch is a state
    assert [b[1] for b in violations(loop % "\tv_readfirstlane_b32 s8, v1\n")[1]] == ["sgpr"]


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
@pytest.mark.parametrize("source,fewest", [("ff_tile", 60), ("ff_sampled", 100), ("spmm_dense", 20)])
def test_loads_into_lds_wait_for_their_scalars(tmp_path, source, fewest):
    csrc = os.path.join(ROOT, "xspmm_amd", "csrc")
    out = str(tmp_path / "out.s")
    subprocess.run([HIPCC, "-std=c++20", "-O3", "-fPIC", "-I" + os.path.join(ROOT, "include"), "-I" + csrc,
                    "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-S", "--cuda-device-only", os.path.join(csrc, source + ".hip"), "-o", out],
                   check=True, capture_output=True)
    with open(out) as f:
        loads, bad = violations(f.read())
    assert loads >= fewest
    assert not bad, (len(bad), bad[:3])
