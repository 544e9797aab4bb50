"""Loads straight into LDS of the 8-bit products' tiles and lists and of the products behind
orthogonalised updates, in the assembly that the sources compile to.

The wait states before each such load, as in test_lds_load_hazards.  And the count
behind the waits of tiles and lists for a window of x: it lets the loads of the last steps' blocks
be under way, so at least as many loads of blocks have to stand between the window's
last load into LDS and the wait, wherever the compiler put them.
"""
from __future__ import annotations

import os
import re
import subprocess

import pytest

from test_lds_load_hazards import HIPCC, ROOT, functions, violations


def assembly(tmp_path, source):
    csrc = os.path.join(ROOT, "xspmm_amd", "csrc")
    out = str(tmp_path / "out.s")
    subprocess.run([HIPCC, "-std=c++20", "-O3", "-fPIC", "-I" + os.path.join(ROOT, "include"), "-I" + csrc,
                    "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-S", "--cuda-device-only", os.path.join(csrc, source + ".hip"), "-o", out],
                   check=True, capture_output=True)
    with open(out) as f:
        return f.read()


def is_lds(line):
    return line.startswith("buffer_load") and line.endswith(" lds")


def is_block(line):
    return line.startswith("buffer_load_dwordx4") and not line.endswith(" lds")


def fewest_blocks_since(code, before, wait):
    """The fewest loads of blocks on any way back from a wait to a load into LDS (None: no way to one)."""
    best, seen = None, {}
    ways = [(j, 0) for j in before[wait]]
    while ways:
        j, blocks = ways.pop()
        if seen.get(j, 1 << 30) <= blocks:
            continue
        seen[j] = blocks
        if is_lds(code[j]):
            best = blocks if best is None else min(best, blocks)
            continue
        blocks += is_block(code[j])
        ways += [(k, blocks) for k in before[j]]
    return best


def test_the_check_sees_what_it_looks_for():
    text = ("_Zk:\n.LBB0_1:\n\tbuffer_load_dwordx4 v1, s[8:11], 0 offen lds\n%s\ts_waitcnt vmcnt(2)\n\ts_barrier\n"
            "\ts_cbranch_scc1 .LBB0_1\n\ts_endpgm\n.Lfunc_end0:\n")
    load = "\tbuffer_load_dwordx4 v[2:5], v6, s[8:11], 0 offen\n"
    for n in (0, 1, 2):
        (_, code, before), = functions(text % (load * n))
        wait = next(i for i, line in enumerate(code) if line.startswith("s_waitcnt"))
        assert fewest_blocks_since(code, before, wait) == n


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_tiles_wait_for_their_window(tmp_path):
    text = assembly(tmp_path, "ff_int8_tile")
    loads, bad = violations(text)
    assert loads >= 60 and not bad, (len(bad), bad[:3])
    kernels = 0
    for name, code, before in functions(text):
        if "ff_int8_tile_kernel" not in name:
            continue
        kernels += 1
        # the wait that stands in the source: vmcnt(12) next to a barrier
        waits = [i for i, line in enumerate(code) if line == "s_waitcnt vmcnt(12)"
                 and any("s_barrier" in c for c in code[i:i + 12])]
        assert waits, name
        found = [fewest_blocks_since(code, before, w) for w in waits]
        assert any(f is not None for f in found) and all(f is None or f >= 12 for f in found), (name, found)
    assert kernels == 6


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_lists_wait_for_their_window(tmp_path):
    text = assembly(tmp_path, "ff_int8_list")
    loads, bad = violations(text)
    assert loads >= 18 * 8 and not bad, (len(bad), bad[:3])
    kernels = 0
    for name, code, before in functions(text):
        found = re.search(r"ff_int8_list_kernelI.*Lb[01]ELi([123])EE", name)
        if not found:
            continue
        kernels += 1
        # two rows' blocks may be under way: vmcnt(2 Q) next to a barrier
        most = 2 * int(found.group(1))
        waits = [i for i, line in enumerate(code) if line == f"s_waitcnt vmcnt({most})"
                 and any("s_barrier" in c for c in code[i:i + 12])]
        assert waits, name
        fewest = [fewest_blocks_since(code, before, w) for w in waits]
        assert any(f is not None for f in fewest) and all(f is None or f >= most for f in fewest), (name, fewest)
    assert kernels == 18


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_products_of_updates_wait_for_their_scalars(tmp_path):
    loads, bad = violations(assembly(tmp_path, "ff_orthogonal"))
    assert loads >= 200 and not bad, (len(bad), bad[:3])
