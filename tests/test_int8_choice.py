"""Which kernel a product in 8-bit integers takes, asked of the library (no GPU is)."""
from __future__ import annotations

import ctypes as C
import itertools
import math
import os
import re
import shutil
import subprocess

import pytest

import xspmm_amd as X
from test_feed_forward_capi import BAD, BF16, refused

FEW, WALK, LISTS, TILES = range(4)
CODES = {"f16": X.F16, "bf16": BF16, "f32": X.F32}


@pytest.fixture(scope="module")
def lib():
    from xspmm_amd import int8

    return int8._load()


def blocks(M, K, density):
    return round(-(-M // 16) * -(-K // 16) * density)


def chosen(lib, weights, M, K, N, density, up=None, quantized=False, kind="bf16"):
    """(kernel, its two numbers) of a product of weights with that share of their blocks."""
    k = (C.c_int32 * 3)(-1, -1, -1)
    up = blocks(M, K, density if up is None else up) if weights == 2 else 0
    X._check(lib.xspmm_int8_kernel(weights, CODES[kind], M, K, N, blocks(M, K, density), up, int(quantized), k))
    return tuple(k)


SIDES = (16, 200, 1000, 2048, 4096, 7000, 9000, 14336, 20000, 33000, 70000)
NS = (1, 2, 5, 16, 17, 31, 33, 64, 100, 256, 700, 1100, 2048, 9000)


def instance(weights, N, kernel, a, b):
    """The template's arguments that a choice stands for."""
    return {FEW: ("few", weights, a, b, N == 1), WALK: ("walk", a, weights, b), LISTS: ("list", weights - 1, a),
            TILES: ("tile", weights - 1)}[kernel]


def instances_built():
    if not shutil.which("nm"):
        pytest.skip("needs nm")
    names = subprocess.run(["nm", X.LIB_PATH], check=True, capture_output=True, text=True).stdout
    built = {}
    for kernel, value, rest in re.findall(r"__device_stub__ff_int8_(few|walk|list|tile)_kernelI(f|DF16_|DF16b)((?:L[ib]\d+E)+)E",
                                          names):
        built.setdefault(value, set()).add((kernel, *(int(n) for n in re.findall(r"\d+", rest))))
    assert len(built) == 3
    return built


def test_every_kernel_that_is_built_can_be_chosen(lib):
    """And no other is chosen."""
    built, wanted = instances_built(), set()
    for weights, M, K, N, density, quantized in itertools.product(
            (1, 2), SIDES, SIDES, NS, (0.01, 0.03, 0.1, 0.3, 0.7, 1.0), (False, True)):
        wanted.add(instance(weights, N, *chosen(lib, weights, M, K, N, density, quantized=quantized)))
    for of in built.values():
        assert of == wanted, (sorted(of - wanted), sorted(wanted - of))


def test_every_kernel_that_is_built_has_a_test_on_the_gpu():
    from test_gpu_int8_kernels import CASES

    tested = {instance(weights, N, *which) for which, weights, _, _, N, _ in CASES}
    for of in instances_built().values():
        assert of == tested, (sorted(of - tested), sorted(tested - of))


def test_what_windows_need(lib):
    """Lists and tiles take weights with a map of their grid, and at most 2^21 tokens."""
    windows = lambda *a, **k: chosen(lib, *a, **k)[0] in (LISTS, TILES)
    assert windows(1, 14336, 4096, 2048, 0.2) and windows(1, 14336, 4096, 2048, 1.0)
    # a weight without blocks, or with hardly any, has none
    assert not windows(2, 14336, 4096, 2048, 0.2, up=0.0) and not windows(2, 14336, 4096, 2048, 0.01, up=0.5)
    for density in (0.2, 1.0):
        assert windows(1, 64, 48, 1 << 21, density) and not windows(1, 64, 48, (1 << 21) + 1, density)
    # 2^31 bytes of blocks, 2^24 blocks of a grid
    assert not windows(1, 16 * 2900, 16 * 2900, 2048, 1.0) and windows(1, 16 * 2800, 16 * 2800, 2048, 1.0)
    assert windows(1, 16 * 4096, 16 * 4096, 2048, 0.3) and not windows(1, 16 * 4097, 16 * 4096, 2048, 0.3)


def test_refusals(lib):
    k = (C.c_int32 * 3)()
    call = lambda weights, M, K, N, a, b, out=k, vtype=X.F16: (
        lambda: lib.xspmm_int8_kernel(weights, vtype, M, K, N, a, b, 0, out))
    assert "type" in refused(lib, call(1, 64, 64, 1, 4, 0, vtype=BAD))
    assert "null" in refused(lib, call(1, 64, 64, 1, 4, 0, None))
    assert "one weight or two" in refused(lib, call(0, 64, 64, 1, 4, 0))
    assert "one weight or two" in refused(lib, call(3, 64, 64, 1, 4, 4))
    for M, K, N in ((0, 64, 1), (64, 64, 0), (-1, 64, 1), (64, -1, 1), (64, 133137, 1), (1 << 30, 64, 1), (64, 64, 1 << 31)):
        assert "size" in refused(lib, call(1, M, K, N, 0, 0))
    for a, b in ((17, 0), (-1, 0), (4, 17), (4, -1)):
        assert "blocks" in refused(lib, call(2, 64, 64, 1, a, b))


# in one launch where that is the faster way for every type, in two where that is (times beside the rule)
@pytest.mark.parametrize("K,N,launches", [(4096, 30, 1), (1000, 2288, 1), (64, 8192, 1), (4999, 31, 1), (1936, 90, 1),
                                          (2060, 2048, 2), (4096, 512, 2), (14336, 64, 2), (64, 65536, 2), (8200, 33, 2)])
def test_tokens_launches(lib, K, N, launches):
    n = C.c_int64(-1)
    assert lib.xspmm_quantize_tokens_scratch(K, N, C.byref(n)) == X.OK
    assert (n.value > 0) == (launches == 2)


# the walk's widths and splits at sizes where it is chosen: us of 1 tile and 4 waves, 1 and 16, 4 and 1, 4 and 4
WALKS = [
    (1, 14336, 4096, 64, 0.03, (5.65, 13.28, 7.31, 4.55)), (2, 14336, 4096, 64, 0.03, (7.01, 18.07, 10.15, 5.8)),
    (1, 5003, 4999, 31, 0.8, (12.83, 11.91, 21.14, 8.67)), (1, 4096, 14336, 31, 0.3, (12.96, 9.35, 23.93, 8.51)),
    (2, 2048, 2048, 96, 0.06, (3.93, 6.17, 9.71, 4.87)), (2, 512, 8192, 512, 0.015, (4.08, 6.95, 9.63, 4.87)),
    (1, 512, 8192, 300, 0.8, (16.44, 12.11, 55.87, 17.18)), (2, 1024, 1024, 300, 0.1, (4.35, 8.25, 9.69, 5.16)),
    (1, 16384, 1024, 96, 0.1, (7.61, 20.72, 7.83, 6.69)), (1, 14336, 4096, 2, 0.8, (12.14, 11.52, 27.25, 13.35)),
    (1, 4096, 14336, 33, 0.2, (11.07, 10.81, 18.54, 7.1)), (2, 4096, 14336, 24, 0.3, (21.85, 14.39, 72.98, 21.98)),
    (2, 50000, 300, 24, 0.06, (9.14, 28.01, 7.14, 10.83)),
]


@pytest.mark.parametrize("weights,M,K,N,density,times", WALKS)
def test_walks(lib, weights, M, K, N, density, times):
    """The fastest or, of ways that are near to each other, one within a quarter of it."""
    kernel, a, b = chosen(lib, weights, M, K, N, density, quantized=True)
    assert kernel == WALK
    assert times[[(1, 4), (1, 16), (4, 1), (4, 4)].index((a, b))] <= 1.25 * min(times)


# tokens rounded within: us of one, two and four block-rows a workgroup, and rounded ahead
FEWS = [
    (1, 14336, 4096, 2, 0.05, (22.3, 12.9, 9.4, 9.2)),
    (1, 14336, 4096, 4, 0.05, (19.8, 11.9, 8.7, 10.2)),
    (2, 14336, 4096, 1, 0.25, (14.6, 9.8, 10.9, 11.8)),
    (2, 14336, 4096, 2, 0.25, (26.4, 16.6, 13.9, 13.2)),
    (2, 14336, 4096, 4, 0.25, (22.7, 14.7, 13.0, 14.1)),
    (2, 14336, 4096, 4, 0.8, (30.4, 21.4, 23.1, 25.6)),
    (1, 4096, 14336, 1, 0.25, (7.6, 8.2, 9.7, 9.3)),
    (2, 16384, 1024, 8, 0.25, (14.5, 8.6, 7.2, 9.3)),
    (2, 16384, 1024, 16, 0.25, (19.1, 10.8, 8.2, 9.5)),
    (2, 16384, 1024, 32, 0.25, (34.7, 19.0, 11.1, 11.2)),
    (2, 16384, 1024, 64, 0.25, (72.9, 39.3, 23.5, 12.5)),
    (2, 16384, 1024, 2, 0.8, (16.1, 10.6, 10.5, 9.9)),
    (1, 9000, 20000, 1, 0.05, (17.9, 13.9, 8.7, 19.4)),
    (1, 5120, 4096, 4, 0.05, (11.9, 8.5, 8.7, 9.9)),
    (1, 8192, 4096, 4, 0.05, (12.3, 8.7, 8.6, 9.9)),
    (1, 5000, 30000, 1, 0.8, (39.1, 31.0, 49.8, 41.8)),
]


@pytest.mark.parametrize("weights,M,K,N,density,times", FEWS)
def test_few_tokens(lib, weights, M, K, N, density, times):
    """The fastest way or, of those that are near to each other, one within a sixth of it."""
    kernel, rows, _ = chosen(lib, weights, M, K, N, density)
    assert times[[1, 2, 4].index(rows) if kernel == FEW else 3] <= 7 / 6 * min(times)


def timed():
    """(weights, type, M, K, N, stored, us of the walk, lists and tiles) of products that were timed."""
    with open(os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "profiles", "int8_kernel_choice.txt")) as f:
        for line in f:
            v = line.split()
            if len(v) == 9 and v[1] in CODES:
                yield int(v[0]), v[1], *(int(t) for t in v[2:5]), *(float(t) for t in v[5:])


def test_kernels_go_by_their_times(lib):
    """What is chosen is the fastest, or near to it, at sizes where all three kernels were timed."""
    ratios = []
    for weights, kind, M, K, N, density, *us in timed():
        kernel = chosen(lib, weights, M, K, N, density, quantized=True, kind=kind)[0]
        ratios.append((us[[WALK, LISTS, TILES].index(kernel)] / min(us), weights, kind, M, K, N, density))
    assert len(ratios) > 300
    assert math.prod(r[0] ** (1 / len(ratios)) for r in ratios) < 1.01
    assert max(ratios)[0] < 1.3, max(ratios)
    # lists from a tenth on, at the size whose times stand beside the kernels
    assert [chosen(lib, 1, 14336, 4096, 2048, d, quantized=True)[0] for d in (0.04, 0.1, 0.25, 0.4, 1.0)] == [
        WALK, LISTS, LISTS, LISTS, TILES]
