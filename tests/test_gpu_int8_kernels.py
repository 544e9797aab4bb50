"""Every kernel of the 8-bit products, width, split and number of weights, against the formula in
64 bits with the bounds of test_gpu_int8_reach: each case states which kernel it is for, and
asks the library whether that is the one that runs."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import xspmm_amd as X
from test_gpu_feed_forward import EPS32, TINY, TYPES
from test_gpu_int8_reach import units, weight
from test_int8_choice import CODES, FEW, LISTS, TILES, WALK
from xspmm_amd import int8

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def kernel(parts, kind, N):
    k = (C.c_int32 * 3)()
    (M, K), n = parts[0].shape, [W.num_blocks for W in parts]
    X._check(int8._load().xspmm_int8_kernel(len(parts), CODES[kind], M, K, N, n[0], n[-1], 0, k))
    return tuple(k)


CASES = [
    # one token: one, two and four block-rows a workgroup, one piece of the token a thread and two
    ((FEW, 1, 1), 1, 4090, 1030, 1, 0.3), ((FEW, 2, 1), 1, 8190, 1030, 1, 0.3), ((FEW, 2, 1), 1, 9000, 2047, 1, 0.9), ((FEW, 4, 1), 1, 9001, 2047, 1, 0.05),
    ((FEW, 4, 1), 1, 20000, 64, 1, 0.5), ((FEW, 1, 2), 1, 700, 20000, 1, 0.2), ((FEW, 2, 2), 1, 5000, 17000, 1, 0.1),
    ((FEW, 4, 2), 1, 9000, 20000, 1, 0.05), ((FEW, 2, 2), 1, 8300, 16500, 1, 0.5),
    ((FEW, 1, 1), 2, 300, 1024, 1, 0.5), ((FEW, 2, 1), 2, 9000, 500, 1, 0.7), ((FEW, 4, 1), 2, 9001, 2047, 1, 0.03),
    ((FEW, 1, 2), 2, 501, 17001, 1, 0.1), ((FEW, 2, 2), 2, 4200, 20000, 1, 0.1), ((FEW, 4, 2), 2, 9000, 20000, 1, 0.05),
    # more: the same of up to sixteen, a last tile of few tokens
    ((FEW, 1, 1), 1, 4000, 1000, 9, 0.4), ((FEW, 1, 1), 1, 1000, 1000, 50, 0.2), ((FEW, 2, 1), 1, 8000, 1024, 13, 0.5),
    ((FEW, 4, 1), 1, 9001, 1000, 10, 0.1), ((FEW, 4, 1), 1, 4100, 333, 47, 0.5), ((FEW, 2, 1), 1, 16000, 3000, 2, 0.9),
    ((FEW, 1, 1), 2, 1024, 1024, 64, 0.2), ((FEW, 2, 1), 2, 8000, 1024, 13, 0.5), ((FEW, 4, 1), 2, 9001, 1000, 10, 0.1),
    ((FEW, 2, 1), 2, 16000, 1000, 3, 1.0), ((FEW, 4, 1), 2, 5400, 1001, 33, 0.05),
    # the walk: one tile of sixteen tokens and four, one, four and sixteen waves to a block-row
    ((WALK, 1, 4), 1, 3000, 3000, 20, 0.1), ((WALK, 1, 16), 1, 130, 9000, 20, 0.9), ((WALK, 1, 16), 1, 8000, 4001, 12, 0.9),
    ((WALK, 4, 4), 1, 9001, 2000, 21, 0.05), ((WALK, 4, 4), 1, 4200, 9000, 50, 0.25), ((WALK, 4, 1), 1, 9000, 400, 700, 0.01),
    ((WALK, 4, 1), 1, 40000, 200, 19, 0.3),
    ((WALK, 1, 4), 2, 1000, 3001, 20, 0.1), ((WALK, 1, 16), 2, 500, 9000, 20, 0.4), ((WALK, 4, 4), 2, 9001, 2000, 21, 0.05),
    ((WALK, 4, 1), 2, 9000, 400, 700, 0.01), ((WALK, 4, 1), 2, 40000, 200, 19, 0.2),
    # lists: one, two and three fours of blocks fetched ahead, rows with more, a last window of few
    ((LISTS, 1, 0), 1, 14336, 1020, 2048, 0.07), ((LISTS, 2, 0), 1, 14336, 4096, 2000, 0.12), ((LISTS, 2, 0), 1, 5003, 4999, 1900, 0.2),
    ((LISTS, 3, 0), 1, 4100, 3000, 1500, 0.35), ((LISTS, 3, 0), 1, 14336, 4096, 515, 0.3),
    ((LISTS, 1, 0), 2, 14336, 4090, 1990, 0.07), ((LISTS, 2, 0), 2, 14336, 4096, 2000, 0.12), ((LISTS, 2, 0), 2, 4091, 3030, 1100, 0.24),
    ((LISTS, 3, 0), 2, 4100, 3000, 1500, 0.35),
    # tiles: windows of 16 block-columns whole and in part, fewer block-columns than one
    ((TILES, 0, 0), 1, 4001, 1030, 1029, 1.0), ((TILES, 0, 0), 1, 14336, 4096, 1000, 0.7), ((TILES, 0, 0), 1, 4096, 200, 16400, 1.0),
    ((TILES, 0, 0), 2, 4096, 1024, 1152, 1.0), ((TILES, 0, 0), 2, 8000, 1500, 1100, 0.7),
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("which,weights,M,K,N,density", CASES)
def test_kernels(kind, which, weights, M, K, N, density):
    print(kind, which, weights, M, K, N, density, flush=True)
    dtype, u = TYPES[kind]
    parts = [weight(M, K, density, dtype, s) for s in range(weights)]
    assert kernel([p[0] for p in parts], kind, N) == which
    g = torch.Generator(device=DEV).manual_seed(7)
    x = torch.randn((K, N), generator=g, device=DEV).to(dtype)
    b = torch.randn(M, generator=g, device=DEV).to(dtype)
    r = torch.randn((M, N), generator=g, device=DEV).to(dtype)
    most = x.double().abs().amax(0)
    q = (x.double() * 127 / most).round()
    z = [(w @ q) * s * (most / 127) + b.double()[:, None] for _, w, s in parts]
    err = [EPS32 * (8 * v.abs() + 8 * b.double().abs()[:, None]) for v in z]
    if weights == 2:
        y = X.int8_gated(parts[0][0], parts[1][0], x, bias_gate=b, bias_up=b, activation="relu")
        want = z[0].clamp(min=0) * z[1]
        bound = err[0] * (z[1].abs() + err[1]) + z[0].abs() * err[1]
    else:
        y = X.int8_linear(parts[0][0], x, bias=b, activation="relu", residual=r)
        want = z[0].clamp(min=0) + r.double()
        bound = err[0] + EPS32 * want.abs()
    bad = (y.double() - want).abs() > bound + u * want.abs() * 1.01 + TINY
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


def some_of_the_grid(M, K, density, seed):
    """Some blocks of -1, 0 and 1, with a 1 in every block and row: its whole numbers are 127 times those."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    Mb, Kb = M // 16, K // 16
    on = torch.rand((Mb, Kb), generator=g, device=DEV) < density
    on[:, 0] = True
    d = units((M, K), seed, torch.float16)
    d.view(Mb, 16, Kb, 16)[:, :, :, 0] = 1
    d *= on.repeat_interleave(16, 0).repeat_interleave(16, 1)
    rows, cols = torch.nonzero(on, as_tuple=True)
    ptr = torch.zeros(Mb + 1, dtype=torch.int32, device=DEV)
    ptr[1:] = torch.cumsum(on.sum(1), 0)
    v = d.view(Mb, 16, Kb, 16).transpose(1, 2)[rows, cols].reshape(-1).contiguous()
    return X.Int8Weight(X.SparseWeight(X.BCSRMatrix(Mb, Kb, 16, 16, M, K, ptr, cols.int(), v))), d


@pytest.mark.parametrize("density,which", [(0.2, LISTS), (1.0, TILES)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N", [(1 << 21) - 67, 1 << 21, (1 << 21) + 1])
def test_offsets_at_their_largest(density, which, gated, N):
    """Lists and tiles take 2^21 tokens, whose windows of x (32 and 16 block-columns) are 2^30 and 2^29
    bytes, the walk what is past that."""
    M, K = 512, 1024
    W, d = some_of_the_grid(M, K, density, 1)
    assert kernel([W, W] if gated else [W], "f16", N)[0] == (which if N <= 1 << 21 else WALK)
    x = units((K, N), 2, torch.float16)
    x[0] = 1
    y = X.int8_gated(W, W, x, activation="none") if gated else X.int8_linear(W, x)
    for n in range(0, N, 1 << 18):
        c = slice(n, n + (1 << 18))
        want = d.float() @ x[:, c].float()
        got = y[:, c].float()
        if gated:
            # the square of 127^2 times a whole number and two scales of 1 / 127, where fp16 holds it
            small = want.abs() < 200
            want = want * want
            assert ((got - want).abs() <= want * (2.0 ** -11 + 2.0 ** -20))[small].all(), n
        else:
            assert ((got - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -21)).all(), n
