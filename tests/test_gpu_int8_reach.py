"""The 8-bit products at sizes that reach each of their kernels and widths, past 2 GiB
and past what one launch holds.

Sums of whole numbers are exact, so two kernels can differ in nothing but what the
formula leaves: results are compared with the formula in 64 bits on the GPU, with the
bounds of test_gpu_int8.
"""
from __future__ import annotations

import pytest
import torch

import xspmm_amd as X
from test_gpu_feed_forward import EPS32, TINY, TYPES

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def weight(M, K, density, dtype, seed):
    """A weight, its whole numbers (M x K, 64 bits) and its rows' scales."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    Mb, Kb = -(-M // 16), -(-K // 16)
    on = torch.rand((Mb, Kb), generator=g, device=DEV) < density
    on[Mb // 2] = False
    full = torch.zeros((Mb * 16, Kb * 16), dtype=dtype, device=DEV)
    full[:M, :K] = torch.randn((M, K), generator=g, device=DEV).to(dtype)
    full *= on.repeat_interleave(16, 0).repeat_interleave(16, 1)
    rows, cols = torch.nonzero(on, as_tuple=True)
    ptr = torch.zeros(Mb + 1, dtype=torch.int32, device=DEV)
    ptr[1:] = torch.cumsum(on.sum(1), 0)
    v = full.view(Mb, 16, Kb, 16).transpose(1, 2)[rows, cols].reshape(-1).contiguous()
    A = X.BCSRMatrix(Mb, Kb, 16, 16, M, K, ptr, cols.int(), v)
    d = full[:M, :K].double()
    most = d.abs().amax(1, keepdim=True)
    return X.Int8Weight(X.SparseWeight(A)), torch.where(most > 0, d * 127 / most, 0).round(), most / 127


def check(kind, M, K, N, density, gated=False):
    print(kind, M, K, N, density, gated, flush=True)
    dtype, u = TYPES[kind]
    parts = [weight(M, K, density, dtype, s) for s in range(1 + gated)]
    g = torch.Generator(device=DEV).manual_seed(7)
    x = torch.randn((K, N), generator=g, device=DEV).to(dtype)
    b = torch.randn(M, generator=g, device=DEV).to(dtype)
    r = torch.randn((M, N), generator=g, device=DEV).to(dtype)
    most = x.double().abs().amax(0)
    q = (x.double() * 127 / most).round()
    z = [(w @ q) * s * (most / 127) + b.double()[:, None] for _, w, s in parts]
    err = [EPS32 * (8 * v.abs() + 8 * b.double().abs()[:, None]) for v in z]
    if gated:
        y = X.int8_gated(parts[0][0], parts[1][0], x, bias_gate=b, bias_up=b, activation="relu")
        want = z[0].clamp(min=0) * z[1]
        bound = err[0] * (z[1].abs() + err[1]) + z[0].abs() * err[1]
    else:
        y = X.int8_linear(parts[0][0], x, bias=b, activation="relu", residual=r)
        want = z[0].clamp(min=0) + r.double()
        bound = err[0] + EPS32 * want.abs()
    bad = (y.double() - want).abs() > bound + u * want.abs() * 1.01 + TINY
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


# tokens rounded within the product: one and two block-rows a workgroup and four, one and
# two blocks of features a thread, a last tile of few tokens
FEW = [(300, 1024, 1, 0.5), (9000, 100, 1, 0.7), (20000, 64, 1, 1.0), (700, 20000, 1, 0.2), (9001, 200, 17, 0.6),
       (17000, 90, 33, 0.8), (500, 2047, 16, 0.4), (260, 2000, 64, 0.3), (4000, 500, 47, 0.1)]
# the walk: 16 and 64 tokens a wave, one, four and sixteen waves to a block-row
WALK = [(130, 9000, 20, 0.9), (3000, 3000, 20, 0.1), (500, 4000, 100, 0.05), (9000, 700, 100, 0.9), (9000, 400, 700, 0.02),
        (640, 2500, 150, 0.6)]
# tiles: windows of 16 block-columns whole and in part, fewer block-columns than one
TILES = [(4001, 1030, 1029, 1.0), (4096, 1024, 1152, 1.0), (2048, 100, 16400, 1.0), (8000, 1500, 1100, 0.6),
         (14336, 4096, 1000, 0.3)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,K,N,density", FEW + WALK + TILES)
def test_kernels(kind, M, K, N, density, gated):
    check(kind, M, K, N, density, gated)


# one weight without blocks; lists of rows with more blocks than are fetched ahead, which
# is chosen by both weights' blocks together
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,K,N,gate,up", [(300, 500, 1, 0.3, 0.0), (300, 500, 9, 0.0, 0.3), (300, 500, 40, 0.3, 0.0),
                                           (2048, 1000, 1030, 0.0, 0.5), (4096, 2048, 1030, 0.9, 0.02),
                                           (4096, 2000, 2048, 0.02, 0.6), (4096, 2000, 2048, 0.1, 0.0)])
def test_weights_of_two_densities(kind, M, K, N, gate, up):
    dtype, u = TYPES[kind]
    (G, g, gs), (U, w, us) = weight(M, K, gate, dtype, 1), weight(M, K, up, dtype, 2)
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn((K, N), generator=gen, device=DEV).to(dtype)
    b = torch.randn(M, generator=gen, device=DEV).to(dtype)
    most = x.double().abs().amax(0)
    q = (x.double() * 127 / most).round()
    z = [(d @ q) * s * (most / 127) + b.double()[:, None] for d, s in ((g, gs), (w, us))]
    err = [EPS32 * (8 * v.abs() + 8 * b.double().abs()[:, None]) for v in z]
    want = z[0].clamp(min=0) * z[1]
    bound = err[0] * (z[1].abs() + err[1]) + z[0].abs() * err[1]
    y = X.int8_gated(G, U, x, bias_gate=b, bias_up=b, activation="relu")
    bad = (y.double() - want).abs() > bound + u * want.abs() * 1.01 + TINY
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


def units(shape, seed, dtype):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = torch.randint(-1, 2, shape, generator=g, device=DEV, dtype=torch.int8).to(dtype)
    return t


def whole_grid(M, K, dtype, seed):
    """All blocks of -1, 0 and 1, every row's largest magnitude 1: its whole numbers are 127 times those."""
    d = units((M, K), seed, dtype)
    d[:, 0] = 1
    Mb, Kb = M // 16, K // 16
    v = d.view(Mb, 16, Kb, 16).transpose(1, 2).reshape(-1).contiguous()
    ptr = torch.arange(Mb + 1, device=DEV, dtype=torch.int32) * Kb
    col = torch.arange(Kb, device=DEV, dtype=torch.int32).repeat(Mb)
    return X.Int8Weight(X.SparseWeight(X.BCSRMatrix(Mb, Kb, 16, 16, M, K, ptr, col, v))), d


@pytest.mark.parametrize("K,N", [(64, (1 << 26) + 5), (256, (1 << 24) + 3), (48, 1 << 22)])
def test_tokens_past_four_gib(K, N):
    """Whole numbers of tokens past 2^32 bytes (by the walk) and just around tiles' limit of tokens."""
    W, d = whole_grid(64, K, torch.float16, 1)
    x = units((K, N), 2, torch.float16)
    x[0] = 1
    y = X.int8_linear(W, x)
    for n in range(0, N, 1 << 22):
        c = slice(n, n + (1 << 22))
        want = d.float() @ x[:, c].float()
        # 127^2 times a whole number of at most 256, two scales of 1 / 127: three roundings, then 2^-11
        assert ((y[:, c].float() - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -21)).all(), n


@pytest.mark.parametrize("N", [1, 40, 300])
def test_block_values_past_two_gib(N):
    M, K = 16 * 1600, 16 * 5300
    W, d = whole_grid(M, K, torch.float16, 1)
    assert W.values.numel() > 1 << 31
    x = units((K, N), 2, torch.float16)
    x[0] = 1
    want = d.float() @ x.float()
    y = X.int8_linear(W, x)
    assert ((y.float() - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -21)).all()
    h = X.int8_gated(W, W, x, activation="none").float()
    # (where fp16 holds the square)
    small = want.abs() < 200
    assert ((h - want * want).abs() <= want * want * (2.0 ** -11 + 2.0 ** -20))[small].all()


def test_tokens_past_one_launch():
    W, _ = whole_grid(16, 16, torch.float16, 1)
    x = torch.empty((16, 1 << 30), dtype=torch.float16, device=DEV)
    with pytest.raises(X.XspmmInvalidArgument, match="one launch"):
        X.quantize_tokens(x)
    with pytest.raises(X.XspmmInvalidArgument, match="one launch"):
        X.int8_linear(W, x)
    with pytest.raises(X.XspmmInvalidArgument):
        X.quantize_tokens(torch.empty((16, (1 << 30) + 1), dtype=torch.float16, device=DEV))
