"""The feed-forward layer's operators on the GPU against plain 64-bit forms.

Bounds, derived from the arithmetic: a sum of n products is taken in fp32, so it
is off by at most n 2^-24 times the sum of the products' magnitudes; an
activation stretches that by at most 1.13 (2 for the slopes' own change) and
adds a few fp32 roundings of its own; the result is rounded once to its type
(unit roundoff u).  A backward product takes its gradient rounded to the type,
which adds u times the products' magnitudes.
"""
from __future__ import annotations

import math

import pytest
import torch

import xspmm_amd as X

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f16": (torch.float16, 2.0 ** -11), "bf16": (torch.bfloat16, 2.0 ** -8), "f32": (torch.float32, 2.0 ** -24)}
EPS32 = 2.0 ** -24
TINY = 2.0 ** -24  # half's smallest subnormal


def weight(M, K, density, dtype, seed, empty_rows=(), index=torch.int32):
    """A SparseWeight, its dense 64-bit matrix (CPU) and its block coordinates."""
    g = torch.Generator().manual_seed(seed)
    Mb, Kb = -(-M // 16), -(-K // 16)
    on = torch.rand((Mb, Kb), generator=g) < density
    for r in empty_rows:
        on[r] = False
    rows, cols = torch.nonzero(on, as_tuple=True)
    n = rows.numel()
    v = torch.randn((n, 16, 16), generator=g)
    inside = ((16 * rows[:, None, None] + torch.arange(16)[None, :, None] < M)
              & (16 * cols[:, None, None] + torch.arange(16)[None, None, :] < K))
    v = (v * inside).to(dtype)
    ptr = torch.zeros(Mb + 1, dtype=torch.int64)
    ptr[1:] = torch.cumsum(on.sum(1), 0)
    A = X.BCSRMatrix(Mb, Kb, 16, 16, M, K, ptr.to(DEV, index), cols.to(DEV, index), v.reshape(-1).to(DEV))
    d = torch.zeros((Mb, Kb, 16, 16), dtype=torch.float64)
    d[rows, cols] = v.double()
    dense = d.permute(0, 2, 1, 3).reshape(Mb * 16, Kb * 16)[:M, :K].contiguous()
    return X.SparseWeight(A), dense, (rows, cols, inside)


def at_blocks(dense, where):
    rows, cols, inside = where
    M, K = dense.shape
    Mb, Kb = -(-M // 16), -(-K // 16)
    full = torch.zeros((Mb * 16, Kb * 16), dtype=dense.dtype)
    full[:M, :K] = dense
    return full.view(Mb, 16, Kb, 16).permute(0, 2, 1, 3)[rows, cols].reshape(-1)


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def f64(t):
    return t.double().cpu()


def act64(name, z):
    z = z.clone().requires_grad_(True)
    F = torch.nn.functional
    y = {"none": lambda v: v * 1, "relu": F.relu, "silu": F.silu, "gelu": F.gelu,
         "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}[name](z)
    (slope,) = torch.autograd.grad(y.sum(), z)
    return y.detach(), slope


def close(got, want, bound, what):
    got = f64(got)
    assert got.shape == want.shape, what
    bad = (got - want).abs() > bound
    bad |= ~torch.isfinite(got)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs().max()), bad.nonzero()[:3].tolist())


# tokens: one, few, about every tile width, odd ones, several tiles
TOKENS = [1, 2, 7, 15, 16, 17, 31, 32, 33, 64, 65, 127, 128, 129, 200, 257]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("N", TOKENS)
def test_linear_tokens(kind, N):
    dtype, u = TYPES[kind]
    M, K = 85, 150
    W, A, _ = weight(M, K, 0.4, dtype, N, empty_rows=(2,))
    x, b, r = normal((K, N), dtype, 1), normal((M,), dtype, 2), normal((M, N), dtype, 3)
    y, z = X.sparse_linear(W, x, bias=b, activation="silu", residual=r, keep=True)
    S = A.abs() @ f64(x).abs() + f64(b).abs()[:, None]
    z64 = A @ f64(x) + f64(b)[:, None]
    err = (K + 2) * EPS32 * S
    close(z, z64, err + u * z64.abs() + TINY, "kept")
    y64 = act64("silu", z64)[0] + f64(r)
    close(y, y64, 1.13 * err + 16 * EPS32 * (z64.abs() + f64(r).abs()) + u * y64.abs() * (1 + 2 ** -8) + TINY, "y")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,K", [(1, 1), (16, 16), (17, 15), (15, 33), (64, 1000), (1000, 64), (333, 517)])
@pytest.mark.parametrize("N", [1, 24, 77])
@pytest.mark.parametrize("density", [0.03, 1.0])
def test_linear_shapes(kind, M, K, N, density):
    dtype, u = TYPES[kind]
    W, A, _ = weight(M, K, density, dtype, M + K, index=torch.int64)
    x = normal((K, N), dtype, 1)
    y = X.sparse_linear(W, x)
    y64 = A @ f64(x)
    close(y, y64, (K + 2) * EPS32 * (A.abs() @ f64(x).abs()) + u * y64.abs() + TINY, "y")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("N", [1, 13, 48, 160])
def test_gated(kind, act, N):
    dtype, u = TYPES[kind]
    M, K = 120, 201
    G, Ga, _ = weight(M, K, 0.3, dtype, 5, empty_rows=(0, 4))
    U, Ua, _ = weight(M, K, 0.5, dtype, 6, empty_rows=(4, 7))
    x, bg, bu = normal((K, N), dtype, 1), normal((M,), dtype, 2), normal((M,), dtype, 3)
    h, zg, zu = X.sparse_gated(G, U, x, bg, bu, activation=act, keep=True)
    xa = f64(x).abs()
    g64, u64 = Ga @ f64(x) + f64(bg)[:, None], Ua @ f64(x) + f64(bu)[:, None]
    eg = (K + 2) * EPS32 * (Ga.abs() @ xa + f64(bg).abs()[:, None])
    eu = (K + 2) * EPS32 * (Ua.abs() @ xa + f64(bu).abs()[:, None])
    close(zg, g64, eg + u * g64.abs() + TINY, "gate")
    close(zu, u64, eu + u * u64.abs() + TINY, "up")
    a64 = act64(act, g64)[0]
    ea = 1.13 * eg + 16 * EPS32 * g64.abs()
    close(h, a64 * u64, ea * (u64.abs() + eu) + a64.abs() * eu + u * (a64 * u64).abs() * 1.01 + TINY, "h")
    again = X.sparse_gated(G, U, x, bg, bu, activation=act)
    assert torch.equal(again, h)
    bare = X.sparse_gated(G, U, x, activation=act)
    g0 = act64(act, Ga @ f64(x))[0]
    close(bare, g0 * (Ua @ f64(x)), ea * (u64.abs() + eu + 4) + (g0.abs() + 4) * eu
          + u * (g0 * (Ua @ f64(x))).abs() * 1.01 + TINY, "h without biases")


GRAD_TOKENS = [1, 3, 8, 31, 32, 100, 129, 600]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("N", GRAD_TOKENS)
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_backward(kind, N, act):
    dtype, u = TYPES[kind]
    M, K = 150, 85
    W, A, where = weight(M, K, 0.4, dtype, N, empty_rows=(3,))
    x, z, dy = normal((K, N), dtype, 1), normal((M, N), dtype, 2), normal((M, N), dtype, 3)
    dx, dv, db = X.sparse_linear_backward(W, x, z if act != "none" else None, dy, activation=act, bias=True)
    dz = f64(dy) * act64(act, f64(z))[1]
    ez = (u if act != "none" else 0) + 32 * EPS32
    want = A.t() @ dz
    S = A.abs().t() @ dz.abs()
    edge = A.abs().t() @ (16 * EPS32 * f64(dy).abs() + TINY)
    close(dx, want, ((M + 2) * EPS32 + ez) * S + edge + u * want.abs() * 1.01 + TINY, "dx")
    want = at_blocks(dz @ f64(x).t(), where)
    S = at_blocks(dz.abs() @ f64(x).abs().t(), where)
    edge = at_blocks((16 * EPS32 * f64(dy).abs() + TINY) @ f64(x).abs().t(), where)
    close(dv, want, ((N + 2) * EPS32 + ez) * S + edge + u * want.abs() * 1.01 + TINY, "dvalues")
    assert not dv.cpu()[~where[2].reshape(-1)].any()
    close(db, dz.sum(1), ((N + 2) * EPS32 + 32 * EPS32) * dz.abs().sum(1) + 16 * EPS32 * f64(dy).abs().sum(1)
          + u * dz.sum(1).abs() + TINY, "dbias")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("N", [1, 40, 131])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu_tanh"])
def test_gated_backward(kind, N, act):
    dtype, u = TYPES[kind]
    M, K = 101, 140
    G, Ga, wg = weight(M, K, 0.3, dtype, 5, empty_rows=(1,))
    U, Ua, wu = weight(M, K, 0.5, dtype, 6, empty_rows=(1, 2))
    x, zg, zu, dh = (normal((K, N), dtype, 1), normal((M, N), dtype, 2), normal((M, N), dtype, 3),
                     normal((M, N), dtype, 4))
    dx, dg, du, bg, bu = X.sparse_gated_backward(G, U, x, zg, zu, dh, activation=act, bias=True)
    value, slope = act64(act, f64(zg))
    g, up = f64(dh) * f64(zu) * slope, f64(dh) * value
    # what the slope and the value may be off by before they are rounded
    og, ou = 32 * EPS32 * (f64(dh) * f64(zu)).abs() + TINY, 32 * EPS32 * f64(dh).abs() * (1 + f64(zg).abs()) + TINY
    want = Ga.t() @ g + Ua.t() @ up
    S = Ga.abs().t() @ g.abs() + Ua.abs().t() @ up.abs()
    edge = Ga.abs().t() @ og + Ua.abs().t() @ ou
    close(dx, want, ((2 * M + 2) * EPS32 + u) * S + edge + u * want.abs() * 1.01 + TINY, "dx")
    for got, d, o, where, name in ((dg, g, og, wg, "dgate"), (du, up, ou, wu, "dup")):
        want = at_blocks(d @ f64(x).t(), where)
        S, edge = at_blocks(d.abs() @ f64(x).abs().t(), where), at_blocks(o @ f64(x).abs().t(), where)
        close(got, want, ((N + 2) * EPS32 + u) * S + edge + u * want.abs() * 1.01 + TINY, name)
    for got, d, o, name in ((bg, g, og, "dbias gate"), (bu, up, ou, "dbias up")):
        close(got, d.sum(1), (N + 2) * EPS32 * d.abs().sum(1) + o.sum(1) + u * d.sum(1).abs() + TINY, name)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,K,N", [(300, 290, 72), (300, 290, 67), (257, 600, 64), (600, 257, 200), (2100, 2060, 136),
                                   (2100, 2060, 75), (3000, 1400, 8)])
@pytest.mark.parametrize("density", [0.02, 0.3])
def test_weight_gradient_tiles(kind, M, K, N, density):
    """Several tiles of either size, ragged edges, tokens in whole chunks and not, sparse and denser tiles."""
    dtype, u = TYPES[kind]
    W, A, where = weight(M, K, density, dtype, N, empty_rows=(1,))
    x, dy = normal((K, N), dtype, 1), normal((M, N), dtype, 2)
    _, dv, _ = X.sparse_linear_backward(W, x, None, dy, need=(False, True))
    want = at_blocks(f64(dy) @ f64(x).t(), where)
    S = at_blocks(f64(dy).abs() @ f64(x).abs().t(), where)
    close(dv, want, (N + 2) * EPS32 * S + u * want.abs() * 1.01 + TINY, "dvalues")
    assert not dv.cpu()[~where[2].reshape(-1)].any()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,K,N", [(100, 90, 601), (300, 290, 1031), (20, 10, 77), (90, 100, 64), (70, 200, 33), (33, 50, 1)])
@pytest.mark.parametrize("density", [0.3, 0.9])
def test_weight_gradient_of_few_blocks(kind, M, K, N, density):
    """Blocks by fours, of rows on 16-byte boundaries and off them, shorter than a line and long."""
    test_weight_gradient_tiles(kind, M, K, N, density)


def test_weight_gradient_leaves_other_rows_alone():
    """What is not finite in the rows after a block's, which share its last line, does not reach it."""
    M, K = 64, 64
    for N in (65, 71, 127, 600, 601):
        W, A, where = weight(M, K, 0.5, torch.float16, N)
        x, dy = normal((K, N), torch.float16, 1), normal((M, N), torch.float16, 2)
        whole = X.sparse_linear_backward(W, x, None, dy, need=(False, True))[1].reshape(-1, 16, 16)
        x[16:32], dy[32:48] = math.nan, math.inf
        part = X.sparse_linear_backward(W, x, None, dy, need=(False, True))[1].reshape(-1, 16, 16)
        rows, cols, _ = where
        clean = ((rows != 2) & (cols != 1)).to(DEV)
        assert 0 < clean.sum() < len(rows) and torch.equal(part[clean], whole[clean])
        assert not part[~clean].isfinite().any()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,K,N", [(4090, 2040, 136), (2040, 4090, 8), (4090, 2040, 75)])
@pytest.mark.parametrize("density", [0.3, 0.7])
def test_weight_gradient_tiles_of_a_full_chip(kind, M, K, N, density):
    """The same where there are tiles enough for every compute unit."""
    test_weight_gradient_tiles(kind, M, K, N, density)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("M,K,N", [(300, 290, 136), (290, 300, 131), (64, 2100, 128), (2100, 64, 264), (1100, 1300, 200),
                                   (700, 90, 257)])
@pytest.mark.parametrize("density", [0.2, 0.6, 1.0])
def test_product_tiles(kind, M, K, N, density):
    """Sizes at which several tiles meet: more block-columns than a window of positions, one and two of a pair of
    blocks stored, ragged edges, tokens in whole chunks and not."""
    dtype, u = TYPES[kind]
    G, Ga, _ = weight(M, K, density, dtype, N, empty_rows=(1,))
    U, Ua, _ = weight(M, K, density / 2, dtype, N + 1, empty_rows=(0,))
    x, dy, b, r = normal((K, N), dtype, 1), normal((M, N), dtype, 2), normal((M,), dtype, 3), normal((M, N), dtype, 4)
    y, z = X.sparse_linear(G, x, bias=b, activation="relu", residual=r, keep=True)
    z64 = Ga @ f64(x) + f64(b)[:, None]
    err = (K + 2) * EPS32 * (Ga.abs() @ f64(x).abs() + f64(b).abs()[:, None])
    close(z, z64, err + u * z64.abs() + TINY, "kept")
    y64 = z64.clamp(min=0) + f64(r)
    close(y, y64, err + 4 * EPS32 * f64(r).abs() + u * y64.abs() * 1.01 + TINY, "y")
    h, zg, zu = X.sparse_gated(G, U, x, None, b, activation="none", keep=True)
    g64, u64 = Ga @ f64(x), Ua @ f64(x) + f64(b)[:, None]
    eu = (K + 2) * EPS32 * (Ua.abs() @ f64(x).abs() + f64(b).abs()[:, None])
    close(zg, g64, err + u * g64.abs() + TINY, "gate")
    close(zu, u64, eu + u * u64.abs() + TINY, "up")
    close(h, g64 * u64, err * (u64.abs() + eu) + g64.abs() * eu + u * (g64 * u64).abs() * 1.01 + TINY, "h")
    dx, _, _ = X.sparse_linear_backward(G, x, None, dy, need=(True, False))
    want = Ga.t() @ f64(dy)
    close(dx, want, (M + 2) * EPS32 * (Ga.abs().t() @ f64(dy).abs()) + u * want.abs() * 1.01 + TINY, "dx")
    one = torch.ones_like(dy)
    dx = X.sparse_gated_backward(G, U, x, one, dy, dy, activation="none", need=(True, False, False))[0]
    g = (f64(dy) ** 2).to(dtype).double()
    want = Ga.t() @ g + Ua.t() @ f64(dy)
    S = Ga.abs().t() @ g + Ua.abs().t() @ f64(dy).abs()
    close(dx, want, (2 * M + 2) * EPS32 * S + 2 * u * (Ga.abs().t() @ g) + u * want.abs() * 1.01 + TINY, "gated dx")


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("M,K,N", [(2100, 300, 2056), (300, 2100, 2051), (2100, 4200, 2056), (4200, 520, 4104),
                                   (520, 4200, 4099)])
@pytest.mark.parametrize("density", [0.3, 1.0])
def test_product_tiles_of_a_full_chip(kind, M, K, N, density):
    """The same where there are tiles enough for every compute unit, of eight block-rows and of sixteen."""
    test_product_tiles(kind, M, K, N, density)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("M,K,N", [(2064, 512, 2056), (4208, 512, 4099)])
def test_product_tiles_leave_absent_blocks_alone(kind, M, K, N):
    """Infinities and NaN in rows of x reach the block-rows that store a block there, and no others."""
    dtype, _ = TYPES[kind]
    W, A, _ = weight(M, K, 0.4, dtype, 5)
    x, dy = normal((K, N), dtype, 1), normal((M, N), dtype, 2)
    x[37], dy[53] = math.nan, math.inf
    stored = A.reshape(M // 16, 16, K // 16, 16).abs().sum((1, 3)) > 0
    assert 0 < stored[:, 2].sum() < M // 16 and 0 < stored[3].sum() < K // 16
    y = X.sparse_linear(W, x)
    hit = stored[:, 2].repeat_interleave(16)
    assert y[hit].isnan().all() and y[~hit].isfinite().all()
    dx = X.sparse_linear_backward(W, x, None, dy, need=(True, False))[0]
    hit = stored[3].repeat_interleave(16)
    assert not dx[hit].isfinite().any() and dx[~hit].isfinite().all()


def test_wanted_gradients_only():
    W, _, _ = weight(64, 64, 0.5, torch.float16, 1)
    x, z, dy = (normal((64, 20), torch.float16, s) for s in (1, 2, 3))
    whole = X.sparse_linear_backward(W, x, z, dy, activation="silu", bias=True)
    for need in ((True, False), (False, True), (False, False)):
        part = X.sparse_linear_backward(W, x, z, dy, activation="silu", need=need)
        for i in range(2):
            assert (part[i] is None) if not need[i] else torch.equal(part[i], whole[i])
        assert part[2] is None


def test_gradients_are_the_differences():
    """fp32: directional differences of the forward pass against the gradients."""
    M, K, N = 70, 90, 24
    G, Ga, wg = weight(M, K, 0.4, torch.float32, 1)
    U, Ua, wu = weight(M, K, 0.4, torch.float32, 2)
    x, dh = normal((K, N), torch.float32, 3) * 0.3, normal((M, N), torch.float32, 4)
    bg, bu = normal((M,), torch.float32, 5), normal((M,), torch.float32, 6)
    h, zg, zu = X.sparse_gated(G, U, x, bg, bu, activation="gelu", keep=True)
    grads = X.sparse_gated_backward(G, U, x, zg, zu, dh, activation="gelu", bias=True)
    step = 2.0 ** -7
    for i, (dirn, where) in enumerate(((normal((K, N), torch.float32, 7), None),
                                       (normal(G.values.shape, torch.float32, 8), wg),
                                       (normal(U.values.shape, torch.float32, 9), wu),
                                       (normal((M,), torch.float32, 10), None), (normal((M,), torch.float32, 11), None))):
        if where is not None:
            dirn = dirn * where[2].reshape(-1).to(DEV)
        ends = []
        for sign in (1, -1):
            old = G.values.clone(), U.values.clone()
            args = [x, None, None, bg, bu]
            if i == 1:
                G.values = G.values + sign * step * dirn
            elif i == 2:
                U.values = U.values + sign * step * dirn
            else:
                args[i] = args[i] + sign * step * dirn
            ends.append((f64(X.sparse_gated(G, U, args[0], args[3], args[4], activation="gelu")) * f64(dh)).sum())
            G.values, U.values = old
        slope = float(ends[0] - ends[1]) / (2 * step)
        want = float((f64(grads[i]) * f64(dirn)).sum())
        # central differences: third derivatives times step^2, and the outputs' fp32 roundings over the step
        scale = float((f64(grads[i]).abs() * f64(dirn).abs()).sum())
        assert abs(slope - want) <= 2e-3 * scale, (i, slope, want, scale)


@pytest.mark.parametrize("kind", list(TYPES))
def test_no_blocks_and_no_tokens(kind):
    dtype, _ = TYPES[kind]
    W, _, _ = weight(40, 50, 0.0, dtype, 1)
    assert W.num_blocks == 0
    x, b = normal((50, 9), dtype, 1), normal((40,), dtype, 2)
    assert torch.equal(X.sparse_linear(W, x, bias=b), b[:, None].expand(40, 9))
    dx, dv, db = X.sparse_linear_backward(W, x, None, normal((40, 9), dtype, 3), bias=True)
    assert not dx.any() and dv.numel() == 0 and db.shape == (40,)
    W, _, _ = weight(40, 50, 0.5, dtype, 1)
    none = torch.empty((50, 0), dtype=dtype, device=DEV)
    zero = torch.empty((40, 0), dtype=dtype, device=DEV)
    assert X.sparse_linear(W, none).shape == (40, 0)
    assert X.sparse_gated(W, W, none).shape == (40, 0)
    dx, dv, db = X.sparse_linear_backward(W, none, zero, zero, activation="gelu", bias=True)
    assert dx.shape == (50, 0) and not dv.any() and not db.any()
    got = X.sparse_gated_backward(W, W, none, zero, zero, zero, bias=True)
    assert got[0].shape == (50, 0) and not any(t.any() for t in got[1:])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("N", [1, 5, 33, 136, 141])
def test_what_is_not_finite_stays_in_its_token(kind, N):
    """Inf and NaN reach the results of their own token and of the rows whose blocks read them, no others;
    rows past the last of a ragged weight read nothing."""
    dtype, _ = TYPES[kind]
    M, K = 90, 75  # K ends inside a block
    W, A, where = weight(M, K, 0.5, dtype, 1)
    x = normal((K, N), dtype, 2)
    clean = X.sparse_linear(W, x)
    bad = x.clone()
    bad[70, N // 2] = float("nan")
    y = X.sparse_linear(W, bad)
    others = torch.arange(N) != N // 2
    assert torch.equal(y[:, others], clean[:, others])
    reads = torch.zeros(M, dtype=torch.bool)
    for r, c in zip(where[0].tolist(), where[1].tolist()):
        if c == 70 // 16:
            reads[16 * r:16 * r + 16] = True
    col = y[:, N // 2].cpu()
    assert col[reads].isnan().all()
    assert torch.equal(col[~reads], clean[:, N // 2].cpu()[~reads])
    # memory after x does not reach the result: the same x at the end of a buffer of NaN
    room = torch.full((K * N + 4096,), float("nan"), dtype=dtype, device=DEV)
    room[:K * N] = x.reshape(-1)
    assert torch.equal(X.sparse_linear(W, room[:K * N].view(K, N)), clean)
    dy = normal((M, N), dtype, 3)
    room = torch.full((M * N + 4096,), float("nan"), dtype=dtype, device=DEV)
    room[:M * N] = dy.reshape(-1)
    a = X.sparse_linear_backward(W, x, None, dy, bias=True)
    b = X.sparse_linear_backward(W, x, None, room[:M * N].view(M, N), bias=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_nothing_past_the_results_is_written():
    for dtype in (torch.float16, torch.float32):
        for M, K, N in ((33, 47, 1), (70, 90, 37), (47, 64, 130)):
            W, _, _ = weight(M, K, 0.6, dtype, 1)
            x = normal((K, N), dtype, 2)
            room = torch.full((M * N + 512,), 7.0, dtype=dtype, device=DEV)
            X.sparse_linear(W, x, out=room[:M * N].view(M, N))
            assert torch.equal(room[:M * N].view(M, N), X.sparse_linear(W, x))
            assert (room[M * N:] == 7).all()


def test_other_stream_and_repeats():
    W, _, _ = weight(500, 700, 0.2, torch.float16, 1)
    x, z, dy = normal((700, 75), torch.float16, 1), normal((500, 75), torch.float16, 2), normal((500, 75), torch.float16, 3)
    y = X.sparse_linear(W, x, activation="gelu")
    grads = X.sparse_linear_backward(W, x, z, dy, activation="gelu", bias=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            y2 = X.sparse_linear(W, x, activation="gelu")
            g2 = X.sparse_linear_backward(W, x, z, dy, activation="gelu", bias=True)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(grads, g2))


def test_a_graph_of_the_layer():
    """Captured forward and backward passes, replayed on new inputs with other work between the replays."""
    G, U, D = (weight(M, K, 0.3, torch.bfloat16, i)[0] for i, (M, K) in enumerate([(400, 300), (400, 300), (300, 400)]))
    x, dy = normal((300, 70), torch.bfloat16, 1), normal((300, 70), torch.bfloat16, 2)
    w, b = normal((300,), torch.bfloat16, 3), normal((300,), torch.bfloat16, 4)

    def passes():
        n, mean, rstd = X.layer_norm(x, w, b, keep=True)
        h, zg, zu = X.sparse_gated(G, U, n, activation="silu", keep=True)
        y = X.sparse_linear(D, h, residual=x)
        dh, dd, _ = X.sparse_linear_backward(D, h, None, dy)
        dn, dg, du, _, _ = X.sparse_gated_backward(G, U, n, zg, zu, dh, activation="silu")
        return (y, dd, dg, du) + tuple(X.layer_norm_backward(dn, x, w, mean, rstd))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        passes()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = passes()
    for seed in range(5, 9):
        x.copy_(normal((300, 70), torch.bfloat16, seed))
        dy.copy_(normal((300, 70), torch.bfloat16, seed + 10))
        want = [t.clone() for t in passes()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------

NORM_SIZES = [(1, 1), (1, 40), (64, 1), (100, 3), (4096, 1), (777, 17), (64, 64), (500, 130), (130, 1000), (2000, 257),
              (16, 5000), (4096, 33), (1000, 9), (300, 70), (5000, 40), (9000, 21), (20000, 19), (20000, 300)]


def norm64(x, w, b, eps):
    m = x.mean(0)
    r = 1 / torch.sqrt((x - m).square().mean(0) + eps)
    return (x - m) * r * w[:, None] + b[:, None], m, r


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("K,N", NORM_SIZES)
def test_layer_norm(kind, K, N):
    dtype, u = TYPES[kind]
    x = normal((K, N), dtype, 1)
    if K > 8:
        x[5] *= 60  # one feature far off the others
    w, b = normal((K,), dtype, 2), normal((K,), dtype, 3)
    eps = 1e-5
    y, mean, rstd = X.layer_norm(x, w, b, eps=eps, keep=True)
    y64, m64, r64 = norm64(f64(x), f64(w), f64(b), eps)
    size = f64(x).abs().mean(0)
    # joins of parts: a few roundings per level, at most 40 levels deep
    close(mean, m64, 64 * EPS32 * (size + m64.abs()) + 1e-30, "mean")
    # the relative error of rstd is half the variance's: that of its sum, and the mean's error squared
    close(rstd, r64, 64 * EPS32 * r64 + r64 * (64 * EPS32 * size) ** 2 * r64 ** 2, "rstd")
    xhat = (f64(x) - m64).abs() * r64
    off = 128 * EPS32 * (xhat + (size + m64.abs()) * r64) * f64(w).abs()[:, None]
    close(y, y64, off + 4 * EPS32 * f64(b).abs()[:, None] + u * y64.abs() * 1.01 + TINY, "y")
    assert torch.equal(X.layer_norm(x, w, b, eps=eps), y)
    close(X.layer_norm(x, eps=eps), (f64(x) - m64) * r64,
          128 * EPS32 * (xhat + (size + m64.abs()) * r64) + u * xhat * 1.01 + TINY, "without weight and bias")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("K,N", NORM_SIZES)
def test_layer_norm_backward(kind, K, N):
    dtype, u = TYPES[kind]
    x, w, dy = normal((K, N), dtype, 1), normal((K,), dtype, 2), normal((K, N), dtype, 3)
    _, m64, r64 = norm64(f64(x), f64(w), f64(w), 1e-5)
    mean, rstd = m64.float().to(DEV), r64.float().to(DEV)
    for weighted in (True, False):
        dx, dw, db = X.layer_norm_backward(dy, x, w if weighted else None, mean, rstd)
        h = (f64(x) - f64(mean)) * f64(rstd)
        g = f64(dy) * (f64(w)[:, None] if weighted else 1.0)
        want = f64(rstd) * (g - g.mean(0) - h * (g * h).mean(0))
        parts = f64(rstd) * (g.abs() + g.abs().mean(0) + h.abs() * (g * h).abs().mean(0))
        close(dx, want, (K + 16) * EPS32 * parts + u * want.abs() * 1.01 + TINY, "dx")
        close(dw, (f64(dy) * h).sum(1), (N + 16) * EPS32 * (f64(dy) * h).abs().sum(1)
              + 8 * EPS32 * (f64(dy).abs() * (f64(x).abs() + f64(mean).abs()) * f64(rstd)).sum(1)
              + u * (f64(dy) * h).sum(1).abs() + TINY, "dweight")
        close(db, f64(dy).sum(1), (N + 16) * EPS32 * f64(dy).abs().sum(1) + u * f64(dy).sum(1).abs() + TINY, "dbias")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("K,N", [(300, 3001), (1100, 2050), (130, 8001)])
def test_layer_norm_wide(kind, K, N):
    """Tiles of every width, and the parameters' gradients without dx."""
    test_layer_norm(kind, K, N)
    test_layer_norm_backward(kind, K, N)
    x, w, dy = (normal(s, TYPES[kind][0], i) for i, s in enumerate([(K, N), (K,), (K, N)]))
    _, mean, rstd = X.layer_norm(x, w, keep=True)
    _, dw, db = X.layer_norm_backward(dy, x, w, mean, rstd)
    none, dw2, db2 = X.layer_norm_backward(dy, x, w, mean, rstd, need=(False, True, True))
    assert none is None and torch.equal(dw, dw2) and torch.equal(db, db2)
    dx, none, db2 = X.layer_norm_backward(dy, x, w, mean, rstd, need=(True, False, True))
    assert none is None and torch.equal(db, db2)


def test_layer_norm_constant_and_not_finite():
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        for N in (5, 300):
            x = normal((200, N), dtype, 1)
            x[:, 2] = 3.0
            clean = X.layer_norm(x)
            assert not clean[:, 2].any()  # no variance: eps alone, and exact zeros
            bad = x.clone()
            bad[7, 1] = float("inf")
            bad[9, 4] = float("nan")
            y = X.layer_norm(bad)
            rest = torch.tensor([n not in (1, 4) for n in range(N)])
            assert torch.equal(y[:, rest], clean[:, rest]) and y[:, 4].isnan().all()


def test_layer_norm_no_tokens():
    x = torch.empty((30, 0), dtype=torch.float16, device=DEV)
    e = torch.empty(0, device=DEV)
    assert X.layer_norm(x).shape == (30, 0)
    dx, dw, db = X.layer_norm_backward(x, x, None, e, e)
    assert dx.shape == (30, 0) and not dw.any() and not db.any()


# ---------------------------------------------------------------------------
# refusals: before anything is launched
# ---------------------------------------------------------------------------

def test_refusals():
    h = torch.float16
    W, _, _ = weight(64, 48, 0.5, h, 1)
    V, _, _ = weight(64, 64, 0.5, h, 1)
    B, _, _ = weight(64, 48, 0.5, torch.bfloat16, 1)
    x = normal((48, 10), h, 1)
    off = torch.zeros(48 * 10 + 1, dtype=h, device=DEV)[1:].view(48, 10)
    for bad in (x.float(), x[:, 0]):
        with pytest.raises((TypeError, ValueError)):
            X.sparse_linear(W, bad)
    with pytest.raises(TypeError):
        X.sparse_linear(W, x.cpu().numpy())
    for bad in (x.cpu(), x[:47], x.t().contiguous().t(), normal((48, 20), h, 1)[:, ::2], off):
        with pytest.raises(ValueError):
            X.sparse_linear(W, bad)
    with pytest.raises(ValueError, match="activation"):
        X.sparse_linear(W, x, activation="tanh")
    with pytest.raises(ValueError):
        X.sparse_linear(W, x, bias=normal((63,), h, 1))
    with pytest.raises(ValueError):
        X.sparse_linear(W, x, residual=normal((64, 9), h, 1))
    with pytest.raises(TypeError):
        X.sparse_linear(W, x, out=torch.empty((64, 10), device=DEV))
    for other in (V, B):
        with pytest.raises(ValueError, match="differ"):
            X.sparse_gated(W, other, x)
    with pytest.raises(TypeError):
        X.sparse_linear_backward(W, x, None, normal((64, 10), h, 1), activation="relu")  # needs what was kept
    with pytest.raises(ValueError):
        X.sparse_linear_backward(W, x, None, normal((64, 11), h, 1))
    with pytest.raises(ValueError):
        W.values = normal((256,), h, 1)
    W.close()
    with pytest.raises(RuntimeError, match="closed"):
        X.sparse_linear(W, x)
    for bad in (normal((0, 4), h, 1), normal((4,), h, 1), normal((4, 4), h, 1).cpu()):
        with pytest.raises(ValueError):
            X.layer_norm(bad)
    with pytest.raises(TypeError):
        X.layer_norm(torch.zeros((4, 4), dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        X.layer_norm(normal((4, 4), h, 1), eps=-1.0)


@pytest.mark.parametrize("ptr,col", [([0, 1, 3], [0, 1, 1]), ([0, 1, 3], [0, 2, 1]), ([0, 1, 3], [0, 1, 3]),
                                     ([0, 1, 3], [-1, 0, 1]), ([0, 2, 1], [0, 1, 2]), ([1, 1, 3], [0, 1, 2]),
                                     ([0, 4, 3], [0, 1, 2])])
def test_arrays_that_are_no_weight(ptr, col):
    A = X.BCSRMatrix(2, 3, 16, 16, 32, 48, torch.tensor(ptr, dtype=torch.int32, device=DEV),
                     torch.tensor(col, dtype=torch.int32, device=DEV), torch.zeros(768, dtype=torch.float16, device=DEV))
    with pytest.raises(X.XspmmInvalidArgument):
        X.SparseWeight(A)


def test_framework_matrix_as_weight():
    """A matrix from csr_to_bcsr, and the framework's own product of it."""
    from xspmm_amd import synth
    import numpy as np

    p = synth.random_csr(300, 200, 40, 0.05, seed=3, dtype=np.float16, unsorted=True)
    Bm = X.csr_to_bcsr(X.CSRMatrix.from_host(p.M, p.K, p.rp, p.ci, p.vals, device=DEV))
    W = X.SparseWeight(Bm)
    B = torch.as_tensor(p.B).to(DEV)
    want = f64(X.spmm(Bm, B))
    close(X.sparse_linear(W, B), want, 2.0 ** -11 * want.abs() + 200 * EPS32 * 20 + TINY, "y")
    assert math.isfinite(float(want.abs().max()))


# ---------------------------------------------------------------------------
# the layer as a module
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("N", [1, 50, 260])
def test_feed_forward_module(N):
    """fp32: outputs and all gradients against the same layer on the unpacked weights in 64 bits.  The bounds are
    those of a chain of four sums of up to K products, relative to the largest value."""
    feats, hidden = 96, 200
    gen = torch.Generator(device=DEV).manual_seed(3)
    mats = [X.prune_blocks(torch.randn(s, generator=gen, device=DEV) * 0.1, 0.5)
            for s in ((hidden, feats), (hidden, feats), (feats, hidden))]
    layer = X.FeedForward(*mats, activation="gelu")
    x = normal((feats, N), torch.float32, 1).requires_grad_(True)
    dy = normal((feats, N), torch.float32, 2)
    with torch.no_grad():
        served = layer(x)
    y = layer(x)
    assert torch.equal(y, served)
    y.backward(dy)

    def unpack(A, v):
        rows = torch.repeat_interleave(torch.arange(A.num_block_rows), torch.diff(A.row_ptr.cpu()).long())
        d = torch.zeros((A.num_block_rows, A.num_block_cols, 16, 16), dtype=torch.float64)
        d = d.index_put((rows, A.col_ind.cpu().long()), v.view(-1, 16, 16))
        return d.permute(0, 2, 1, 3).reshape(A.num_block_rows * 16, -1)[:A.num_rows, :A.num_cols]

    vals = [f64(p.detach()).requires_grad_(True) for p in (layer.gate, layer.up, layer.down)]
    w64, b64 = (f64(p.detach()).requires_grad_(True) for p in (layer.norm_weight, layer.norm_bias))
    x64 = f64(x.detach()).requires_grad_(True)
    G, U, D = (unpack(A, v) for A, v in zip(mats, vals))
    n = norm64(x64, w64, b64, 1e-5)[0]
    y64 = x64 + D @ (torch.nn.functional.gelu(G @ n) * (U @ n))
    y64.backward(f64(dy))
    for got, want in ((y.detach(), y64.detach()), (x.grad, x64.grad), (layer.gate.grad, vals[0].grad),
                      (layer.up.grad, vals[1].grad), (layer.down.grad, vals[2].grad),
                      (layer.norm_weight.grad, w64.grad), (layer.norm_bias.grad, b64.grad)):
        close(got, want, 4 * (hidden + N) * EPS32 * float(want.abs().max()), "module")


def test_feed_forward_demo():
    from xspmm_amd import feed_forward_demo

    out = feed_forward_demo.run(features=128, hidden=320, tokens=256, density=0.4, steps=40, dtype="f16")
    assert out["error_after"] < 0.7 * out["error_before"], out
    assert out["served_vs_batch"] < 4 * 2.0 ** -11, out


def test_prune_blocks_keeps_the_largest():
    w = normal((50, 70), torch.float32, 1)
    A = X.prune_blocks(w, 0.3)
    assert A.num_blocks == round(0.3 * 4 * 5) and int(A.row_ptr[-1]) == A.num_blocks
    norms = torch.stack([w[16 * i:16 * i + 16, 16 * j:16 * j + 16].square().sum() for i in range(4) for j in range(5)])
    rows = torch.repeat_interleave(torch.arange(4), torch.diff(A.row_ptr.cpu()).long())
    kept = rows * 5 + A.col_ind.cpu()
    assert set(kept.tolist()) == set(torch.topk(norms, A.num_blocks).indices.tolist())
    with pytest.raises(ValueError):
        X.FeedForward(A, A, A)
