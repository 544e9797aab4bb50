"""Orthogonalised updates on the GPU against the formula in 64 bits.

The bound of a case comes from the arithmetic itself: the same formula in 64 bits with
the operands of its products rounded as the operator states (fp16, or two fp16 halves
each for fp16 and fp32 updates, whose sums are then fp32) is off by some rms; another order of
the same roundings is off by about as much, and twice that (four times with halves, where
the sums' order counts) is allowed, beside the result's own rounding.  A single
element may be off by eight times the rms: a sum of thousands of independent roundings
is near normal, and 8 deviations are past any number of elements here.  Roundings are
relative to what is rounded: in X' = (a + d) X + Y X the error of row i goes by the
elements of row i of Y and X, that of column j by column j of X.  Where rows or
columns differ in size (at rank 1 by 4 times the rms and more, both) an element's share
is as much larger as its row and its column are than the rms of them.
"""
from __future__ import annotations

import copy

import pytest
import torch

import xspmm_amd as X
from test_gpu_feed_forward import TYPES, at_blocks, f64, normal, weight

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
ABC = (3.4445, -4.7750, 2.0315)


def exact(U, steps=5, abc=ABC, eps=1e-7):
    a, b, c = abc
    x = U.to(DEV)
    if U.shape[0] > U.shape[1]:
        x = x.t().contiguous()
    x = x / (x.norm() + eps)
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.t() if U.shape[0] > U.shape[1] else x).cpu()


def rounded(U, kind, steps=5, abc=ABC, eps=1e-7):
    """The formula with the operands of its products rounded."""
    a, b, c = abc
    x = U.to(DEV)
    if U.shape[0] > U.shape[1]:
        x = x.t().contiguous()
    x = x / (x.norm() + eps) * 4096
    hi = lambda t: t.half().double()
    both = lambda t: hi(t) + hi(t - hi(t))

    def product(p, q):
        if kind == "bf16":
            return hi(p) @ hi(q)
        ph, qh = hi(p), hi(q)
        pl, ql = hi(p - ph), hi(q - qh)
        return (ph.float() @ qh.float() + ph.float() @ ql.float() + pl.float() @ qh.float()).double()

    held = hi if kind == "bf16" else both
    for _ in range(steps):
        x = both(x)
        s = held(product(x, x.t().contiguous()) / 4096)
        y = b * s + c * product(s, s) / 4096
        d = torch.diagonal(y).clone() / 4096
        y.fill_diagonal_(0)
        x = (a + d)[:, None] * x + product(y, x) / 4096
    x = x / 4096
    return (x.t() if U.shape[0] > U.shape[1] else x).cpu()


def check(got, U, where, kind, **how):
    want, near = exact(U, **how), rounded(U, kind, **how)
    u = TYPES[kind][1]
    rms = lambda t: float(t.square().mean().sqrt())
    w, got = at_blocks(want, where), f64(got)
    assert got.shape == w.shape and torch.isfinite(got).all()
    # values below fp16's normal numbers round by up to 2^-25
    allowed = (2 if kind == "bf16" else 4) * rms(near - want) + u * rms(w) + 2.0 ** -25
    assert rms(got - w) <= allowed, (rms(got - w), allowed, rms(w))
    size = [want.square().mean(d, keepdim=True).sqrt() for d in (0, 1)]
    size = [(t / (t.square().mean().sqrt() + 1e-300)).clamp(min=1) for t in size]
    assert ((got - w).abs() <= 8 * allowed * at_blocks(size[0] * size[1], where) + u * w.abs()).all()
    rows, cols, inside = where
    assert not got.view(-1, 16, 16)[~inside].any()


def update(M, K, density, kind, seed, rank=None, **more):
    """(weight, its positions, an update of its blocks, the dense one in 64 bits)"""
    W, _, where = weight(M, K, density, TYPES[kind][0], seed, **more)
    g = torch.Generator().manual_seed(seed + 1)
    if rank:
        d = torch.randn((M, rank), generator=g) @ torch.randn((rank, K), generator=g)
    else:
        d = torch.randn((M, K), generator=g)
    v = at_blocks(d * 1e-2, where).to(TYPES[kind][0])
    rows, cols, inside = where
    Mb, Kb = -(-M // 16), -(-K // 16)
    full = torch.zeros((Mb, Kb, 16, 16), dtype=torch.float64)
    full[rows, cols] = v.double().view(-1, 16, 16)
    return W, where, v.to(DEV), full.permute(0, 2, 1, 3).reshape(Mb * 16, Kb * 16)[:M, :K].contiguous()


SHAPES = [(1, 1), (16, 16), (1, 300), (300, 1), (17, 15), (128, 128), (127, 129), (129, 127), (200, 700), (700, 200),
          (513, 1025), (1024, 1100), (1025, 1040), (1300, 1100)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,K", SHAPES)
@pytest.mark.parametrize("density", [0.2, 1.0])
def test_shapes(kind, M, K, density):
    W, where, v, U = update(M, K, density, kind, M + K)
    if W.num_blocks == 0:
        assert X.orthogonalize(W, v).numel() == 0
        return
    check(X.orthogonalize(W, v), U, where, kind)


# tiles of 128 rows (bf16) and of 256, whole and in part
@pytest.mark.parametrize("kind,M,K", [("bf16", 2000, 2200), ("bf16", 2048, 2304), ("bf16", 2900, 3100), ("bf16", 3100, 2830),
                                      ("f16", 2050, 2300), ("f32", 2050, 2300), ("f32", 2600, 2049)])
@pytest.mark.parametrize("density", [0.1, 1.0])
def test_larger_tiles(kind, M, K, density):
    W, where, v, U = update(M, K, density, kind, M + K)
    check(X.orthogonalize(W, v), U, where, kind)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_past_four_gib(kind):
    """X of 2^32 bytes and more, against the polynomial of S in 64 bits: X = Q X0, Q <- B Q and
    S <- B S B with B = a + b S + c S S.  bf16 results are off by up to 1e-3 of their rms and
    their rounding, fp32 ones by 1e-5; twice that is allowed."""
    M, K, per = 2100, (1 << 20) - 5, 130
    dtype, u = TYPES[kind]
    Mb, Kb = -(-M // 16), -(-K // 16)
    g = torch.Generator().manual_seed(1)
    cols = torch.stack([torch.randperm(Kb, generator=g)[:per].sort().values for _ in range(Mb)])
    ptr = torch.arange(Mb + 1, dtype=torch.int32, device=DEV) * per
    v = torch.randn(Mb * per * 256, generator=g).to(dtype).to(DEV)
    rows, col = torch.arange(Mb, device=DEV).repeat_interleave(per), cols.reshape(-1).to(DEV)
    inside = (16 * rows[:, None] + torch.arange(16, device=DEV) < M)[:, :, None] & (
        16 * col[:, None] + torch.arange(16, device=DEV) < K)[:, None, :]
    v *= inside.reshape(-1)
    W = X.SparseWeight(X.BCSRMatrix(Mb, Kb, 16, 16, M, K, ptr, col.int(), v))
    got = X.orthogonalize(W, v).view(-1, 16, 16)
    a, b, c = ABC
    v64 = v.double().view(-1, 16, 16)
    S = torch.zeros((Mb * 16, Mb * 16), dtype=torch.float64, device=DEV)
    step, slabs = 4096, []
    v64 = v64 / (v64.norm() + 1e-7)
    for c0 in range(0, Kb, step):  # block-columns
        on = ((col >= c0) & (col < c0 + step)).nonzero().flatten()
        d = torch.zeros((Mb, step, 16, 16), dtype=torch.float64, device=DEV)
        d[rows[on], col[on] - c0] = v64[on]
        d = d.permute(0, 2, 1, 3).reshape(Mb * 16, step * 16)
        S += d @ d.t()
        slabs.append((c0, on))
    Q = torch.eye(Mb * 16, dtype=torch.float64, device=DEV)
    for _ in range(5):
        B = b * S + c * (S @ S)
        B.diagonal().add_(a)
        Q, S = B @ Q, B @ S @ B
    error = size = 0.0
    for c0, on in slabs:
        d = torch.zeros((Mb, step, 16, 16), dtype=torch.float64, device=DEV)
        d[rows[on], col[on] - c0] = v64[on]
        want = (Q @ d.permute(0, 2, 1, 3).reshape(Mb * 16, step * 16)).view(Mb, 16, step, 16).transpose(1, 2)
        want = want[rows[on], col[on] - c0] * inside[on]
        error += float((got[on].double() - want).square().sum())
        size += float(want.square().sum())
    assert error ** 0.5 <= 2 * ((1e-3 if kind == "bf16" else 1e-5) + u) * size ** 0.5


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rank", [1, 16, 100])
def test_low_rank(kind, rank):
    W, where, v, U = update(600, 900, 1.0, kind, rank, rank=rank)
    check(X.orthogonalize(W, v), U, where, kind)


@pytest.mark.parametrize("kind", list(TYPES))
def test_empty_rows_and_columns(kind):
    W, where, v, U = update(330, 250, 0.3, kind, 7, empty_rows=(0, 3, 20))
    check(X.orthogonalize(W, v), U, where, kind)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("how", [dict(steps=1), dict(steps=2), dict(steps=9), dict(steps=3, abc=(1.5, -0.5, 0.0)),
                                 dict(steps=2, abc=(0.0, 1.0, -2.0)), dict(steps=4, eps=0.0), dict(steps=5, eps=3.0)])
def test_coefficients(kind, how):
    W, where, v, U = update(200, 333, 0.7, kind, 3)
    got = X.orthogonalize(W, v, steps=how["steps"], coefficients=how.get("abc", ABC), eps=how.get("eps", 1e-7))
    check(got, U, where, kind, **how)


def test_singular_values():
    W, where, v, U = update(400, 640, 1.0, "f32", 1)
    rows, cols, _ = where
    d = torch.zeros((25, 40, 16, 16), dtype=torch.float64)
    d[rows, cols] = f64(X.orthogonalize(W, v)).view(-1, 16, 16)
    sv = torch.linalg.svdvals(d.permute(0, 2, 1, 3).reshape(400, 640))
    # what five steps make of the singular values of such a matrix lies in 0.68 .. 1.21
    assert sv.min() > 0.6 and sv.max() < 1.25


def test_sparse_grid_without_a_map():
    """One block in 100: positions are searched for, not read from a map of the grid."""
    W, where, v, U = update(1600, 1900, 0.01, "bf16", 5)
    check(X.orthogonalize(W, v), U, where, "bf16")


@pytest.mark.parametrize("kind,scale", [("f32", 1e-30), ("f32", 1e30), ("bf16", 1e-30), ("bf16", 1e36), ("f16", 1e-3)])
def test_scale(kind, scale):
    W, where, v, U = update(200, 150, 1.0, kind, 3)
    v = (v.double() * scale).to(v.dtype)
    rows, cols, _ = where
    d = torch.zeros((13, 10, 16, 16), dtype=torch.float64)
    d[rows, cols] = f64(v).view(-1, 16, 16)
    U = d.permute(0, 2, 1, 3).reshape(208, 160)[:200, :150].contiguous()
    eps = 0.0 if scale < 1e-20 else 1e-7
    check(X.orthogonalize(W, v, eps=eps), U, where, kind, eps=eps)


@pytest.mark.parametrize("kind", list(TYPES))
def test_zero_and_not_finite(kind):
    W, where, v, U = update(100, 180, 0.5, kind, 3)
    for eps in (0.0, 1e-7):
        assert not X.orthogonalize(W, torch.zeros_like(v), eps=eps).any()
    rows, cols, inside = where
    for bad in (float("inf"), float("-inf"), float("nan")):
        w = v.clone()
        w[int(inside.reshape(-1).nonzero()[40])] = bad
        got = X.orthogonalize(W, w).cpu().view(-1, 16, 16)
        assert torch.isnan(got[inside]).all() and not got[~inside].any()
    # past the edges there is nothing to read
    w = v.clone().view(-1, 16, 16)
    w[(~inside).to(DEV)] = float("nan")
    assert torch.equal(X.orthogonalize(W, w.reshape(-1)), X.orthogonalize(W, v))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,K", [(300, 500), (1100, 1200)])
def test_repeats_and_in_place(kind, M, K):
    W, where, v, U = update(M, K, 0.4, kind, 9)
    want = X.orthogonalize(W, v)
    assert torch.equal(X.orthogonalize(W, v), want)
    out = torch.full_like(v, float("nan"))
    assert X.orthogonalize(W, v, out=out) is out and torch.equal(out, want)
    mine = v.clone()
    assert X.orthogonalize(W, mine, out=mine) is mine and torch.equal(mine, want)


def test_refusals():
    W, where, v, U = update(100, 180, 0.5, "bf16", 3)
    big = torch.empty(v.numel() + 8, dtype=v.dtype, device=DEV)
    bad = [
        (TypeError, lambda: X.orthogonalize(W.matrix, v)),
        (TypeError, lambda: X.orthogonalize(W, v.float())),
        (TypeError, lambda: X.orthogonalize(W, v.tolist())),
        (ValueError, lambda: X.orthogonalize(W, v[:-256])),
        (ValueError, lambda: X.orthogonalize(W, v.view(-1, 256))),
        (ValueError, lambda: X.orthogonalize(W, v.cpu())),
        (ValueError, lambda: X.orthogonalize(W, v, steps=0)),
        (ValueError, lambda: X.orthogonalize(W, v, eps=-1.0)),
        (ValueError, lambda: X.orthogonalize(W, v, eps=float("nan"))),
        (ValueError, lambda: X.orthogonalize(W, v, coefficients=(1.0, float("inf"), 0.0))),
        (ValueError, lambda: X.orthogonalize(W, v, coefficients=(1.0, 2.0))),
        (ValueError, lambda: X.orthogonalize(W, big[:-8], out=big[8:])),
        (RuntimeError, lambda: X.orthogonalize(W, v.clone().requires_grad_())),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()
    W.close()
    with pytest.raises(RuntimeError, match="closed"):
        X.orthogonalize(W, v)


def test_too_many_columns():
    ptr, col = torch.tensor([0, 1], dtype=torch.int32, device=DEV), torch.tensor([0], dtype=torch.int32, device=DEV)
    K = (1 << 20) + 16
    W = X.SparseWeight(X.BCSRMatrix(1, K // 16, 16, 16, 16, K, ptr, col, torch.ones(256, device=DEV)))
    with pytest.raises(X.XspmmInvalidArgument, match="2\\^20"):
        X.orthogonalize(W, W.values)


@pytest.mark.parametrize("M,K", [(300, 500), (1100, 1200)])
def test_captured(M, K):
    W, where, v, U = update(M, K, 0.4, "bf16", 9)
    v = v.clone()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        X.orthogonalize(W, v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = X.orthogonalize(W, v)
    for seed in range(4):
        v.copy_(normal(v.shape, v.dtype, seed))
        graph.replay()
        want = X.orthogonalize(W, v)
        torch.cuda.synchronize()
        assert torch.equal(y, want), seed


def test_streams_at_once():
    sets = [update(200 + 100 * i, 300, 0.5, "f16", i) for i in range(3)]
    want = [X.orthogonalize(W, v) for W, _, v, _ in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(3):
        for s, (W, _, v, _) in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(X.orthogonalize(W, v))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 3]) for i, g in enumerate(got))


def layer(dtype):
    return X.FeedForward(*(weight(m, k, 0.4, dtype, s)[0].matrix for m, k, s in ((144, 96, 1), (144, 96, 2), (96, 144, 3))))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("nesterov", [True, False])
def test_optimiser(kind, nesterov):
    dtype = TYPES[kind][0]
    L = layer(dtype)
    opt = X.OrthogonalMomentum(L, lr=0.1, momentum=0.8, nesterov=nesterov, weight_decay=0.5)
    x = normal((96, 64), dtype, 1)
    params = [L.gate, L.up, L.down]
    master = [p.detach().float() for p in params]
    velocity = [torch.zeros_like(m) for m in master]
    for step in range(3):
        L(x).float().square().mean().backward()
        for i, p in enumerate(params):
            g = p.grad.float()
            velocity[i] = 0.8 * velocity[i] + g
            # with one rounding, as the optimiser has it: a bit of u in 16 bits that falls to the
            # other side is 2^-8 of an element, which the small singular values' growth (3.4 a
            # step) makes more of than any bound on the weights allows
            u = torch.add(g, velocity[i], alpha=0.8) if nesterov else velocity[i]
            if kind != "f32":
                u = u / u.abs().max()
            W = L._weights[i]
            o = X.orthogonalize(W, u.to(dtype)).float()
            ratio = max(1.0, W.shape[0] / W.shape[1])
            master[i] = master[i] * (1 - 0.1 * 0.5) - 0.1 * ratio ** 0.5 * o
        opt.step()
        opt.zero_grad()
        L.zero_grad()
        for p, m in zip(params, master):
            # fused or separate multiplications and additions: a few roundings
            assert torch.allclose(p.float(), m.to(dtype).float(), rtol=2 * TYPES[kind][1] * 2, atol=1e-5)
        # the next step from the same state
        master = [opt.state[p].get("master", p.detach()).clone() for p in params]
        velocity = [opt.state[p]["momentum"].clone() for p in params]


@pytest.mark.parametrize("kind", list(TYPES))
def test_optimiser_of_a_weight_without_blocks(kind):
    dtype = TYPES[kind][0]
    sides = ((144, 96, 0.4), (144, 96, 0.0), (96, 144, 0.4))
    L = X.FeedForward(*(weight(m, k, d, dtype, 1)[0].matrix for m, k, d in sides))
    opt = X.OrthogonalMomentum(L, lr=0.1, weight_decay=0.5)
    was = L.down.detach().clone()
    L(normal((96, 64), dtype, 1)).float().square().mean().backward()
    opt.step()
    # up gives zeros: the others' gradients are zero, and so are their updates
    assert L.up.numel() == 0 and torch.equal(L.down, (was.float() * (1 - 0.1 * 0.5)).to(dtype))


def test_optimiser_resumes():
    """State saved and loaded gives the same next step, bit for bit."""
    x = normal((96, 64), torch.bfloat16, 1)

    def steps(L, opt, n):
        for _ in range(n):
            opt.zero_grad()
            L(x).float().square().mean().backward()
            opt.step()

    A = layer(torch.bfloat16)
    a = X.OrthogonalMomentum([A], lr=0.003)
    steps(A, a, 3)
    B = layer(torch.bfloat16)
    B.load_state_dict(A.state_dict())
    b = X.OrthogonalMomentum([B], lr=0.5)
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    assert all(v.dtype is torch.float32 for s in b.state.values() for v in s.values())
    steps(A, a, 2)
    steps(B, b, 2)
    assert all(torch.equal(p, q) for p, q in zip(A.parameters(), B.parameters()))


def test_optimiser_refusals():
    L = layer(torch.float16)
    with pytest.raises(TypeError):
        X.OrthogonalMomentum(torch.nn.Linear(2, 2))
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            X.OrthogonalMomentum(L, **bad)
    opt = X.OrthogonalMomentum(L)
    with pytest.raises(RuntimeError):
        opt.add_param_group({"params": [L.norm_weight]})
    opt.step()  # without gradients nothing moves
    assert not opt.state
