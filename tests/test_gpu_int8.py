"""The 8-bit operators on the GPU against plain 64-bit forms.

Whole numbers are compared exactly.  Given them, a sum is exact; turning it to fp32,
two products with scales and the bias's addition are off by at most 2^-24 each
(scales by 2^-24 of their own), an activation stretches that by at most 1.13 and
adds a few fp32 roundings, and the result is rounded once (unit roundoff u).
"""
from __future__ import annotations

import copy
import math
import pickle

import pytest
import torch

import xspmm_amd as X
from test_gpu_feed_forward import EPS32, TINY, TYPES, act64, close, f64, normal, weight

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def whole64(v, dim):
    """Whole numbers and scales (64 bits, CPU) along a dimension."""
    most = v.abs().amax(dim, keepdim=True) if v.shape[dim] else v.new_zeros(v.sum(dim, keepdim=True).shape)
    return torch.where(most > 0, v * 127 / most, 0).round(), most / 127


def blocked(q):
    K, N = q.shape
    full = torch.zeros((-(-K // 16) * 16, N), dtype=torch.int8)
    full[:K] = q.to(torch.int8)
    return full.view(-1, 16, N).permute(0, 2, 1).contiguous()


def same_tokens(t, x):
    q, scale = whole64(f64(x), 0)
    assert t.shape == tuple(x.shape) and t.values.dtype == torch.int8
    assert torch.equal(t.values.cpu(), blocked(q))
    assert torch.equal(t.scale.cpu(), (f64(x).abs().amax(0).float() / 127))
    assert t.values.is_contiguous()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("K", [1, 15, 16, 17, 200, 1024, 1500, 14336])
@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 63, 64, 65, 129, 511, 512, 515, 1030])
def test_tokens(kind, K, N):
    x = normal((K, N), TYPES[kind][0], K + N)
    x *= torch.linspace(0.01, 30, N, device=DEV).to(x.dtype)
    same_tokens(X.quantize_tokens(x), x)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("N", [1, 40, 700])
def test_borders(kind, N):
    """Every value is a border of the rounding, exactly or next to it."""
    dtype = TYPES[kind][0]
    K = 508
    half = torch.arange(-127, 127, dtype=torch.float64) + 0.5
    col = torch.cat([half, half])
    x = torch.empty((K, N), dtype=torch.float64)
    for n in range(N):
        step = 2.0 ** (n % 9 - 4) * (1 + (n // 9) % 3) * (1.1 if n % 2 else 1.0)
        x[:, n] = col * step
        x[3, n] = 127 * step
    x = x.to(dtype)
    x = x.to(DEV)
    same_tokens(X.quantize_tokens(x), x)


def test_scales_of_any_size():
    most = torch.tensor([1e-45, 1e-40, 1.2e-38, 3e-37, 1e-30, 1e30, 3.3e38, 0.0, 2.0 ** -126, 127.0])
    x = (torch.rand((200, 10), generator=torch.Generator().manual_seed(0), dtype=torch.float64) * 2 - 1) * most.double()
    x = x.float()
    x[7] = most
    x = x.to(DEV)
    t = X.quantize_tokens(x)
    assert torch.equal(t.values.cpu(), blocked(whole64(f64(x), 0)[0]))
    assert torch.equal(t.scale.cpu(), x.cpu().abs().amax(0) / 127)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("N", [3, 80, 600])
def test_infinities_stay_in_their_token(kind, N):
    dtype = TYPES[kind][0]
    x = normal((300, N), dtype, 4)
    clean = x.clone()
    x[299, 0], x[5, 1], x[17, 2] = float("inf"), float("nan"), float("-inf")
    t = X.quantize_tokens(x)
    assert torch.isnan(t.scale[:3]).all() and not t.values[:, :3].any()
    if N > 3:
        q, scale = whole64(f64(clean), 0)
        assert torch.equal(t.values[:, 3:].cpu(), blocked(q)[:, 3:])
    W = X.Int8Weight(weight(40, 300, 0.5, dtype, 1)[0])
    y = X.int8_linear(W, x, activation="relu")
    assert torch.isnan(y[:, :3]).all() and not torch.isnan(y[:, 3:]).any()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("K", [16383, 16384, 16385, 32768, 32769, 100003])
def test_one_long_token(kind, K):
    """In one workgroup's registers or, past 16384 features, in slices; a product rounds
    up to 32768 itself.  The largest value stands last, in the last slice."""
    dtype = TYPES[kind][0]
    x = normal((K, 1), dtype, K)
    x[-1] = 9
    same_tokens(X.quantize_tokens(x), x)
    W, A, _ = weight(40, K, 0.05, dtype, K)
    check_linear(W, A, x, None, None, None, kind)
    bad = x.clone()
    bad[K // 2] = math.inf
    t = X.quantize_tokens(bad)
    assert t.scale.isnan().all() and not t.values.any()
    assert X.int8_linear(X.Int8Weight(W), bad).isnan().all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,K", [(1, 1), (16, 16), (17, 15), (85, 150), (16, 3000), (200, 33)])
def test_weights(kind, M, K):
    dtype = TYPES[kind][0]
    W, A, (rows, cols, inside) = weight(M, K, 0.6, dtype, M * K, empty_rows=(2,) if M > 48 else ())
    W8 = X.Int8Weight(W)
    q, scale = whole64(A, 1)
    assert torch.equal(W8.scale.cpu(), A.abs().amax(1).float() / 127)
    Mb, Kb = -(-M // 16), -(-K // 16)
    full = torch.zeros((Mb * 16, Kb * 16), dtype=torch.float64)
    full[:M, :K] = q
    want = full.view(Mb, 16, Kb, 16).permute(0, 2, 1, 3)[rows, cols].reshape(-1).to(torch.int8)
    assert torch.equal(W8.values.cpu(), want)


def test_weight_values_past_the_edge_count_for_nothing():
    W, A, (rows, cols, inside) = weight(21, 37, 1.0, torch.float16, 3)
    v = W.values.clone().view(-1, 16, 16)
    v[(~inside).to(DEV)] = 1000.0
    a, b = X.Int8Weight(W), X.Int8Weight(W, values=v.reshape(-1))
    assert torch.equal(a.values, b.values) and torch.equal(a.scale, b.scale)


def reference(A, x, bias, act):
    """(activation's argument, its error, value) of a product in 64 bits."""
    (qa, sa), (qx, sx) = whole64(A, 1), whole64(x, 0)
    p = (qa @ qx) * sa * sx
    z = p if bias is None else p + f64(bias)[:, None]
    return z, EPS32 * (6 * p.abs() + 2 * z.abs())


def check_linear(W, A, x, bias, act, residual, kind):
    u = TYPES[kind][1]
    y = X.int8_linear(X.Int8Weight(W), x, bias=bias, activation=act, residual=residual)
    z, err = reference(A, f64(x), bias, act)
    r = 0 if residual is None else f64(residual)
    y64 = act64(act or "none", z)[0] + r
    size = z.abs() + (0 if residual is None else r.abs())
    close(y, y64, 1.13 * err + 16 * EPS32 * size + u * y64.abs() * (1 + 2 ** -8) + TINY, "y")
    return y


TOKENS = [1, 2, 7, 15, 16, 17, 31, 32, 33, 64, 65, 127, 128, 129, 200, 257]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("N", TOKENS)
def test_linear_tokens(kind, N):
    dtype = TYPES[kind][0]
    M, K = 85, 150
    W, A, _ = weight(M, K, 0.4, dtype, N, empty_rows=(2,))
    x, b, r = normal((K, N), dtype, 1), normal((M,), dtype, 2), normal((M, N), dtype, 3)
    check_linear(W, A, x, b, "silu", r, kind)
    check_linear(W, A, x, None, None, None, kind)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("M,K", [(1, 1), (16, 16), (17, 15), (15, 33), (64, 1000), (1000, 64), (333, 517), (40, 9000)])
@pytest.mark.parametrize("N", [1, 24, 77, 300])
@pytest.mark.parametrize("density", [0.03, 0.3, 1.0])
def test_linear_shapes(kind, M, K, N, density):
    dtype = TYPES[kind][0]
    W, A, _ = weight(M, K, density, dtype, M + K, index=torch.int64)
    check_linear(W, A, normal((K, N), dtype, 1), None, None, None, kind)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("N", [1, 13, 48, 160])
def test_gated(kind, act, N):
    dtype, u = TYPES[kind]
    M, K = 120, 201
    G, Ga, _ = weight(M, K, 0.3, dtype, 5, empty_rows=(0, 4))
    U, Ua, _ = weight(M, K, 0.5, dtype, 6, empty_rows=(4, 7))
    x, bg, bu = normal((K, N), dtype, 1), normal((M,), dtype, 2), normal((M,), dtype, 3)
    G8, U8 = X.Int8Weight(G), X.Int8Weight(U)
    for biases in ((None, None), (bg, bu)):
        h = X.int8_gated(G8, U8, x, *biases, activation=act)
        (g64, eg), (u64, eu) = (reference(a, f64(x), b, act) for a, b in zip((Ga, Ua), biases))
        a64 = act64(act, g64)[0]
        ea = 1.13 * eg + 16 * EPS32 * g64.abs()
        close(h, a64 * u64, ea * (u64.abs() + eu) + a64.abs() * eu + u * (a64 * u64).abs() * 1.01 + TINY, "h")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("N", [1, 50, 700])
def test_tokens_given(kind, N):
    """Tokens that several products share give what each makes by itself."""
    dtype = TYPES[kind][0]
    W, _, _ = weight(100, 500, 0.4, dtype, 1)
    V, _, _ = weight(100, 500, 0.2, dtype, 2)
    x, r = normal((500, N), dtype, 3), normal((100, N), dtype, 4)
    t = X.quantize_tokens(x)
    W8, V8 = X.Int8Weight(W), X.Int8Weight(V)
    assert torch.equal(X.int8_linear(W8, t, residual=r), X.int8_linear(W8, x, residual=r))
    assert torch.equal(X.int8_gated(W8, V8, t), X.int8_gated(W8, V8, x))
    back = (t.dequantize().double() - x.double()).abs()
    # half a step, and the fp32 roundings of the scale and the product
    assert (back <= t.scale.double() * 0.5 + 2 * EPS32 * x.double().abs()).all()


def test_sums_at_their_largest():
    """127 * 127 in every one of the most features that a weight may have."""
    K = 133136
    one = torch.ones
    ptr, col = torch.tensor([0, K // 16], dtype=torch.int32), torch.arange(K // 16, dtype=torch.int32)
    A = X.BCSRMatrix(1, K // 16, 16, 16, 16, K, ptr.to(DEV), col.to(DEV), one(K * 16, device=DEV))
    W = X.Int8Weight(X.SparseWeight(A))
    for N in (1, 20):
        y = X.int8_linear(W, one((K, N), device=DEV))
        assert torch.allclose(y, torch.full_like(y, K), rtol=1e-6, atol=0)
        y = X.int8_linear(W, -one((K, N), device=DEV))
        assert torch.allclose(y, torch.full_like(y, -K), rtol=1e-6, atol=0)


@pytest.mark.parametrize("M,K,N", [(0, 40, 5), (40, 0, 5), (40, 40, 0), (40, 0, 700)])
def test_empty(M, K, N):
    ptr = torch.zeros(-(-M // 16) + 1, dtype=torch.int32, device=DEV)
    A = X.BCSRMatrix(-(-M // 16), -(-K // 16), 16, 16, M, K, ptr, ptr[:0], torch.empty(0, device=DEV))
    W = X.Int8Weight(X.SparseWeight(A))
    x, b, r = torch.randn((K, N), device=DEV), torch.randn(M, device=DEV), torch.randn((M, N), device=DEV)
    t = X.quantize_tokens(x)
    assert t.values.shape == (-(-K // 16), N, 16) and t.scale.shape == (N,) and (K or not t.scale.any())
    for v in (x, t):
        assert torch.equal(X.int8_linear(W, v, bias=b, residual=r), b[:, None] + r)
        assert X.int8_gated(W, W, v).shape == (M, N)
        assert not X.int8_gated(W, W, v).any()


def test_no_blocks():
    W, A, _ = weight(60, 90, 0.0, torch.bfloat16, 1)
    W8 = X.Int8Weight(W)
    assert not W8.scale.any()
    x, b = normal((90, 33), torch.bfloat16, 2), normal((60,), torch.bfloat16, 3)
    assert torch.equal(X.int8_linear(W8, x, bias=b), b[:, None].expand(60, 33))


def test_out():
    W, _, _ = weight(64, 96, 0.5, torch.float16, 1)
    W8 = X.Int8Weight(W)
    for N in (1, 40, 300):
        x, r = normal((96, N), torch.float16, 2), normal((64, N), torch.float16, 3)
        want = X.int8_linear(W8, x, residual=r)
        out = torch.empty_like(want)
        assert X.int8_linear(W8, x, residual=r, out=out) is out and torch.equal(out, want)
        mine = r.clone()
        assert torch.equal(X.int8_linear(W8, x, residual=mine, out=mine), want)
        h = torch.empty_like(want)
        assert torch.equal(X.int8_gated(W8, W8, x, out=h), X.int8_gated(W8, W8, x))
        with pytest.raises(ValueError, match="overlaps x"):
            X.int8_linear(W8, x, out=x[:64])
        big = torch.empty(64 * N + 8, dtype=torch.float16, device=DEV)
        with pytest.raises(ValueError, match="overlaps residual"):
            X.int8_linear(W8, x, residual=big[:64 * N].view(64, N), out=big[8:].view(64, N))


def test_refusals():
    W, _, _ = weight(64, 96, 0.5, torch.float16, 1)
    W8 = X.Int8Weight(W)
    V8 = X.Int8Weight(weight(64, 80, 0.5, torch.float16, 1)[0])
    x = normal((96, 8), torch.float16, 2)
    bad = [
        (TypeError, lambda: X.Int8Weight(W8)),
        (TypeError, lambda: X.Int8Weight(W, values=W.values.float())),
        (ValueError, lambda: X.Int8Weight(W, values=W.values[:-256])),
        (TypeError, lambda: X.int8_linear(W8, x.float())),
        (ValueError, lambda: X.int8_linear(W8, x.t().contiguous())),
        (ValueError, lambda: X.int8_linear(W8, x.t().contiguous().t())),
        (ValueError, lambda: X.int8_linear(W8, x.cpu())),
        (TypeError, lambda: X.int8_linear(W8, x.tolist())),
        (ValueError, lambda: X.int8_linear(W8, x[0])),
        (ValueError, lambda: X.int8_linear(W8, x, bias=x[:, 0].contiguous())),
        (ValueError, lambda: X.int8_linear(W8, x, residual=x)),
        (ValueError, lambda: X.int8_linear(W8, x, activation="tanh")),
        (ValueError, lambda: X.int8_linear(V8, X.quantize_tokens(x))),
        (ValueError, lambda: X.int8_gated(W8, V8, x)),
        (TypeError, lambda: X.quantize_tokens(x.double())),
        (ValueError, lambda: X.quantize_tokens(x.cpu())),
        (ValueError, lambda: X.quantize_tokens(x[0])),
        (RuntimeError, lambda: X.int8_linear(W8, x.clone().requires_grad_())),
        (RuntimeError, lambda: X.int8_linear(W8, x, bias=torch.zeros(64, dtype=x.dtype, device=DEV, requires_grad=True))),
        (RuntimeError, lambda: X.int8_gated(W8, W8, x.clone().requires_grad_())),
        (RuntimeError, lambda: X.quantize_tokens(x.clone().requires_grad_())),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()
    with torch.no_grad():
        X.int8_linear(W8, x.clone().requires_grad_())
    W.close()
    with pytest.raises(RuntimeError, match="closed"):
        X.int8_linear(W8, x)


def test_too_many_features():
    K = 133136 + 16
    ptr, col = torch.tensor([0, 1], dtype=torch.int32, device=DEV), torch.tensor([0], dtype=torch.int32, device=DEV)
    W = X.SparseWeight(X.BCSRMatrix(1, K // 16, 16, 16, 16, K, ptr, col, torch.ones(256, device=DEV)))
    with pytest.raises(X.XspmmInvalidArgument, match="133136"):
        X.Int8Weight(W)


def layer(dtype, density=0.4, features=96, hidden=144):
    parts = [weight(m, k, density, dtype, s)[0].matrix for m, k, s in ((hidden, features, 1), (hidden, features, 2),
                                                                       (features, hidden, 3))]
    for A in parts:
        A.values.mul_(0.2)
    return X.FeedForward(*parts)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("N", [1, 37, 300])
def test_served_layer(kind, N):
    dtype = TYPES[kind][0]
    L = layer(dtype)
    S = X.Int8FeedForward(L)
    x = normal((96, N), dtype, 5)
    with torch.no_grad():
        want = L(x)
        y = S(x)
        n = X.layer_norm(x, L.norm_weight, L.norm_bias, L.eps)
        h = X.int8_gated(S.gate, S.up, n)
        assert torch.equal(y, X.int8_linear(S.down, h, residual=x))
        # the layer's weights go on changing, the served ones do not
        for p in L.parameters():
            p.mul_(2)
        assert torch.equal(S(x), y)
    # roundings are spread evenly over a step, 1 / 127 of the largest value, which is some four
    # times their rms: 4 / (127 sqrt 12) = 0.9 % of each operand's norm, 1.3 % of a product,
    # 1.8 % of two multiplied, 2.2 % after the third
    assert (y.float() - want.float()).norm() < 0.05 * (want.float() - x.float()).norm()


def test_copies():
    S = X.Int8FeedForward(layer(torch.bfloat16))
    x = normal((96, 20), torch.bfloat16, 5)
    y = S(x)
    for other in (copy.deepcopy(S), pickle.loads(pickle.dumps(S))):
        assert torch.equal(other(x), y)
    del other
    assert torch.equal(S(x), y)


@pytest.mark.parametrize("N", [1, 64, 700])
def test_captured(N):
    """Calls in a graph, replayed with other inputs and eager work between."""
    S = X.Int8FeedForward(layer(torch.float16))
    x = normal((96, N), torch.float16, 1)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        S(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = S(x)
    for seed in range(4):
        x.copy_(normal((96, N), torch.float16, 10 + seed))
        graph.replay()
        want = S(x)
        torch.cuda.synchronize()
        assert torch.equal(y, want), seed


def test_two_streams_at_once():
    S = X.Int8FeedForward(layer(torch.bfloat16, features=512, hidden=1024))
    xs = [normal((512, n), torch.bfloat16, n) for n in (1, 600, 1, 90)]
    want = [S(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(3):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(S(x))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 4]) for i, g in enumerate(got))
