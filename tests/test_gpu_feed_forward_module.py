"""The feed-forward module and the operators' gradients through autograd: weights
that share a matrix, second derivatives, gradients as other layers hand them over,
what is kept for the backward pass, copies.

Bounds as in the operators' own tests: chains of fp32 sums, relative to the
largest value."""
from __future__ import annotations

import copy
import io
import threading

import pytest
import torch

import xspmm_amd as X

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
EPS32 = 2.0 ** -24


def normal(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def pruned(M, K, seed, dtype=torch.float32, density=0.5):
    return X.prune_blocks(normal((M, K), seed, dtype) * 0.1, density)


def unpack(A, v):
    """The M x K matrix of block values v, differentiable."""
    rows = torch.repeat_interleave(torch.arange(A.num_block_rows), torch.diff(A.row_ptr.cpu()).long())
    d = torch.zeros((A.num_block_rows, A.num_block_cols, 16, 16), dtype=torch.float64)
    d = d.index_put((rows, A.col_ind.cpu().long()), v.view(-1, 16, 16))
    return d.permute(0, 2, 1, 3).reshape(A.num_block_rows * 16, -1)[:A.num_rows, :A.num_cols]


def f64(t):
    return t.detach().double().cpu()


def near(got, want, bound, what):
    got = f64(got)
    off = float((got - want).abs().max())
    assert got.shape == want.shape and off <= bound * float(want.abs().max()), (what, off)


def layer64(mats, layer, x):
    """The layer on the unpacked weights, and everything that has a gradient."""
    leaves = [f64(p).requires_grad_(True) for p in (layer.gate, layer.up, layer.down, layer.norm_weight,
                                                    layer.norm_bias, x)]
    G, U, D = (unpack(A, v) for A, v in zip(mats, leaves))
    w, b, xx = leaves[3:]
    m = xx.mean(0)
    n = (xx - m) / torch.sqrt((xx - m).square().mean(0) + 1e-5) * w[:, None] + b[:, None]
    return xx + D @ (torch.nn.functional.silu(G @ n) * (U @ n)), leaves


# ---------------------------------------------------------------------------
# one matrix, several weights
# ---------------------------------------------------------------------------

def check_shared(mats):
    feats, N = mats[0].num_cols, 40
    before = [A.values.clone() for A in mats]
    at = [A.values.data_ptr() for A in mats]
    layer = X.FeedForward(*mats)
    with torch.no_grad():  # as after an update
        for i, p in enumerate((layer.gate, layer.up, layer.down)):
            p.add_(0.1 * normal(p.shape, 10 + i))
    x = normal((feats, N), 3).requires_grad_(True)
    dy = normal((feats, N), 4)
    with torch.no_grad():
        served = layer(x)
    y = layer(x)
    y.backward(dy)
    y64, leaves = layer64(mats, layer, x)
    y64.backward(f64(dy))
    assert torch.equal(y.detach(), served)
    bound = 4 * (mats[0].num_rows + N) * EPS32
    near(y, y64.detach(), bound, "y")
    for name, p, want in zip(("gate", "up", "down", "weight", "bias", "x"),
                             (layer.gate, layer.up, layer.down, layer.norm_weight, layer.norm_bias, x), leaves):
        near(p.grad, want.grad, bound, name)
    for A, v, a in zip(mats, before, at):  # the matrices are the caller's
        assert A.values.data_ptr() == a and torch.equal(A.values, v)


def test_gate_and_up_of_one_matrix():
    A = pruned(200, 96, 1)
    check_shared((A, A, pruned(96, 200, 2)))


def test_three_weights_of_one_square_matrix():
    A = pruned(96, 96, 1)
    check_shared((A, A, A))


def test_operators_of_one_matrix():
    A = pruned(64, 48, 1)
    G, U = X.SparseWeight(A), X.SparseWeight(A)
    x = normal((48, 10), 2)
    first = A.values
    U.values = A.values * 2
    assert A.values is first and G.values is first
    assert torch.equal(X.sparse_linear(U, x), 2 * X.sparse_linear(G, x))
    # until set, they are the matrix's, read at every call
    y = X.sparse_linear(G, x)
    A.values = A.values * 4
    assert torch.equal(X.sparse_linear(G, x), 4 * y) and torch.equal(X.sparse_linear(U, x), 2 * y)
    # and a call can bring its own
    assert torch.equal(X.sparse_linear(G, x, values=first), y)
    h = X.sparse_gated(G, U, x, values=(first, first))
    assert torch.equal(h, X.sparse_gated(X.SparseWeight(A), G, x, values=(first, first)))
    for bad in (first[:-256], first.half(), first.cpu()):
        with pytest.raises((TypeError, ValueError)):
            X.sparse_linear(G, x, values=bad)


def test_layers_of_one_matrix_in_threads():
    A, D = pruned(200, 96, 1), pruned(96, 200, 2)
    x = normal((96, 33), 3)
    layers = [X.FeedForward(A, A, D) for _ in range(2)]
    with torch.no_grad():
        for i, layer in enumerate(layers):
            layer.gate.mul_(1 + i)
        alone = [layer(x) for layer in layers]
    torch.cuda.synchronize()
    wrong = []

    def work(layer, want):
        with torch.no_grad():
            for _ in range(50):
                if not torch.equal(layer(x), want):
                    wrong.append(1)

    threads = [threading.Thread(target=work, args=p) for p in zip(layers, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ---------------------------------------------------------------------------
# second derivatives
# ---------------------------------------------------------------------------

def second_order(f, inputs, through):
    """Asks for the gradient of a first gradient."""
    y = f()
    first = torch.autograd.grad(y.square().sum() if through == "square" else y.sum(), inputs[0], create_graph=True)[0]
    penalty = first.square().sum() + sum(t.sum() for t in inputs)
    if through == "backward":
        penalty.backward()
    else:
        torch.autograd.grad(penalty, inputs)


@pytest.mark.parametrize("through", ["square", "sum", "backward"])
def test_second_derivatives_are_refused(through):
    """A gradient penalty would get a wrong value: what the kernels compute has no graph of its own."""
    A, D = pruned(64, 48, 1), pruned(48, 64, 2)
    layer = X.FeedForward(A, A, D)
    x = normal((48, 20), 3).requires_grad_(True)
    for inputs in ([x], [layer.gate, x], [layer.down, x], [layer.norm_weight, x]):
        with pytest.raises(RuntimeError, match="second derivative"):
            second_order(lambda: layer(x), inputs, through)
    # first derivatives with a graph kept are as without
    want = torch.autograd.grad(layer(x).sum(), [x, layer.gate])
    got = torch.autograd.grad(layer(x).sum(), [x, layer.gate], create_graph=True)
    assert all(torch.equal(a.detach(), b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# gradients as other layers hand them over
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_gradients_off_sixteen_bytes(dtype):
    """The backward pass of torch.cat hands over a contiguous view that starts anywhere."""
    A, D = pruned(64, 48, 1, dtype), pruned(48, 64, 2, dtype)
    layer = X.FeedForward(A, A, D)
    head = normal((3, 5), 4, dtype)
    dy = normal((51, 5), 5, dtype)
    grads = []
    for joined in (True, False):
        layer.zero_grad()
        x = normal((48, 5), 3, dtype).requires_grad_(True)
        y = layer(x)
        if joined:
            torch.cat([head, y]).backward(dy)
        else:
            y.backward(dy[3:].clone())
        grads.append([x.grad] + [p.grad for p in layer.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_nothing_is_kept_that_no_pass_reads():
    """The down projection has no activation, so its sum is neither written nor saved."""
    A, D = pruned(64, 48, 1), pruned(512, 64, 2)
    W = X.SparseWeight(D)
    h = normal((64, 1024), 3).requires_grad_(True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = X.feed_forward._Linear.apply(W, W.values, h, None, None, None)
    assert torch.cuda.memory_allocated() - before <= 512 * 1024 * 4 + (64 << 10)
    y.sum().backward()
    want = torch.autograd.grad((unpack(D, f64(D.values)) @ (h64 := f64(h).requires_grad_(True))).sum(), h64)[0]
    near(h.grad, want, 600 * EPS32, "dx")


# ---------------------------------------------------------------------------
# the operators themselves through autograd
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("activation", [None, "gelu"])
def test_linear_through_autograd(activation):
    A = pruned(64, 48, 1)
    W = X.SparseWeight(A)
    W.values = A.values.clone().requires_grad_(True)
    x, b, r = (normal(s, i).requires_grad_(True) for i, s in enumerate([(48, 20), (64,), (64, 20)]))
    dy = normal((64, 20), 5)
    y, kept = X.sparse_linear(W, x, bias=b, activation=activation, residual=r, keep=True)
    with torch.no_grad():
        y2, kept2 = X.sparse_linear(W, x, bias=b, activation=activation, residual=r, keep=True)
    assert torch.equal(y, y2) and torch.equal(kept, kept2) and y.requires_grad and not kept.requires_grad
    got = torch.autograd.grad(y, [W.values, x, b, r], dy)
    leaves = [f64(t).requires_grad_(True) for t in (W.values, x, b, r)]
    z = unpack(A, leaves[0]) @ leaves[1] + leaves[2][:, None]
    y64 = (torch.nn.functional.gelu(z) if activation else z) + leaves[3]
    for name, g, w in zip(("values", "x", "bias", "residual"), got, torch.autograd.grad(y64, leaves, f64(dy))):
        near(g, w, 400 * EPS32, name)
    # one at a time
    for i, t in enumerate((x, b, r)):
        args = [t if j == i else u.detach() for j, u in enumerate((x, b, r))]
        y = X.sparse_linear(W, args[0], bias=args[1], activation=activation, residual=args[2], values=W.values.detach())
        assert torch.equal(torch.autograd.grad(y, t, dy)[0], got[1 + i])


def test_gated_through_autograd():
    A, B = pruned(64, 48, 1), pruned(64, 48, 2)
    G, U = X.SparseWeight(A), X.SparseWeight(B)
    gv, uv = (m.values.clone().requires_grad_(True) for m in (A, B))
    x, bg, bu = (normal(s, i).requires_grad_(True) for i, s in enumerate([(48, 20), (64,), (64,)]))
    dh = normal((64, 20), 5)
    h = X.sparse_gated(G, U, x, bg, bu, values=(gv, uv))
    got = torch.autograd.grad(h, [gv, uv, x, bg, bu], dh)
    leaves = [f64(t).requires_grad_(True) for t in (gv, uv, x, bg, bu)]
    zg = unpack(A, leaves[0]) @ leaves[2] + leaves[3][:, None]
    zu = unpack(B, leaves[1]) @ leaves[2] + leaves[4][:, None]
    h64 = torch.nn.functional.silu(zg) * zu
    near(h, h64.detach(), 200 * EPS32, "h")
    for name, g, w in zip(("gate", "up", "x", "bias gate", "bias up"), got, torch.autograd.grad(h64, leaves, f64(dh))):
        near(g, w, 400 * EPS32, name)
    h, zg, zu = X.sparse_gated(G, U, x, bg, bu, keep=True)
    assert h.requires_grad and not zg.requires_grad and not zu.requires_grad
    h = X.sparse_gated(G, U, x.detach(), None, bu)
    assert torch.equal(torch.autograd.grad(h, bu, dh)[0], torch.autograd.grad(
        X.sparse_gated(G, U, x, None, bu), bu, dh)[0])


def test_norm_through_autograd():
    x, w, b = (normal(s, i).requires_grad_(True) for i, s in enumerate([(96, 20), (96,), (96,)]))
    dy = normal((96, 20), 5)
    y, mean, rstd = X.layer_norm(x, w, b, keep=True)
    assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad
    got = torch.autograd.grad(y, [x, w, b], dy)
    want = X.layer_norm_backward(dy, x.detach(), w.detach(), mean, rstd)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    y = X.layer_norm(x.detach(), None, b)
    assert torch.equal(torch.autograd.grad(y, b, dy)[0], got[2])


def test_no_graph_where_none_is_wanted():
    A = pruned(64, 48, 1)
    W = X.SparseWeight(A)
    x = normal((48, 20), 1)
    assert not X.sparse_linear(W, x).requires_grad and not X.layer_norm(x).requires_grad
    x.requires_grad_(True)
    with torch.no_grad():
        assert not X.sparse_linear(W, x).requires_grad
        assert not X.sparse_gated(W, W, x).requires_grad
        assert not X.layer_norm(x).requires_grad
    out = torch.empty((64, 20), device=DEV)
    for call in (lambda: X.sparse_linear(W, x, out=out), lambda: X.sparse_gated(W, W, x, out=out),
                 lambda: X.layer_norm(x, out=torch.empty_like(x))):
        with pytest.raises(RuntimeError, match="out"):
            call()
        with torch.no_grad():
            call()


# ---------------------------------------------------------------------------
# copies
# ---------------------------------------------------------------------------

def test_copies_have_handles_of_their_own():
    A = pruned(64, 48, 1)
    W = X.SparseWeight(A)
    W.values = A.values * 2
    x = normal((48, 20), 1)
    y = X.sparse_linear(W, x)
    shallow, deep = copy.copy(W), copy.deepcopy(W)
    assert shallow.matrix is A and deep.matrix is not A
    W.close()
    for V in (shallow, deep):
        assert torch.equal(X.sparse_linear(V, x), y)
    assert deep.values.data_ptr() != shallow.values.data_ptr()
    shallow.close()
    assert torch.equal(X.sparse_linear(deep, x), y)


def test_copy_of_a_layer():
    A, D = pruned(64, 48, 1), pruned(48, 64, 2)
    layer = X.FeedForward(A, A, D)
    x = normal((48, 20), 1)
    with torch.no_grad():
        want = layer(x)
        other = copy.deepcopy(layer)
        layer.gate.zero_()
        assert torch.equal(other(x), want) and torch.equal(layer(x), x)
        buffer = io.BytesIO()
        torch.save(other, buffer)
        buffer.seek(0)
        again = torch.load(buffer, weights_only=False)  # what this test wrote itself
        assert torch.equal(again(x), want)


def test_a_layer_holds_its_values_once():
    """The caller's matrices are not kept alive by the layers made from them."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    A, D = pruned(1024, 512, 1), pruned(512, 1024, 2)
    layer = X.FeedForward(A, A, D)
    x = normal((512, 16), 3)
    with torch.no_grad():
        want = layer(x)
    size = sum(p.numel() * 4 for p in layer.parameters())
    del A, D
    held = torch.cuda.memory_allocated() - before
    assert size <= held <= 1.1 * size + 2 * x.numel() * 4 + (256 << 10)
    with torch.no_grad():
        assert torch.equal(layer(x), want)
        layer.up.zero_()
        assert torch.equal(layer(x), x)
