"""OrthogonalMomentum: copies of it, gradients of any size, values that come from elsewhere,
a captured step."""
from __future__ import annotations

import copy
import io

import pytest
import torch

import xspmm_amd as X
from test_gpu_feed_forward import TYPES, normal, weight

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def layer(dtype, features=96, hidden=144, density=0.4):
    sides = ((hidden, features, 1), (hidden, features, 2), (features, hidden, 3))
    return X.FeedForward(*(weight(m, k, density, dtype, s)[0].matrix for m, k, s in sides))


def weights(L):
    return [L.gate, L.up, L.down]


def gradients(L, seed, scale=1.0):
    """Whole numbers of at most 8 times `scale`, which every type holds."""
    g = torch.Generator().manual_seed(seed)
    for p in weights(L):
        p.grad = (torch.randint(-8, 9, p.shape, generator=g).double() * scale).to(p.dtype).to(DEV)


def same(A, B):
    return all(torch.equal(p, q) for p, q in zip(weights(A), weights(B)))


def pickled(t):
    f = io.BytesIO()
    torch.save(t, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("duplicate", [copy.deepcopy, pickled])
@pytest.mark.parametrize("before", [0, 2])
def test_copies(kind, duplicate, before):
    """A layer copied with its optimiser goes on as the first ones do, apart from them."""
    A = layer(TYPES[kind][0])
    a = X.OrthogonalMomentum(A, lr=0.01, weight_decay=0.1)
    for i in range(before):
        gradients(A, i)
        a.step()
    B, b = duplicate((A, a))
    assert all(p is q for p, q in zip(weights(B), b.param_groups[0]["params"]))
    assert same(A, B)
    was = [p.detach().clone() for p in weights(A)]
    gradients(B, 9)
    b.step()
    assert all(torch.equal(p, w) for p, w in zip(weights(A), was)) and not same(A, B)
    gradients(A, 9)
    a.step()
    assert same(A, B)
    for o in (a, b):
        with pytest.raises(RuntimeError, match="layers' weights"):
            o.add_param_group({"params": [A.norm_weight]})


# (fp16's smallest number is 2^-24)
@pytest.mark.parametrize("kind,scale", [("f16", 2.0 ** -24), ("bf16", 2.0 ** -60), ("bf16", 2.0 ** -115), ("f32", 2.0 ** -24),
                                        ("f32", 2.0 ** -60), ("f32", 2.0 ** -115), ("f32", 2.0 ** 100)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_gradients_of_any_size(kind, scale, nesterov):
    """The size of the gradients does not matter: powers of two, so that nothing but the size differs."""
    A, B = layer(TYPES[kind][0]), layer(TYPES[kind][0])
    a, b = (X.OrthogonalMomentum(L, lr=0.01, nesterov=nesterov) for L in (A, B))
    for i in range(2):
        gradients(A, i)
        gradients(B, i, scale)
        a.step()
        b.step()
        assert same(A, B)


@pytest.mark.parametrize("kind", list(TYPES))
def test_gradients_of_zero(kind):
    A = layer(TYPES[kind][0])
    was = [p.detach().clone() for p in weights(A)]
    a = X.OrthogonalMomentum(A, lr=0.5)
    gradients(A, 0, 0.0)
    a.step()
    assert all(torch.equal(p, w) for p, w in zip(weights(A), was))


@pytest.mark.parametrize("kind", list(TYPES))
def test_values_from_elsewhere(kind):
    """Values that a layer is given between two steps are what the next one moves."""
    A, B = layer(TYPES[kind][0]), layer(TYPES[kind][0])
    a = X.OrthogonalMomentum(A, lr=0.01)
    gradients(A, 0)
    a.step()
    with torch.no_grad():
        for p in weights(B):
            p.mul_(3)
    A.load_state_dict(B.state_dict())
    A.up.data.mul_(2)  # past torch's count of changes
    B.up.data.mul_(2)
    for group in a.param_groups:
        group["lr"] = 0.0
    gradients(A, 1)
    a.step()
    assert same(A, B)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_small_steps_add_up(kind):
    """What a 16-bit weight cannot show of a step is kept for the next ones."""
    dtype, u = TYPES[kind]
    A = layer(dtype)
    was = A.gate.detach().float()
    # an element of an update is at most 1.3 and some 0.08, of a weight some 1, whose neighbours are 2 u away:
    # one step moves hardly any, 64 most
    a = X.OrthogonalMomentum(A, lr=u / 4, momentum=0.0, nesterov=False)
    for _ in range(64):
        gradients(A, 0)
        a.step()
        assert torch.equal(a.state[A.gate]["master"].to(dtype), A.gate.detach())
    moved = A.gate.detach().float() - was
    assert (moved != 0).float().mean() > 0.5


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sides", [(96, 144), (1024, 4096)])
def test_captured(kind, sides):
    """A step in a graph, replayed with other gradients and eager work between."""
    A, B = layer(TYPES[kind][0], *sides), layer(TYPES[kind][0], *sides)
    a, b = (X.OrthogonalMomentum(L, lr=0.01) for L in (A, B))
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        gradients(A, 0)
        a.step()
    torch.cuda.synchronize()
    gradients(B, 0)
    b.step()
    assert same(A, B)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        a.step()
    for i in range(1, 6):
        gradients(B, i)
        for p, q in zip(weights(A), weights(B)):
            p.grad.copy_(q.grad)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert same(A, B), i


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_state_of_a_layer_in_fp32(kind):
    """It holds no copy of the weights in fp32: a 16-bit layer that takes it up has one of its own."""
    dtype, u = TYPES[kind]
    A, B = layer(torch.float32), layer(dtype)
    a, b = X.OrthogonalMomentum(A), X.OrthogonalMomentum(B)
    gradients(A, 0)
    a.step()
    b.load_state_dict(a.state_dict())
    for group in b.param_groups:
        group.update(lr=u / 4, momentum=0.0, nesterov=False)
    was = B.gate.detach().clone()
    for _ in range(64):
        gradients(B, 0)
        b.step()
    # steps that a 16-bit weight cannot show one by one
    assert (B.gate != was).float().mean() > 0.5


def test_a_layer_given_twice():
    A = layer(torch.float16)
    with pytest.raises(ValueError, match="twice"):
        X.OrthogonalMomentum([A, A])


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("share", [1.0, 0.1, 0.01])
def test_updates_as_small_as_eps(kind, share):
    """orthogonalize itself adds eps to the norm: down to a hundredth of it as many digits are right."""
    dtype, u = TYPES[kind]
    W, A, (rows, cols, inside) = weight(200, 333, 1.0, dtype, 3)
    norm = A.norm()
    eps = float(norm) / share  # (an fp16 update of a size that the type holds)
    x = A / (norm + eps)
    for _ in range(5):
        s = x @ x.t()
        x = 3.4445 * x + (-4.775 * s + 2.0315 * (s @ s)) @ x
    got = X.orthogonalize(W, W.values, eps=eps).double().cpu().view(-1, 16, 16)
    full = torch.zeros((13 * 16, 21 * 16), dtype=torch.float64)
    full[:200, :333] = x
    want = full.view(13, 16, 21, 16).permute(0, 2, 1, 3)[rows, cols]
    rms = lambda t: float(t.square().mean().sqrt())
    # 1e-5 of the rms as stated, and the result's rounding (below 2^-14 by up to 2^-25 in fp16)
    assert rms(got - want) <= (1e-5 + u) * rms(want) + (2.0 ** -25 if kind == "f16" else 0.0)
