"""Results in memory of the caller's: what they may share with the operands."""
from __future__ import annotations

import pytest
import torch

import xspmm_amd as X

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def normal(shape, seed, dtype=torch.float16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def square(K, seed, dtype=torch.float16, density=0.4):
    return X.SparseWeight(X.prune_blocks(normal((K, K), seed, dtype), density))


def test_out_apart_from_the_operands():
    """A workgroup would read what another one has written already."""
    K, N = 64, 24
    W = square(K, 1)
    room = normal((4 * K, N), 2)
    x, r, b = room[K:2 * K], normal((K, N), 3), normal((K,), 4)
    for out in (x, room[K + 8:2 * K + 8], room[8:K + 8]):
        for call in (lambda: X.sparse_linear(W, x, out=out), lambda: X.sparse_gated(W, W, x, out=out),
                     lambda: X.layer_norm(x, out=out)):
            with pytest.raises(ValueError, match="overlaps"):
                call()
    with pytest.raises(ValueError, match="residual"):
        X.sparse_linear(W, r, residual=x, out=room[K + 8:2 * K + 8])
    many = normal((K * N + 512,), 5)
    out = many[:K * N].view(K, N)
    for call in (lambda: X.sparse_linear(W, x, bias=many[8:8 + K], out=out),
                 lambda: X.sparse_gated(W, W, x, None, many[8:8 + K], out=out),
                 lambda: X.layer_norm(x, weight=many[8:8 + K], out=out),
                 lambda: X.layer_norm(x, None, many[K * N - 8:K * N - 8 + K], out=out)):
        with pytest.raises(ValueError, match="overlaps"):
            call()
    values = W.values.clone()
    with pytest.raises(ValueError, match="values"):
        X.sparse_linear(W, x, values=values, out=values[:K * N].view(K, N))
    # next to each other is apart
    want = X.sparse_linear(W, x, bias=b)
    assert torch.equal(X.sparse_linear(W, x, bias=b, out=room[:K]), want)
    assert torch.equal(X.layer_norm(x, out=room[2 * K:3 * K]), X.layer_norm(x))
    none = torch.empty((K, 0), dtype=torch.float16, device=DEV)
    assert X.sparse_linear(W, none, out=none).shape == (K, 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("K,N", [(64, 1), (64, 24), (96, 37), (320, 130), (2048, 1024), (2048, 1029)])
def test_the_residual_in_place(dtype, K, N):
    """Each of its values is read by the thread that writes the result there: in walks and in tiles, ragged or not."""
    W = square(K, 1, dtype, 0.9)
    x, r = normal((K, N), 2, dtype), normal((K, N), 3, dtype)
    want = X.sparse_linear(W, x, activation="relu", residual=r)
    again = r.clone()
    assert X.sparse_linear(W, x, activation="relu", residual=again, out=again) is again
    assert torch.equal(again, want)
