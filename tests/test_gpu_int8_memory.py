"""What an Int8Weight keeps: its whole numbers and where they stand, not the values that it was
made from."""
from __future__ import annotations

import copy
import gc
import pickle

import pytest
import torch

import xspmm_amd as X
from test_gpu_feed_forward import TYPES, normal
from test_gpu_int8_reach import whole_grid

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def held():
    gc.collect()
    torch.cuda.synchronize()
    return torch.cuda.memory_allocated()


def grid(M, K, dtype, seed):
    """A matrix whose blocks are all stored."""
    Mb, Kb = M // 16, K // 16
    g = torch.Generator(device=DEV).manual_seed(seed)
    v = torch.randn(M * K, generator=g, device=DEV).to(dtype)
    ptr = torch.arange(Mb + 1, device=DEV, dtype=torch.int32) * Kb
    col = torch.arange(Kb, device=DEV, dtype=torch.int32).repeat(Mb)
    return X.BCSRMatrix(Mb, Kb, 16, 16, M, K, ptr, col, v)


@pytest.mark.parametrize("kind", list(TYPES))
def test_a_weight_lets_its_values_go(kind):
    dtype = TYPES[kind][0]
    M, K = 1024, 2048
    x = normal((K, 5), dtype, 1)
    before = held()
    W = X.SparseWeight(grid(M, K, dtype, 3))
    W8 = X.Int8Weight(W)
    y = X.int8_linear(W8, x)
    del W
    # a byte of each value, the rows' scales and the blocks' positions; the result; allocations in whole 512 bytes
    assert held() - before <= M * K + 4 * M + 4 * (M * K // 256 + M // 16 + 1) + y.numel() * y.element_size() + 8 * 512
    assert torch.equal(X.int8_linear(W8, x), y)


def test_a_served_layer_lets_its_layer_go():
    F, H = 512, 1024
    x = normal((F, 40), torch.bfloat16, 1)
    before = held()
    L = X.FeedForward(*(grid(m, k, torch.bfloat16, s) for m, k, s in ((H, F, 1), (H, F, 2), (F, H, 3))))
    S = X.Int8FeedForward(L)
    want = S(x)
    del L
    assert held() - before <= 3 * F * H * 1.1
    assert torch.equal(S(x), want)
    # copies have what they need, too
    for other in (copy.deepcopy(S), pickle.loads(pickle.dumps(S))):
        assert torch.equal(other(x), want)
    assert len(pickle.dumps(S)) <= 3 * F * H * 1.1
    del S
    assert torch.equal(other(x), want)


def test_the_weight_goes_first():
    """A weight's end does not take the positions from what was made from it; closing it does."""
    W8, d = whole_grid(64, 96, torch.float16, 1)
    x = normal((96, 3), torch.float16, 2)
    want = X.int8_linear(W8, x)
    gc.collect()
    assert torch.equal(X.int8_linear(W8, x), want)
    W = X.SparseWeight(grid(64, 96, torch.float16, 1))
    a, b = X.Int8Weight(W), X.Int8Weight(W)
    del a
    gc.collect()
    X.int8_linear(b, x)
    X.sparse_linear(W, x)
    W.close()
    W.close()
    for call in (lambda: X.int8_linear(b, x), lambda: X.int8_gated(b, b, x), lambda: X.sparse_linear(W, x)):
        with pytest.raises(RuntimeError, match="closed"):
            call()
    # a copy lays its positions out again
    for c in (copy.deepcopy(b), pickle.loads(pickle.dumps(b))):
        assert X.int8_linear(c, x).shape == (64, 3)


def test_tokens_after_the_weight_on_another_stream():
    """The last one that holds the positions may go while a product on them is under way."""
    x = normal((1024, 600), torch.float16, 2)
    want = X.int8_linear(X.Int8Weight(X.SparseWeight(grid(1024, 1024, torch.float16, 1))), x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [X.int8_linear(X.Int8Weight(X.SparseWeight(grid(1024, 1024, torch.float16, 1))), x) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
