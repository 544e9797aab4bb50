"""The C entry points of the 8-bit products and of orthogonalised updates: what they
refuse, and their scratch, from sizes alone (no GPU is asked)."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import xspmm_amd as X
from test_feed_forward_capi import BAD, BF16, refused


@pytest.fixture(scope="module")
def lib():
    from xspmm_amd import int8, orthogonal

    int8._load()
    return orthogonal._load()


def scratch(f, *sizes):
    n = C.c_int64(-1)
    assert f(*sizes, C.byref(n)) == X.OK
    return n.value


@pytest.mark.parametrize("K,N", [(1, 1), (14336, 1), (16385, 1), (20000, 3), (4096, 64), (4999, 301), (14336, 2048), (64, 1 << 20)])
def test_scratch(lib, K, N):
    maxima = scratch(lib.xspmm_quantize_tokens_scratch, K, N)
    # a maximum of every token and slice, a small share of what is read
    assert maxima % 4 == 0 and 0 <= maxima <= 4 * N * (-(-K // 16)) and (maxima == 0 or maxima >= 4 * N)
    for weights, M in ((1, 4096), (2, 14336), (2, 16)):
        whole = scratch(lib.xspmm_int8_scratch, weights, M, K, N)
        # none where the product rounds its tokens itself, else the whole numbers, the scales and the maxima
        if N == 1 and K <= 32768:
            assert whole == 0
        assert whole == 0 or whole >= -(-K // 16) * 16 * N + 4 * N + maxima


def test_scratch_empty_and_refused(lib):
    whole = lambda K, N, out: lib.xspmm_int8_scratch(1, 64, K, N, out)
    for f in (lib.xspmm_quantize_tokens_scratch, whole):
        for K, N in ((0, 5), (5, 0), (0, 0)):
            assert scratch(f, K, N) >= 0
        n = C.c_int64(0)
        for K, N in ((-1, 5), (5, -1), (1 << 31, 5), (5, (1 << 30) + 1)):
            refused(lib, lambda: f(K, N, C.byref(n)))
        refused(lib, lambda: f(5, 5, None))
    for weights, M in ((0, 5), (3, 5), (1, -1)):
        refused(lib, lambda: lib.xspmm_int8_scratch(weights, M, 5, 5, C.byref(n)))


def test_null_weights(lib):
    n = C.c_int64(0)
    assert "null" in refused(lib, lambda: lib.xspmm_int8_weight(None, X.F16, None, None, None, None))
    assert "null" in refused(lib, lambda: lib.xspmm_int8_linear(None, X.F16, 0, *[None] * 8, 4, None, 0, None))
    assert "null" in refused(lib, lambda: lib.xspmm_int8_gated(None, None, X.F16, 0, *[None] * 10, 4, None, 0, None))
    assert "null" in refused(lib, lambda: lib.xspmm_orthogonalize_scratch(None, X.F16, C.byref(n)))
    assert "null" in refused(lib, lambda: lib.xspmm_orthogonalize(None, X.F16, None, None, 5, 1.0, 1.0, 1.0, 0.0, None, 0,
                                                                  None))


def test_token_arguments(lib):
    # addresses are looked at, never read
    call = lambda *a: lib.xspmm_quantize_tokens(*a)
    assert "type" in refused(lib, lambda: call(BAD, 5, 1, 256, 256, 256, None, 0, None))
    assert "null" in refused(lib, lambda: call(X.F16, 5, 1, None, 256, 256, None, 0, None))
    assert "null" in refused(lib, lambda: call(X.F16, 5, 1, 256, None, 256, None, 0, None))
    assert "scale" in refused(lib, lambda: call(X.F16, 5, 1, 256, 256, None, None, 0, None))
    assert "boundary" in refused(lib, lambda: call(BF16, 5, 1, 258, 256, 256, None, 0, None))
    assert "boundary" in refused(lib, lambda: call(BF16, 5, 1, 256, 260, 256, None, 0, None))
    need = scratch(lib.xspmm_quantize_tokens_scratch, 14336, 2048)
    assert "scratch" in refused(lib, lambda: call(X.F32, 14336, 2048, 256, 256, 256, 256, need - 1, None))
    assert "scratch" in refused(lib, lambda: call(X.F32, 14336, 2048, 256, 256, 256, None, need, None))
    assert "boundary" in refused(lib, lambda: call(X.F32, 14336, 2048, 256, 256, 256, 128, need, None))


def test_view_without_gpu_tensors():
    x = torch.zeros((4, 4))
    with pytest.raises(ValueError, match="GPU"):
        X.quantize_tokens(x)
    with pytest.raises(TypeError):
        X.quantize_tokens([[1.0]])
    with pytest.raises(TypeError):
        X.Int8Weight(x)
    with pytest.raises(TypeError):
        X.orthogonalize(x, x)
    with pytest.raises(TypeError):
        X.OrthogonalMomentum(torch.nn.Linear(2, 2))
    t = X.Int8Tokens(torch.tensor([[[1, 2] + [0] * 14, [3, -4] + [0] * 14]], dtype=torch.int8), torch.tensor([0.5, 2.0]), (2, 2))
    assert t.dequantize().tolist() == [[0.5, 6.0], [1.0, -8.0]]
