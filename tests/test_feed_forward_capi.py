"""The feed-forward layer's C entry points: what they refuse, and their scratch,
from sizes alone (no GPU is asked)."""
from __future__ import annotations

import ctypes as C
import threading

import pytest

import xspmm_amd as X

BF16, BAD = 2, 7


@pytest.fixture(scope="module")
def lib():
    from xspmm_amd import feed_forward

    return feed_forward._load()


def refused(L, call):
    """The call's message; in a thread of its own, as the library keeps the last error per thread."""
    out = []

    def run():
        out.append(call())
        out.append(L.xspmm_last_error().decode())

    t = threading.Thread(target=run)
    t.start()
    t.join()
    assert out[0] == X.ERR_INVALID, out
    assert out[1]
    return out[1]


@pytest.mark.parametrize("vtype", [X.F32, X.F16, BF16])
@pytest.mark.parametrize("K,N", [(1, 1), (4096, 1), (4096, 2048), (4096, 8001), (64, 16384), (16385, 300)])
def test_norm_scratch(lib, vtype, K, N):
    n = C.c_int64(-1)
    assert lib.xspmm_layer_norm_scratch(vtype, K, N, 0, C.byref(n)) == X.OK
    forward = n.value
    assert forward >= 0 and (forward == 0 or forward >= 8 * N)  # a pair of floats per token and slice
    assert lib.xspmm_layer_norm_scratch(vtype, K, N, 1, C.byref(n)) == X.OK
    assert n.value >= 8 * (N + K)  # sums per token and per feature
    # a small share of what the pass reads
    assert n.value <= 4096 + max(64 * (N + K), K * N)


def test_norm_scratch_empty_and_refused(lib):
    n = C.c_int64(-1)
    for K, N in ((0, 5), (5, 0), (0, 0)):
        for backward in (0, 1):
            assert lib.xspmm_layer_norm_scratch(X.F16, K, N, backward, C.byref(n)) == X.OK and n.value == 0
    for K, N in ((-1, 5), (5, -1), (1 << 31, 5), (5, (1 << 30) + 1)):
        refused(lib, lambda: lib.xspmm_layer_norm_scratch(X.F16, K, N, 0, C.byref(n)))
    assert "type" in refused(lib, lambda: lib.xspmm_layer_norm_scratch(BAD, 5, 5, 0, C.byref(n)))
    refused(lib, lambda: lib.xspmm_layer_norm_scratch(X.F16, 5, 5, 0, None))


def test_null_weights(lib):
    n = C.c_int64(0)
    assert "null" in refused(lib, lambda: lib.xspmm_linear(None, X.F16, 0, *[None] * 6, 4, None))
    assert "null" in refused(lib, lambda: lib.xspmm_gated(None, None, X.F16, 0, *[None] * 8, 4, None))
    refused(lib, lambda: lib.xspmm_linear_backward_scratch(None, X.F16, 0, 4, C.byref(n)))
    refused(lib, lambda: lib.xspmm_gated_backward_scratch(None, X.F16, 4, C.byref(n)))
    refused(lib, lambda: lib.xspmm_linear_backward(None, X.F16, 0, *[None] * 7, 4, None, 0, None))
    refused(lib, lambda: lib.xspmm_gated_backward(None, None, X.F16, 0, *[None] * 11, 4, None, 0, None))
    assert lib.xspmm_weight_destroy(None) == X.OK


@pytest.mark.parametrize("M,K,Mb,Kb,nnzb", [(-1, 16, 0, 1, 0), (16, -1, 1, 0, 0), (16, 16, 1, 1, -1), (17, 16, 1, 1, 1),
                                            (16, 33, 1, 2, 1), (1 << 31, 16, 1 << 27, 1, 1),
                                            (16, 16, 1, 1, (1 << 31) - 1)])
def test_weight_sizes(lib, M, K, Mb, Kb, nnzb):
    h = C.c_void_p(1)
    refused(lib, lambda: lib.xspmm_weight_create(X.I32, M, K, Mb, Kb, nnzb, 16, 16, None, C.byref(h)))
    assert h.value is None


def test_weight_arguments(lib):
    h = C.c_void_p()
    assert "index" in refused(lib, lambda: lib.xspmm_weight_create(5, 16, 16, 1, 1, 1, 16, 16, None, C.byref(h)))
    refused(lib, lambda: lib.xspmm_weight_create(X.I32, 16, 16, 1, 1, 1, None, 16, None, C.byref(h)))
    refused(lib, lambda: lib.xspmm_weight_create(X.I32, 16, 16, 1, 1, 1, 16, None, None, C.byref(h)))
    refused(lib, lambda: lib.xspmm_weight_create(X.I32, 16, 16, 1, 1, 1, 16, 16, None, None))


def test_norm_arguments(lib):
    # addresses are looked at, never read
    ok = [256, None, None]
    assert "null" in refused(lib, lambda: lib.xspmm_layer_norm(X.F16, 5, 1, None, None, None, 1e-5, 256, None, None, None,
                                                               0, None))
    assert "boundary" in refused(lib, lambda: lib.xspmm_layer_norm(X.F16, 5, 1, 258, None, None, 1e-5, 256, None, None,
                                                                   None, 0, None))
    assert "eps" in refused(lib, lambda: lib.xspmm_layer_norm(X.F16, 5, 1, *ok, -1.0, 256, None, None, None, 0, None))
    assert "eps" in refused(lib, lambda: lib.xspmm_layer_norm(X.F16, 5, 1, *ok, float("nan"), 256, None, None, None, 0,
                                                              None))
    assert "both" in refused(lib, lambda: lib.xspmm_layer_norm(X.F16, 5, 1, *ok, 1e-5, 256, 256, None, None, 0, None))
    assert "scratch" in refused(lib, lambda: lib.xspmm_layer_norm(X.F16, 4096, 4096, *ok, 1e-5, 256, None, None, None, 0,
                                                                  None))
    assert "statistics" in refused(lib, lambda: lib.xspmm_layer_norm_backward(X.F16, 5, 1, 256, 256, None, None, None,
                                                                              256, None, None, 256, 1 << 20, None))
    assert "scratch" in refused(lib, lambda: lib.xspmm_layer_norm_backward(X.F16, 5, 1, 256, 256, None, 256, 256, 256,
                                                                           None, None, None, 0, None))


def test_view_without_gpu_tensors():
    import torch

    x = torch.zeros((4, 4))
    with pytest.raises(ValueError, match="GPU"):
        X.layer_norm(x)
    A = X.BCSRMatrix(1, 1, 16, 16, 16, 16, torch.tensor([0, 1], dtype=torch.int32), torch.tensor([0], dtype=torch.int32),
                     torch.zeros(256))
    with pytest.raises(ValueError, match="GPU"):
        X.SparseWeight(A)
    with pytest.raises(AttributeError):
        X.no_such_operator
