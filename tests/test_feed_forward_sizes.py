"""Sizes past what one launch holds, refused before anything is allocated."""
from __future__ import annotations

import ctypes as C
import threading

import pytest

import xspmm_amd as X


@pytest.mark.parametrize("M,K", [((1 << 30) - 63, 16), (16, (1 << 30) - 63), (1 << 30, 16), (0x7ffffff0 - 1, 16)])
def test_weights_past_a_launch(M, K):
    from xspmm_amd import feed_forward

    L, out = feed_forward._load(), []

    def run():  # the library keeps the last error per thread
        h = C.c_void_p(1)
        out.append(L.xspmm_weight_create(X.I32, M, K, -(-M // 16), -(-K // 16), 1, 16, 16, None, C.byref(h)))
        out.append((L.xspmm_last_error().decode(), h.value))

    t = threading.Thread(target=run)
    t.start()
    t.join()
    assert out[0] == X.ERR_INVALID and "2^30" in out[1][0] and out[1][1] is None, out
