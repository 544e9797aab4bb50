"""The feed-forward products at sizes that reach every kernel, width and split.

Which one a product takes follows from its number of block-rows, of stored blocks
a block-row and of tokens; the sizes here were chosen by those rules, each at both
products, linear and gated, and their gradients' (the bounds are those of the forms
they share with the operators' other tests).
"""
from __future__ import annotations

import pytest
import torch

import xspmm_amd as X
from test_gpu_feed_forward import TYPES, normal, weight
from test_gpu_feed_forward import test_product_tiles as product_forms

pytestmark = pytest.mark.gpu

ALL, SHORT = ["f16", "bf16", "f32"], ["f16", "bf16"]


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("M,K", [(100, 2100), (2100, 100)])
@pytest.mark.parametrize("N", [1, 2, 7, 20])
def test_sixteen_waves_a_block_row(kind, M, K, N):
    """64 blocks a block-row (block-column) and more, up to 16 tokens a wave."""
    product_forms(kind, M, K, N, 0.6)


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("M,K,N,density", [(4100, 1030, 33, 0.3), (4100, 1030, 40, 0.03), (1030, 4100, 47, 0.3),
                                           (1030, 4100, 33, 0.03), (2100, 4100, 40, 0.3), (2100, 4100, 33, 0.3),
                                           (4100, 2100, 63, 0.3)])
def test_thirty_two_tokens_a_wave(kind, M, K, N, density):
    """One wave, four and sixteen a block-row."""
    product_forms(kind, M, K, N, density)


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("M,K,N,density", [(2064, 2060, 130, 0.3), (2060, 2064, 128, 0.03), (2100, 2100, 201, 0.1),
                                           (4200, 90, 64, 0.2), (90, 4200, 67, 0.2), (4200, 1040, 1025, 0.03)])
def test_sixty_four_tokens_a_wave(kind, M, K, N, density):
    """One wave and four a block-row; in 16 bits where there are too few for more tokens."""
    product_forms(kind, M, K, N, density)


@pytest.mark.parametrize("kind", SHORT)
@pytest.mark.parametrize("M,K,N,density", [(4200, 520, 4104, 0.05), (520, 4200, 4099, 0.05), (2100, 4200, 1100, 0.05),
                                           (4200, 2100, 1101, 0.05)])
def test_hundred_and_twenty_eight_tokens_a_wave(kind, M, K, N, density):
    """One wave and four a block-row, where blocks are rare."""
    product_forms(kind, M, K, N, density)


@pytest.mark.parametrize("kind", SHORT)
@pytest.mark.parametrize("M,K,N", [(4200, 300, 4099), (4200, 300, 4104), (300, 400, 4096), (300, 400, 4099),
                                   (400, 300, 4096)])
@pytest.mark.parametrize("density", [0.3, 1.0])
def test_tiles_of_sixteen_and_eight(kind, M, K, N, density):
    """Sixteen slots and eight, gated and not, rows on 16-byte boundaries and off them."""
    product_forms(kind, M, K, N, density)


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("N", [1, 200, 2056, 2051])
def test_gradients_repeat(kind, N):
    """Bit for bit, with other work in between: sums have one order, and no pass keeps anything for the next."""
    dtype, M, K = TYPES[kind][0], 2100, 1040
    G, U = weight(M, K, 0.3, dtype, 1)[0], weight(M, K, 0.6, dtype, 2)[0]
    x, zg, zu, dh = (normal(s, dtype, i) for i, s in enumerate([(K, N), (M, N), (M, N), (M, N)]))
    first = X.sparse_gated_backward(G, U, x, zg, zu, dh, bias=True)
    for i in range(3):
        X.sparse_gated_backward(U, G, x * 2, zu, zg, dh, bias=True)
        torch.full((1 << 22,), float("nan"), device=x.device)  # what scratch may hold
        again = X.sparse_gated_backward(G, U, x, zg, zu, dh, bias=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
