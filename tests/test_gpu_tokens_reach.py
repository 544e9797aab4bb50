"""Tokens to whole numbers at sizes that reach each way of reading them: whole tokens by four
and by sixteen lanes, slices of their features by sixteen and by 64, of four tokens a lane
each where they are many."""
from __future__ import annotations

import pytest
import torch

import xspmm_amd as X
from test_gpu_feed_forward import TYPES

pytestmark = pytest.mark.gpu

DEV = "cuda:0"

SIZES = [
    # whole tokens by four lanes, one and two pieces of 16 features a thread, around its bounds
    (4096, 2), (3520, 1023), (3521, 112), (4097, 70), (5000, 33), (8192, 23), (8191, 48), (640, 1024), (8180, 5),
    # by sixteen lanes
    (641, 1024), (1023, 1025), (1536, 1500), (1521, 8191), (2048, 1025), (2033, 200), (64, 8192), (17, 4001),
    # slices of features: by sixteen lanes and by 64, one of them and several rounds of workgroups
    (8208, 63), (14336, 17), (20000, 5), (100003, 3), (2049, 1025), (4999, 301), (14336, 515), (16, 8193), (300, 20000),
    (14336, 1171), (65537, 257), (2048, 8200), (16400, 1024), (3000, 9001), (40, 70000),
    # more than 48 MB of 16-bit values: four tokens a thread for the maxima
    (14336, 1771), (98500, 257), (2999, 8401), (12290, 2049)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("K,N", SIZES)
def test_sizes(kind, K, N):
    print(kind, K, N, flush=True)
    g = torch.Generator(device=DEV).manual_seed(K + N)
    x = torch.randn((K, N), generator=g, device=DEV) * torch.linspace(0.01, 30, N, device=DEV)
    x[-1, ::3] = 200  # the largest in a slice's last row
    x = x.to(TYPES[kind][0])
    t = X.quantize_tokens(x)
    d = x.double()
    most = d.abs().amax(0)
    full = torch.zeros((-(-K // 16) * 16, N), dtype=torch.int8, device=DEV)
    full[:K] = (d * 127 / most).round().to(torch.int8)
    assert torch.equal(t.values, full.view(-1, 16, N).permute(0, 2, 1))
    assert torch.equal(t.scale.cpu(), x.abs().amax(0).float().cpu() / 127)
    # one token that holds no number leaves the others as they are
    n = N // 2
    x[K // 2, n] = float("nan")
    bad = X.quantize_tokens(x)
    assert bad.scale[n].isnan() and not bad.values[:, n].any()
    others = torch.arange(N, device=DEV) != n
    assert torch.equal(bad.values[:, others], t.values[:, others]) and torch.equal(bad.scale[others], t.scale[others])
