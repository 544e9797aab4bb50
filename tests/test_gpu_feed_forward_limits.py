"""The feed-forward layer where sums are infinite, activations vanish and means are
large, against the limits and 64-bit forms.

A weight without blocks makes the sums the biases, so that an activation sees
exactly what it is given; with one token and dy = 1, the bias's gradient is its
slope.  Bounds: fp32 roundings (2^-24 each), some per function (erfc and exp are
good for 16 units in the last place at most) and those of the functions'
arguments, stretched by how steep they are there.
"""
from __future__ import annotations

import math

import pytest
import torch

import xspmm_amd as X

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
EPS32 = 2.0 ** -24
KINDS = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ACTS = ["relu", "silu", "gelu", "gelu_tanh"]


def no_blocks(M, K, dtype):
    Mb, Kb = -(-M // 16), -(-K // 16)
    return X.SparseWeight(X.BCSRMatrix(Mb, Kb, 16, 16, M, K, torch.zeros(Mb + 1, dtype=torch.int32, device=DEV),
                                       torch.zeros(0, dtype=torch.int32, device=DEV),
                                       torch.zeros(0, dtype=dtype, device=DEV)))


def value(act, z):
    W = no_blocks(z.numel(), 16, z.dtype)
    return X.sparse_linear(W, torch.zeros((16, 1), dtype=z.dtype, device=DEV), bias=z, activation=act)[:, 0]


def slope(act, z):
    W = no_blocks(z.numel(), 16, z.dtype)
    x = torch.zeros((16, 1), dtype=z.dtype, device=DEV)
    return X.sparse_linear_backward(W, x, z[:, None], torch.ones_like(z[:, None]), activation=act, bias=True)[2]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("act", ACTS)
def test_infinite_sums_give_the_limits(kind, act):
    big = torch.finfo(KINDS[kind]).max
    z = torch.tensor([-math.inf, -big, -big / 2, math.inf, big, math.nan], dtype=KINDS[kind], device=DEV)
    y, s = value(act, z), slope(act, z)
    assert not y[:3].any() and torch.equal(y[3:5], z[3:5]) and y[5].isnan(), y
    assert not s[:3].any() and (s[3:5] == 1).all() and s[5].isnan(), s


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("act", ACTS)
def test_gradients_of_infinite_sums(kind, act):
    """dz of a gate that is off for good is zero, and so is what it multiplies."""
    dtype = KINDS[kind]
    W = no_blocks(3, 16, dtype)
    x = torch.zeros((16, 9), dtype=dtype, device=DEV)
    z = torch.tensor([-math.inf, math.inf, 0.0], dtype=dtype, device=DEV)[:, None].expand(3, 9).contiguous()
    up, dh = torch.full_like(z, 3), torch.full_like(z, 2)
    _, _, _, bg, bu = X.sparse_gated_backward(W, W, x, z, up, dh, activation=act, bias=True)
    assert bg[0] == 0 and bg[1] == 54 and bu[0] == 0 and bu[1] == math.inf and bu[2] == 0


def test_activations_keep_their_digits_where_they_vanish():
    """Relative to the result: an activation that takes 1 + erf, or 1 - p, from a difference loses them."""
    z = torch.cat([torch.linspace(-12, -2, 4001), torch.linspace(-80, -12, 1001)]).to(DEV)
    zz = z.double().cpu()
    root, a, b = math.sqrt(0.5), math.sqrt(8 / math.pi), 0.044715
    near = zz >= -12
    # silu
    p = torch.special.expit(zz)
    for got, want in ((value("silu", z), zz * p), (slope("silu", z), p * (1 + zz * (1 - p)))):
        off = (got.double().cpu() - want).abs()
        assert (off <= 64 * EPS32 * want.abs()).all(), float((off / want.abs()).max())
    # gelu: erfc's own logarithmic slope is about z, that of exp(-z z / 2) is -z z / 2
    p, density = 0.5 * torch.special.erfc(-zz * root), torch.exp(-zz * zz / 2) / math.sqrt(2 * math.pi)
    for got, want in ((value("gelu", z), zz * p), (slope("gelu", z), p + zz * density)):
        off = (got.double().cpu() - want).abs()
        bound = (64 + 4 * zz * zz) * EPS32 * want.abs()
        assert (off <= bound)[near].all(), float((off / want.abs())[near].max())
        assert (got.double().cpu().abs() <= 1e-30)[zz < -13].all()
    # gelu_tanh: p = sigmoid(u)
    u = a * (zz + b * zz ** 3)
    p = torch.special.expit(u)
    within = u > -85
    for got, want in ((value("gelu_tanh", z), zz * p),
                      (slope("gelu_tanh", z), p + zz * p * (1 - p) * a * (1 + 3 * b * zz * zz))):
        off = (got.double().cpu() - want).abs()
        bound = (64 + 8 * u.abs()) * EPS32 * want.abs()
        assert (off <= bound)[within].all(), float((off / want.abs())[within].max())


@pytest.mark.parametrize("K,N", [(1000, 100), (130, 1000), (4000, 20)])
def test_norm_of_large_means(K, N):
    """A mean whose square is past fp32's range, deviations whose squares are not."""
    j = torch.randint(0, 8, (K, N), generator=torch.Generator().manual_seed(1)).double()
    x64 = 2.0 ** 65 * (1 + j * 2.0 ** -12)
    x = x64.float().to(DEV)
    assert torch.equal(x.double().cpu(), x64)
    y, mean, rstd = X.layer_norm(x, keep=True)
    m = x64.mean(0)
    r = 1 / torch.sqrt((x64 - m).square().mean(0) + 1e-5)
    assert ((mean.double().cpu() - m).abs() <= 64 * EPS32 * m).all()
    want = (x64 - m) * r
    off = (y.double().cpu() - want).abs()
    assert (off <= 128 * EPS32 * (want.abs() + 2 * m * r)).all(), float(off.max())
    # of one sign throughout, and of a feature far off
    x[5] = -2.0 ** 66
    assert X.layer_norm(x).isfinite().all()


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("N", [1, 40])
def test_weights_of_no_rows_and_of_no_columns(kind, N):
    dtype = KINDS[kind]
    tall, wide = no_blocks(40, 0, dtype), no_blocks(0, 40, dtype)
    none, x = torch.empty((0, N), dtype=dtype, device=DEV), torch.ones((40, N), dtype=dtype, device=DEV)
    b = torch.arange(40, device=DEV).to(dtype)
    assert torch.equal(X.sparse_linear(tall, none, bias=b), b[:, None].expand(40, N))
    assert X.sparse_linear(wide, x).shape == (0, N) and X.sparse_gated(wide, wide, x).shape == (0, N)
    dx, dv, db = X.sparse_linear_backward(tall, none, x, x, activation="relu", bias=True)
    assert dx.shape == (0, N) and dv.numel() == 0 and (db == N).all()
    dx, dv, db = X.sparse_linear_backward(wide, x, none, none, activation="relu", bias=True)
    assert dx.shape == (40, N) and not dx.any() and db.numel() == 0
    assert not X.sparse_gated_backward(wide, wide, x, none, none, none)[0].any()
