"""Operands past 2 GiB, just below it, and at what one launch holds.  Values of
-1, 0 and 1 keep every sum exact, so the results equal the dense products'."""
from __future__ import annotations

import pytest
import torch

import xspmm_amd as X

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def units(shape, seed, dtype):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-1, 2, shape, generator=g, device=DEV, dtype=torch.int8).to(dtype)


def grid(M, K, dtype, seed, absent=()):
    """A weight of all blocks but those listed, and its dense matrix in fp32."""
    Mb, Kb = -(-M // 16), -(-K // 16)
    full = torch.zeros((Mb * 16, Kb * 16), device=DEV)
    full[:M, :K] = units((M, K), seed, torch.float32)
    on = torch.ones((Mb, Kb), dtype=torch.bool, device=DEV)
    for i, j in absent:
        on[i, j] = False
    blocks = full.view(Mb, 16, Kb, 16).transpose(1, 2)[on]
    dense = torch.where(on.repeat_interleave(16, 0).repeat_interleave(16, 1), full, 0.0)[:M, :K]
    rows, cols = torch.nonzero(on, as_tuple=True)
    ptr = torch.zeros(Mb + 1, dtype=torch.int32, device=DEV)
    ptr[1:] = torch.cumsum(on.sum(1), 0)
    A = X.BCSRMatrix(Mb, Kb, 16, 16, M, K, ptr, cols.int(), blocks.reshape(-1).to(dtype))
    return X.SparseWeight(A), dense, (rows, cols)


def same_columns(got, want_of, N, step=1 << 22):
    for n in range(0, N, step):
        cols = slice(n, min(N, n + step))
        assert torch.equal(got[:, cols], want_of(cols).to(got.dtype)), n


def check_long(kind, M, K, N):
    print(kind, M, K, N, flush=True)
    dtype = TYPES[kind]
    G, A, _ = grid(M, K, dtype, 1, absent=[(0, 1)])
    U, B, _ = grid(M, K, dtype, 2, absent=[(1, 0)])
    x, dy = units((K, N), 3, dtype), units((M, N), 4, dtype)
    same_columns(X.sparse_linear(G, x, residual=dy), lambda c: A @ x[:, c].float() + dy[:, c].float(), N)
    h = X.sparse_gated(G, U, x, activation="none")
    same_columns(h, lambda c: (A @ x[:, c].float()) * (B @ x[:, c].float()), N)
    del h
    dx, dv, db = X.sparse_linear_backward(G, x, None, dy, bias=True)
    same_columns(dx, lambda c: A.t() @ dy[:, c].float(), N)
    del dx
    total = sum(dy[:, n:n + (1 << 22)].double().sum(1) for n in range(0, N, 1 << 22))
    assert torch.equal(db, total.to(dtype))
    check_blocks(G, dv, dy, x, dtype)
    one = torch.ones_like(dy)
    dx, dg, du, _, _ = X.sparse_gated_backward(G, U, x, one, dy, dy, activation="none")
    # dg = dh up = dy * dy, du = dh act(1) = dy
    same_columns(dx, lambda c: A.t() @ dy[:, c].float().square() + B.t() @ dy[:, c].float(), N)
    del dx, one
    check_blocks(G, dg, dy * dy, x, dtype)
    check_blocks(U, du, dy, x, dtype)


def check_blocks(W, got, left, right, dtype):
    """The stored blocks of left right^T, summed exactly."""
    (M, K), N = W.shape, left.shape[1]
    Mb, Kb = -(-M // 16), -(-K // 16)
    full = torch.zeros((Mb * 16, Kb * 16), dtype=torch.float64, device=DEV)
    for n in range(0, N, 1 << 20):  # parts that fp32 holds exactly
        full[:M, :K] += (left[:, n:n + (1 << 20)].float() @ right[:, n:n + (1 << 20)].float().t()).double()
    A = W.matrix
    rows = torch.repeat_interleave(torch.arange(Mb, device=DEV), torch.diff(A.row_ptr).long())
    want = full.view(Mb, 16, Kb, 16).transpose(1, 2)[rows, A.col_ind.long()].reshape(-1)
    assert float(want.abs().max()) < 2 ** 24 and torch.equal(got, want.to(dtype))


# 48 rows (33 and what fills their last block) of N values reach 2 GiB at 22369622 tokens in 16 bits and 11184811
# in 32: rows past it, and the last that are not, in whole chunks of 16 bytes and off them
@pytest.mark.parametrize("kind,N", [("f16", 22369625), ("bf16", 22369632), ("f32", 11184813), ("f16", 22369621),
                                    ("bf16", 22369616), ("f32", 11184810), ("f32", 11184808)])
@pytest.mark.parametrize("M,K", [(17, 33), (33, 17)])
def test_activations_around_two_gib(kind, M, K, N):
    check_long(kind, M, K, N)


# block values past 2 GiB
@pytest.mark.parametrize("kind,blocks", [("f16", 2050), ("bf16", 2050), ("f32", 1450)])
@pytest.mark.parametrize("N", [1, 33, 65])
def test_block_values_past_two_gib(kind, blocks, N):
    print(kind, blocks, N, flush=True)
    dtype = TYPES[kind]
    M = K = 16 * blocks - 3
    W, A, (rows, cols) = grid(M, K, dtype, 1, absent=[(1, 2), (blocks - 1, blocks - 1)])
    assert W.values.numel() * W.values.element_size() >= 1 << 31
    x, dy = units((K, N), 3, dtype), units((M, N), 4, dtype)
    assert torch.equal(X.sparse_linear(W, x), (A @ x.float()).to(dtype))
    h = X.sparse_gated(W, W, x, activation="relu")
    assert torch.equal(h, ((A @ x.float()).clamp(min=0) * (A @ x.float())).to(dtype))
    dx, dv, _ = X.sparse_linear_backward(W, x, None, dy)
    assert torch.equal(dx, (A.t() @ dy.float()).to(dtype))
    del A, dx
    full = torch.zeros((16 * blocks, 16 * blocks), dtype=dtype, device=DEV)
    full[:M, :K] = (dy.float() @ x.float().t()).to(dtype)
    want = full.view(blocks, 16, blocks, 16).transpose(1, 2)
    dv = dv.view(-1, 16, 16)
    for b in range(0, dv.shape[0], 1 << 20):
        part = slice(b, b + (1 << 20))
        assert torch.equal(dv[part], want[rows[part], cols[part]]), b


def test_tokens_of_one_launch():
    """64 rows of 64 tokens a workgroup of 256 threads: 2^24 workgroups are one too many threads."""
    W, A, _ = grid(16, 16, torch.float16, 1)
    N = ((1 << 24) - 8) * 64 - 3
    x = units((16, N), 3, torch.float16)
    y = X.sparse_linear(W, x)
    same_columns(y, lambda c: A @ x[:, c].float(), N, 1 << 24)
    del x, y
    x = torch.empty((16, 1 << 30), dtype=torch.float16, device=DEV)
    with pytest.raises(X.XspmmInvalidArgument, match="one launch"):
        X.sparse_linear(W, x)
    with pytest.raises(X.XspmmInvalidArgument, match="2\\^30"):
        X.sparse_linear(W, torch.empty((16, (1 << 30) + 1), dtype=torch.float16, device=DEV))
