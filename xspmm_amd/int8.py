"""Serving a block-sparse feed-forward layer in 8-bit integers.

Weights and activations are rounded to whole numbers of at most 127, a weight's
rows and the tokens each with a scale of their own:

  q = round(127 v / m), half to even, scale = m / 127, m the largest |v|

Products of whole numbers are summed in 32 bits, exactly; then a result is
float(sum) * row's scale * token's scale, bias, activation and residual in fp32,
rounded once to the weight's value type.

  Int8Weight        a SparseWeight's block values in 8 bits, made once
  quantize_tokens   activations in 8 bits
  int8_linear       y = act(A x + bias) + residual
  int8_gated        h = act(G x + bias_gate) * (U x + bias_up)
  Int8FeedForward   a FeedForward layer with its weights in 8 bits

The products take activations in the weight's value type, features x tokens as
``sparse_linear`` does, and round them themselves, or an ``Int8Tokens`` that several
products share.  A token or a weight's row that holds an infinity or a NaN has the
scale NaN, and so NaN results.  They run on torch's current stream, allocate with
torch, and have no gradients: an operand that wants one is refused.  An
``Int8Weight`` does not keep the wide values that it was made from.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

import xspmm_amd as X

from .feed_forward import (_TYPES, SparseWeight, _activation, _apart, _call, _check, _load as _load_layer, _grad_enabled,
                           _pair, _scratch, _Tensor, layer_norm)

_lib = None


def _load():
    global _lib
    if _lib is None:
        L = _load_layer()
        p, i64, i32 = C.c_void_p, C.c_int64, C.c_int
        out = C.POINTER(C.c_int64)
        for name, args in {
            "xspmm_int8_weight": [p, i32, p, p, p, p],
            "xspmm_quantize_tokens_scratch": [i64, i64, out],
            "xspmm_quantize_tokens": [i32, i64, i64, p, p, p, p, i64, p],
            "xspmm_int8_scratch": [i32, i64, i64, i64, out],
            "xspmm_int8_kernel": [i32, i32, i64, i64, i64, i64, i64, i32, C.POINTER(C.c_int32)],
            "xspmm_int8_linear": [p, i32, i32, p, p, p, p, p, p, p, p, i64, p, i64, p],
            "xspmm_int8_gated": [p, p, i32, i32, p, p, p, p, p, p, p, p, p, p, i64, p, i64, p],
        }.items():
            f = getattr(L, name)
            f.restype, f.argtypes = i32, args
        _lib = L
    return _lib


@functools.lru_cache(maxsize=1024)
def _bytes(query, *sizes):
    n = C.c_int64(0)
    X._check(getattr(_load(), query)(*sizes, C.byref(n)))
    return n.value


def _no_gradients(*operands):
    for t in operands:
        if t is not None and t.requires_grad and _grad_enabled():
            raise RuntimeError("the 8-bit operators have no gradients: call them under torch.no_grad()")


class Int8Weight:
    """The block values of a SparseWeight in 8 bits, with a scale for each row:
    ``values`` (num_blocks * 256 whole numbers, where the weight's values stand) and
    ``scale`` (fp32, one for each row).  Made once from the weight's values or from
    others (``values=``).  Neither they nor the weight are kept, only where its blocks
    stand: the values' memory is free when the weight goes.  Closing the weight closes
    what was made from it."""

    def __init__(self, W, values=None):
        if not isinstance(W, SparseWeight):
            raise TypeError("W must be a SparseWeight")
        _, vals = W._values(None if values is None else values.detach())
        self.shape, self.dtype, self.device, self.num_blocks = W.shape, W.dtype, W.device, W.num_blocks
        self._positions, self._code = W._positions, W.code
        self.values = torch.empty(W.num_blocks * 256, dtype=torch.int8, device=W.device)
        self.scale = torch.empty(W.shape[0], dtype=torch.float32, device=W.device)
        self._flat, self._rows = (W.num_blocks * 256,), (W.shape[0],)
        _call(W.device.index, _load().xspmm_int8_weight, W._h, W.code, vals, self.values.data_ptr() or None,
              self.scale.data_ptr() or None)

    def _operands(self):
        h = self._positions.h
        if h is None:
            raise RuntimeError("SparseWeight is closed")
        return (h, _check(self.values, "values", self._flat, torch.int8, self.device),
                _check(self.scale, "scale", self._rows, torch.float32, self.device, 3))


class Int8Tokens:
    """Activations (``shape``: features x tokens) in 8 bits: ``values``,
    ceil(features / 16) x tokens x 16 with 16 consecutive features of a token side by
    side and zeros past the last, and ``scale``, one for each token."""

    __slots__ = ("values", "scale", "shape")

    def __init__(self, values, scale, shape):
        self.values, self.scale, self.shape = values, scale, tuple(shape)

    def dequantize(self):
        """The activations that the whole numbers stand for, features x tokens in fp32."""
        K, N = self.shape
        return self.values.permute(0, 2, 1).reshape(-1, N)[:K].float() * self.scale


def _columns(x):
    if not isinstance(x, _Tensor):
        raise TypeError("x must be a torch tensor or Int8Tokens")
    if x.dim() != 2:
        raise ValueError(f"x must be features x tokens, got {x.dim()} dimensions")
    return x.shape


def quantize_tokens(x):
    """x (features x tokens) as ``Int8Tokens``."""
    K, N = _columns(x)
    dt, dev = x.dtype, x.device
    if dt not in _TYPES:
        raise TypeError(f"unsupported dtype {dt}")
    if dev.type != "cuda":
        raise ValueError("x is not on the GPU")
    xp = _check(x, "x", (K, N), dt, dev)
    _no_gradients(x)
    q = torch.empty((-(-K // 16), N, 16), dtype=torch.int8, device=dev)
    scale = torch.empty(N, dtype=torch.float32, device=dev)
    n = _bytes("xspmm_quantize_tokens_scratch", K, N)
    ws = _scratch(n, dev)
    _call(dev.index, _load().xspmm_quantize_tokens, _TYPES[dt], K, N, xp, q.data_ptr() or None,
          scale.data_ptr() or None, None if ws is None else ws.data_ptr(), n)
    return Int8Tokens(q, scale, (K, N))


def _tokens(x, weights, M, K, dtype, device):
    """(tokens, the addresses of x, of whole numbers and of scales, scratch, its
    bytes, what must stay alive) of a product's activations."""
    if isinstance(x, Int8Tokens):
        N = x.shape[1]
        if x.shape[0] != K:
            raise ValueError(f"x has shape {x.shape}, expected {(K, N)}")
        q = _check(x.values, "x.values", (-(-K // 16), N, 16), torch.int8, device)
        s = _check(x.scale, "x.scale", (N,), torch.float32, device, 3)
        return N, None, q, s, None, 0, x
    N = _columns(x)[1]
    xp = _check(x, "x", (K, N), dtype, device)
    if xp is None and N:  # no features: zeros
        s = torch.zeros(N, dtype=torch.float32, device=device)
        return N, None, None, s.data_ptr(), None, 0, s
    n = _bytes("xspmm_int8_scratch", weights, M, K, N)
    ws = _scratch(n, device)
    return N, xp, None, None, None if ws is None else ws.data_ptr(), n, ws


def _result(out, M, N, dtype, device, residual=None, **operands):
    if out is None:
        y = torch.empty((M, N), dtype=dtype, device=device)
        return y, y.data_ptr() or None
    yp = _check(out, "out", (M, N), dtype, device)
    if residual is not None and residual.data_ptr() == out.data_ptr():
        residual = None
    _apart(out, residual=residual, **operands)
    return out, yp


def _parts(x):
    return {"x": x.values, "x.scale": x.scale} if isinstance(x, Int8Tokens) else {"x": x}


def int8_linear(W, x, bias=None, activation=None, residual=None, out=None):
    """act(A x + bias) + residual of an ``Int8Weight``, M x N in its value type.  x:
    activations of that type, or ``Int8Tokens``.  out: memory for the result, apart
    from every operand, or the residual itself."""
    act = _activation(activation)
    (M, K), dt, dev = W.shape, W.dtype, W.device
    h, vals, scale = W._operands()
    N, xp, q, s, ws, n, held = _tokens(x, 1, M, K, dt, dev)
    bp = None if bias is None else _check(bias, "bias", (M,), dt, dev, 0)
    rp = None if residual is None else _check(residual, "residual", (M, N), dt, dev)
    _no_gradients(None if held is x else x, bias, residual)
    y, yp = _result(out, M, N, dt, dev, **({} if out is None else dict(
        residual=residual, bias=bias, values=W.values, scale=W.scale, **_parts(x))))
    _call(dev.index, _load().xspmm_int8_linear, h, W._code, act, vals, scale, xp, q, s, bp, rp, yp, N,
          ws, n)
    return y


def int8_gated(G, U, x, bias_gate=None, bias_up=None, activation="silu", out=None):
    """act(G x + bias_gate) * (U x + bias_up) of two ``Int8Weight``, M x N in their
    value type.  x as in ``int8_linear``; out: memory for the result, apart from every
    operand."""
    act = _activation(activation)
    (M, K), dt, dev = _pair(G, U), G.dtype, G.device
    (gh, gv, gs), (uh, uv, us) = G._operands(), U._operands()
    N, xp, q, s, ws, n, held = _tokens(x, 2, M, K, dt, dev)
    gb = None if bias_gate is None else _check(bias_gate, "bias_gate", (M,), dt, dev, 0)
    ub = None if bias_up is None else _check(bias_up, "bias_up", (M,), dt, dev, 0)
    _no_gradients(None if held is x else x, bias_gate, bias_up)
    h, hp = _result(out, M, N, dt, dev, **({} if out is None else dict(
        bias_gate=bias_gate, bias_up=bias_up, gate=G.values, gate_scale=G.scale, up=U.values, up_scale=U.scale,
        **_parts(x))))
    _call(dev.index, _load().xspmm_int8_gated, gh, uh, G._code, act, gv, gs, uv, us, xp, q, s,
          gb, ub, hp, N, ws, n)
    return h


class Int8FeedForward:
    """A ``FeedForward`` layer as it is served: its weights in 8 bits as they are now,
    its norm's weight and bias, x + D (act(G n) * (U n)) without gradients."""

    def __init__(self, layer):
        self.gate, self.up, self.down = (Int8Weight(W, v) for W, v in
                                         zip(layer._weights, (layer.gate, layer.up, layer.down)))
        self.norm_weight, self.norm_bias = layer.norm_weight.detach().clone(), layer.norm_bias.detach().clone()
        self.activation, self.eps = layer.activation, layer.eps

    def __call__(self, x):
        _no_gradients(x)
        n = layer_norm(x, self.norm_weight, self.norm_bias, self.eps)
        h = int8_gated(self.gate, self.up, n, activation=self.activation)
        return int8_linear(self.down, h, residual=x)
