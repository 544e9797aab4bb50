"""The feed-forward layer of a model on block-sparse weights, and layer norm.

Activations are features x tokens, contiguous, as the B and C of ``spmm``; a
weight is a ``BCSRMatrix`` of 16x16 blocks (``csr_to_bcsr``) whose block
positions a ``SparseWeight`` lays out once.  Every array of a call has the
weight's value type: float16, float32, or bfloat16, which the operators here
take besides the framework's two.  Sums are fp32, rounded once.  The products of
the backward pass take the sums' gradient (dy act', gated dy up act' and dy act)
rounded to the value type, as their matrix instructions have 16-bit operands: in 16
bits that adds as much error again as the results' own rounding, and fp16's range
holds for it (past 65504 it is infinite, below 6e-8 zero).

  sparse_linear            y = act(A x + bias) + residual
  sparse_gated             h = act(G x + bias_gate) * (U x + bias_up)
  layer_norm               over the features of every token
  *_backward               their gradients

The operators run on torch's current stream and allocate their results and
scratch with torch.  Where an operand has a gradient, the first three go through
autograd, to the same kernels; what they keep, and the results of the backward
operators, have none.  ``FeedForward`` puts them together as a module.
"""
from __future__ import annotations

import ctypes as C
import dataclasses
import functools

import torch

import xspmm_amd as X

BF16 = 2
ACTIVATIONS = {"none": 0, None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_TYPES = {torch.float32: X.F32, torch.float16: X.F16, torch.bfloat16: BF16}


def _prototypes(L):
    p, i64, i32, f32 = C.c_void_p, C.c_int64, C.c_int, C.c_float
    out = C.POINTER(C.c_int64)
    for name, args in {
        "xspmm_weight_create": [i32, i64, i64, i64, i64, i64, p, p, p, C.POINTER(C.c_void_p)],
        "xspmm_weight_destroy": [p],
        "xspmm_linear": [p, i32, i32, p, p, p, p, p, p, i64, p],
        "xspmm_gated": [p, p, i32, i32, p, p, p, p, p, p, p, p, i64, p],
        "xspmm_linear_backward_scratch": [p, i32, i32, i64, out],
        "xspmm_linear_backward": [p, i32, i32, p, p, p, p, p, p, p, i64, p, i64, p],
        "xspmm_gated_backward_scratch": [p, i32, i64, out],
        "xspmm_gated_backward": [p, p, i32, i32, p, p, p, p, p, p, p, p, p, p, p, i64, p, i64, p],
        "xspmm_layer_norm_scratch": [i32, i64, i64, i32, out],
        "xspmm_layer_norm": [i32, i64, i64, p, p, p, f32, p, p, p, p, i64, p],
        "xspmm_layer_norm_backward": [i32, i64, i64, p, p, p, p, p, p, p, p, p, i64, p],
    }.items():
        f = getattr(L, name)
        f.restype, f.argtypes = i32, args
    return L


_lib = None


def _load():
    global _lib
    if _lib is None:
        _lib = _prototypes(X.load())
    return _lib


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


# without the check of an initialized GPU, which what has an operand there needs none of
_current = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_grad_enabled = torch.is_grad_enabled
_Tensor = torch.Tensor
_PLAIN = (_Tensor, torch.nn.Parameter)


def _call(index, f, *args):
    """f(*args, stream) on torch's current stream of device `index`."""
    if _current() == index:
        rc = f(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _raw_stream(index))
    if rc:
        X._check(rc)


def _check(t, name, shape, dtype, device, mask=15):
    """The address of an operand that the kernels can take as given (None: no
    elements); raises otherwise.  mask: low bits that the address may not have."""
    if (t.__class__ in _PLAIN and t.dtype is dtype and t.shape == shape and t.device == device
            and t.is_contiguous()):
        at = t.data_ptr()
        if not at & mask:
            return at or None
    if not isinstance(t, _Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.data_ptr() & mask:
        raise ValueError(f"{name} must start on a 16-byte boundary")
    return t.data_ptr() or None


def _activation(name):
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"unknown activation {name!r}: one of {', '.join(k for k in ACTIVATIONS if k)}") from None


def _no_out(out):
    if out is not None:
        raise RuntimeError("out= has no gradient: call it under torch.no_grad(), or without out")


def _apart(out, **operands):
    """Raises where a result shares memory with an operand: workgroups read the
    operands after others have written."""
    lo = out.data_ptr()
    hi = lo + out.numel() * out.element_size()
    for name, t in operands.items():
        if t is not None and t.data_ptr() < hi and lo < t.data_ptr() + t.numel() * t.element_size():
            raise ValueError(f"out overlaps {name}")


def _scratch(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


class SparseWeight:
    """Where the 16x16 blocks of a BCSR matrix stand, laid out once for products
    with the matrix and with its transpose.  The positions are read once, here,
    and synchronize torch's current stream.  The block values (``values``,
    num_blocks * 256 of them) may change between calls: they are the matrix's,
    read at every call, until others are set here, which leaves the matrix as it
    is; and a call can bring its own (``values=``)."""

    def __init__(self, A):
        self._h = self._own = None
        if A.r_block != 16 or A.c_block != 16:
            raise ValueError("a weight has 16x16 blocks")
        if A.values.dtype not in _TYPES:
            raise TypeError(f"unsupported value dtype {A.values.dtype}")
        rp, ci = A.row_ptr, A.col_ind
        device = rp.device
        if device.type != "cuda":
            raise ValueError("a weight's arrays are on the GPU")
        X.icode(rp.dtype)
        _check(rp, "row_ptr", (int(A.num_block_rows) + 1,), rp.dtype, device, mask=0)
        _check(ci, "col_ind", (int(ci.numel()),), rp.dtype, device, mask=0)
        self.device = device
        self.shape = (int(A.num_rows), int(A.num_cols))
        self.num_blocks = int(ci.numel())
        self.dtype = A.values.dtype
        self.code = _TYPES[self.dtype]
        self.matrix = A
        self._flat = (self.num_blocks * 256,)
        _check(A.values, "values", (self.num_blocks * 256,), self.dtype, device)
        h = C.c_void_p()
        self._L = _load()
        with torch.cuda.device(device):
            X._check(self._L.xspmm_weight_create(X.icode(rp.dtype), *self.shape, int(A.num_block_rows),
                                                 int(A.num_block_cols), self.num_blocks, X._ptr(rp), X._ptr(ci),
                                                 _raw_stream(device.index), C.byref(h)))
        self._h = h

    @property
    def values(self):
        return self.matrix.values if self._own is None else self._own

    @values.setter
    def values(self, v):
        _check(v, "values", (self.num_blocks * 256,), self.dtype, self.device)
        self._own = v

    def _values(self, v=None):
        """The block values of a call, v or the weight's, and their address."""
        if self._h is None:
            raise RuntimeError("SparseWeight is closed")
        if v is None:
            v = self._own
            if v is None:
                v = self.matrix.values
        return v, _check(v, "values", self._flat, self.dtype, self.device)

    def close(self):
        if self._h is not None:
            self._L.xspmm_weight_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __reduce__(self):
        # copies lay their matrix out again: two that held one handle would free it twice
        return SparseWeight, (self.matrix,), {"_own": self._own}


def _tokens(x, name="x"):
    if not isinstance(x, _Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    shape = x.shape
    if len(shape) != 2:
        raise ValueError(f"{name} must be features x tokens, got {len(shape)} dimensions")
    return shape[1]


def _at(t):
    return None if t is None else t.data_ptr() or None


def sparse_linear(W, x, bias=None, activation=None, residual=None, keep=False, out=None, values=None):
    """act(W x + bias) + residual, M x N; with keep also W x + bias, which
    ``sparse_linear_backward`` takes where there is an activation.  values: block
    values in the place of W's.  out: memory for the result, apart from every
    operand, or the residual itself."""
    act = _activation(activation)
    (M, K), N, dt, dev = W.shape, _tokens(x), W.dtype, W.device
    v, vals = W._values(values)
    xp = _check(x, "x", (K, N), dt, dev)
    bp = None if bias is None else _check(bias, "bias", (M,), dt, dev, 0)
    rp = None if residual is None else _check(residual, "residual", (M, N), dt, dev)
    if (x.requires_grad or v.requires_grad or (bias is not None and bias.requires_grad)
            or (residual is not None and residual.requires_grad)) and _grad_enabled():
        _no_out(out)
        return _Linear.apply(W, v, x, bias, activation, residual, keep)
    if out is None:
        y = x.new_empty((M, N))
        yp = y.data_ptr() or None
    else:
        y, yp = out, _check(out, "out", (M, N), dt, dev)
        _apart(out, x=x, values=v, bias=bias, residual=None if yp == rp else residual)
    if not keep:
        _call(dev.index, W._L.xspmm_linear, W._h, W.code, act, vals, xp, bp, rp, yp, None, N)
        return y
    z = x.new_empty((M, N))
    _call(dev.index, W._L.xspmm_linear, W._h, W.code, act, vals, xp, bp, rp, yp, _at(z), N)
    return y, z


def sparse_linear_backward(W, x, kept, dy, activation=None, bias=False, need=(True, True), values=None):
    """(dx, dvalues, dbias) from dy = the gradient of ``sparse_linear``'s result
    and `kept` = W x + bias (not read, and may be None, without an activation).
    bias: whether the layer has one (dbias is None otherwise); need: whether dx
    and dvalues are wanted (None otherwise); values as in the forward pass.  The
    residual's gradient is dy.  dx and dvalues are products of dy act'(kept) rounded
    to the value type, dbias is its sum before that."""
    act = _activation(activation)
    (M, K), N, dt, dev = W.shape, _tokens(dy, "dy"), W.dtype, W.device
    _, vals = W._values(values)
    xp = _check(x, "x", (K, N), dt, dev)
    zp = _check(kept, "kept", (M, N), dt, dev) if act else None
    gp = _check(dy, "dy", (M, N), dt, dev)
    dx = x.new_empty((K, N)) if need[0] else None
    dv = x.new_empty(W._flat) if need[1] else None
    db = x.new_empty((M,)) if bias else None
    n = C.c_int64(0)
    rc = W._L.xspmm_linear_backward_scratch(W._h, W.code, act, N, C.byref(n))
    if rc:
        X._check(rc)
    ws = _scratch(n.value, dev)
    _call(dev.index, W._L.xspmm_linear_backward, W._h, W.code, act, vals, xp, zp, gp, _at(dx), _at(dv), _at(db), N,
          _at(ws), n.value)
    return dx, dv, db


def _pair(G, U):
    if G.shape != U.shape or G.dtype is not U.dtype or G.device != U.device:
        raise ValueError(f"gate ({G.shape}, {G.dtype}, {G.device}) and up ({U.shape}, {U.dtype}, {U.device}) differ")
    return G.shape


def sparse_gated(G, U, x, bias_gate=None, bias_up=None, activation="silu", keep=False, out=None,
                 values=(None, None)):
    """act(G x + bias_gate) * (U x + bias_up), M x N; with keep also the two
    sums, which ``sparse_gated_backward`` takes.  G and U have blocks of their
    own.  values: block values in the place of G's and U's (None: theirs).  out:
    memory for the result, apart from every operand."""
    act = _activation(activation)
    (M, K), N, dt, dev = _pair(G, U), _tokens(x), G.dtype, G.device
    (g, gv), (u, uv) = G._values(values[0]), U._values(values[1])
    xp = _check(x, "x", (K, N), dt, dev)
    gb = None if bias_gate is None else _check(bias_gate, "bias_gate", (M,), dt, dev, 0)
    ub = None if bias_up is None else _check(bias_up, "bias_up", (M,), dt, dev, 0)
    if (x.requires_grad or g.requires_grad or u.requires_grad or (bias_gate is not None and bias_gate.requires_grad)
            or (bias_up is not None and bias_up.requires_grad)) and _grad_enabled():
        _no_out(out)
        return _Gated.apply(G, U, g, u, x, bias_gate, bias_up, activation, keep)
    if out is None:
        h = x.new_empty((M, N))
        hp = h.data_ptr() or None
    else:
        h, hp = out, _check(out, "out", (M, N), dt, dev)
        _apart(out, x=x, gate_values=g, up_values=u, bias_gate=bias_gate, bias_up=bias_up)
    if not keep:
        _call(dev.index, G._L.xspmm_gated, G._h, U._h, G.code, act, gv, uv, xp, gb, ub, hp, None, None, N)
        return h
    zg, zu = x.new_empty((M, N)), x.new_empty((M, N))
    _call(dev.index, G._L.xspmm_gated, G._h, U._h, G.code, act, gv, uv, xp, gb, ub, hp, _at(zg), _at(zu), N)
    return h, zg, zu


def sparse_gated_backward(G, U, x, kept_gate, kept_up, dh, activation="silu", bias=False, need=(True, True, True),
                          values=(None, None)):
    """(dx, dvalues of G, dvalues of U, dbias_gate, dbias_up) from dh = the
    gradient of ``sparse_gated``'s result and the two sums it kept.  bias:
    whether the biases' gradients are wanted; need: whether the first three are
    (None otherwise); values as in the forward pass.  As in
    ``sparse_linear_backward``, the products take dh up act'(gate) and dh act(gate)
    rounded to the value type, the biases' gradients do not."""
    act = _activation(activation)
    (M, K), N, dt, dev = _pair(G, U), _tokens(dh, "dh"), G.dtype, G.device
    (_, gv), (_, uv) = G._values(values[0]), U._values(values[1])
    xp = _check(x, "x", (K, N), dt, dev)
    zg = _check(kept_gate, "kept_gate", (M, N), dt, dev)
    zu = _check(kept_up, "kept_up", (M, N), dt, dev)
    hp = _check(dh, "dh", (M, N), dt, dev)
    dx = x.new_empty((K, N)) if need[0] else None
    dg = x.new_empty(G._flat) if need[1] else None
    du = x.new_empty(U._flat) if need[2] else None
    bg = x.new_empty((M,)) if bias else None
    bu = x.new_empty((M,)) if bias else None
    n = C.c_int64(0)
    rc = G._L.xspmm_gated_backward_scratch(G._h, G.code, N, C.byref(n))
    if rc:
        X._check(rc)
    ws = _scratch(n.value, dev)
    _call(dev.index, G._L.xspmm_gated_backward, G._h, U._h, G.code, act, gv, uv, xp, zg, zu, hp, _at(dx), _at(dg),
          _at(du), _at(bg), _at(bu), N, _at(ws), n.value)
    return dx, dg, du, bg, bu


@functools.lru_cache(maxsize=1024)
def _norm_scratch(code, K, N, backward):
    """Bytes of scratch, from the sizes alone."""
    n = C.c_int64(0)
    X._check(_load().xspmm_layer_norm_scratch(code, K, N, backward, C.byref(n)))
    return n.value


def _norm_operands(x, weight):
    if not isinstance(x, _Tensor):
        raise TypeError("x must be a torch tensor")
    if x.dim() != 2:
        raise ValueError(f"x must be features x tokens, got {x.dim()} dimensions")
    dt, dev, (K, N) = x.dtype, x.device, x.shape
    if dt not in _TYPES:
        raise TypeError(f"unsupported dtype {dt}")
    if dev.type != "cuda":
        raise ValueError("x is not on the GPU")
    if K == 0:
        raise ValueError("a norm needs at least one feature")
    return K, N, dt, dev, _check(x, "x", (K, N), dt, dev), (
        None if weight is None else _check(weight, "weight", (K,), dt, dev, 0))


def layer_norm(x, weight=None, bias=None, eps=1e-5, keep=False, out=None):
    """Layer norm over the features (rows) of every token (column) of x; with
    keep also the tokens' mean and 1 / sqrt(variance + eps) in fp32, which
    ``layer_norm_backward`` takes.  out: memory for the result, apart from
    every operand."""
    K, N, dt, dev, xp, wp = _norm_operands(x, weight)
    bp = None if bias is None else _check(bias, "bias", (K,), dt, dev, 0)
    if (x.requires_grad or (weight is not None and weight.requires_grad)
            or (bias is not None and bias.requires_grad)) and _grad_enabled():
        _no_out(out)
        return _Norm.apply(x, weight, bias, eps, keep)
    if out is None:
        y = x.new_empty((K, N))
        yp = y.data_ptr() or None
    else:
        y, yp = out, _check(out, "out", (K, N), dt, dev)
        _apart(out, x=x, weight=weight, bias=bias)
    mean = torch.empty(N, dtype=torch.float32, device=dev) if keep else None
    rstd = torch.empty(N, dtype=torch.float32, device=dev) if keep else None
    code = _TYPES[dt]
    n = _norm_scratch(code, K, N, 0)
    ws = _scratch(n, dev)
    _call(dev.index, _load().xspmm_layer_norm, code, K, N, xp, wp, bp, eps, yp, _at(mean), _at(rstd), _at(ws), n)
    return (y, mean, rstd) if keep else y


def layer_norm_backward(dy, x, weight, mean, rstd, need=(True, True, True)):
    """(dx, dweight, dbias) of ``layer_norm`` from dy and the statistics it
    kept; weight may be None (ones).  need: which of them are wanted (None
    otherwise)."""
    K, N, dt, dev, xp, wp = _norm_operands(x, weight)
    gp = _check(dy, "dy", (K, N), dt, dev)
    mp = _check(mean, "mean", (N,), torch.float32, dev, 3)
    sp = _check(rstd, "rstd", (N,), torch.float32, dev, 3)
    dx = x.new_empty((K, N)) if need[0] else None
    dw = x.new_empty((K,)) if need[1] else None
    db = x.new_empty((K,)) if need[2] else None
    code = _TYPES[dt]
    n = _norm_scratch(code, K, N, 1)
    ws = _scratch(n, dev)
    _call(dev.index, _load().xspmm_layer_norm_backward, code, K, N, gp, xp, wp, mp, sp, _at(dx), _at(dw), _at(db),
          _at(ws), n)
    return dx, dw, db


# ---------------------------------------------------------------------------
# as a module
# ---------------------------------------------------------------------------

def prune_blocks(dense, density):
    """The 16x16 blocks of a dense M x K weight with the largest norms, a share
    `density` of them (at least one), as a BCSRMatrix on the weight's device."""
    M, K = dense.shape
    Mb, Kb = -(-M // 16), -(-K // 16)
    padded = dense.new_zeros((Mb * 16, Kb * 16))
    padded[:M, :K] = dense
    blocks = padded.view(Mb, 16, Kb, 16).permute(0, 2, 1, 3).reshape(Mb * Kb, 256)
    norms = blocks.float().square().sum(1)
    keep = torch.topk(norms, max(1, round(density * Mb * Kb))).indices.sort().values
    row_ptr = torch.zeros(Mb + 1, dtype=torch.int32, device=dense.device)
    row_ptr[1:] = torch.cumsum(torch.bincount(keep // Kb, minlength=Mb), 0)
    return X.BCSRMatrix(Mb, Kb, 16, 16, M, K, row_ptr, (keep % Kb).int(), blocks[keep].reshape(-1).contiguous())


class _NoSecond(torch.autograd.Function):
    """Gradients as they are, with a derivative that is refused: `n` of them, then
    all that they depend on, so that every way back to it comes through here."""

    @staticmethod
    def forward(ctx, n, *tensors):
        return tuple(t.view_as(t) for t in tensors[:n])

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("the feed-forward operators have no second derivatives")


def _incoming(g):
    """An incoming gradient as the kernels take it: other layers may hand over any
    strides, and contiguous views that start anywhere."""
    g = g.contiguous()
    return g.clone() if g.data_ptr() & 15 else g


def _first_order(backward):
    """A backward pass whose results come from kernels and so have no graph.  Where
    one is asked for (create_graph), their derivative raises instead of being taken
    for zero."""
    @functools.wraps(backward)
    def first_order(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            found = backward(ctx, *grads)
        given = [t for t in found if t is not None]
        on = [t for t in (*grads, *ctx.saved_tensors) if t is not None and t.requires_grad]
        if not on:
            return found
        marked = iter(_NoSecond.apply(len(given), *given, *on))
        return tuple(None if t is None else next(marked) for t in found)

    return first_order


def _result(ctx, y, *kept):
    """Results of a forward pass, of which the kept ones have no gradient."""
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(*kept)
    return (y, *kept)


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep=False):
        y, mean, rstd = layer_norm(x, weight, bias, eps, keep=True)
        ctx.save_for_backward(x, weight, mean, rstd)
        return _result(ctx, y, mean, rstd) if keep else y

    @staticmethod
    @_first_order
    def backward(ctx, dy, *_):
        x, weight, mean, rstd = ctx.saved_tensors
        return (*layer_norm_backward(_incoming(dy), x, weight, mean, rstd, need=ctx.needs_input_grad[:3]), None, None)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, W, values, x, bias, activation, residual, keep=False):
        # without an activation the backward pass does not read W x + bias
        wanted = keep or _activation(activation) != 0
        y = sparse_linear(W, x, bias, activation, residual, keep=wanted, values=values)
        y, z = y if wanted else (y, None)
        ctx.W, ctx.activation, ctx.bias = W, activation, bias is not None
        ctx.save_for_backward(values, x, z if _activation(activation) else None, bias)
        return _result(ctx, y, z) if keep else y

    @staticmethod
    @_first_order
    def backward(ctx, dy, *_):
        values, x, z, _bias = ctx.saved_tensors
        dy = _incoming(dy)
        need = ctx.needs_input_grad
        dx, dv, db = sparse_linear_backward(ctx.W, x, z, dy, ctx.activation, ctx.bias and need[3], (need[2], need[1]),
                                            values=values)
        return None, dv, dx, db, None, dy if need[5] else None, None


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, G, U, gate, up, x, bias_gate, bias_up, activation, keep=False):
        h, zg, zu = sparse_gated(G, U, x, bias_gate, bias_up, activation, keep=True, values=(gate, up))
        ctx.G, ctx.U, ctx.activation = G, U, activation
        ctx.save_for_backward(gate, up, x, zg, zu, bias_gate, bias_up)
        return _result(ctx, h, zg, zu) if keep else h

    @staticmethod
    @_first_order
    def backward(ctx, dh, *_):
        gate, up, x, zg, zu, _bg, _bu = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dg, du, bg, bu = sparse_gated_backward(ctx.G, ctx.U, x, zg, zu, _incoming(dh), ctx.activation,
                                                   need[5] or need[6], (need[4], need[2], need[3]), (gate, up))
        return None, None, dg, du, dx, bg if need[5] else None, bu if need[6] else None, None, None


class FeedForward(torch.nn.Module):
    """x + D (act(G n) * (U n)), n = layer_norm(x): a model's feed-forward layer
    on three BCSR matrices (G and U hidden x features, D features x hidden), with
    their block values and the norm's weight and bias as parameters.  The matrices
    are read, not kept up to date; weights may share one.  Which blocks are stored
    does not change, and is not in the state dict.  x is features x tokens.  There
    are no second derivatives: asking for one raises."""

    def __init__(self, gate, up, down, activation="silu", eps=1e-5):
        super().__init__()
        # matrices of its own, whose values the parameters share
        self._weights = [SparseWeight(dataclasses.replace(A, values=A.values.detach().clone()))
                         for A in (gate, up, down)]
        G, U, D = self._weights
        features = _pair(G, U)[1]
        if D.shape != (features, G.shape[0]) or D.dtype is not G.dtype or D.device != G.device:
            raise ValueError(f"down is {D.shape}, {D.dtype}, expected {(features, G.shape[0])}, {G.dtype}")
        _activation(activation)
        self.activation, self.eps = activation, eps
        self.gate, self.up, self.down = (torch.nn.Parameter(W.values) for W in self._weights)
        like = dict(dtype=G.dtype, device=G.device)
        self.norm_weight = torch.nn.Parameter(torch.ones(features, **like))
        self.norm_bias = torch.nn.Parameter(torch.zeros(features, **like))

    def forward(self, x):
        G, U, D = self._weights
        n = layer_norm(x, self.norm_weight, self.norm_bias, self.eps)
        h = sparse_gated(G, U, n, activation=self.activation, values=(self.gate, self.up))
        return sparse_linear(D, h, residual=x, values=self.down)
