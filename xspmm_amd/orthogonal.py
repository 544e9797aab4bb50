"""Orthogonalised updates for training block-sparse feed-forward layers.

An update whose singular values differ by orders moves a weight along a few
directions only.  ``orthogonalize`` brings them near 1 by an odd polynomial of the
matrix, applied several times (quintic Newton-Schulz iteration):

  X = U / (|U| + eps),  X <- a X + (b S + c S S) X,  S = X X^T

U is the dense matrix of a weight's stored blocks, zeros elsewhere; the result is X at
the stored blocks.  ``OrthogonalMomentum`` is the optimiser that uses it for the
weights of ``FeedForward`` layers.
"""
from __future__ import annotations

import ctypes as C

import torch

import xspmm_amd as X

from .feed_forward import FeedForward, SparseWeight, _apart, _call, _check, _grad_enabled, _load as _load_layer, _scratch

COEFFICIENTS = (3.4445, -4.7750, 2.0315)

_lib = None


def _load():
    global _lib
    if _lib is None:
        L = _load_layer()
        p, i64, i32, f32 = C.c_void_p, C.c_int64, C.c_int, C.c_float
        for name, args in {
            "xspmm_orthogonalize_scratch": [p, i32, C.POINTER(C.c_int64)],
            "xspmm_orthogonalize": [p, i32, p, p, i32, f32, f32, f32, f32, p, i64, p],
        }.items():
            f = getattr(L, name)
            f.restype, f.argtypes = i32, args
        _lib = L
    return _lib


def orthogonalize(W, update, steps=5, coefficients=COEFFICIENTS, eps=1e-7, out=None):
    """An update of the block values of W (a ``SparseWeight``; its own values are not
    read), orthogonalised: values as W's, num_blocks * 256 in its value type, zeros past
    the weight's edges.  Products take fp16 operands, of fp16 and fp32 updates two halves of
    each; the result is off by its own rounding and up to 1e-3 (bf16), 1e-5 (fp16, fp32)
    of its rms.  (X is held to 2^-37, which leaves fewer digits of an update whose norm is
    less than a hundredth of eps.)  With coefficients of one's own, the elements of X, S and
    b S + c S S have to stay below 16.  An update that holds an infinity or a NaN gives NaN.
    out: memory for the result, apart from the update or the update itself.  Scratch of
    several dense matrices of W's size is allocated for the call.  No gradients."""
    if not isinstance(W, SparseWeight):
        raise TypeError("W must be a SparseWeight")
    if W._h is None:
        raise RuntimeError("SparseWeight is closed")
    steps = int(steps)
    if not 1 <= steps < 1 << 31:
        raise ValueError(f"steps must be at least 1, got {steps}")
    a, b, c = coefficients
    dev = W.device
    up = _check(update, "update", W._flat, W.dtype, dev)
    if update.requires_grad and _grad_enabled():
        raise RuntimeError("orthogonalize has no gradient: call it under torch.no_grad()")
    if out is None:
        out = torch.empty(W._flat, dtype=W.dtype, device=dev)
        op = out.data_ptr() or None
    else:
        op = _check(out, "out", W._flat, W.dtype, dev)
        if op != up:
            _apart(out, update=update)
    L, n = _load(), C.c_int64(0)
    rc = L.xspmm_orthogonalize_scratch(W._h, W.code, C.byref(n))
    if rc:
        X._check(rc)
    ws = _scratch(n.value, dev)
    _call(dev.index, L.xspmm_orthogonalize, W._h, W.code, up, op, steps, a, b, c, eps,
          None if ws is None else ws.data_ptr(), n.value)
    return out


class OrthogonalMomentum(torch.optim.Optimizer):
    """Momentum whose updates are orthogonalised, for the weights (gate, up, down) of
    ``FeedForward`` layers; their norms' weights and biases are another optimiser's.

      v <- momentum v + g,   u = g + momentum v (nesterov) or v
      w <- (1 - lr weight_decay) w - lr sqrt(max(1, rows / columns)) orthogonalize(u)

    The size of u does not matter, however small.  v and, for 16-bit weights, a master
    copy of w are kept in fp32; where a weight is not what its copy rounds to, as after
    loading another, the weight counts."""

    def __init__(self, layers, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5):
        layers = [layers] if isinstance(layers, torch.nn.Module) else list(layers)
        for layer in layers:
            if not isinstance(layer, FeedForward):
                raise TypeError("OrthogonalMomentum takes FeedForward layers")
        if lr < 0 or weight_decay < 0 or not 0 <= momentum < 1:
            raise ValueError("lr and weight_decay must not be negative, momentum lies in [0, 1)")
        params = [p for layer in layers for p in (layer.gate, layer.up, layer.down)]
        if len(set(map(id, params))) < len(params):
            raise ValueError("a layer's weights are given twice")
        self._weights = None
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      steps=steps))
        self._weights = [W for layer in layers for W in layer._weights]

    def __getstate__(self):
        # copies and pickles: torch's own state leaves the weights out
        return {**super().__getstate__(), "_weights": self._weights}

    def add_param_group(self, group):
        if getattr(self, "_weights", None) is not None:
            raise RuntimeError("the parameters of OrthogonalMomentum are its layers' weights")
        super().add_param_group(group)

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # which takes the state to the parameters' type
        saved = (i for g in state_dict["param_groups"] for i in g["params"])
        for i, p in zip(saved, (p for g in self.param_groups for p in g["params"])):
            for name, v in state_dict["state"].get(i, {}).items():
                self.state[p][name] = v.detach().to(p.device, torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        weights = iter(self._weights)
        for group in self.param_groups:
            lr, momentum = group["lr"], group["momentum"]
            for p in group["params"]:
                W = next(weights)
                if p.grad is None or not p.numel():  # a weight without blocks
                    continue
                state = self.state[p]
                if "momentum" not in state:
                    state["momentum"] = torch.zeros_like(p, dtype=torch.float32)
                if "master" not in state and p.dtype is not torch.float32:  # nor in the state of an fp32 layer
                    state["master"] = p.detach().float()
                g, v = p.grad.float(), state["momentum"]
                v.mul_(momentum).add_(g)
                u = g.add(v, alpha=momentum) if group["nesterov"] else v
                # The size of u does not matter, nor may eps damp it: beside a 16-bit u, scaled to fit
                # its type with a largest element of 1, it is nothing, in fp32 it is left out.
                eps = 0.0
                if W.dtype is not torch.float32:
                    u, eps = u / u.abs().amax().clamp_min(torch.finfo(torch.float32).tiny), 1e-7
                # a copy in W's type: the result goes where it stood
                u = u.to(W.dtype, copy=True)
                orthogonalize(W, u, steps=group["steps"], eps=eps, out=u)
                master = state.get("master", p)
                if master is not p:  # values that the weight has been given since the last step count
                    master.copy_(torch.where(master.to(p.dtype) == p, master, p.float()))
                if group["weight_decay"]:
                    master.mul_(1 - lr * group["weight_decay"])
                rows, columns = W.shape
                master.add_(u, alpha=-lr * max(1.0, rows / max(1, columns)) ** 0.5)
                if master is not p:
                    p.copy_(master)
        return loss
