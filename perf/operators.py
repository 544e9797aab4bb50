"""The feed-forward layer of a model with block-sparse weights, as timed cases.

A case is one call of an operator of that layer, on inputs made from a seed.
Activations are features x tokens, weights are 16x16 blocks (block-CSR):

  linear       y = act(A x + b) + residual; with keep also z = A x + b
  linear_grad  from z and dy: dx, the gradient of A's stored blocks, db
  gated        h = act(Ag x + bg) * (Au x + bu); with keep also both sums
  gated_grad   from both sums and dh: dx, both block gradients, dbg, dbu
  norm         layer norm over the features of every token; with keep also the
               mean and the reciprocal standard deviation
  norm_grad    from those and dy: dx, dweight, dbias

`density` is the share of a weight's blocks that are stored, `empty` the share
of its block-rows that hold none (neurons pruned away).  Every value of a
stored block is a weight.  Where `own` is false the operators are computed in
elementary operations in 32 bits on the unpacked weight.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
_VALUES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-5


def listed():
    return [
        # one token through a down projection whose weight has a quarter of
        # its blocks, added to the residual stream
        _matrix("linear_token", "linear", "f16", 4096, 14336, 1, 0.25, "none", residual=True),
        # block-structured weights, 5 % of the blocks, a batch of 256
        _matrix("linear_blocks", "linear", "f16", 8192, 8192, 256, 0.05, "relu", bias=True),
        # an up projection pruned entry by entry (no block falls out) over a
        # long prompt
        _matrix("linear_pruned", "linear", "f16", 14336, 4096, 2048, 1.0, "gelu", bias=True),
        # odd sizes everywhere, in the reference's value type: a head's 31 columns
        _matrix("linear_ragged", "linear", "f32", 5003, 4999, 31, 0.1, "silu", bias=True, residual=True),
        # training such a layer in single precision
        _matrix("linear_grad_f32", "linear_grad", "f32", 4096, 4096, 512, 0.1, "gelu_tanh", bias=True),
        # one token through the gate and up projections
        _matrix("gated_token", "gated", "bf16", 14336, 4096, 1, 0.25, "silu"),
        # a small layer and few tokens: launch and latency
        _matrix("gated_small", "gated", "f16", 1024, 1024, 64, 0.2, "gelu", bias=True, empty=0.1),
        # a long prompt through gate and up
        _matrix("gated_prompt", "gated", "bf16", 14336, 4096, 2048, 0.25, "silu"),
        # the same in training: everything the backward pass returns
        _matrix("gated_grad", "gated_grad", "bf16", 14336, 4096, 2048, 0.25, "silu", bias=True),
        # the norm of one token
        _norm("norm_token", "norm", "f16", 4096, 1),
        # the norm of a long prompt, its statistics kept
        _norm("norm_prompt", "norm", "f16", 4096, 2048, keep=True),
        # its backward pass over packed sequences of odd length
        _norm("norm_grad", "norm_grad", "bf16", 4096, 8001),
    ]


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        # 32-bit products run at a sixteenth of the 16-bit rate
        flops = w["flops"] * (16 if case["values"] == "f32" and "density" in case else 1)
        if flops <= 2.4e11 and w["bytes"] <= 4e8:
            return case


def _draw_once(rng):
    kind = rng.choice(["linear", "linear", "linear_grad", "gated", "gated", "gated_grad", "norm", "norm_grad"])
    values = rng.choice(["f16", "bf16", "f32"])
    if kind.startswith("norm"):
        N = 1 if rng.random() < 0.15 else _size(rng, 2, 16384)
        return _norm(None, kind, values, _size(rng, 64, 16384), N, keep=rng.random() < 0.5)
    N = 1 if rng.random() < 0.15 else _size(rng, 2, 2048)
    if rng.random() < 0.4:
        N = max(8, N // 8 * 8)
    act = rng.choice(["silu", "gelu", "gelu_tanh", "relu"] + ([] if kind.startswith("gated") else ["none"]))
    density = math.exp(rng.uniform(math.log(0.02), 0.0))
    empty = rng.choice([0.0, 0.0, rng.uniform(0.02, 0.3)])
    return _matrix(None, kind, values, _size(rng, 256, 14336), _size(rng, 256, 14336), N, density, act,
                   bias=rng.random() < 0.5, residual=kind == "linear" and rng.random() < 0.5,
                   keep=kind in ("linear", "gated") and rng.random() < 0.3, empty=empty)


def _size(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def _matrix(name, kind, values, M, K, N, density, act, bias=False, residual=False, keep=False, empty=0.0):
    case = dict(kind=kind, values=values, M=M, K=K, N=N, density=density, act=act, bias=bias,
                residual=residual, keep=keep, empty=empty)
    if name:
        case["name"] = name
    return case


def _norm(name, kind, values, K, N, keep=False):
    case = dict(kind=kind, values=values, K=K, N=N, keep=keep)
    if name:
        case["name"] = name
    return case


# ---------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------

def _stored(case):
    """Stored blocks of one weight."""
    Mb, Kb = -(-case["M"] // 16), -(-case["K"] // 16)
    return max(1, round((Mb - round(Mb * case["empty"])) * Kb * case["density"]))


def work(case):
    s = 4 if case["values"] == "f32" else 2
    kind, K, N = case["kind"], case["K"], case["N"]
    if kind == "norm":
        return {"bytes": float(2 * K * N * s + 2 * K * s + case["keep"] * 8 * N), "flops": 8.0 * K * N}
    if kind == "norm_grad":
        return {"bytes": float(3 * K * N * s + 3 * K * s + 8 * N), "flops": 12.0 * K * N}
    M = case["M"]
    weights = 2 if kind.startswith("gated") else 1
    blocks = weights * _stored(case)
    index = 4 * blocks + weights * 4 * (-(-M // 16) + 1)
    bias = case["bias"] * weights * M * s
    if kind in ("linear", "gated"):
        dense = K * N + M * N + case["residual"] * M * N + case["keep"] * weights * M * N
        return {"bytes": float(blocks * 256 * s + index + dense * s + bias), "flops": 512.0 * blocks * N}
    # the weights and x are read, dx and the blocks' gradients written; the
    # kept sums (not needed without an activation) and the incoming gradient
    # are read
    kept = 0 if case["act"] == "none" else weights
    dense = 2 * K * N + (kept + 1) * M * N
    return {"bytes": float(2 * blocks * 256 * s + index + dense * s + bias), "flops": 1024.0 * blocks * N}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _weight(case, g):
    """row_ptr, col_ind and block values of one weight; entries past the last
    row or column are zero, the products have about unit variance."""
    M, K = case["M"], case["K"]
    Mb, Kb = -(-M // 16), -(-K // 16)
    # as many blocks for every seed: those of the lowest draws outside the
    # block-rows that were pruned away
    full = Mb - round(Mb * case["empty"])
    kept = torch.randperm(Mb, generator=g, device=DEVICE)[:full].sort().values
    pick = torch.randperm(full * Kb, generator=g, device=DEVICE)[:_stored(case)]
    on = torch.zeros((Mb, Kb), dtype=torch.bool, device=DEVICE)
    on[kept[pick // Kb], pick % Kb] = True
    rows, cols = torch.nonzero(on, as_tuple=True)
    ptr = torch.zeros(Mb + 1, dtype=torch.int64, device=DEVICE)
    ptr[1:] = torch.cumsum(on.sum(1), 0)
    v = torch.randn((cols.numel(), 16, 16), generator=g, device=DEVICE)
    v *= 1.0 / math.sqrt(max(1.0, case["density"] * K))
    if M % 16:
        v[rows == Mb - 1, M % 16:, :] = 0
    if K % 16:
        v[cols == Kb - 1, :, K % 16:] = 0
    return {"M": M, "K": K, "ptr": ptr.int(), "col": cols.int(), "v": v.reshape(-1).to(_VALUES[case["values"]])}


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    vt = _VALUES[case["values"]]

    def normal(*shape, scale=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device=DEVICE) * scale + mean).to(vt)

    K, N, kind = case["K"], case["N"], case["kind"]
    s = {"case": case}
    if kind.startswith("norm"):
        # a residual stream: tokens of different scale and a small offset
        scale = torch.rand((1, N), generator=g, device=DEVICE) * 2 + 0.5
        s["x"] = (torch.randn((K, N), generator=g, device=DEVICE) * scale + 0.1).to(vt)
        s["weight"] = normal(K, scale=0.2, mean=1.0)
        s["bias"] = normal(K, scale=0.1)
        if kind == "norm_grad":
            s["dy"] = normal(K, N)
            xd = s["x"].double()
            mean = xd.mean(0)
            s["mean"] = mean.float()
            s["rstd"] = ((xd - mean).square().mean(0) + _EPS).rsqrt().float()
        return s
    M = case["M"]
    weights = 2 if kind.startswith("gated") else 1
    s["x"] = normal(K, N)
    s["w"] = [_weight(case, g) for _ in range(weights)]
    s["b"] = [normal(M, scale=0.1) if case["bias"] else None for _ in range(weights)]
    s["residual"] = normal(M, N) if case["residual"] else None
    if kind.endswith("grad"):
        s["z"] = [normal(M, N) for _ in range(weights)]
        s["dy"] = normal(M, N)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and "w" in s:
        import xspmm_amd as X

        def weight(w):
            Mb, Kb = -(-w["M"] // 16), -(-w["K"] // 16)
            return X.SparseWeight(X.BCSRMatrix(Mb, Kb, 16, 16, w["M"], w["K"], w["ptr"], w["col"], w["v"]))

        s["W"] = [weight(w) for w in s["w"]]
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    out = _run_own(state) if own else _run_plain(state)
    return [t for t in out if t is not None] if isinstance(out, tuple) else out


def _run_own(s):
    import xspmm_amd as X

    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        return X.layer_norm(s["x"], s["weight"], s["bias"], eps=_EPS, keep=case["keep"])
    if kind == "norm_grad":
        return X.layer_norm_backward(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"])
    W, b, act = s["W"], s["b"], case["act"]
    if kind == "linear":
        return X.sparse_linear(W[0], s["x"], bias=b[0], activation=act, residual=s["residual"], keep=case["keep"])
    if kind == "gated":
        return X.sparse_gated(W[0], W[1], s["x"], bias_gate=b[0], bias_up=b[1], activation=act, keep=case["keep"])
    if kind == "linear_grad":
        return X.sparse_linear_backward(W[0], s["x"], s["z"][0], s["dy"], activation=act, bias=case["bias"])
    return X.sparse_gated_backward(W[0], W[1], s["x"], s["z"][0], s["z"][1], s["dy"], activation=act,
                                   bias=case["bias"])


def _unpack(w):
    """The weight as an M x K matrix in 32 bits."""
    M, K = w["M"], w["K"]
    Mb, Kb = -(-M // 16), -(-K // 16)
    n = w["col"].numel()
    rows = torch.repeat_interleave(torch.arange(Mb, device=DEVICE), torch.diff(w["ptr"]).long(), output_size=n)
    d = torch.zeros((Mb, Kb, 16, 16), device=DEVICE)
    d[rows, w["col"].long()] = w["v"].view(n, 16, 16).float()
    return d.permute(0, 2, 1, 3).reshape(Mb * 16, Kb * 16)[:M, :K]


def _at_blocks(w, d):
    """The stored blocks of an M x K matrix, zero past its edges."""
    M, K = w["M"], w["K"]
    Mb, Kb = -(-M // 16), -(-K // 16)
    n = w["col"].numel()
    rows = torch.repeat_interleave(torch.arange(Mb, device=DEVICE), torch.diff(w["ptr"]).long(), output_size=n)
    full = torch.zeros((Mb * 16, Kb * 16), device=DEVICE)
    full[:M, :K] = d
    return full.view(Mb, 16, Kb, 16).permute(0, 2, 1, 3)[rows, w["col"].long()].reshape(-1)


def _act(name, z):
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return z * 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _run_plain(s):
    case = s["case"]
    kind, vt = case["kind"], s["x"].dtype
    x = s["x"].float()
    if kind == "norm":
        mean = x.mean(0)
        c = x - mean
        rstd = 1 / torch.sqrt((c * c).mean(0) + _EPS)
        y = (c * rstd * s["weight"].float()[:, None] + s["bias"].float()[:, None]).to(vt)
        return (y, mean, rstd) if case["keep"] else y
    if kind == "norm_grad":
        dy, rstd = s["dy"].float(), s["rstd"]
        xhat = (x - s["mean"]) * rstd
        g = dy * s["weight"].float()[:, None]
        dx = (g - g.mean(0) - xhat * (g * xhat).mean(0)) * rstd
        return dx.to(vt), (dy * xhat).sum(1).to(vt), dy.sum(1).to(vt)
    act = case["act"]
    w = [_unpack(m) for m in s["w"]]
    if kind in ("linear", "gated"):
        z = [m @ x for m in w]
        z = [v if b is None else v + b.float()[:, None] for v, b in zip(z, s["b"])]
        y = _act(act, z[0])
        if kind == "gated":
            y = y * z[1]
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return (y.to(vt), *[v.to(vt) for v in z]) if case["keep"] else y.to(vt)
    z, dy = [v.float() for v in s["z"]], s["dy"].float()
    if kind == "linear_grad":
        dz = [dy * _act_slope(act, z[0])]
    else:
        dz = [dy * z[1] * _act_slope(act, z[0]), dy * _act(act, z[0])]
    dx = w[0].t() @ dz[0]
    for m, d in zip(w[1:], dz[1:]):
        dx = dx + m.t() @ d
    dw = [_at_blocks(m, d @ x.t()) for m, d in zip(s["w"], dz)]
    db = [d.sum(1).to(vt) if case["bias"] else None for d in dz]
    return (dx.to(vt), *[d.to(vt) for d in dw], *db)


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    x = s["x"].double()
    if kind == "norm":
        var, mean = torch.var_mean(x, 0, correction=0)
        sigma = (var + _EPS).sqrt()
        y = torch.addcmul(s["bias"].double()[:, None], (x - mean) / sigma, s["weight"].double()[:, None])
        return (y, mean, 1 / sigma) if case["keep"] else y
    if kind == "norm_grad":
        dy, r = s["dy"].double(), s["rstd"].double()
        h = (x - s["mean"].double()) * r
        g = s["weight"].double()[:, None] * dy
        K = case["K"]
        dx = r / K * (K * g - g.sum(0) - h * (g * h).sum(0))
        return dx, torch.linalg.vecdot(dy, h), dy.sum(1)
    act = case["act"]
    if kind in ("linear", "gated"):
        z = []
        for w, b in zip(s["w"], s["b"]):
            v = _gather(w, x, False)
            z.append(v if b is None else v + b.double()[:, None])
        y = _value64(act, z[0])[0]
        if kind == "gated":
            y = y * z[1]
        if s["residual"] is not None:
            y = y + s["residual"].double()
        return (y, *z) if case["keep"] else y
    dy = s["dy"].double()
    value, slope = _value64(act, s["z"][0].double())
    dz = [dy * slope] if kind == "linear_grad" else [dy * slope * s["z"][1].double(), dy * value]
    dx = sum(_gather(w, d, True) for w, d in zip(s["w"], dz))
    dw = [_sampled(w, d, x) for w, d in zip(s["w"], dz)]
    return (dx, *dw, *[d.sum(1) for d in dz if case["bias"]])


def _value64(act, z):
    """An activation and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, z, 0), torch.where(z > 0, 1.0, 0.0).double()
    if act == "silu":
        p = torch.special.expit(z)
        return z * p, p + z * p * torch.special.expit(-z)
    if act == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    a = math.sqrt(8 / math.pi)
    p = torch.special.expit(a * (z + 0.044715 * z ** 3))
    return z * p, p + z * p * (1 - p) * a * (1 + 0.134145 * z * z)


def _padded(d, rows):
    out = torch.zeros((rows, d.shape[1]), dtype=torch.float64, device=DEVICE)
    out[:d.shape[0]] = d
    return out


def _coordinates(w):
    Mb = w["ptr"].numel() - 1
    counts = (w["ptr"][1:] - w["ptr"][:-1]).cpu().tolist()
    rows = torch.tensor([i for i in range(Mb) for _ in range(counts[i])], dtype=torch.int64, device=DEVICE)
    return rows, w["col"].long()


def _gather(w, d, transposed):
    """A d, or its transpose's product, one output block-row at a time."""
    rows, cols = _coordinates(w)
    v = w["v"].double().view(-1, 16, 16)
    out_len, in_len = (w["K"], w["M"]) if transposed else (w["M"], w["K"])
    to, of = (cols, rows) if transposed else (rows, cols)
    if transposed:
        v = v.transpose(1, 2)
    order = torch.argsort(to, stable=True)
    ends = torch.cumsum(torch.bincount(to, minlength=-(-out_len // 16)), 0).cpu().tolist()
    slabs = _padded(d, -(-in_len // 16) * 16).view(-1, 16, d.shape[1])
    out = torch.zeros((len(ends) * 16, d.shape[1]), dtype=torch.float64, device=DEVICE)
    begin = 0
    for i, end in enumerate(ends):
        if end > begin:
            pick = order[begin:end]
            left = v[pick].permute(1, 0, 2).reshape(16, -1)
            out[16 * i:16 * i + 16] = left @ slabs[of[pick]].reshape(-1, d.shape[1])
        begin = end
    return out[:out_len]


def _sampled(w, d, x):
    """The stored blocks of d x^T."""
    rows, cols = _coordinates(w)
    N = d.shape[1]
    left = _padded(d, -(-w["M"] // 16) * 16).view(-1, 16, N)
    right = _padded(x, -(-w["K"] // 16) * 16).view(-1, 16, N)
    out = torch.empty((cols.numel(), 16, 16), dtype=torch.float64, device=DEVICE)
    step = max(1, (1 << 25) // (16 * N))
    for b in range(0, cols.numel(), step):
        pick = slice(b, b + step)
        out[pick] = torch.bmm(left[rows[pick]], right[cols[pick]].transpose(1, 2).contiguous())
    return out.reshape(-1)
