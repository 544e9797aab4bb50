"""Serving a block-sparse feed-forward layer in 8 bits, and orthogonalised
updates for training it, as timed cases.

A case is one call of an operator, on inputs made from a seed.  Activations are
features x tokens, weights are 16x16 blocks (block-CSR):

  tokens      q = round(127 x / max|x|) and max|x| / 127 of every token
  linear      y = act(A x + b) + residual, A in 8-bit integers with a scale for
              each row, x taken to 8-bit integers with a scale for each token
  gated       h = act(Ag x + bg) * (Au x + bu), likewise
  orthogonal  an update of a weight's stored blocks, orthogonalised: X = U / |U|,
              then `steps` times X <- aX + (bS + cSS) X with S = X X^T (of the
              transpose where that is smaller), at the stored blocks

`density` is the share of a weight's blocks that are stored, `empty` the share
of its block-rows that hold none.  Where `own` is false the operators are
computed in elementary operations in 32 bits on the unpacked weight, quotients
next to a border in 64.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
_VALUES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_STEPS = 5
_EPS = 1e-7


def listed():
    return [
        # one served token ahead of the down projection
        _tokens("tokens_one", "f16", 14336, 1),
        # a prompt's hidden activations
        _tokens("tokens_prompt", "bf16", 14336, 2048),
        # odd sizes, single precision
        _tokens("tokens_ragged", "f32", 4999, 301),
        # one token through a down projection with a quarter of its blocks,
        # added to the residual stream
        _matrix("linear_token", "linear", "f16", 4096, 14336, 1, 0.25, "none", residual=True),
        # an up projection whose blocks are all stored over a long prompt
        _matrix("linear_full", "linear", "f16", 14336, 4096, 2048, 1.0, "gelu", bias=True),
        # odd sizes everywhere, single precision, few blocks
        _matrix("linear_ragged", "linear", "f32", 5003, 4999, 31, 0.1, "silu", bias=True, residual=True),
        # one token through gate and up
        _matrix("gated_token", "gated", "bf16", 14336, 4096, 1, 0.25, "silu"),
        # a small layer and a batch of served tokens: launch and latency
        _matrix("gated_small", "gated", "f16", 1024, 1024, 64, 0.2, "gelu", bias=True, empty=0.1),
        # a long prompt through gate and up
        _matrix("gated_prompt", "gated", "bf16", 14336, 4096, 2048, 0.25, "silu"),
        # a training step's update of a small layer's gate
        _update("orthogonal_small", "bf16", 1792, 512, 0.25),
        # of a large layer's down projection
        _update("orthogonal_large", "bf16", 4096, 14336, 0.25),
        # odd sizes in single precision, some block-rows pruned away
        _update("orthogonal_ragged", "f32", 999, 2500, 0.5, empty=0.1),
    ]


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        # an orthogonalised update in single precision takes about three times
        # as many operations as one in 16 bits
        if case["kind"] == "orthogonal":
            ok = w["flops"] * (3 if case["values"] == "f32" else 1) <= 3.9e12
        else:
            ok = w["flops"] <= 2.5e11
        if ok and w["bytes"] <= 4e8:
            return case


def _draw_once(rng):
    kind = rng.choice(["tokens", "linear", "linear", "gated", "gated", "orthogonal", "orthogonal"])
    values = rng.choice(["f16", "bf16", "f32"])
    if kind == "tokens":
        N = 1 if rng.random() < 0.15 else _size(rng, 2, 16384)
        return _tokens(None, values, _size(rng, 64, 16384), N)
    density = math.exp(rng.uniform(math.log(0.02), 0.0))
    empty = rng.choice([0.0, 0.0, rng.uniform(0.02, 0.3)])
    if kind == "orthogonal":
        return _update(None, values, _size(rng, 128, 14336), _size(rng, 128, 14336), density, empty=empty)
    N = 1 if rng.random() < 0.15 else _size(rng, 2, 2048)
    if rng.random() < 0.4:
        N = max(8, N // 8 * 8)
    act = rng.choice(["silu", "gelu", "gelu_tanh", "relu"] + (["none"] if kind == "linear" else []))
    return _matrix(None, kind, values, _size(rng, 256, 14336), _size(rng, 256, 14336), N, density, act,
                   bias=rng.random() < 0.5, residual=kind == "linear" and rng.random() < 0.5, empty=empty)


def _size(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def _named(name, case):
    return {"name": name, **case} if name else case


def _tokens(name, values, K, N):
    return _named(name, dict(kind="tokens", values=values, K=K, N=N))


def _matrix(name, kind, values, M, K, N, density, act, bias=False, residual=False, empty=0.0):
    return _named(name, dict(kind=kind, values=values, M=M, K=K, N=N, density=density, act=act, bias=bias,
                             residual=residual, empty=empty))


def _update(name, values, M, K, density, empty=0.0):
    return _named(name, dict(kind="orthogonal", values=values, M=M, K=K, density=density, empty=empty))


# ---------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------

def _stored(case):
    """Stored blocks of one weight."""
    Mb, Kb = -(-case["M"] // 16), -(-case["K"] // 16)
    return max(1, round((Mb - round(Mb * case["empty"])) * Kb * case["density"]))


def work(case):
    s = 4 if case["values"] == "f32" else 2
    kind, K = case["kind"], case["K"]
    if kind == "tokens":
        N = case["N"]
        return {"bytes": float(K * N * s + K * N + 4 * N), "flops": 3.0 * K * N}
    M = case["M"]
    blocks = _stored(case)
    index = 4 * blocks + 4 * (-(-M // 16) + 1)
    if kind == "orthogonal":
        m, k = min(M, K), max(M, K)
        share = blocks / ((-(-M // 16)) * (-(-K // 16)))
        # the two products with symmetric results need half of them, the last
        # product the stored blocks
        flops = _STEPS * (m * m * k + m ** 3) + 2.0 * m * m * k * (_STEPS - 1 + share)
        return {"bytes": float(2 * blocks * 256 * s + index), "flops": flops}
    N, weights = case["N"], 2 if kind == "gated" else 1
    dense = (K * N + M * N + case["residual"] * M * N) * s
    each = blocks * 256 + index + 4 * M + case["bias"] * M * s
    return {"bytes": float(weights * each + dense), "flops": 512.0 * weights * blocks * N}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _positions(case, g):
    """Block coordinates of one weight and its row pointers: as many blocks for
    every seed, outside the block-rows that were pruned away."""
    Mb, Kb = -(-case["M"] // 16), -(-case["K"] // 16)
    full = Mb - round(Mb * case["empty"])
    kept = torch.randperm(Mb, generator=g, device=DEVICE)[:full].sort().values
    pick = torch.randperm(full * Kb, generator=g, device=DEVICE)[:_stored(case)]
    on = torch.zeros((Mb, Kb), dtype=torch.bool, device=DEVICE)
    on[kept[pick // Kb], pick % Kb] = True
    rows, cols = torch.nonzero(on, as_tuple=True)
    ptr = torch.zeros(Mb + 1, dtype=torch.int64, device=DEVICE)
    ptr[1:] = torch.cumsum(on.sum(1), 0)
    return rows, cols, ptr


def _clip_edges(case, rows, cols, v):
    """Block values with zeros past the weight's last row and column."""
    M, K = case["M"], case["K"]
    if M % 16:
        v[rows == -(-M // 16) - 1, M % 16:, :] = 0
    if K % 16:
        v[cols == -(-K // 16) - 1, :, K % 16:] = 0
    return v.reshape(-1).to(_VALUES[case["values"]])


def _weight(case, g):
    """A weight whose products with unit activations have about unit variance and
    whose rows differ in scale."""
    rows, cols, ptr = _positions(case, g)
    v = torch.randn((cols.numel(), 16, 16), generator=g, device=DEVICE)
    scale = torch.rand((-(-case["M"] // 16), 16, 1), generator=g, device=DEVICE) + 0.5
    v *= scale[rows] / math.sqrt(max(1.0, case["density"] * case["K"]))
    return {"M": case["M"], "K": case["K"], "rows": rows, "ptr": ptr.int(), "col": cols.int(),
            "v": _clip_edges(case, rows, cols, v)}


def _gradient(case, g):
    """An update as momentum holds it: a few dozen strong directions of falling
    weight, and noise."""
    M, K = case["M"], case["K"]
    rows, cols, ptr = _positions(case, g)
    rank = min(48, M, K)
    left = torch.randn((M, rank), generator=g, device=DEVICE)
    left /= torch.arange(1, rank + 1, device=DEVICE).float().sqrt()
    d = torch.zeros((-(-M // 16) * 16, -(-K // 16) * 16), device=DEVICE)
    d[:M, :K] = left @ torch.randn((rank, K), generator=g, device=DEVICE)
    d[:M, :K] += 0.3 * torch.randn((M, K), generator=g, device=DEVICE)
    v = d.view(d.shape[0] // 16, 16, d.shape[1] // 16, 16).permute(0, 2, 1, 3)[rows, cols] * 1e-3
    return {"M": M, "K": K, "rows": rows, "ptr": ptr.int(), "col": cols.int(), "v": _clip_edges(case, rows, cols, v)}


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    vt = _VALUES[case["values"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(vt)

    s = {"case": case}
    if case["kind"] == "orthogonal":
        s["w"] = [_gradient(case, g)]
        return s
    K, N = case["K"], case["N"]
    # tokens of different scale, with a few features that stand out
    x = torch.randn((K, N), generator=g, device=DEVICE)
    x *= torch.rand((1, N), generator=g, device=DEVICE) * 2 + 0.5
    x[torch.randint(K, (max(1, K // 1000),), generator=g, device=DEVICE)] *= 4
    s["x"] = x.to(vt)
    if case["kind"] == "tokens":
        return s
    M, weights = case["M"], 2 if case["kind"] == "gated" else 1
    s["w"] = [_weight(case, g) for _ in range(weights)]
    s["b"] = [normal(M, scale=0.1) if case["bias"] else None for _ in range(weights)]
    s["residual"] = normal(M, N) if case["residual"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if "w" not in s:
        return s
    if own:
        import xspmm_amd as X

        def weight(w):
            Mb, Kb = -(-w["M"] // 16), -(-w["K"] // 16)
            return X.SparseWeight(X.BCSRMatrix(Mb, Kb, 16, 16, w["M"], w["K"], w["ptr"], w["col"], w["v"]))

        s["W"] = [weight(w) for w in s["w"]]
        if case["kind"] != "orthogonal":
            # what serves the weights from now on
            s["W"] = [X.Int8Weight(W) for W in s["W"]]
    elif case["kind"] != "orthogonal":
        s["w8"] = [_weight8(w) for w in s["w"]]
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import xspmm_amd as X

    case = s["case"]
    kind = case["kind"]
    if kind == "tokens":
        t = X.quantize_tokens(s["x"])
        return t.values, t.scale
    if kind == "orthogonal":
        return X.orthogonalize(s["W"][0], s["w"][0]["v"], steps=_STEPS, coefficients=_COEFFICIENTS, eps=_EPS)
    W, b, act = s["W"], s["b"], case["act"]
    if kind == "linear":
        return X.int8_linear(W[0], s["x"], bias=b[0], activation=act, residual=s["residual"])
    return X.int8_gated(W[0], W[1], s["x"], bias_gate=b[0], bias_up=b[1], activation=act)


def _blocks_of_features(q):
    """Whole numbers K x N as 16 consecutive features of a token side by side, the
    last ones filled up with zeros: ceil(K / 16) x N x 16."""
    K, N = q.shape
    full = torch.zeros((-(-K // 16) * 16, N), dtype=torch.int8, device=DEVICE)
    full[:K] = q.to(torch.int8)
    return full.view(-1, 16, N).permute(0, 2, 1).contiguous()


def _round8(v, dim):
    """Whole numbers of at most 127 and the scale (32 bits) that they go by, along
    a dimension of v."""
    most = v.abs().amax(dim, keepdim=True)
    q = torch.round(v.double() * 127 / torch.where(most == 0, 1, most).double())
    return q, most.float() / 127


def _unpack(w, v):
    """Block values as an M x K matrix in 32 bits."""
    M, K = w["M"], w["K"]
    Mb, Kb = -(-M // 16), -(-K // 16)
    d = torch.zeros((Mb, Kb, 16, 16), device=DEVICE)
    d[w["rows"], w["col"].long()] = v.view(-1, 16, 16).float()
    return d.permute(0, 2, 1, 3).reshape(Mb * 16, Kb * 16)[:M, :K]


def _at_blocks(w, d):
    """The stored blocks of an M x K matrix, zero past its edges."""
    M, K = w["M"], w["K"]
    Mb, Kb = -(-M // 16), -(-K // 16)
    full = torch.zeros((Mb * 16, Kb * 16), dtype=d.dtype, device=DEVICE)
    full[:M, :K] = d
    return full.view(Mb, 16, Kb, 16).permute(0, 2, 1, 3)[w["rows"], w["col"].long()].reshape(-1)


def _weight8(w):
    """A weight's whole numbers (at the blocks, 8 bits) and its rows' scales."""
    q, scale = _round8(_unpack(w, w["v"]), 1)
    return {**w, "q": _at_blocks(w, q).to(torch.int8), "scale": scale}


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


def _run_plain(s):
    case = s["case"]
    kind, vt = case["kind"], _VALUES[case["values"]]
    if kind == "orthogonal":
        w = s["w"][0]
        a, b, c = _COEFFICIENTS
        x = _unpack(w, w["v"])
        wide = w["M"] <= w["K"]
        x = x if wide else x.t().contiguous()
        x = x / (x.double().square().sum().sqrt() + _EPS).float()
        for _ in range(_STEPS):
            S = x @ x.t()
            x = a * x + (b * S + c * (S @ S)) @ x
        return _at_blocks(w, x if wide else x.t()).to(vt)
    q, scale = _round8(s["x"], 0)
    if kind == "tokens":
        return _blocks_of_features(q), scale[0]
    q = q.float()
    z = [(_unpack(w, w["q"]) @ q) * scale * w["scale"] for w in s["w8"]]
    z = [v if b is None else v + b.float()[:, None] for v, b in zip(z, s["b"])]
    y = _act(case["act"], z[0])
    if kind == "gated":
        y = y * z[1]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(vt)


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "orthogonal":
        return _orthogonal64(s["w"][0])
    x = s["x"].double()
    peak = torch.linalg.vector_norm(x, math.inf, dim=0)
    q = torch.where(peak > 0, x * 127 / peak, 0).round()
    if kind == "tokens":
        K, N = q.shape
        whole = torch.nn.functional.pad(q, (0, 0, 0, -K % 16))
        return torch.stack([whole[i::16] for i in range(16)], 2).to(torch.int8), peak / 127
    sums = [_product64(w, q) * (peak / 127) for w in s["w"]]
    for i, b in enumerate(s["b"]):
        if b is not None:
            sums[i] = sums[i] + b.double().unsqueeze(1)
    y = _value64(case["act"], sums[0])
    if kind == "gated":
        y = y * sums[1]
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return y


def _value64(act, z):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z > 0, z, 0)
    if act == "silu":
        return z * torch.special.expit(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z * torch.special.expit(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))


def _slabs(w):
    """(block-row, its block-columns, its values 16 x 16n in 64 bits) of every
    block-row that holds blocks."""
    v = w["v"].double().view(-1, 16, 16)
    ends = w["ptr"].cpu().tolist()
    for i in range(len(ends) - 1):
        if ends[i + 1] > ends[i]:
            pick = slice(ends[i], ends[i + 1])
            yield i, w["col"][pick].long(), v[pick].permute(1, 0, 2).reshape(16, -1)


def _product64(w, q):
    """A q with A's rows rounded to whole numbers of at most 127, times their scales."""
    N = q.shape[1]
    blocks = torch.nn.functional.pad(q, (0, 0, 0, -w["K"] % 16)).view(-1, 16, N)
    out = torch.zeros((w["ptr"].numel() - 1, 16, N), dtype=torch.float64, device=DEVICE)
    for i, cols, v in _slabs(w):
        peak = torch.linalg.vector_norm(v, math.inf, dim=1, keepdim=True)
        whole = torch.where(peak > 0, v * 127 / peak, 0).round()
        out[i] = (whole @ blocks[cols].reshape(-1, N)) * (peak / 127)
    return out.reshape(-1, N)[:w["M"]]


def _orthogonal64(w):
    M, K = w["M"], w["K"]
    Mb, Kb = -(-M // 16), -(-K // 16)
    x = torch.zeros((Mb, 16, Kb, 16), dtype=torch.float64, device=DEVICE)
    for i, cols, v in _slabs(w):
        x[i, :, cols] = v.view(16, -1, 16)
    x = x.view(Mb * 16, Kb * 16)
    a, b, c = _COEFFICIENTS
    x = x / (torch.linalg.matrix_norm(x) + _EPS)
    for _ in range(_STEPS):
        # the polynomial one factor at a time, from the side with fewer rows
        if Mb <= Kb:
            S = x @ x.t()
            y = S @ x
            x = a * x + b * y + c * (S @ y)
        else:
            S = x.t() @ x
            y = x @ S
            x = a * x + b * y + c * (y @ S)
    x = x.view(Mb, 16, Kb, 16)
    return torch.cat([x[i, :, cols].permute(1, 0, 2).reshape(-1) for i, cols, _ in _slabs(w)])
