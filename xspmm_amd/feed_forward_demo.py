"""A feed-forward layer pruned to blocks, trained back and served.

    python -m xspmm_amd.feed_forward_demo [--features 512] [--hidden 1792]
        [--tokens 1024] [--density 0.25] [--steps 60] [--dtype bf16]
        [--orthogonal]

A dense layer with random weights is the teacher.  Its three weights are pruned
to the blocks of the largest norms, trained for some steps to give the teacher's
outputs again, and the trained layer then serves the last tokens one by one, as it
is and with its weights in 8 bits.  With --orthogonal the weights' updates are
orthogonalised (``OrthogonalMomentum``).
Prints the error before and after the training, the time of a training step
(forward, backward, update) and of a served token, how far the tokens served one by
one are from the same tokens in one batch, and the last two again in 8 bits.
"""
from __future__ import annotations

import argparse
import json
import time

import torch

from .feed_forward import FeedForward, prune_blocks
from .int8 import Int8FeedForward
from .orthogonal import OrthogonalMomentum

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def run(features=512, hidden=1792, tokens=1024, density=0.25, steps=60, dtype="bf16", seed=0, device="cuda:0",
        orthogonal=False):
    g = torch.Generator(device=device).manual_seed(seed)
    dt = DTYPES[dtype]
    # weights whose blocks differ in size, as trained ones' do
    scale = lambda m, k: torch.rand((-(-m // 16), -(-k // 16)), generator=g, device=device).square().repeat_interleave(
        16, 0).repeat_interleave(16, 1)[:m, :k]
    dense = lambda m, k: torch.randn((m, k), generator=g, device=device) * scale(m, k) * (2 / k ** 0.5)
    gate, up, down = dense(hidden, features), dense(hidden, features), dense(features, hidden)
    x = torch.randn((features, tokens), generator=g, device=device)
    n = (x - x.mean(0)) / torch.sqrt(x.var(0, correction=0) + 1e-5)
    a = gate @ n
    want = x + down @ (a / (1 + torch.exp(-a)) * (up @ n))
    layer = FeedForward(*(prune_blocks(w.to(dt), density) for w in (gate, up, down)))
    # master copies in fp32: an update is small against a 16-bit weight
    optimiser = OrthogonalMomentum(layer, lr=2e-3) if orthogonal else None
    params = [layer.norm_weight, layer.norm_bias] if orthogonal else list(layer.parameters())
    master = [p.detach().float() for p in params]
    moments = [torch.zeros_like(p) for p in master]
    x = x.to(dt)
    error = lambda y: float((y.float() - want).norm() / (want - x.float()).norm())
    with torch.no_grad():
        before = error(layer(x))
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(steps):
        y = layer(x)
        y.backward((2 * (y.detach().float() - want)).to(dt))
        for p, m, v in zip(params, master, moments):
            grad = p.grad.float()
            v.mul_(0.9).add_(grad.square(), alpha=0.1)
            m.sub_(2e-3 * grad / (v.sqrt() + 1e-6))
            p.data.copy_(m)
            p.grad = None
        if optimiser is not None:
            optimiser.step()
            optimiser.zero_grad()
    torch.cuda.synchronize()
    step_ms = (time.perf_counter() - start) / max(steps, 1) * 1e3
    with torch.no_grad():
        batch = layer(x)
        after = error(batch)
        last = [x[:, i:i + 1].contiguous() for i in range(tokens - min(tokens, 32), tokens)]

        def serve(f, batch):
            """us of a token served alone, its distance from the same token of a batch."""
            f(last[0])
            torch.cuda.synchronize()
            start = time.perf_counter()
            served = [f(t) for t in last]
            torch.cuda.synchronize()
            us = (time.perf_counter() - start) / len(last) * 1e6
            apart = (torch.cat(served, 1) - batch[:, -len(last):]).float().norm() / batch[:, -len(last):].float().norm()
            return us, float(apart)

        token_us, apart = serve(layer, batch)
        token8_us, apart8 = serve(Int8FeedForward(layer), batch)
    return {"error_before": before, "error_after": after, "step_ms": step_ms, "token_us": token_us,
            "served_vs_batch": apart, "token_int8_us": token8_us, "served_int8_vs_batch": apart8, "blocks": [int(w.num_blocks) for w in layer._weights]}


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--features", type=int, default=512)
    ap.add_argument("--hidden", type=int, default=1792)
    ap.add_argument("--tokens", type=int, default=1024)
    ap.add_argument("--density", type=float, default=0.25)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--orthogonal", action="store_true")
    ap.add_argument("--dtype", choices=list(DTYPES), default="bf16")
    print(json.dumps(run(**vars(ap.parse_args()))))


if __name__ == "__main__":
    main()
