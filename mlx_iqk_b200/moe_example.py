"""A routed layer from logits to output: train its router, then serve it.

    python -m mlx_iqk_b200.moe_example [--experts 64] [--hidden 1024] [--inter 512] \\
        [--tokens 512] [--top-k 4] [--steps 30]

The experts are frozen MXFP4 matrices. The router is a linear map to one logit
per expert, tilted towards a few experts at the start. A training step chooses experts, weights and the balance loss in
one pass (``route_balanced``), takes each pair's output from the experts
(``MxSwitchGLU`` without scores), and sums them with the weights, through which
the gradient reaches the logits; the balance loss spreads the tokens. Serving runs the same layer
with the weights inside (``route``, ``MxSwitchGLU`` with scores): a prefill, and
its first tokens again as decode steps of one token.
"""

from __future__ import annotations

import argparse

import torch

from .mx import MxSwitchGLU
from .router import route, route_balanced


def make_layer(experts: int, hidden: int, inter: int, gen) -> MxSwitchGLU:
    """A layer of random experts, quantised on the device."""
    layer = MxSwitchGLU(experts, hidden, inter, device="cuda")
    for name, shape in (("gate", (experts, inter, hidden)), ("up", (experts, inter, hidden)),
                        ("down", (experts, hidden, inter))):
        fan = shape[-1]
        layer.load_weights(name, torch.randn(shape, generator=gen, device="cuda") / fan ** 0.5)
    return layer


def run(experts: int = 64, hidden: int = 1024, inter: int = 512, tokens: int = 512,
        top_k: int = 4, steps: int = 30, decode: int = 4) -> dict:
    """Trains the router for ``steps`` and serves; returns what each showed."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    layer = make_layer(experts, hidden, inter, gen)
    router = torch.randn((hidden, experts), generator=gen, device="cuda") / hidden ** 0.5
    router[:, : experts // 8] += 4.0 / hidden  # tokens have a mean: these draw most of them
    router.requires_grad_()
    target = torch.randn((hidden, hidden), generator=gen, device="cuda") * (0.1 / hidden ** 0.5)
    optimizer = torch.optim.Adam([router], lr=2e-3)
    seen = {"balance": [], "busiest": []}
    # packed sequences: ragged ends, and padding after the last
    offsets = torch.tensor([0, tokens // 3, tokens // 2, tokens], dtype=torch.int32, device="cuda")
    mask = torch.arange(tokens, device="cuda") < tokens - tokens // 16
    for _ in range(steps):
        x = (torch.randn((tokens, hidden), generator=gen, device="cuda") + 0.5).to(torch.bfloat16)
        logits = x.float() @ router
        indices, weights, balance, counts = route_balanced(logits, top_k, mask=mask,
                                                           offsets=offsets)
        pairs = layer(x, indices)  # [tokens, top_k, hidden], no gradient: the experts are frozen
        y = (weights[..., None] * pairs).sum(1)
        loss = ((y - x.float() @ target) * mask[:, None]).square().mean() + balance
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        seen["balance"].append(balance.detach())
        seen["busiest"].append(counts.sum(0).amax())
    with torch.no_grad():
        x = torch.randn((tokens, hidden), generator=gen, device="cuda").to(torch.bfloat16)
        indices, weights = route(x.float() @ router, top_k)
        seen["prefill"] = layer(x, indices, weights)
        rows = []
        for t in range(decode):
            indices, weights = route(x[t:t + 1].float() @ router, top_k)
            rows.append(layer(x[t:t + 1], indices, weights))
        seen["decode"] = torch.cat(rows)
    return seen


def main() -> None:
    ap = argparse.ArgumentParser()
    for name, value in (("experts", 64), ("hidden", 1024), ("inter", 512), ("tokens", 512),
                        ("top-k", 4), ("steps", 30)):
        ap.add_argument(f"--{name}", type=int, default=value)
    args = ap.parse_args()
    seen = run(args.experts, args.hidden, args.inter, args.tokens, args.top_k, args.steps)
    print(f"balance loss {float(seen['balance'][0]):.3f} -> {float(seen['balance'][-1]):.3f}, "
          f"busiest expert {int(seen['busiest'][0])} -> {int(seen['busiest'][-1])} pairs of "
          f"{args.tokens * args.top_k}")
    decode, prefill = seen["decode"], seen["prefill"][: len(seen["decode"])]
    print(f"decode against prefill: {float((decode - prefill).norm() / prefill.norm()):.2e}")


if __name__ == "__main__":
    main()
