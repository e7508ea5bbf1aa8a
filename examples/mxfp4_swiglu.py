"""Train a stack of gated feed-forward blocks on MXFP4 matrices, then serve it from
4-bit weights.

    python examples/mxfp4_swiglu.py [--steps 60]

Training: ``Linear`` projections with float32 masters under
``PrecisionConfig.mxfp4_mixed()``; ``swiglu_mlp`` runs both input projections, the
activation and the product in one kernel, and every product of the backward is over
4-bit operands. Serving: each projection's weight encoded once (``MXFP4Linear``), a
single token through the one-launch kernels.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), os.pardir))

import representax_amd as rx  # noqa: E402


class Block(torch.nn.Module):
    """``x + down(silu(gate(n)) * up(n))``, n = x over its root mean square."""

    def __init__(self, hidden: int, ffn: int, key: int, device: str) -> None:
        super().__init__()
        make = lambda i, k, n: rx.Linear.init(k, n, key=8 * key + i, scale=k ** -0.5,  # noqa: E731
                                              device=device)
        self.gate, self.up, self.down = make(0, hidden, ffn), make(1, hidden, ffn), make(2, ffn, hidden)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        n = x.float()
        n = (n * torch.rsqrt(n.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)
        return x + rx.swiglu_mlp(n, self.gate, self.up, self.down)


def serving_copy(model: torch.nn.Module) -> torch.nn.Module:
    """The same blocks over kept 4-bit weights."""

    import copy

    served = copy.deepcopy(model)
    for block in served:
        for name in ("gate", "up", "down"):
            setattr(block, name, rx.MXFP4Linear.from_linear(getattr(block, name)))
    return served


def main(steps: int = 60, tokens: int = 2048, hidden: int = 512, ffn: int = 1536, layers: int = 2,
         device: str = "cuda") -> dict:
    torch.manual_seed(0)
    policy = rx.resolve_precision_policy(rx.PrecisionConfig.mxfp4_mixed())
    model = torch.nn.Sequential(*[Block(hidden, ffn, i, device) for i in range(layers)])
    teacher = torch.nn.Sequential(*[Block(hidden, ffn, 100 + i, device) for i in range(layers)])
    optimizer = torch.optim.AdamW(model.parameters(), lr=2e-3)
    losses = []
    for step in range(steps):
        x = torch.randn((tokens, hidden), device=device).to(torch.bfloat16)
        with torch.no_grad():
            target = teacher(x.float()) - x.float()  # float32: plain products
        with rx.precision_context(policy):
            loss = ((model(x) - x).float() - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
        if step % 10 == 0 or step + 1 == steps:
            print(f"step {step:4d}  loss {losses[-1]:.4f}", flush=True)

    x = torch.randn((64, hidden), device=device).to(torch.bfloat16)
    with rx.precision_context(policy), torch.no_grad():
        served = serving_copy(model)
        batch = model(x)
        off = max(float((served(x[i:i + 1]) - batch[i:i + 1]).float().norm()
                        / batch[i:i + 1].float().norm()) for i in range(8))
    dense = sum(p.numel() * 2 for p in model.parameters())
    kept = sum(b.numel() for b in served.buffers())
    print(f"served token by token from {kept / 1e6:.2f} MB of weights (bf16: {dense / 1e6:.2f}): "
          f"within {off:.1e} of the training forward")
    return {"losses": losses, "off": off, "kept_bytes": kept, "dense_bytes": dense}


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=60)
    main(parser.parse_args().steps)
