"""The feed-forward half of a transformer layer on the operators of ``easy_as_amd.ops``:

    y = x + down(act(gate(h)) * up(h)),  h = layer_norm(x)

forward and backward on buffers made once, plain SGD with an ``@eas.kernel`` for the update, and the
block on a single token as a decoding step runs it.  ``python examples/feed_forward.py`` fits a small
block to another one's outputs and times both uses.
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import eas
from eas import mk, ops


@eas.kernel
def sgd_kernel(w, g, rate, N, BLOCK: eas.constexpr):
    """w += rate g"""
    offs = mk.program_id(0) * BLOCK + mk.arange(0, BLOCK)
    mask = offs < N
    mk.store(w, offs, mk.load(w, offs, mask) + rate * mk.load(g, offs, mask), mask)


@eas.kernel
def add_kernel(a, b, c, N, BLOCK: eas.constexpr):
    offs = mk.program_id(0) * BLOCK + mk.arange(0, BLOCK)
    mask = offs < N
    mk.store(c, offs, mk.load(a, offs, mask) + mk.load(b, offs, mask), mask)


class FeedForward:
    """The block's parameters, their gradients and the buffers of one batch size.  All calls are asynchronous on
    torch's current stream, so a step can be captured in a graph."""

    def __init__(self, width: int, hidden: int, rows: int, *, dtype: torch.dtype = torch.float32,
                 activation: str = "silu", seed: int = 0) -> None:
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weights(k: int, n: int) -> torch.Tensor:
            return torch.randn(k, n, generator=g, device="cuda") * k ** -0.5

        def buffer(*shape: int, of: torch.dtype = dtype) -> torch.Tensor:
            return torch.empty(*shape, device="cuda", dtype=of)

        self.activation = activation
        # the parameters and their gradients in 32 bits; the products read weights in their own type
        self.params = {"norm_w": torch.ones(width, device="cuda"), "norm_b": torch.zeros(width, device="cuda"),
                       "gate": weights(width, hidden), "up": weights(width, hidden), "down": weights(hidden, width)}
        self.grads = {k: torch.empty_like(v) for k, v in self.params.items()}
        self.read = {k: v if k.startswith("norm") else v.to(dtype) for k, v in self.params.items()}
        # what the forward pass leaves for the backward one, and the backward pass's own
        self.h, self.y, self.dh, self.dx = (buffer(rows, width) for _ in range(4))
        self.a, self.gate, self.up, self.da = (buffer(rows, hidden) for _ in range(4))
        self.mean, self.rstd = (buffer(rows, of=torch.float32) for _ in range(2))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        p, rows = self.read, x.shape[0]
        h, a, y = self.h[:rows], self.a[:rows], self.y[:rows]
        ops.layer_norm(x, p["norm_w"], p["norm_b"], h, self.mean[:rows], self.rstd[:rows], _sync=False)
        ops.gated_linear(h, p["gate"], p["up"], a, activation=self.activation, gate=self.gate[:rows],
                         up=self.up[:rows], _sync=False)
        ops.linear(a, p["down"], y, residual=x, _sync=False)
        return y

    def backward(self, x: torch.Tensor, dy: torch.Tensor) -> torch.Tensor:
        """The parameters' gradients into ``grads``, x's returned; after ``forward(x)``."""
        p, g, rows = self.read, self.grads, x.shape[0]
        h, a, da, dh, dx = self.h[:rows], self.a[:rows], self.da[:rows], self.dh[:rows], self.dx[:rows]
        ops.linear_backward(dy, a, p["down"], dx=da, dw=g["down"], _sync=False)
        ops.gated_linear_backward(da, h, p["gate"], p["up"], self.gate[:rows], self.up[:rows], dx=dh,
                                  dw_gate=g["gate"], dw_up=g["up"], activation=self.activation, _sync=False)
        ops.layer_norm_backward(dh, x, p["norm_w"], self.mean[:rows], self.rstd[:rows], dx, g["norm_w"], g["norm_b"],
                                _sync=False)
        add_kernel(dx, dy, dx, dx.numel(), BLOCK=256, _sync=False)  # the residual's
        return dx

    def step(self, lr: float) -> None:
        for name, w in self.params.items():
            sgd_kernel(w, self.grads[name], -float(lr), w.numel(), BLOCK=256, _sync=False)
            if self.read[name] is not w:
                self.read[name].copy_(w)

    def token(self, x: torch.Tensor) -> torch.Tensor:
        """One row or a few of a decoding step: nothing is kept for a backward pass."""
        p, rows = self.read, x.shape[0]
        h, a, y = self.h[:rows], self.a[:rows], self.y[:rows]
        ops.layer_norm(x, p["norm_w"], p["norm_b"], h, _sync=False)
        ops.gated_linear(h, p["gate"], p["up"], a, activation=self.activation, _sync=False)
        ops.linear(a, p["down"], y, residual=x, _sync=False)
        return y


def fit(block: FeedForward, x: torch.Tensor, goal: torch.Tensor, steps: int, lr: float = 0.1) -> list[float]:
    """Mean squared distance to ``goal`` before each step of gradient descent on it."""
    losses = []
    for _ in range(steps):
        off = block.forward(x) - goal
        losses.append(off.float().square().mean().item())
        block.backward(x, off * (2.0 / x.shape[0]))
        block.step(lr)
    return losses


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--width", type=int, default=1024)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--rows", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=20)
    args = ap.parse_args()
    target, block = (FeedForward(args.width, args.hidden, args.rows, dtype=torch.bfloat16, seed=s) for s in (1, 2))
    x = torch.randn(args.rows, args.width, device="cuda").to(torch.bfloat16)
    dy = torch.randn_like(x)
    losses = fit(block, x, target.forward(x), args.steps)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {len(losses)} steps")

    def timed(call, turns: int = 50) -> float:
        for _ in range(3):
            call()
        torch.cuda.synchronize()
        began = time.perf_counter()
        for _ in range(turns):
            call()
        torch.cuda.synchronize()
        return (time.perf_counter() - began) / turns * 1e6

    def train() -> None:
        block.forward(x)
        block.backward(x, dy)
        block.step(0.0)

    print(f"training step, {args.rows} rows, bf16: {timed(train):.1f} us; one token: {timed(lambda: block.token(x[:1])):.1f} us")


if __name__ == "__main__":
    main()
