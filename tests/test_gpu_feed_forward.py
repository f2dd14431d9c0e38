"""The feed-forward example: the operators together, against the same block in 64 bits."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

import ops_reference as ref

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

pytestmark = pytest.mark.gpu


def forward(x, p):
    mean = x.mean(1, keepdim=True)
    h = (x - mean) * ((x - mean).square().mean(1, keepdim=True) + 1e-5) ** -0.5 * p["norm_w"] + p["norm_b"]
    return x + ref.act(h @ p["gate"], "silu") * (h @ p["up"]) @ p["down"]


def parameters(block):
    return {k: v.detach().cpu().double().requires_grad_() for k, v in block.params.items()}


def test_block_gradients_match_64_bits():
    from feed_forward import FeedForward

    rows, width, hidden = 37, 72, 200
    block = FeedForward(width, hidden, rows)
    x, dy = (torch.randn(rows, width, generator=torch.Generator().manual_seed(s)).cuda() for s in (5, 6))
    y = block.forward(x).clone()
    dx = block.backward(x, dy)
    torch.cuda.synchronize()
    p = parameters(block)
    xd = x.cpu().double().requires_grad_()
    want = forward(xd, p)
    want.backward(dy.cpu().double())
    # fp32 through three products, a norm and back: sums of at most 272 terms of order 1, each off by 2^-23 of its
    # size at most, four deep; 64 times that leaves room for the largest element
    tol = 64 * 272 * 2.0 ** -23
    for got, exact in [(y, want.detach()), (dx, xd.grad)] + [(block.grads[k], p[k].grad) for k in p]:
        scale = exact.abs().max()
        assert (got.cpu().double() - exact).abs().max() <= tol * scale


def test_steps_follow_the_64_bit_ones():
    from feed_forward import FeedForward, fit

    rows, width, hidden, steps, lr = 128, 64, 160, 12, 0.5
    target, block = (FeedForward(width, hidden, rows, seed=s) for s in (1, 2))
    x = torch.randn(rows, width, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    p, xd = parameters(block), x.cpu().double()
    goal = forward(xd, parameters(target)).detach()
    losses = fit(block, x, target.forward(x).clone(), steps, lr)
    assert losses[-1] < 0.6 * losses[0]
    for got in losses:
        off = forward(xd, p) - goal
        want = off.square().mean().item()
        # sums of 200 terms are off by about 14 * 2^-24 each; a step of this length can double what it starts from,
        # so twelve leave 4096 times that
        assert abs(got - want) <= 4096 * 14 * 2.0 ** -24 * want
        for v in p.values():
            v.grad = None
        (off.square().sum() / rows).backward()
        with torch.no_grad():
            for v in p.values():
                v -= lr * v.grad


def test_a_token_matches_the_batch():
    from feed_forward import FeedForward

    block = FeedForward(96, 256, 40, dtype=torch.bfloat16)
    x = torch.randn(40, 96, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    whole = block.forward(x).float()
    row = block.token(x[7:8]).float()
    torch.cuda.synchronize()
    # both round h and a to bf16 from sums that differ in their last bits: a unit of bf16 each way
    assert (row - whole[7:8]).abs().max() <= 4 * 2.0 ** -8 * (1 + whole[7].abs().max())
