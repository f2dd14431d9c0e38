"""The conversion to 8 bits and the 8-bit product where values and scales are small or large, against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import fp8_reference as ref
from easy_as_amd import ops
from test_gpu_fp8_ops import COLUMNS, E4M3, ROWS, SQUARES, TYPES, empty, rnd, scales

pytestmark = pytest.mark.gpu


def act(z: torch.Tensor, name: str) -> torch.Tensor:
    """The activations in 64 bits, in forms that keep their digits for every z."""
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * torch.erfc(-z * math.sqrt(0.5))
    return z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))


# where a block's gates lie: its scale and every code go by the activation there, down to values below 32 bits' normal ones
PLACES = [("silu", z) for z in (-3.0, -20.0, -60.0, -80.0, -88.5, -96.0)] + \
         [("gelu", z) for z in (-1.0, -5.0, -9.0, -12.5, -13.25)] + [("gelu_tanh", z) for z in (-1.0, -5.0, -8.0, -9.5, -10.25)]


@pytest.mark.parametrize("block", [ROWS, COLUMNS, SQUARES])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gated", [False, True])
def test_quantize_keeps_the_activations_digits(block, dtype, gated):
    """act(z) within 2^-20 of itself: 13 units of 2^-24 by the roundings of its steps, and one of the product with x.  What lies
    below 2^-126 is a multiple of 2^-149, rounded twice."""
    m, n = 131, 390
    for i, (name, place) in enumerate(PLACES):
        g = torch.Generator().manual_seed(i)
        z = (place - 0.25 * torch.rand(m, n, generator=g)).to(dtype)
        if place > -4:  # and the ordinary ones
            z = (2 * torch.randn(m, n, generator=g)).to(dtype)
        x = rnd(i, m, n, dtype=dtype)
        q, s = empty(m, n, dtype=E4M3), scales(m, n, block)
        if gated:
            ops.quantize(x, q, s, gate=z.cuda(), activation=name)
        else:
            ops.quantize(z.cuda(), q, s, activation=name)
        a, by = act(z.double(), name), x.cpu().double() if gated else torch.ones(())
        want = a * by
        ref.check_fp8(f"{name} at {place}", want, 2.0 ** -20 * want.abs() + 2.0 ** -148 * (1 + by.abs()), q, s, block)


@pytest.mark.parametrize("block", [ROWS, COLUMNS, SQUARES])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
def test_quantize_of_gates_beyond_the_exponentials_range(block, dtype, name):
    """Gates of every size beside each other, infinities and NaN among them: those are NaN, and the others as if they were not there."""
    m, n = 260, 390
    g = torch.Generator().manual_seed(7)
    z = 30 * torch.randn(m, n, generator=g)
    odd = torch.tensor([float("inf"), -float("inf"), float("nan"), 6e4, -6e4, 0.0, -0.0, 1e-7, -1e-7, -87.0, -90.0, -200.0, 13.0, -13.0])
    at = torch.randint(0, 8 * len(odd), (m, n), generator=g)
    z = torch.where(at < len(odd), odd[at.clamp(max=len(odd) - 1)], z).to(dtype)
    if dtype != torch.float16:
        z[5, 7], z[140, 200] = 3e38, -3e38
    x = rnd(8, m, n, dtype=dtype)
    q, s = empty(m, n, dtype=E4M3), scales(m, n, block)
    ops.quantize(x, q, s, gate=z.cuda(), activation=name)
    by = x.cpu().double()
    # what leaves the range of 32 bits is infinite in them: only act(3e38) x may be
    want = act(z.double(), name) * by
    want = torch.where(want.abs() < 2.0 ** 128, want, torch.full_like(want, float("inf")))
    slack = torch.where(want.isfinite(), 2.0 ** -20 * want.abs() + 2.0 ** -148 * (1 + by.abs()), torch.zeros_like(want))
    ref.check_fp8(name, want, slack, q, s, block)
