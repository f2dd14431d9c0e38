"""Scales of the 8-bit product that are large on one side and small on the other: only their product has to be within range."""

from __future__ import annotations

import pytest
import torch

import fp8_reference as ref
from easy_as_amd import ops
from test_gpu_fp8_ops import BF16, COLUMNS, E4M3, F32, ROWS, SQUARES, empty, rnd

pytestmark = pytest.mark.gpu


def matrix(seed: int, rows: int, cols: int, size: float, lying: str) -> torch.Tensor:
    """8-bit values of about `size`; `lying`: memory's rows are its rows or its columns."""
    q = rnd(seed, rows, cols, scale=size).to(E4M3)
    return q if lying == "rows" else q.t().contiguous().t()


def scale(seed: int, rows: int, cols: int) -> torch.Tensor:
    """Scales in [1, 2): times any power of two within the range they are as exact."""
    return 1 + torch.rand(rows, cols, generator=torch.Generator().manual_seed(seed)).cuda()


# w's scales times 2^up and x's times 2^-up, over values so large that a block's sum times w's scale would leave the range, or so
# small that it would lose its last digits
@pytest.mark.parametrize("up,size", [(120, 60.0), (-125, 0.03)])
@pytest.mark.parametrize("plan", ["", "tile64:1", "tile128:1", "tile128:2", "tile256:1"])
@pytest.mark.parametrize("m,k,n", [(1, 384, 70), (5, 200, 130), (40, 512, 96), (130, 400, 300)])
@pytest.mark.parametrize("lying", ["y", "dx", "dw"])
@pytest.mark.parametrize("block", [SQUARES, COLUMNS])
def test_scales_that_make_up_for_each_other(monkeypatch, up, size, plan, m, k, n, lying, block):
    if plan:
        monkeypatch.setenv("EAS_HIP_OPS_GEMM", plan)
    x = matrix(0, m, k, size, "columns" if lying == "dw" else "rows")
    w = matrix(1, k, n, size, "columns" if lying == "y" else "rows")
    xs, ws = scale(2, m, ref.blocks(k)), scale(3, ref.blocks(k), ref.blocks(n) if block == SQUARES else n)
    for dtype in (BF16, F32):
        y, same = empty(m, n, dtype=dtype), empty(m, n, dtype=dtype)
        ops.linear_fp8(x, xs, w, ws, same)
        ops.linear_fp8(x, xs * 2.0 ** -up, w, ws * 2.0 ** up, y)
        ref.check_linear_fp8(ref.values(x, xs, ROWS), ref.values(w, ws, block), same)
        assert torch.equal(y, same)  # each product of two scales is the same number
