"""The feed-forward operators on the GPU against their definitions in 64 bits."""

from __future__ import annotations

import itertools

import numpy as np
import pytest
import torch

import ops_reference as ref
from easy_as_amd import ops

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TYPES = [F16, BF16, F32]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def rnd(seed: int, *shape: int, dtype=F32, scale: float = 1.0, mean: float = 0.0) -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + mean).to(dtype).cuda()


def spaced(t: torch.Tensor, ld: int, offset: int = 0, fill: float = float("nan")) -> torch.Tensor:
    """t's values with a row stride of `ld` elements from `offset` on, `fill` between the rows."""
    rows, cols = t.shape
    whole = torch.full((rows * ld + offset + cols,), fill, dtype=t.dtype, device=t.device)
    view = whole.as_strided((rows, cols), (ld, 1), offset)
    view.copy_(t)
    return view


def empty(*shape: int, dtype) -> torch.Tensor:
    return torch.full(shape, float("nan"), dtype=dtype, device="cuda")


# -- layer norm -----------------------------------------------------------------

# one vector, the edges of each register kernel, and rows beyond them
NORM_N = [1, 7, 8, 9, 511, 512, 513, 1024, 1031, 2048, 2049, 4096, 4099, 8192, 8193, 16384, 16385, 40003]


@pytest.mark.parametrize("n", NORM_N)
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_row_lengths(n, dtype):
    m = 5
    x = rnd(n, m, n, dtype=dtype, scale=2.0, mean=0.7)
    w, b = rnd(n + 1, n, dtype=dtype, mean=1.0), rnd(n + 2, n, dtype=dtype)
    y, mean, rstd = empty(m, n, dtype=dtype), empty(m, dtype=F32), empty(m, dtype=F32)
    ops.layer_norm(x, w, b, y, mean, rstd)
    ref.check_norm(x, w, b, 1e-5, y, mean, rstd)
    dy = rnd(n + 3, m, n, dtype=dtype)
    dx, dw, db = empty(m, n, dtype=dtype), empty(n, dtype=dtype), empty(n, dtype=dtype)
    ops.layer_norm_backward(dy, x, w, mean, rstd, dx, dw, db)
    ref.check_norm_backward(dy, x, w, mean, rstd, dx, dw, db)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 63, 1031, 2500])
@pytest.mark.parametrize("n", [64, 257, 3000])
def test_norm_row_counts(m, n):
    x = rnd(m, m, n, dtype=BF16, mean=-1.0)
    w, b = rnd(1, n, mean=1.0), rnd(2, n)  # f32 parameters of a bf16 row
    y, mean, rstd = empty(m, n, dtype=BF16), empty(m, dtype=F32), empty(m, dtype=F32)
    ops.layer_norm(x, w, b, y, mean, rstd, eps=1e-3)
    ref.check_norm(x, w, b, 1e-3, y, mean, rstd)
    dy = rnd(m + 1, m, n, dtype=BF16)
    dx, dw, db = empty(m, n, dtype=BF16), empty(n, dtype=F32), empty(n, dtype=F32)
    ops.layer_norm_backward(dy, x, w, mean, rstd, dx, dw, db)
    ref.check_norm_backward(dy, x, w, mean, rstd, dx, dw, db)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ld,offset", [(261, 1), (264, 8), (300, 3)])
def test_norm_strides(dtype, ld, offset):
    m, n = 17, 259
    x = spaced(rnd(0, m, n, dtype=dtype), ld, offset)
    dy = spaced(rnd(1, m, n, dtype=dtype), ld + 3, offset)
    y, dx = spaced(empty(m, n, dtype=dtype), ld + 1, offset, 7.0), spaced(empty(m, n, dtype=dtype), ld + 2, offset, 7.0)
    mean, rstd = empty(m, dtype=F32), empty(m, dtype=F32)
    ops.layer_norm(x, None, None, y, mean, rstd)
    ref.check_norm(x, None, None, 1e-5, y, mean, rstd)
    ops.layer_norm_backward(dy, x, None, mean, rstd, dx)
    ref.check_norm_backward(dy, x, None, mean, rstd, dx)
    for t, s in ((y, ld + 1), (dx, ld + 2)):  # nothing written between the rows
        gap = t.as_strided((m - 1, s - n), (s, 1), offset + n)
        assert bool((gap == 7.0).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("wdtype", [None, F32])
@pytest.mark.parametrize("n,ld,offset", [(2, 6, 2), (262, 262, 0), (262, 266, 6), (2054, 2060, 4), (5000, 5002, 2), (9002, 9010, 0)])
def test_norm_even_rows(dtype, wdtype, n, ld, offset):
    """16-bit rows of whole 4 bytes that end inside a vector of 8."""
    m = 19
    x, dy = spaced(rnd(0, m, n, dtype=dtype), ld, offset), spaced(rnd(1, m, n, dtype=dtype), ld + 2, offset)
    w, b = rnd(2, n, dtype=wdtype or dtype), rnd(3, n, dtype=wdtype or dtype)
    y, dx = spaced(empty(m, n, dtype=dtype), ld + 2, offset, 7.0), spaced(empty(m, n, dtype=dtype), ld + 4, offset, 7.0)
    mean, rstd = empty(m, dtype=F32), empty(m, dtype=F32)
    ops.layer_norm(x, w, b, y, mean, rstd)
    ref.check_norm(x, w, b, 1e-5, y, mean, rstd)
    dw, db = empty(n, dtype=wdtype or dtype), empty(n, dtype=wdtype or dtype)
    ops.layer_norm_backward(dy, x, w, mean, rstd, dx, dw, db)
    ref.check_norm_backward(dy, x, w, mean, rstd, dx, dw, db)
    for t, s in ((y, ld + 2), (dx, ld + 4)):  # nothing written between the rows
        assert bool((t.as_strided((m - 1, s - n), (s, 1), offset + n) == 7.0).all())


@pytest.mark.parametrize("parts", list(itertools.product([False, True], repeat=3)))
def test_norm_backward_parts(parts):
    for n in (100, 20000):
        x, dy, w = rnd(0, 33, n), rnd(1, 33, n), rnd(2, n)
        y, mean, rstd = empty(33, n, dtype=F32), empty(33, dtype=F32), empty(33, dtype=F32)
        ops.layer_norm(x, w, None, y, mean, rstd)
        dx = empty(33, n, dtype=F32) if parts[0] else None
        dw, db = (empty(n, dtype=F32) if p else None for p in parts[1:])
        ops.layer_norm_backward(dy, x, w, mean, rstd, dx, dw, db)
        ref.check_norm_backward(dy, x, w, mean, rstd, dx, dw, db)


def test_norm_in_place():
    for n in (384, 17000):
        x, w, b = rnd(0, 9, n), rnd(1, n), rnd(2, n)
        y, mean, rstd = x.clone(), empty(9, dtype=F32), empty(9, dtype=F32)
        ops.layer_norm(y, w, b, y, mean, rstd)
        ref.check_norm(x, w, b, 1e-5, y, mean, rstd)
        dy = rnd(3, 9, n)
        for over in (dy.clone(), x.clone()):
            a, c = (over, x) if torch.equal(over, dy) else (dy, over)
            dw, db = empty(n, dtype=F32), empty(n, dtype=F32)
            ops.layer_norm_backward(a, c, w, mean, rstd, over, dw, db)
            ref.check_norm_backward(dy, x, w, mean, rstd, over, dw, db)


def test_norm_constant_infinite_and_nan_rows():
    x = rnd(0, 6, 1000)
    x[1] = 3.0            # no variance: rstd is eps ** -0.5
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    x[4] = 1e4
    x[4, ::2] = -1e4
    y, mean, rstd = empty(6, 1000, dtype=F32), empty(6, dtype=F32), empty(6, dtype=F32)
    ops.layer_norm(x, None, None, y, mean, rstd)
    fine = [0, 1, 4, 5]
    ref.check_norm(x[fine], None, None, 1e-5, y[fine], mean[fine], rstd[fine])
    assert bool(y[2:4].isnan().all()) and mean[2].item() == float("inf") and bool(mean[3].isnan())


def test_norm_large_offset_keeps_the_variance():
    # rows of mean 1000 and deviation 1: a sum of squares about 0 would lose the variance's digits
    x = rnd(0, 8, 4096, mean=1000.0)
    y, mean, rstd = empty(8, 4096, dtype=F32), empty(8, dtype=F32), empty(8, dtype=F32)
    ops.layer_norm(x, None, None, y, mean, rstd)
    ref.check_norm(x, None, None, 1e-5, y, mean, rstd)


def test_norm_no_rows():
    w = rnd(0, 64)
    x, mean = empty(0, 64, dtype=F32), empty(0, dtype=F32)
    ops.layer_norm(x, w, w, empty(0, 64, dtype=F32), mean, mean.clone())
    dw, db = empty(64, dtype=F32), empty(64, dtype=F32)
    ops.layer_norm_backward(x, x, w, mean, mean, empty(0, 64, dtype=F32), dw, db)
    assert bool((dw == 0).all()) and bool((db == 0).all())


# -- linear ------------------------------------------------------------------------

# few rows, each few-row kernel's edges, tiles' edges; k and n around the stages and the chunks
SHAPES = [(1, 64, 64), (1, 1, 1), (3, 129, 70), (16, 256, 200), (17, 40, 333), (33, 520, 64), (64, 64, 65), (65, 63, 127),
          (100, 7, 9), (128, 300, 256), (257, 33, 259), (300, 512, 515), (513, 1031, 64), (2, 4100, 96)]


def layer(seed, k, n, dtype, trans):
    w = rnd(seed, n, k, dtype=dtype, scale=k ** -0.5).t() if trans else rnd(seed, k, n, dtype=dtype, scale=k ** -0.5)
    return w


def like(w, dtype):
    return torch.full_like(w, float("nan"), dtype=dtype)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("trans", [False, True])
def test_linear_shapes(shape, dtype, trans):
    m, k, n = shape
    x, w, b, r = rnd(0, m, k, dtype=dtype), layer(1, k, n, dtype, trans), rnd(2, n, dtype=dtype), rnd(3, m, n, dtype=dtype)
    act = ACTS[(m + n) % 5]
    y, pre = empty(m, n, dtype=dtype), empty(m, n, dtype=dtype)
    ops.linear(x, w, y, bias=b, residual=r, activation=act, pre=pre)
    ref.check_linear(x, w, y, b, r, act, pre)
    dy, dx, dw, db = rnd(4, m, n, dtype=dtype), empty(m, k, dtype=dtype), like(w, dtype), empty(n, dtype=dtype)
    ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db, activation=act, pre=pre)
    ref.check_linear_backward(dy, x, w, dx, dw, db, act, pre)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [5, 80])
def test_linear_activations(act, dtype, m):
    k, n = 96, 136
    x, w = rnd(0, m, k, dtype=dtype, scale=3.0), layer(1, k, n, dtype, False)
    y, pre = empty(m, n, dtype=dtype), empty(m, n, dtype=dtype)
    ops.linear(x, w, y, activation=act, pre=pre)
    ref.check_linear(x, w, y, activation=act, pre=pre)
    dy, dx, dw, db = rnd(4, m, n, dtype=dtype), empty(m, k, dtype=dtype), like(w, dtype), empty(n, dtype=dtype)
    ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db, activation=act, pre=pre)
    ref.check_linear_backward(dy, x, w, dx, dw, db, act, pre)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m", [9, 140])
def test_linear_f32_results_of_16_bit_operands(dtype, m):
    k, n = 200, 150
    x, w, r = rnd(0, m, k, dtype=dtype), layer(1, k, n, dtype, False), rnd(3, m, n)
    y, pre = empty(m, n, dtype=F32), empty(m, n, dtype=F32)
    ops.linear(x, w, y, residual=r, activation="silu", pre=pre)
    ref.check_linear(x, w, y, None, r, "silu", pre)
    dy, dw, db = rnd(4, m, n, dtype=dtype), like(w, F32), empty(n, dtype=F32)
    ops.linear_backward(dy, x, None, dw=dw, dbias=db)
    ref.check_linear_backward(dy, x, w, None, dw, db)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [7, 150])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("pad,offset", [(8, 0), (16, 8), (1, 0), (3, 1), (0, 5)])
def test_linear_strides_and_alignments(dtype, m, trans, pad, offset):
    k, n = 104, 144  # NaN between the rows: what is read past a row's end must not reach a sum
    x = spaced(rnd(0, m, k, dtype=dtype), k + pad, offset)
    w = spaced(rnd(1, n, k, dtype=dtype) if trans else rnd(1, k, n, dtype=dtype), (k if trans else n) + pad, offset)
    w = w.t() if trans else w
    r, y = spaced(rnd(2, m, n, dtype=dtype), n + pad, offset), spaced(empty(m, n, dtype=dtype), n + pad, offset, 7.0)
    pre = spaced(empty(m, n, dtype=dtype), n + pad + 2, offset, 7.0)
    ops.linear(x, w, y, residual=r, activation="gelu", pre=pre)
    ref.check_linear(x, w, y, None, r, "gelu", pre)
    dy = spaced(rnd(3, m, n, dtype=dtype), n + pad, offset)
    dx = spaced(empty(m, k, dtype=dtype), k + pad, offset, 7.0)
    dw = spaced(empty(n, k, dtype=dtype) if trans else empty(k, n, dtype=dtype), (k if trans else n) + pad, offset, 7.0)
    dw = dw.t() if trans else dw
    for act in ("gelu", "none"):
        ops.linear_backward(dy, x, w, dx=dx, dw=dw, activation=act, pre=pre)
        ref.check_linear_backward(dy, x, w, dx, dw, None, act, pre)
    if pad:
        for t in (y, dx):
            rows, cols = t.shape
            assert bool((t.as_strided((rows - 1, pad), (cols + pad, 1), offset + cols) == 7.0).all())


@pytest.mark.parametrize("m,k,n", [(20, 100, 52), (200, 52, 100)])
def test_linear_k_not_a_multiple_of_8_beside_nan(m, k, n):
    # rows aligned to 16 bytes whose length is not: the last chunk of a row holds what lies after it
    for dtype in TYPES:
        kp, np_ = (k + 15) // 8 * 8, (n + 15) // 8 * 8
        x, w = spaced(rnd(0, m, k, dtype=dtype), kp), spaced(rnd(1, n, k, dtype=dtype), kp).t()
        y = empty(m, n, dtype=dtype)
        ops.linear(x, w, y)
        ref.check_linear(x, w, y)
        w2 = spaced(rnd(1, k, n, dtype=dtype), np_)
        ops.linear(x, w2, y)
        ref.check_linear(x, w2, y)


@pytest.mark.parametrize("parts", list(itertools.product([False, True], repeat=3)))
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_backward_parts(parts, act):
    m, k, n = 70, 90, 110
    x, w, dy, pre = rnd(0, m, k, dtype=BF16), layer(1, k, n, BF16, False), rnd(2, m, n, dtype=BF16), rnd(3, m, n, dtype=BF16)
    dx = empty(m, k, dtype=BF16) if parts[0] else None
    dw = like(w, BF16) if parts[1] else None
    db = empty(n, dtype=BF16) if parts[2] else None
    ops.linear_backward(dy, x if parts[1] else None, w if parts[0] else None, dx=dx, dw=dw, dbias=db, activation=act,
                        pre=pre if act != "none" else None)
    ref.check_linear_backward(dy, x, w, dx, dw, db, act, pre)


@pytest.mark.parametrize("m,k,n", [(8, 0, 24), (300, 0, 24), (0, 16, 24), (8, 16, 0)])
def test_linear_empty(m, k, n):
    for dtype in TYPES:
        x, w, b, r = rnd(0, m, k, dtype=dtype), rnd(1, k, n, dtype=dtype), rnd(2, n, dtype=dtype), rnd(3, m, n, dtype=dtype)
        y = empty(m, n, dtype=dtype)
        ops.linear(x, w, y, bias=b, residual=r, activation="silu")
        ref.check_linear(x, w, y, b, r, "silu")
        dy, dx, dw, db = rnd(4, m, n, dtype=dtype), empty(m, k, dtype=dtype), empty(k, n, dtype=dtype), empty(n, dtype=dtype)
        ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db)
        ref.check_linear_backward(dy, x, w, dx, dw, db)


def test_linear_in_place_residual_and_column_halves():
    x, w = rnd(0, 50, 64, dtype=F16), rnd(1, 64, 48, dtype=F16)
    r = rnd(2, 50, 48, dtype=F16)
    y = r.clone()
    ops.linear(x, w, y, residual=y)
    ref.check_linear(x, w, y, None, r)
    both = empty(50, 96, dtype=F16)  # y and pre side by side in one array
    ops.linear(x, w, both[:, :48], activation="relu", pre=both[:, 48:])
    ref.check_linear(x, w, both[:, :48], activation="relu", pre=both[:, 48:])


def test_linear_leading_axes():
    x, w = rnd(0, 3, 5, 32, dtype=F16), rnd(1, 32, 24, dtype=F16)
    y = empty(3, 5, 24, dtype=F16)
    ops.linear(x, w, y)
    ref.check_linear(x.view(15, 32), w, y.view(15, 24))
    v = rnd(2, 32, dtype=F16)
    out = empty(24, dtype=F16)
    ops.linear(v, w, out)
    ref.check_linear(v[None], w, out[None])


def test_linear_infinity_and_nan_stay_in_their_rows_and_columns():
    for m in (10, 200):
        x, w = rnd(0, m, 72, dtype=BF16), rnd(1, 72, 80, dtype=BF16)
        x[3, 5] = float("inf")
        x[7] = float("nan")
        y = empty(m, 80, dtype=BF16)
        ops.linear(x, w, y)
        rows = [i for i in range(m) if i not in (3, 7)]
        ref.check_linear(x[rows], w, y[rows])
        assert bool(y[7].isnan().all()) and not bool(y[3].isfinite().any())


# -- every kernel and a split k -------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 9000, 128), (30, 5000, 70), (96, 8200, 80), (260, 4200, 264)])
def test_long_k(dtype, m, k, n):
    x, w, b = rnd(0, m, k, dtype=dtype), layer(1, k, n, dtype, False), rnd(2, n, dtype=dtype)
    y, pre = empty(m, n, dtype=dtype), empty(m, n, dtype=dtype)
    ops.linear(x, w, y, bias=b, activation="gelu", pre=pre)
    ref.check_linear(x, w, y, b, None, "gelu", pre)
    wt = layer(1, n, k, dtype, False)  # dx over k
    dy, dx = rnd(4, m, k, dtype=dtype), empty(m, n, dtype=dtype)
    ops.linear_backward(dy, None, wt, dx=dx)
    ref.check_linear_backward(dy, None, wt, dx)
    xk, dyk, dw = rnd(5, k, m, dtype=dtype), rnd(6, k, n, dtype=dtype), empty(m, n, dtype=dtype)
    ops.linear_backward(dyk, xk, None, dw=dw)
    ref.check_linear_backward(dyk, xk, None, None, dw)


KERNELS = [f"{tile}{split}" for tile in ("tile64", "tile128", "tile256") for split in ("", ":2", ":3")]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (5, 40, 300), (130, 96, 260), (257, 65, 129), (300, 328, 513), (70, 1000, 90)])
def test_every_kernel(kernel, dtype, m, k, n, monkeypatch):
    """Each tile, whole and split, on sizes around its edges, in all layouts and both epilogues."""
    monkeypatch.setenv("EAS_HIP_OPS_GEMM", kernel)
    for trans in (False, True):
        x, w, wu, b, r = rnd(0, m, k, dtype=dtype), layer(1, k, n, dtype, trans), layer(2, k, n, dtype, trans), rnd(3, n, dtype=dtype), rnd(4, m, n, dtype=dtype)
        y, pre, g, u = (empty(m, n, dtype=dtype) for _ in range(4))
        ops.linear(x, w, y, bias=b, residual=r, activation="gelu", pre=pre)
        ref.check_linear(x, w, y, b, r, "gelu", pre)
        dy, dx, dw = rnd(5, m, n, dtype=dtype), empty(m, k, dtype=dtype), like(w, dtype)
        ops.linear_backward(dy, x, w, dx=dx, dw=dw)
        ref.check_linear_backward(dy, x, w, dx, dw)
        ops.gated_linear(x, w, wu, y, bias_up=b, gate=g, up=u)
        ref.check_gated(x, w, wu, y, None, b, gate=g, up=u)
        dw2 = like(wu, dtype)
        ops.gated_linear_backward(dy, x, w, wu, g, u, dx=dx, dw_gate=dw, dw_up=dw2)
        ref.check_gated_backward(dy, x, w, wu, g, u, dx, dw, dw2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("trans", [False, True])
def test_many_tiles(dtype, trans):
    m, k, n = 1100, 200, 2100
    x, w, b = rnd(0, m, k, dtype=dtype), layer(1, k, n, dtype, trans), rnd(2, n, dtype=dtype)
    y = empty(m, n, dtype=dtype)
    ops.linear(x, w, y, bias=b, activation="relu")
    ref.check_linear(x, w, y, b, None, "relu")
    dy, dx, dw = rnd(4, m, n, dtype=dtype), empty(m, k, dtype=dtype), like(w, dtype)
    ops.linear_backward(dy, x, w, dx=dx, dw=dw)
    ref.check_linear_backward(dy, x, w, dx, dw)


# -- gated linear ------------------------------------------------------------------


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("trans", [False, True])
def test_gated_shapes(shape, dtype, trans):
    m, k, n = shape
    x, wg, wu = rnd(0, m, k, dtype=dtype), layer(1, k, n, dtype, trans), layer(2, k, n, dtype, trans)
    bg, bu = rnd(3, n, dtype=dtype), rnd(4, n, dtype=dtype)
    act = ACTS[(m + k) % 5]
    y, g, u = (empty(m, n, dtype=dtype) for _ in range(3))
    ops.gated_linear(x, wg, wu, y, bias_gate=bg, bias_up=bu, activation=act, gate=g, up=u)
    ref.check_gated(x, wg, wu, y, bg, bu, act, g, u)
    dy, dx, dg, du = rnd(5, m, n, dtype=dtype), empty(m, k, dtype=dtype), like(wg, dtype), like(wu, dtype)
    db, dc = empty(n, dtype=dtype), empty(n, dtype=dtype)
    ops.gated_linear_backward(dy, x, wg, wu, g, u, dx=dx, dw_gate=dg, dw_up=du, dbias_gate=db, dbias_up=dc, activation=act)
    ref.check_gated_backward(dy, x, wg, wu, g, u, dx, dg, du, db, dc, act)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [4, 90])
def test_gated_activations(act, dtype, m):
    k, n = 64, 88
    x, wg, wu = rnd(0, m, k, dtype=dtype, scale=3.0), layer(1, k, n, dtype, False), layer(2, k, n, dtype, False)
    y = empty(m, n, dtype=dtype)
    ops.gated_linear(x, wg, wu, y, activation=act)
    ref.check_gated(x, wg, wu, y, activation=act)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [6, 130])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("pad,offset", [(8, 0), (1, 0), (3, 1)])
def test_gated_strides_and_alignments(dtype, m, trans, pad, offset):
    k, n = 72, 104
    x = spaced(rnd(0, m, k, dtype=dtype), k + pad, offset)
    shape = (n, k) if trans else (k, n)
    wg, wu = spaced(rnd(1, *shape, dtype=dtype), shape[1] + pad, offset), spaced(rnd(2, *shape, dtype=dtype), shape[1] + 2 * pad, offset)
    wg, wu = (wg.t(), wu.t()) if trans else (wg, wu)
    both = empty(m, 2 * n + pad, dtype=dtype)  # gate and up side by side
    g, u, y = both[:, :n], both[:, n:2 * n], spaced(empty(m, n, dtype=dtype), n + pad, offset, 7.0)
    ops.gated_linear(x, wg, wu, y, gate=g, up=u)
    ref.check_gated(x, wg, wu, y, gate=g, up=u)
    dy, dx = spaced(rnd(3, m, n, dtype=dtype), n + pad, offset), empty(m, k, dtype=dtype)
    dg, du = like(wg, dtype), like(wu, dtype)
    ops.gated_linear_backward(dy, x, wg, wu, g, u, dx=dx, dw_gate=dg, dw_up=du)
    ref.check_gated_backward(dy, x, wg, wu, g, u, dx, dg, du)


@pytest.mark.parametrize("parts", list(itertools.product([False, True], repeat=3)))
def test_gated_backward_parts(parts):
    m, k, n = 40, 56, 72
    x, wg, wu = rnd(0, m, k, dtype=F16), layer(1, k, n, F16, True), layer(2, k, n, F16, True)
    dy, g, u = (rnd(3 + i, m, n, dtype=F16) for i in range(3))
    dx = empty(m, k, dtype=F16) if parts[0] else None
    dg, du = (like(wg, F32), like(wu, F32)) if parts[1] else (None, None)
    db, dc = (empty(n, dtype=F32), empty(n, dtype=F32)) if parts[2] else (None, None)
    ops.gated_linear_backward(dy, x if parts[1] else None, wg if parts[0] else None, wu if parts[0] else None, g, u,
                              dx=dx, dw_gate=dg, dw_up=du, dbias_gate=db, dbias_up=dc, activation="gelu")
    ref.check_gated_backward(dy, x, wg, wu, g, u, dx, dg, du, db, dc, "gelu")


@pytest.mark.parametrize("m,k,n", [(8, 0, 24), (0, 16, 24), (8, 16, 0)])
def test_gated_empty(m, k, n):
    x, wg, wu, bg, bu = rnd(0, m, k), rnd(1, k, n), rnd(2, k, n), rnd(3, n), rnd(4, n)
    y, g, u = (empty(m, n, dtype=F32) for _ in range(3))
    ops.gated_linear(x, wg, wu, y, bias_gate=bg, bias_up=bu, gate=g, up=u)
    ref.check_gated(x, wg, wu, y, bg, bu, gate=g, up=u)
    dy, dx, dg, du, db, dc = rnd(5, m, n), empty(m, k, dtype=F32), empty(k, n, dtype=F32), empty(k, n, dtype=F32), empty(n, dtype=F32), empty(n, dtype=F32)
    ops.gated_linear_backward(dy, x, wg, wu, g, u, dx=dx, dw_gate=dg, dw_up=du, dbias_gate=db, dbias_up=dc)
    ref.check_gated_backward(dy, x, wg, wu, g, u, dx, dg, du, db, dc)


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_long_k_and_many_tiles(dtype):
    for m, k, n in ((2, 6000, 64), (80, 5000, 96), (700, 264, 1500)):
        x, wg, wu = rnd(0, m, k, dtype=dtype), layer(1, k, n, dtype, False), layer(2, k, n, dtype, False)
        y = empty(m, n, dtype=dtype)
        ops.gated_linear(x, wg, wu, y, activation="gelu_tanh")
        ref.check_gated(x, wg, wu, y, activation="gelu_tanh")
        g, u, dy, dx = rnd(3, m, n, dtype=dtype), rnd(4, m, n, dtype=dtype), rnd(5, m, n, dtype=dtype), empty(m, k, dtype=dtype)
        dg, du = like(wg, dtype), like(wu, dtype)
        ops.gated_linear_backward(dy, x, wg, wu, g, u, dx=dx, dw_gate=dg, dw_up=du)
        ref.check_gated_backward(dy, x, wg, wu, g, u, dx, dg, du)


# -- gradients against differences --------------------------------------------------


def test_gradients_against_differences():
    """Central differences of the 64-bit forward definitions along random directions, against the kernels' gradients
    in fp32: a step of 1e-4 leaves errors of its square and of 64-bit rounding over it, far below the bound."""
    m, k, n = 12, 20, 28
    x, w, wu, b = rnd(0, m, k), rnd(1, k, n, scale=0.3), rnd(2, k, n, scale=0.3), rnd(3, n)
    dy = rnd(4, m, n)
    step = 1e-4

    def slope(f, inputs, grads, outs_grad):
        for i, g in enumerate(grads):
            v = torch.randn(inputs[i].shape, generator=torch.Generator().manual_seed(9 + i), dtype=torch.float64)
            hi = [ref.d(t) + step * v if j == i else ref.d(t) for j, t in enumerate(inputs)]
            lo = [ref.d(t) - step * v if j == i else ref.d(t) for j, t in enumerate(inputs)]
            want = ((f(*hi) - f(*lo)) * ref.d(outs_grad)).sum() / (2 * step)
            got = (ref.d(g) * v).sum()
            assert abs(got - want) <= 1e-4 * (1 + (ref.d(g).abs() * v.abs()).sum()), (i, got, want)

    for act in ACTS[2:]:
        y, pre = empty(m, n, dtype=F32), empty(m, n, dtype=F32)
        ops.linear(x, w, y, bias=b, activation=act, pre=pre)
        dx, dw, db = empty(m, k, dtype=F32), empty(k, n, dtype=F32), empty(n, dtype=F32)
        ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db, activation=act, pre=pre)
        slope(lambda x, w, b: ref.act(x @ w + b, act), (x, w, b), (dx, dw, db), dy)
        g, u = empty(m, n, dtype=F32), empty(m, n, dtype=F32)
        ops.gated_linear(x, w, wu, y, bias_gate=b, activation=act, gate=g, up=u)
        dg, du, dbg, dbu = empty(k, n, dtype=F32), empty(k, n, dtype=F32), empty(n, dtype=F32), empty(n, dtype=F32)
        ops.gated_linear_backward(dy, x, w, wu, g, u, dx=dx, dw_gate=dg, dw_up=du, dbias_gate=dbg, dbias_up=dbu, activation=act)
        slope(lambda x, w, wu, b: ref.act(x @ w + b, act) * (x @ wu), (x, w, wu, b), (dx, dg, du, dbg), dy)
    gamma, beta = rnd(5, n), rnd(6, n)
    z, y, mean, rstd = rnd(7, m, n), empty(m, n, dtype=F32), empty(m, dtype=F32), empty(m, dtype=F32)
    ops.layer_norm(z, gamma, beta, y, mean, rstd)
    dz, dgamma, dbeta = empty(m, n, dtype=F32), empty(n, dtype=F32), empty(n, dtype=F32)
    ops.layer_norm_backward(dy, z, gamma, mean, rstd, dz, dgamma, dbeta)
    slope(lambda z, g, b: ref.norm(z, g, b, 1e-5)[0], (z, gamma, beta), (dz, dgamma, dbeta), dy)


# -- how they are called --------------------------------------------------------------


def test_repeated_runs_are_bit_identical():
    x, w, dy, pre = rnd(0, 700, 1030, dtype=BF16), layer(1, 1030, 600, BF16, False), rnd(2, 700, 600, dtype=BF16), rnd(3, 700, 600, dtype=BF16)
    first = None
    for _ in range(4):
        dx, dw, db = empty(700, 1030, dtype=BF16), like(w, BF16), empty(600, dtype=BF16)
        ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db, activation="gelu", pre=pre)
        now = [t.clone() for t in (dx, dw, db)]
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_async_calls_on_another_stream_and_the_in_flight_bound(gpu_runtime):
    s = torch.cuda.Stream()
    x, w = rnd(0, 64, 512, dtype=F16), rnd(1, 512, 512, dtype=F16, scale=512 ** -0.5)
    outs = [empty(64, 512, dtype=F16) for _ in range(40)]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for y in outs:
            ops.linear(x, w, y, _sync=False)
    gpu_runtime.synchronize()
    ref.check_linear(x, w, outs[0])
    assert all(torch.equal(outs[0], y) for y in outs)


def test_numpy_and_eas_tensors():
    import eas

    rng = np.random.default_rng(0)
    x, w, r = (rng.standard_normal(s, dtype=np.float32) for s in ((20, 24), (24, 40), (20, 40)))
    y, pre = np.full((20, 40), np.nan, np.float32), np.full((20, 40), np.nan, np.float32)
    ops.linear(x, w, y, residual=r, activation="gelu", pre=pre)
    t = torch.from_numpy
    ref.check_linear(t(x), t(w), t(y), None, t(r), "gelu", t(pre))
    h = eas.tensor(x, device="hip"), eas.tensor(w, device="hip"), eas.empty((20, 40), device="hip")
    ops.linear(*h, _sync=False)
    from easy_as_amd.runtime import get_runtime

    get_runtime().synchronize()
    ref.check_linear(t(x), t(w), t(h[2].numpy()))
    xc = rng.standard_normal((6, 300), dtype=np.float32)
    g, m, s = np.ones(300, np.float32), np.empty(6, np.float32), np.empty(6, np.float32)
    z = xc.copy()
    ops.layer_norm(z, g, None, z, m, s)  # in place on the host
    ref.check_norm(t(xc), t(g), None, 1e-5, t(z), t(m), t(s))


def test_graph_replays_match_eager():
    m, k, n = 48, 520, 264
    x, wg, wu, wd = rnd(0, m, k, dtype=BF16), layer(1, k, n, BF16, False), layer(2, k, n, BF16, False), layer(3, n, k, BF16, False)
    gam, bet = rnd(4, k, dtype=BF16, mean=1.0), rnd(5, k, dtype=BF16)
    dy = rnd(6, m, k, dtype=BF16)
    bufs = {s: empty(m, k, dtype=BF16) for s in ("h", "y", "dh", "dx")}
    mid = {s: empty(m, n, dtype=BF16) for s in ("a", "g", "u", "da")}
    mean, rstd = empty(m, dtype=F32), empty(m, dtype=F32)
    grads = [like(wg, BF16), like(wu, BF16), like(wd, BF16), like(gam, BF16), like(bet, BF16)]

    def step():
        ops.layer_norm(x, gam, bet, bufs["h"], mean, rstd, _sync=False)
        ops.gated_linear(bufs["h"], wg, wu, mid["a"], gate=mid["g"], up=mid["u"], _sync=False)
        ops.linear(mid["a"], wd, bufs["y"], residual=x, _sync=False)
        ops.linear_backward(dy, mid["a"], wd, dx=mid["da"], dw=grads[2], _sync=False)
        ops.gated_linear_backward(mid["da"], bufs["h"], wg, wu, mid["g"], mid["u"], dx=bufs["dh"], dw_gate=grads[0], dw_up=grads[1], _sync=False)
        ops.layer_norm_backward(bufs["dh"], x, gam, mean, rstd, bufs["dx"], grads[3], grads[4], _sync=False)

    outs = list(bufs.values()) + list(mid.values()) + grads
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    with pytest.raises(ValueError, match="_sync=False"):
        capture = torch.cuda.CUDAGraph()
        with torch.cuda.graph(capture):
            step()
            ops.linear(mid["a"], wd, bufs["y"])
    torch.cuda.synchronize()
    for turn in range(4):
        x.copy_(rnd(20 + turn, m, k, dtype=BF16))
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in outs]
        for t in outs:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs))


def test_calls_again_follow_their_arguments(gpu_runtime):
    """A repeated call goes by its tensors as they are now: other values, addresses, sizes, types, layouts and options
    after one another, and refusals where an earlier call of another kind was fine."""
    for turn in range(3):
        for dtype in (F16, F32):
            for m, k, n, act in ((3, 40, 64, "relu"), (3, 40, 64, "silu"), (70, 40, 64, "relu"), (3, 44, 64, "relu")):
                x, w, y = rnd(turn, m, k, dtype=dtype), layer(turn + 9, k, n, dtype, turn == 1), empty(m, n, dtype=dtype)
                ops.linear(x, w, y, activation=act, _sync=turn != 2)
                gpu_runtime.synchronize()
                ref.check_linear(x, w, y, activation=act)
                xs = spaced(x, k + 1, 1)
                ops.linear(xs, w, y, activation=act, pre=None)
                ref.check_linear(x, w, y, activation=act)
        x, w, b = rnd(turn, 4, 96), rnd(1, 96), rnd(2, 96)
        for eps in (1e-5, 1e-2):
            y = empty(4, 96, dtype=F32)
            ops.layer_norm(x, w, b, y, eps=eps)
            ref.check_norm(x, w, b, eps, y)
    x, w, y = rnd(0, 3, 40), rnd(1, 40, 64), empty(3, 64, dtype=F32)
    ops.linear(x, w, y)
    both = empty(3 * 64 + 120, dtype=F32)
    with pytest.raises(ValueError, match="shares"):  # the shapes of the call above, y over x
        ops.linear(both[:120].view(3, 40), w, both[100:292].view(3, 64))
    with pytest.raises(ValueError, match="'y' must hold"):
        ops.linear(x, w, y[:2])
    with pytest.raises(TypeError, match="_sync"):
        ops.linear(x, w, y, _sync=1)


def test_calls_again_on_the_current_stream():
    x, w = rnd(0, 2, 2048, dtype=F16), rnd(1, 2048, 512, dtype=F16, scale=0.02)  # a split k: scratch on each stream
    y0 = empty(2, 512, dtype=F16)
    ops.linear(x, w, y0)
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(12):
        s = streams[turn % 3]
        s.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(s):
            y = torch.zeros(2, 512, dtype=F16, device="cuda")
            ops.linear(x, w, y, _sync=False)
            outs.append(y * 1)  # ordered after it on the same stream
    torch.cuda.synchronize()
    assert all(torch.equal(o, y0) for o in outs)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m", [1, 16, 17, 33, 64])
@pytest.mark.parametrize("k,n", [(1, 1), (7, 9), (129, 131), (1030, 255), (257, 1027)])
@pytest.mark.parametrize("trans", [False, True])
def test_few_rows_of_odd_lengths(dtype, m, k, n, trans):
    """16-bit rows at odd addresses: the few-row kernels' stages through registers, NaN wherever they must not read."""
    shape = (n, k) if trans else (k, n)
    x = spaced(rnd(0, m, k, dtype=dtype), k + 2, 1)
    ws = [spaced(rnd(s, *shape, dtype=dtype, scale=k ** -0.5), shape[1] + 1 + s % 2, 1) for s in (1, 2)]
    w, wu = (t.t() for t in ws) if trans else ws
    y, g, u = (empty(m, n, dtype=dtype) for _ in range(3))
    ops.linear(x, w, y, activation="silu")
    ref.check_linear(x, w, y, None, None, "silu")
    ops.gated_linear(x, w, wu, y, gate=g, up=u)
    ref.check_gated(x, w, wu, y, gate=g, up=u)
    dy, dx = spaced(rnd(3, m, n, dtype=dtype), n + 1, 1), empty(m, k, dtype=dtype)
    ops.linear_backward(dy, None, w, dx=dx)
    ref.check_linear_backward(dy, None, w, dx)
    ops.gated_linear_backward(dy, None, w, wu, g, u, dx=dx)
    ref.check_gated_backward(dy, None, w, wu, g, u, dx)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("trans", [False, True])
def test_a_few_tiles_beyond_a_round(dtype, trans):
    """16 x 16 tiles of 256 and four columns more (and as many of 128 for fp32): the last columns run apart."""
    m, n = (4096, 4100) if dtype != F32 else (2048, 2052)
    k = 768
    x, w, wu, b, r = rnd(0, m, k, dtype=dtype), layer(1, k, n, dtype, trans), layer(2, k, n, dtype, trans), rnd(3, n, dtype=dtype), rnd(4, m, n, dtype=dtype)
    y, pre, u = empty(m, n, dtype=dtype), empty(m, n, dtype=dtype), empty(m, n, dtype=dtype)
    ops.linear(x, w, y, bias=b, residual=r, activation="gelu", pre=pre)
    ref.check_linear(x, w, y, b, r, "gelu", pre)
    ops.gated_linear(x, w, wu, y, bias_gate=b, bias_up=b, gate=pre, up=u)
    ref.check_gated(x, w, wu, y, b, b, gate=pre, up=u)
    xk, dyk = rnd(5, k, n, dtype=dtype), rnd(6, k, m, dtype=dtype)  # dw [n, m], and its transpose
    dw = empty(m, n, dtype=dtype).t() if trans else empty(n, m, dtype=dtype)
    ops.linear_backward(dyk, xk, None, dw=dw)
    ref.check_linear_backward(dyk, xk, None, None, dw)
    dy, wn, dx = rnd(7, m, k, dtype=dtype), layer(8, n, k, dtype, trans), empty(m, n, dtype=dtype)
    ops.linear_backward(dy, None, wn, dx=dx)
    ref.check_linear_backward(dy, None, wn, dx)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,n,ld", [(1, 264, 264), (9, 514, 520), (70, 1030, 1030), (203, 4098, 4100), (1500, 1026, 1032)])
def test_gradients_of_even_rows(dtype, bias, m, n, ld):
    """Rows of whole 4 bytes that end inside a vector of 8 and inside a wave's columns."""
    k = 16
    x, w, wu = rnd(0, m, k, dtype=dtype), layer(1, k, n, dtype, False), layer(2, k, n, dtype, False)
    dy, pre, u = spaced(rnd(3, m, n, dtype=dtype), ld, 2), spaced(rnd(4, m, n, dtype=dtype), ld + 2), rnd(5, m, n, dtype=dtype)
    dx, dw, dwu = empty(m, k, dtype=dtype), like(w, dtype), like(wu, dtype)
    db, dbu = (empty(n, dtype=dtype) if bias else None for _ in range(2))
    ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db, activation="gelu_tanh", pre=pre)
    ref.check_linear_backward(dy, x, w, dx, dw, db, "gelu_tanh", pre)
    ops.gated_linear_backward(dy, x, w, wu, pre, u, dx=dx, dw_gate=dw, dw_up=dwu, dbias_gate=db, dbias_up=dbu, activation="gelu")
    ref.check_gated_backward(dy, x, w, wu, pre, u, dx, dw, dwu, db, dbu, "gelu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("m,k,n", [(65, 64, 64), (130, 70, 2100), (300, 512, 1031), (517, 1023, 201), (700, 130, 132)])
def test_gradients_of_products_that_share_a_launch(dtype, trans, m, k, n):
    """dx and dw of few tiles, dx's sum whole and split, and each of them alone."""
    x, w, wu = rnd(0, m, k, dtype=dtype), layer(1, k, n, dtype, trans), layer(2, k, n, dtype, trans)
    dy, pre, u = rnd(3, m, n, dtype=dtype), rnd(4, m, n, dtype=dtype), rnd(5, m, n, dtype=dtype)
    dx, dw, dwu = empty(m, k, dtype=dtype), like(w, F32), like(wu, F32)
    db, dbu = empty(n, dtype=F32), empty(n, dtype=F32)
    ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db, activation="silu", pre=pre)
    ref.check_linear_backward(dy, x, w, dx, dw, db, "silu", pre)
    ops.gated_linear_backward(dy, x, w, wu, pre, u, dx=dx, dw_gate=dw, dw_up=dwu, dbias_gate=db, dbias_up=dbu)
    ref.check_gated_backward(dy, x, w, wu, pre, u, dx, dw, dwu, db, dbu)
    one, two, three = empty(m, k, dtype=dtype), like(w, F32), like(wu, F32)
    ops.gated_linear_backward(dy, None, w, wu, pre, u, dx=one)
    ref.check_gated_backward(dy, x, w, wu, pre, u, one)
    ops.gated_linear_backward(dy, x, None, None, pre, u, dw_gate=two, dw_up=three)
    ref.check_gated_backward(dy, x, w, wu, pre, u, None, two, three)


def test_gradients_of_inputs_beyond_the_caches():
    k, n = 24, 4100
    for gated in (False, True):
        m = 3500 if gated else 5800  # over 128 MB with dz
        x, w, wu = rnd(0, m, k, dtype=BF16), layer(1, k, n, BF16, False), layer(2, k, n, BF16, False)
        dy, pre = rnd(3, m, n, dtype=BF16), rnd(4, m, n, dtype=BF16)
        dx, dw, dwu, db, dbu = empty(m, k, dtype=BF16), like(w, BF16), like(w, BF16), empty(n, dtype=BF16), empty(n, dtype=BF16)
        if gated:
            u = rnd(5, m, n, dtype=BF16)
            ops.gated_linear_backward(dy, x, w, wu, pre, u, dx=dx, dw_gate=dw, dw_up=dwu, dbias_gate=db, dbias_up=dbu)
            ref.check_gated_backward(dy, x, w, wu, pre, u, dx, dw, dwu, db, dbu)
        else:
            ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db, activation="silu", pre=pre)
            ref.check_linear_backward(dy, x, w, dx, dw, db, "silu", pre)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 128, 520), (16, 1024, 4104), (33, 520, 2050), (64, 256, 16400), (5, 2048, 11011)])
def test_few_rows_even_shares_of_columns(dtype, m, k, n):
    """Weights along k whose columns do not fill the last round of workgroups."""
    x, w, wu, b, r = rnd(0, m, k, dtype=dtype), layer(1, k, n, dtype, True), layer(2, k, n, dtype, True), rnd(3, n, dtype=dtype), rnd(4, m, n, dtype=dtype)
    y, pre = spaced(empty(m, n, dtype=dtype), n + 3, 1, 7.0), empty(m, n, dtype=dtype)
    ops.linear(x, w, y, bias=b, residual=r, activation="silu", pre=pre)
    ref.check_linear(x, w, y, b, r, "silu", pre)
    assert m == 1 or bool((y.as_strided((m - 1, 3), (n + 3, 1), 1 + n) == 7.0).all())
    ops.gated_linear(x, w, wu, y, bias_gate=b, bias_up=b)
    ref.check_gated(x, w, wu, y, b, b)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shifted", ["x", "w", "dy"])
@pytest.mark.parametrize("m", [100, 16])
def test_calls_again_at_other_addresses(dtype, shifted, m):
    """One shape and layout at every place that an array may have within 16 bytes, each after a call at another one."""
    k, n = 64, 72

    def at(name, t, offset):
        return spaced(t, t.shape[1], offset) if name == shifted else t

    for turn, offset in enumerate((2, 1, 3, 8, 2, 5, 0, 1, 4, 7)):
        x, w, wu = at("x", rnd(turn, m, k, dtype=dtype), offset), at("w", layer(1, k, n, dtype, False), offset), layer(2, k, n, dtype, False)
        y, pre, up = (empty(m, n, dtype=dtype) for _ in range(3))
        ops.linear(x, w, y, activation="gelu", pre=pre)
        ref.check_linear(x, w, y, activation="gelu", pre=pre)
        dy, dx, dw, dwu, db = at("dy", rnd(4, m, n, dtype=dtype), offset), empty(m, k, dtype=dtype), like(w, dtype), like(wu, dtype), empty(n, dtype=dtype)
        for act in ("none", "gelu"):
            ops.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db, activation=act, pre=pre)
            ref.check_linear_backward(dy, x, w, dx, dw, db, act, pre)
        ops.gated_linear(x, w, wu, y, gate=pre, up=up)
        ref.check_gated(x, w, wu, y, gate=pre, up=up)
        ops.gated_linear_backward(dy, x, w, wu, pre, up, dx=dx, dw_gate=dw, dw_up=dwu)
        ref.check_gated_backward(dy, x, w, wu, pre, up, dx, dw, dwu)


def long_rows(m, k):
    """Rows of k that are 0 but in forty columns, the first and the last among them, and those columns."""
    at = torch.cat([torch.tensor([0, 1, k - 2, k - 1]), torch.randint(2, k - 2, (36,), generator=torch.Generator().manual_seed(k))]).unique()
    x = torch.zeros(m, k, dtype=F16, device="cuda")
    x[:, at.cuda()] = rnd(m, m, len(at), dtype=F16)
    return x, at.cuda()


@pytest.mark.parametrize("kernel,rows", [("tile256:2", 256), ("tile128:2", 128), ("tile64:2", 64), ("auto", 64)])
def test_rows_at_the_end_of_a_tiles_offsets(kernel, rows, monkeypatch):
    """A tile's last row just within 2^31 bytes of its first one."""
    monkeypatch.setenv("EAS_HIP_OPS_GEMM", kernel)
    m, k, n = rows + 6, (2 ** 31 - 4 - 128) // (rows - 1) // 16 * 8, 16
    x, at = long_rows(m, k)
    w, y = torch.randn(k, n, dtype=F16, device="cuda"), empty(m, n, dtype=F16)
    ops.linear(x, w, y)
    ref.check_linear(x[:, at], w[at], y)  # the other columns' products are 0
    with pytest.raises(ValueError, match="too long"):
        ops.linear(torch.empty_strided((m, k + 16), (k + 16, 1), dtype=F16, device="cuda"), torch.empty(k + 16, n, dtype=F16, device="cuda"), y)


def test_gradient_of_weights_of_long_rows():
    m, k, n = 40, 20000000, 8  # rows of x 40 MB apart: tiles of few k reach them
    x, dy, dw = torch.randn(m, k, dtype=F16, device="cuda"), rnd(1, m, n, dtype=F16), torch.full((k, n), float("nan"), dtype=F16, device="cuda")
    ops.linear_backward(dy, x, None, dw=dw)
    assert not bool(dw.isnan().any())
    for first in (0, 2 ** 20 - 300, 2 ** 24 - 300, k - 600):
        some = slice(first, first + 600)
        ref.check_linear_backward(dy, x[:, some], None, None, dw[some])


# -- the activations' tails ------------------------------------------------------------
#
# Products with one k and a weight of 1 give z itself.  Relative errors: exp of an argument a is off by the 2^-24 that each of
# the three roundings in a may add to it, so by 3 |a| 2^-24 at most, beside a few units of 2^-23 for the functions and the
# arithmetic (16); a = z for silu, z (1.5958 + 0.0714 z^2) for the tanh form and z^2 / 2 for gelu.  16-bit operands' gelu goes
# by a formula within 1.5e-5; that of f32 by erfc, whose argument's two roundings count twice.


def phi(z):
    """The normal integral; torch.special.ndtr has no digits of it left below -8."""
    return 0.5 * torch.special.erfc(z * -0.5 ** 0.5)


def tail_error(z, act, dtype):
    a = {"silu": z.abs(), "gelu_tanh": z.abs() * (1.6 + 0.072 * z.square()), "gelu": z.square() / 2}[act]
    return (4 * a + 16) * 2.0 ** -23 + (1.5e-5 if act == "gelu" and dtype != F32 else 0)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "gelu"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("wide", [False, True])
def test_activations_tails_keep_their_digits(act, dtype, wide):
    z = torch.cat([torch.linspace(-12, -0.5, 4000), torch.linspace(-0.5, 12, 1000)]).to(dtype).cuda()
    n, out = z.numel(), F32 if wide else dtype
    one, ones = torch.ones(1, 1, dtype=dtype, device="cuda"), torch.ones(1, n, dtype=dtype, device="cuda")
    want, err = ref.act(ref.d(z), act)[None], tail_error(ref.d(z), act, dtype)[None]
    if act == "gelu_tanh":  # 1 + tanh cancels in 64 bits too: z sigmoid(2 u)
        u2 = (8 / torch.pi) ** 0.5 * (ref.d(z) + 0.044715 * ref.d(z) ** 3)
        want = (ref.d(z) * torch.sigmoid(u2))[None]
    elif act == "gelu":
        want = (ref.d(z) * phi(ref.d(z)))[None]
    y = empty(1, n, dtype=out)
    ops.linear(one, z[None], y, activation=act)
    ref.check(act, y, want, err * want.abs())
    ops.gated_linear(one, z[None], ones, y, activation=act)
    ref.check(act, y, want, err * want.abs())
    many, ys = torch.ones(70, 1, dtype=dtype, device="cuda"), empty(70, n, dtype=out)  # the tiles' epilogue
    ops.linear(many, z[None], ys, activation=act)
    assert torch.equal(ys, y.expand(70, n))


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "gelu"])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_tails_keep_their_digits(act, dtype):
    z = torch.cat([torch.linspace(-12, -0.5, 4000), torch.linspace(-0.5, 12, 1000)]).to(dtype).cuda()
    zd, n = ref.d(z), z.numel()
    # the slope's terms, s and z s', each with its own error
    if act == "gelu":
        s, ds = phi(zd), torch.exp(-zd.square() / 2) / (2 * torch.pi) ** 0.5
    else:
        a, da = (zd, 1.0) if act == "silu" else ((8 / torch.pi) ** 0.5 * (zd + 0.044715 * zd ** 3), (8 / torch.pi) ** 0.5 * (1 + 3 * 0.044715 * zd.square()))
        s, ds = torch.sigmoid(a), torch.sigmoid(a) * torch.sigmoid(-a) * da
    err = tail_error(zd, act, dtype) * (s + (zd * ds).abs())
    dbias = empty(n, dtype=F32)
    ops.linear_backward(torch.ones(1, n, dtype=dtype, device="cuda"), None, None, dbias=dbias, activation=act, pre=z[None])
    ref.check(act, dbias, s + zd * ds, err)
    dg, du = empty(n, dtype=F32), empty(n, dtype=F32)
    ones = torch.ones(1, n, dtype=dtype, device="cuda")
    ops.gated_linear_backward(ones, None, None, None, z[None], ones, dbias_gate=dg, dbias_up=du, activation=act)
    ref.check(act, dg, s + zd * ds, err)
    ref.check(act, du, zd * s, tail_error(zd, act, dtype) * (zd * s).abs())


def test_norm_sums_of_more_columns_than_a_grid_has_threads_for():
    m, n = 2, 2 ** 26 + 5  # 2^27 sums, 32 to a workgroup of 1024
    g = torch.Generator(device="cuda").manual_seed(0)
    x, dy = (torch.randn(m, n, generator=g, dtype=F16, device="cuda") for _ in range(2))
    mean, rstd = rnd(1, m), rnd(2, m).abs()
    dw, db = (torch.full((n,), float("nan"), dtype=F16, device="cuda") for _ in range(2))
    ops.layer_norm_backward(dy, x, None, mean, rstd, None, dw, db)
    assert not bool(dw.isnan().any()) and not bool(db.isnan().any())
    for first in (0, 2 ** 24 - 300, 2 ** 25 - 300, n - 600):
        some = slice(first, first + 600)
        ref.check_norm_backward(dy[:, some], x[:, some], None, mean, rstd, None, dw[some], db[some])


@pytest.mark.parametrize("trans", [False, True])
def test_few_rows_beyond_a_tiles_offsets(trans):
    m, k, n = 20, 60000000, 8  # rows of x 120 MB apart
    x, at = long_rows(m, k)
    w, y = torch.randn(n, k, dtype=F16, device="cuda").t() if trans else torch.randn(k, n, dtype=F16, device="cuda"), empty(m, n, dtype=F16)
    ops.linear(x, w, y)
    ref.check_linear(x[:, at], w[at], y)
    wn, dx = w.t(), empty(m, n, dtype=F16)  # dx over the same k
    ops.linear_backward(x, None, wn, dx=dx)
    ref.check_linear_backward(x[:, at], None, wn[:, at], dx)
