"""The norm's gradients in the kernels that keep partial sums, each form of them against the definition in 64 bits, and what is read
past the caches."""

from __future__ import annotations

import pytest
import torch

import fp8_reference as ref
from easy_as_amd import ops
from test_gpu_fp8_ops import BF16, E4M3, F16, F32, empty, rnd, scales, spaced

pytestmark = pytest.mark.gpu

# (dy's type, the stream's)
KINDS = [(F16, F16), (BF16, BF16), (F32, F32), (F16, F32), (BF16, F32)]


def case(m: int, n: int, dtype, htype, seed: int = 0):
    h, dy, dt = rnd(seed, m, n, dtype=htype, scale=2.0, mean=0.3), rnd(seed + 1, m, n, dtype=dtype), rnd(seed + 2, m, n, dtype=htype)
    return dy, h, rnd(seed + 3, n, dtype=dtype, mean=1.0), (h.float().square().mean(1) + 1e-5).rsqrt(), dt


# the edges of each number of threads and vectors a row, rows of whole 4 bytes and others; over 2^20 elements in all
@pytest.mark.parametrize("n", [129, 509, 512, 514, 1023, 1024, 1030, 1537, 2048, 2051, 3001, 4096, 4098, 6143, 8192, 8194, 8201, 12288, 12290,
                               12301, 16383, 16384])
@pytest.mark.parametrize("kind", KINDS)
def test_every_width(n, kind):
    m = 2 ** 20 // n + 6
    dtype, htype = kind
    dy, h, w, rstd, dt = case(m, n, dtype, htype, n)
    dx, dw = empty(m, n, dtype=htype), empty(n, dtype=dtype)
    ops.rms_norm_backward(dy, h, w, rstd, dx, dw, dtotal=dt)
    ref.check_rms_backward(dy, h, w, rstd, dx, dw, dt)


@pytest.mark.parametrize("n", [300, 1030, 4096, 8192, 16384])
@pytest.mark.parametrize("kind", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("over", ["dy", "h", "dtotal"])
def test_in_place(n, kind, over):
    """dx over what is read a row or two ahead of it."""
    m = 2 ** 20 // n + 300
    dtype, htype = kind
    if over == "dy" and dtype != htype:
        return
    dy, h, w, rstd, dt = case(m, n, dtype, htype, n)
    args = {"dy": dy.clone(), "h": h.clone(), "dtotal": dt.clone()}
    dw = empty(n)
    ops.rms_norm_backward(args["dy"], args["h"], w.float(), rstd, args[over], dw, dtotal=args["dtotal"])
    ref.check_rms_backward(dy, h, w.float(), rstd, args[over], dw, dt)


@pytest.mark.parametrize("n", [1030, 4096, 12300])
@pytest.mark.parametrize("kind", KINDS)
def test_one_of_the_two(n, kind):
    m = 2 ** 20 // n + 300
    dtype, htype = kind
    dy, h, w, rstd, dt = case(m, n, dtype, htype, n)
    dw, dx = empty(n, dtype=dtype), empty(m, n, dtype=htype)
    ops.rms_norm_backward(dy, h, w, rstd, None, dw)
    ref.check_rms_backward(dy, h, w, rstd, None, dw)
    ops.rms_norm_backward(dy, h, w, rstd, dx)
    ref.check_rms_backward(dy, h, w, rstd, dx)


@pytest.mark.parametrize("n,ld,offset", [(1030, 1033, 1), (4096, 4104, 8), (8194, 8199, 3)])
@pytest.mark.parametrize("kind", KINDS)
def test_strides(n, ld, offset, kind):
    m = 2 ** 20 // n + 300
    dtype, htype = kind
    dy, h, w, rstd, dt = case(m, n, dtype, htype, n)
    dy, h, dt = (spaced(t, ld + e, offset) for t, e in ((dy, 0), (h, 2), (dt, 4)))
    dx, dw = spaced(empty(m, n, dtype=htype), ld + 6, offset), empty(n, dtype=dtype)
    ops.rms_norm_backward(dy, h, w, rstd, dx, dw, dtotal=dt)
    ref.check_rms_backward(dy, h, w, rstd, dx, dw, dt)
    assert bool((dx.as_strided((m - 1, ld + 6 - n), (ld + 6, 1), dx.storage_offset() + n) == 7).all())


# over 128 MB moved, in rows of whole lines: what is read goes past the caches
@pytest.mark.parametrize("m,n,kind", [(4200, 4096, (BF16, BF16)), (2500, 4096, (F16, F32)), (1100, 8192, (F32, F32)), (1300, 8192, (BF16, F32)),
                                      (1100, 16384, (F16, F16))])
def test_large(m, n, kind):
    dtype, htype = kind
    dy, h, w, rstd, dt = case(m, n, dtype, htype, n)
    assert m * n * (dy.element_size() + 3 * h.element_size()) > 128 << 20
    dx, dw = empty(m, n, dtype=htype), empty(n, dtype=dtype)
    ops.rms_norm_backward(dy, h, w, rstd, dx, dw, dtotal=dt)
    ref.check_rms_backward(dy, h, w, rstd, dx, dw, dt)


@pytest.mark.parametrize("m,n,kind", [(8200, 4096, (BF16, BF16)), (2100, 8192, (F16, F32)), (1030, 16384, (F32, F32))])
def test_a_large_batch_as_its_parts(m, n, kind):
    """The norm of over 192 MB moved, past the caches, and of parts of it, within them: a row's results are the same bits."""
    dtype, htype = kind
    x, res, w = rnd(0, m, n, dtype=dtype), rnd(1, m, n, dtype=htype, scale=5.0), rnd(2, n, dtype=dtype, mean=1.0)
    assert m * n * (2 * x.element_size() + 2 * res.element_size() + 1) > 192 << 20

    def norm(a, b):
        rows = b - a
        y, total, rstd = empty(rows, n, dtype=dtype), empty(rows, n, dtype=htype), empty(rows)
        q, s = empty(rows, n, dtype=E4M3), scales(rows, n)
        ops.rms_norm(x[a:b], w, y, rstd, residual=res[a:b], total=total, q=q, q_scale=s)
        return y, total, rstd, q.view(torch.uint8), s

    whole = norm(0, m)
    for a in range(0, m, 300):
        b = min(a + 300, m)
        for one, part in zip(whole, norm(a, b)):
            assert torch.equal(one[a:b], part)
    last = slice(m - 300, m)
    y, total, rstd, q, s = (t[last] for t in whole)
    ref.check_rms(x[last], w, 1e-5, res[last], total, y, rstd, q.view(E4M3), s)
