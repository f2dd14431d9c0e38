"""The operators around 8-bit operands as a program uses them: together, again, on streams, in graphs, on the host, and at sizes
that choose another kernel."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import fp8_reference as ref
from easy_as_amd import ops
from ops_reference import act, act_grad, d, gamma
from test_gpu_fp8_ops import BF16, COLUMNS, E4M3, F16, F32, ROWS, SQUARES, TYPES, empty, operand, rnd, scales, spaced

pytestmark = pytest.mark.gpu


# -- the product's kernels ------------------------------------------------------------------


@pytest.mark.parametrize("plan", ["tile64:1", "tile64:3", "tile128:1", "tile128:2", "tile128:5", "tile256:1", "tile256:3"])
@pytest.mark.parametrize("m,k,n", [(5, 128, 9), (300, 640, 260), (257, 1552, 513), (260, 896, 129)])
@pytest.mark.parametrize("lying", ["y", "dx", "dw"])
def test_every_tile(monkeypatch, plan, m, k, n, lying):
    """Each tile kernel over odd and even counts of blocks, whole and cut, and joined ranges of k."""
    monkeypatch.setenv("EAS_HIP_OPS_GEMM", plan)
    x, xs, xv = operand(0, m, k, ROWS, "columns" if lying == "dw" else "rows")
    w, ws, wv = operand(1, k, n, COLUMNS if lying == "dw" else SQUARES, "columns" if lying == "y" else "rows")
    for dtype in (BF16, F32):
        b, res, pre, y = rnd(2, n, dtype=dtype), rnd(3, m, n, dtype=dtype), empty(m, n, dtype=dtype), empty(m, n, dtype=dtype)
        ops.linear_fp8(x, xs, w, ws, y, bias=b, residual=res, activation="gelu", pre=pre)
        ref.check_linear_fp8(xv, wv, y, b, res, "gelu", pre)


@pytest.mark.parametrize("m,k,n,dtype", [(2900, 208, 5900, BF16), (2597, 256, 6390, F16), (700, 130, 25000, BF16), (2900, 256, 3300, F32),
                                         (130, 200, 33300, F32)])
@pytest.mark.parametrize("lying", ["y", "dx", "dw"])
def test_somewhat_more_than_a_round_of_tiles(m, k, n, dtype, lying):
    """Products whose last rows or columns are a launch of their own, among them so few rows that they have their own kernel."""
    x, xs, xv = operand(0, m, k, ROWS, "columns" if lying == "dw" else "rows")
    w, ws, wv = operand(1, k, n, COLUMNS if lying == "dw" else SQUARES, "columns" if lying == "y" else "rows")
    b, res, pre, y = rnd(2, n, dtype=dtype), rnd(3, m, n, dtype=dtype), empty(m, n, dtype=dtype), spaced(empty(m, n, dtype=dtype), n + 3, 1)
    ops.linear_fp8(x, xs, w, ws, y, bias=b, residual=res, activation="relu", pre=pre)
    ref.check_linear_fp8(xv, wv, y, b, res, "relu", pre)
    ops.linear_fp8(x, xs, w, ws, res, bias=b, residual=res, activation="relu")  # in place
    assert torch.equal(res, y)


@pytest.mark.parametrize("m", [1, 15, 16, 17, 32, 33, 64, 65])
@pytest.mark.parametrize("k,n", [(256, 16), (256, 7), (1024, 3000), (2320, 1100), (8192, 200), (300, 520), (1031, 333)])
def test_few_rows(m, k, n):
    """Every width of the few-row kernels, k in one range or several, rows that are read as they are, shifted or copied."""
    x, xs, xv = operand(m, m, k, ROWS, "rows")
    w, ws, wv = operand(n, k, n, SQUARES, "columns")
    for dtype in (F16, F32):
        y = empty(m, n, dtype=dtype)
        ops.linear_fp8(x, xs, w, ws, y)
        ref.check_linear_fp8(xv, wv, y)


@pytest.mark.parametrize("m", [3, 20, 50])
def test_few_rows_with_a_scale_for_each_column(m):
    for k, n in ((640, 90), (1025, 200)):
        x, xs, xv = operand(m, m, k, ROWS, "rows")
        w, ws, wv = operand(n, k, n, COLUMNS, "columns")
        y = empty(m, n, dtype=BF16)
        ops.linear_fp8(x, xs, w, ws, y)
        ref.check_linear_fp8(xv, wv, y)


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("k", [128, 255, 257, 400])
def test_few_rows_at_every_byte(shift, k):
    """Rows that start at any byte, the last one ending where its storage ends."""
    m, n = 4, 37
    x, xs, xv = operand(0, m, k, ROWS, "rows", k + 1, shift)
    w, ws, wv = operand(1, k, n, SQUARES, "columns", k + 3, shift)
    y = empty(m, n)
    ops.linear_fp8(x, xs, w, ws, y)
    ref.check_linear_fp8(xv, wv, y)


def test_more_columns_than_a_round_of_workgroups():
    m, k, n = 2, 256, 40000
    x, xs, xv = operand(0, m, k, ROWS, "rows")
    w, ws, wv = operand(1, k, n, SQUARES, "columns")
    y = empty(m, n, dtype=F16)
    ops.linear_fp8(x, xs, w, ws, y)
    ref.check_linear_fp8(xv, wv, y)


def test_offsets_beyond_32_bits():
    """Operands and outputs of over 2^31 elements: the last rows are where a 32-bit offset would not reach."""
    m, k = 70016, 32768
    x = torch.zeros(m, k, dtype=torch.uint8, device="cuda")
    x[-5:] = torch.randint(0x30, 0x48, (5, k), dtype=torch.uint8, device="cuda")
    xs = torch.ones(m, k // 128, device="cuda")
    xs[-3:] = 0.5
    w, ws, wv = operand(1, k, 24, SQUARES, "columns")
    y = empty(m, 24, dtype=BF16)
    ops.linear_fp8(x.view(E4M3), xs, w, ws, y)
    ref.check_linear_fp8(ref.values(x[-5:].view(E4M3), xs[-5:], ROWS), wv, y[-5:])
    assert bool((y[:-5] == 0).all())
    # and across the sum: the same matrix as [k, n]
    w1, ws1 = x.view(E4M3), torch.ones(m // 128, k // 128, device="cuda")
    a, as_, av = operand(2, 3, m, ROWS, "rows")
    y = empty(3, k, dtype=F16)
    ops.linear_fp8(a, as_, w1, ws1, y)
    ref.check_linear_fp8(av[:, -5:], w1[-5:].cpu().float().double(), y)
    del x, w1

    m, n = 600000, 4096
    h = torch.zeros(m, n, dtype=F16, device="cuda")
    h[-2:] = rnd(0, 2, n, dtype=F16)
    q, s, rstd, total = torch.empty(m, n, dtype=E4M3, device="cuda"), empty(m, 32), empty(m), torch.empty_like(h)
    wn = rnd(1, n, dtype=F16, mean=1.0)
    ops.rms_norm(h, wn, None, rstd, residual=h, total=total, q=q, q_scale=s)
    ref.check_rms(h[-2:], wn, 1e-5, h[-2:], total[-2:], None, rstd[-2:], q[-2:], s[-2:])
    for block in (ROWS, COLUMNS, SQUARES):
        s = scales(m, n, block)
        ops.quantize(h, q, s)
        last = m // 128 * 128 - 128
        ref.check_quantize(h[last:], q[last:], s[last // block[0]:], block)


# -- again, streams, graphs, the host -----------------------------------------------------------


def test_calls_again_with_other_arrays():
    """The native table's calls: other addresses, and every argument that makes another call of one shape."""
    m, k, n = 9, 400, 136
    for turn in range(3):
        x, xs, xv = operand(turn, m, k, ROWS, "rows")
        w, ws, wv = operand(turn + 9, k, n, SQUARES, "columns")
        y, b = empty(m, n, dtype=BF16), rnd(turn, n, dtype=BF16)
        for a in ("none", "silu"):
            ops.linear_fp8(x, xs, w, ws, y, activation=a, bias=b)
            ref.check_linear_fp8(xv, wv, y, b, None, a)
        v, r, wn = rnd(turn, m, k, dtype=F16), rnd(turn + 1, m, k, dtype=F16), rnd(turn + 2, k, dtype=F16)
        for eps in (1e-5, 0.1):
            out, q, s = empty(m, k, dtype=F16), empty(m, k, dtype=E4M3), scales(m, k)
            ops.rms_norm(v, wn, out, q=q, q_scale=s, eps=eps)
            ref.check_rms(v, wn, eps, y=out, q=q, q_scale=s)
            ops.rms_norm(v, wn, out, residual=r, eps=eps)
            ref.check_rms(v, wn, eps, r, y=out)
        rstd = (v.float().square().mean(1) + 1e-5).rsqrt()
        for over in (False, True):  # of one shape, but read and written in other ways
            dy, dw = rnd(turn + 3, m, k, dtype=F16), empty(k, dtype=F16)
            dx = dy.clone() if over else empty(m, k, dtype=F16)
            ops.rms_norm_backward(dx if over else dy, v, wn, rstd, dx, dw)
            ref.check_rms_backward(dy, v, wn, rstd, dx, dw)
        for block in (ROWS, COLUMNS, SQUARES):
            for a in ("none", "relu"):
                q, s = empty(m, k, dtype=E4M3), scales(m, k, block)
                ops.quantize(v, q, s, activation=a)
                ref.check_quantize(v, q, s, block, None, a)


def test_on_another_stream():
    side = torch.cuda.Stream()
    x, w = rnd(0, 500, 3000, dtype=BF16), rnd(1, 3000, dtype=BF16)
    wq, ws, wv = operand(1, 3000, 700, SQUARES, "columns")
    q, s, y, ready = empty(500, 3000, dtype=E4M3), scales(500, 3000), empty(500, 700, dtype=BF16), torch.cuda.Event()
    ready.record()
    with torch.cuda.stream(side):
        side.wait_event(ready)
        ops.rms_norm(x, w, q=q, q_scale=s, _sync=False)
        ops.linear_fp8(q, s, wq, ws, y, _sync=False)
    side.synchronize()
    ref.check_rms(x, w, 1e-5, q=q, q_scale=s)
    ref.check_linear_fp8(ref.values(q, s, ROWS), wv, y)


def test_captured_and_replayed():
    """Norm, products with a split k and with copies, and conversions in one graph, replayed on other inputs among eager work."""
    m, k, n = 130, 1031, 300
    x, res, w = rnd(0, m, k, dtype=BF16), rnd(1, m, k, dtype=BF16), rnd(2, k, dtype=BF16)
    wq, ws, wv = operand(1, k, n, SQUARES, "columns")
    lq, ls, lv = operand(2, 8192, 64, SQUARES, "columns")
    b, bs, bv = operand(3, m, 8192, ROWS, "rows")
    q, s, total, rstd = empty(m, k, dtype=E4M3), scales(m, k), empty(m, k, dtype=BF16), empty(m)
    y, qc, sc, long = empty(m, n, dtype=BF16), empty(m, n, dtype=E4M3), scales(m, n, COLUMNS), empty(m, 64)
    dx, dw = empty(m, k, dtype=BF16), empty(k, dtype=BF16)

    def work():
        ops.rms_norm(x, w, None, rstd, residual=res, total=total, q=q, q_scale=s, _sync=False)
        ops.linear_fp8(q, s, wq, ws, y, _sync=False)
        ops.quantize(y, qc, sc, activation="silu", _sync=False)
        ops.linear_fp8(b, bs, lq, ls, long, _sync=False)
        ops.rms_norm_backward(x, total, w, rstd, dx, dw, dtotal=res, _sync=False)

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for turn in range(3):
        x.copy_(rnd(10 + turn, m, k, dtype=BF16))
        for t in (y, long, dx, dw, total):
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        ref.check_rms(x, w, 1e-5, res, total, None, rstd, q, s)
        ref.check_linear_fp8(ref.values(q, s, ROWS), wv, y)
        ref.check_quantize(y, qc, sc, COLUMNS, None, "silu")
        ref.check_linear_fp8(bv, lv, long)
        ref.check_rms_backward(x, total, w, rstd, dx, dw, res)
        got = y.clone()
        work()  # eager, the same inputs
        torch.cuda.synchronize()
        assert torch.equal(got, y)


def test_two_graphs_share_nothing():
    """Two captured products with scratch, replayed in turns and together."""
    side = torch.cuda.Stream()
    cases, graphs = [], []
    for i in range(2):
        x, xs, xv = operand(i, 40, 8193, ROWS, "rows")
        w, ws, wv = operand(i + 5, 8193, 50, SQUARES, "columns")
        y = empty(40, 50, dtype=BF16)
        ops.linear_fp8(x, xs, w, ws, y)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.linear_fp8(x, xs, w, ws, y, _sync=False)
        cases.append((x, xs, w, ws, xv, wv, y))
        graphs.append(g)
    for _ in range(3):
        for c in cases:
            c[-1].fill_(float("nan"))
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for c in cases:
            ref.check_linear_fp8(c[4], c[5], c[6])


def test_a_call_that_waits_is_refused_in_a_graph():
    x, q, s = rnd(0, 4, 256), empty(4, 256, dtype=E4M3), scales(4, 256)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(ValueError, match="_sync=False"):
            ops.quantize(x, q, s)
        ops.quantize(x, q, s, _sync=False)
    g.replay()
    torch.cuda.synchronize()
    ref.check_quantize(x, q, s, ROWS)


def test_host_arrays():
    x, w = np.random.default_rng(0).standard_normal((6, 300), dtype=np.float32), np.ones(300, np.float32)
    y, rstd, s = np.zeros_like(x), np.zeros(6, np.float32), np.zeros((6, 3), np.float32)
    q = torch.zeros(6, 300, dtype=torch.uint8).view(E4M3)
    ops.rms_norm(x, w, y, rstd, q=q, q_scale=s)
    t = torch.from_numpy
    ref.check_rms(t(x), t(w), 1e-5, y=t(y), rstd=t(rstd), q=q, q_scale=t(s))
    wq, ws = ref.make(torch.randn(300, 40, generator=torch.Generator().manual_seed(1)), SQUARES)
    out = np.zeros((6, 40), np.float32)
    ops.linear_fp8(q, s, wq, ws, out)
    ref.check_linear_fp8(ref.values(q, t(s), ROWS), ref.values(wq, ws, SQUARES), t(out))
    sc, qc = np.zeros((1, 300), np.float32), torch.zeros(6, 300, dtype=torch.uint8).view(E4M3)
    ops.quantize(x, qc, sc)
    ref.check_quantize(t(x), qc, t(sc), COLUMNS)
    dx, dw = np.zeros_like(x), np.zeros_like(w)
    ops.rms_norm_backward(y, x, w, rstd, dx, dw)
    ref.check_rms_backward(t(y), t(x), t(w), t(rstd), t(dx), t(dw))


def test_the_same_on_every_run():
    """Sums over rows and split ranges of k are added in one order."""
    x, w, rstd = rnd(0, 3000, 1500, dtype=BF16), rnd(1, 1500, dtype=BF16), rnd(2, 3000).abs()
    a, as_, _ = operand(3, 70, 9000, ROWS, "rows")
    b, bs, _ = operand(4, 9000, 80, SQUARES, "columns")
    first = None
    for _ in range(4):
        dx, dw, y = empty(3000, 1500, dtype=BF16), empty(1500, dtype=BF16), empty(70, 80)
        ops.rms_norm_backward(x, x, w, rstd, dx, dw)
        ops.linear_fp8(a, as_, b, bs, y)
        if first is None:
            first = (dx, dw, y)
        assert all(torch.equal(p, q) for p, q in zip(first, (dx, dw, y)))


def test_refusals_on_the_gpu():
    x, q, s = rnd(0, 8, 256), empty(8, 256, dtype=E4M3), scales(8, 256)
    for call, error in ((lambda: ops.quantize(x, q, s[:, :1]), ValueError), (lambda: ops.quantize(x, q.view(torch.uint8), s), TypeError),
                        (lambda: ops.quantize(x, x.view(torch.uint8).view(E4M3)[:, :256], s), ValueError),
                        (lambda: ops.rms_norm(x, None, x[:, :], q=q, q_scale=s.expand(8, 2)[:, :1].expand(8, 2)), ValueError),
                        (lambda: ops.linear_fp8(q, s, empty(256, 8, dtype=E4M3), scales(256, 8, SQUARES), x[:, :8]), None),
                        (lambda: ops.linear_fp8(q, s, q.t(), scales(256, 8, SQUARES), s.view(-1)[:16].view(8, 2)), ValueError)):
        if error is None:
            call()
        else:
            with pytest.raises(error):
                call()


# -- a feed-forward block in 8 bits ------------------------------------------------------------------


def both(v: torch.Tensor, block):
    q, s = empty(*v.shape, dtype=E4M3), scales(*v.shape, block)
    ops.quantize(v, q, s, _sync=False)
    return q, s


@pytest.mark.parametrize("m", [1, 48, 200])
def test_a_feed_forward_block(m):
    """out = total + down(silu(gate(h)) * up(h)), h = norm(x + residual), all operands in 8 bits, forward and backward: each step
    against its definition in 64 bits on what the step before it left."""
    width, hidden = 384, 640
    x, res, wn = rnd(0, m, width, dtype=BF16), rnd(1, m, width, dtype=BF16), rnd(2, width, dtype=BF16, mean=1.0)
    wg, wgs = both(rnd(3, 2 * hidden, width, scale=width ** -0.5), SQUARES)  # gate over up, [outputs, inputs]
    wd, wds = both(rnd(4, width, hidden, scale=hidden ** -0.5), SQUARES)
    gv, dv = ref.values(wg, wgs, SQUARES), ref.values(wd, wds, SQUARES)
    total, rstd, h, hs, h16 = empty(m, width, dtype=BF16), empty(m), empty(m, width, dtype=E4M3), scales(m, width), empty(m, width, dtype=BF16)
    ops.rms_norm(x, wn, h16, rstd, residual=res, total=total, q=h, q_scale=hs, _sync=False)
    gu = empty(m, 2 * hidden, dtype=BF16)
    ops.linear_fp8(h, hs, wg.t(), wgs.t(), gu, _sync=False)
    a, as_ = empty(m, hidden, dtype=E4M3), scales(m, hidden)
    ops.quantize(gu[:, hidden:], a, as_, gate=gu[:, :hidden], activation="silu", _sync=False)
    out = empty(m, width, dtype=BF16)
    ops.linear_fp8(a, as_, wd.t(), wds.t(), out, residual=total, _sync=False)
    torch.cuda.synchronize()
    ref.check_rms(x, wn, 1e-5, res, total, h16, rstd, h, hs)
    ref.check_linear_fp8(ref.values(h, hs, ROWS), gv.t(), gu)
    ref.check_quantize(gu[:, hidden:], a, as_, ROWS, gu[:, :hidden], "silu")
    ref.check_linear_fp8(ref.values(a, as_, ROWS), dv.t(), out, residual=total)

    dy = rnd(5, m, width, dtype=BF16)
    dq, ds = both(dy, ROWS)
    da = empty(m, hidden, dtype=BF16)
    ops.linear_fp8(dq, ds, wd, wds, da, _sync=False)  # dy @ down, as it is stored
    dqc, dsc = both(dy, COLUMNS)
    act_ = (act(d(gu[:, :hidden]), "silu") * d(gu[:, hidden:])).to(BF16).cuda()
    ac, acs = both(act_, COLUMNS)
    dwd = empty(width, hidden)
    ops.linear_fp8(dqc.t(), dsc.t(), ac, acs, dwd, _sync=False)
    g, u, t = d(gu[:, :hidden]), d(gu[:, hidden:]), d(da)
    dgu = torch.cat([t * u * act_grad(g, "silu"), t * act(g, "silu")], 1).to(BF16).cuda()
    gq, gs = both(dgu, ROWS)
    dh = empty(m, width, dtype=BF16)
    ops.linear_fp8(gq, gs, wg, wgs, dh, _sync=False)
    dx, dwn = empty(m, width, dtype=BF16), empty(width, dtype=BF16)
    ops.rms_norm_backward(dh, total, wn, rstd, dx, dwn, dtotal=dy, _sync=False)
    torch.cuda.synchronize()
    ref.check_linear_fp8(ref.values(dq, ds, ROWS), dv, da)
    ref.check_linear_fp8(ref.values(dqc, dsc, COLUMNS).t(), ref.values(ac, acs, COLUMNS), dwd)
    ref.check_linear_fp8(ref.values(gq, gs, ROWS), gv, dh)
    ref.check_rms_backward(dh, total, wn, rstd, dx, dwn, dy)


@pytest.mark.parametrize("at", [0, 5])
def test_one_tokens_scales_among_those_of_others(at):
    """Scales kept as [blocks, tokens], of which a call writes one token's."""
    n, kept = 1100, torch.full((9, 8), 3.0, device="cuda")
    x, w, up = rnd(0, 1, n, dtype=BF16), rnd(1, n, dtype=BF16), rnd(2, 1, n, dtype=BF16)
    for call in (lambda q, s: ops.rms_norm(x, w, q=q, q_scale=s), lambda q, s: ops.quantize(up, q, s, gate=x, activation="relu")):
        q, s, same = empty(1, n, dtype=E4M3), kept.t()[at:at + 1], empty(1, n, dtype=E4M3)
        alone = scales(1, n)
        call(q, s)
        call(same, alone)
        assert torch.equal(s, alone) and torch.equal(q.view(torch.uint8), same.view(torch.uint8))
        assert bool((kept[:, [c for c in range(8) if c != at]] == 3).all())
