"""The feed-forward operators from their definitions in 64 bits, and how far a kernel may be from them.

Every bound is the rounding analysis of the operation in question, worst case over the data: a sum of K
products kept in 32 bits is off by at most (K + 8) 2^-23 of the sum of their magnitudes (the matrix
units may truncate), a result rounded to its type by half a unit, and an intermediate rounded to 16
bits carries half a unit of each term into the sums that read it.
"""

from __future__ import annotations

import math

import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}
SLOPE = 1.13  # no activation is steeper
# of z: the formula for erf is within 1.5e-7, exponentials and reciprocals within a few units of 2^-24
ACT_ERROR = 1e-6


def act(z: torch.Tensor, name: str) -> torch.Tensor:
    if name == "none":
        return z.clone()
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    c = math.sqrt(2 / math.pi)
    return 0.5 * z * (1 + torch.tanh(c * (z + 0.044715 * z ** 3)))


def act_grad(z: torch.Tensor, name: str) -> torch.Tensor:
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def gamma(k: int) -> float:
    return (k + 8) * 2.0 ** -23


def check(name: str, got: torch.Tensor, want: torch.Tensor, slack: torch.Tensor) -> None:
    """|got - want| within half a unit of got's type and `slack`, element by element; NaN where want is NaN."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    g = got.detach().cpu().double()
    tol = UNIT[got.dtype] * (want.abs() + slack) + slack + TINY[got.dtype]
    same = (g == want) | (g.isnan() & want.isnan())
    bad = ~(same | ((g - want).abs() <= tol))
    if bad.any():
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{name}{list(at)}: got {g[at].item()!r}, want {want[at].item()!r} +- {tol[at].item():.3g} "
                             f"({int(bad.sum())} of {bad.numel()} off)")


def d(t: torch.Tensor | None) -> torch.Tensor | None:
    return None if t is None else t.detach().cpu().double()


# -- layer norm -----------------------------------------------------------------


def norm(x, w, b, eps):
    x = d(x)
    mean = x.mean(1)
    var = (x - mean[:, None]).square().mean(1)
    rstd = (var + eps) ** -0.5
    xh = (x - mean[:, None]) * rstd[:, None]
    y = xh * (1 if w is None else d(w)) + (0 if b is None else d(b))
    return y, mean, rstd, xh


def check_norm(x, w, b, eps, y, mean=None, rstd=None):
    want, m, r, xh = norm(x, w, b, eps)
    n = x.shape[1]
    big = d(x).abs().mean(1)
    e_mean = gamma(n) * big                                          # of the mean
    # the centred sum of squares: each term relative, and the mean's error moves it by its square only
    e_rstd = r * (gamma(n) + 2.0 ** -21) + r ** 3 * e_mean.square()
    if mean is not None:
        check("mean", mean, m, e_mean)
    if rstd is not None:
        check("rstd", rstd, r, e_rstd)
    slack = (xh.abs() * (e_rstd / r + 2.0 ** -22)[:, None] + (e_mean * r)[:, None]
             + 2.0 ** -23 * d(x).abs() * r[:, None])
    check("y", y, want, slack * (1 if w is None else d(w).abs()) + 2.0 ** -23 * want.abs())


def norm_backward(dy, x, w, mean, rstd):
    dy, x, mean, rstd = d(dy), d(x), d(mean), d(rstd)
    xh = (x - mean[:, None]) * rstd[:, None]
    g = dy * (1 if w is None else d(w))
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0), xh, g


def check_norm_backward(dy, x, w, mean, rstd, dx=None, dw=None, db=None):
    want, wdw, wdb, xh, g = norm_backward(dy, x, w, mean, rstd)
    m, n = x.shape
    e_xh = 2.0 ** -22 * (xh.abs() + (d(x).abs() + d(mean).abs()[:, None]) * d(rstd).abs()[:, None])
    if dx is not None:
        a = g.abs().mean(1, keepdim=True)
        b = (g * xh).abs().mean(1, keepdim=True)
        e_b = gamma(n) * b + (g.abs() * e_xh).mean(1, keepdim=True)
        slack = d(rstd).abs()[:, None] * (2.0 ** -21 * (g.abs() + a + xh.abs() * b) + gamma(n) * a + xh.abs() * e_b + e_xh * b)
        check("dx", dx, want, slack)
    if dw is not None:
        check("dweight", dw, wdw, gamma(m) * (d(dy) * xh).abs().sum(0) + (d(dy).abs() * e_xh).sum(0))
    if db is not None:
        check("dbias", db, wdb, gamma(m) * d(dy).abs().sum(0))


# -- linear ------------------------------------------------------------------------


def product(x, w, b):
    """x @ w + b and the error of its sums."""
    x, w = d(x), d(w)
    z = x @ w + (0 if b is None else d(b))
    return z, gamma(x.shape[1]) * (x.abs() @ w.abs() + (0 if b is None else d(b).abs()))


def check_linear(x, w, y, bias=None, residual=None, activation="none", pre=None):
    z, e = product(x, w, bias)
    if pre is not None:
        check("pre", pre, z, e)
    want = act(z, activation)
    slack = e if activation == "none" else SLOPE * e + ACT_ERROR * z.abs()
    if residual is not None:
        want = want + d(residual)
        slack = slack + 2.0 ** -23 * want.abs()
    check("y", y, want, slack)


def dz_error(dy, factor, z, dtype):
    """The error of dy * factor: of the activation's slope, and of its rounding to 16 bits."""
    dz = dy * factor
    e = dy.abs() * (ACT_ERROR * (1 + z.abs() + z.square())) + 2.0 ** -22 * dz.abs()
    return e, e + (UNIT[dtype] * (dz.abs() + e) + TINY[dtype] if dtype != torch.float32 else 0)


def check_products(dzs, errors, x, ws, dx, dws):
    """dx and dws from dz's in 64 bits, each of which the kernel has within `errors`."""
    k_dx = sum(dz.shape[1] for dz in dzs)
    if dx is not None:
        want = sum(dz @ d(w).t() for dz, w in zip(dzs, ws))
        slack = sum(gamma(k_dx) * (dz.abs() @ d(w).t().abs()) + (1 + gamma(k_dx)) * (e @ d(w).t().abs()) for dz, w, e in zip(dzs, ws, errors))
        check("dx", dx, want, slack)
    for dz, e, dw in zip(dzs, errors, dws):
        if dw is not None:
            xt = d(x).t()
            g = gamma(dz.shape[0])
            check("dw", dw, xt @ dz, g * (xt.abs() @ dz.abs()) + (1 + g) * (xt.abs() @ e))


def check_linear_backward(dy, x, w, dx=None, dw=None, dbias=None, activation="none", pre=None):
    g = d(dy)
    if activation == "none":
        dz, e, e16 = g, torch.zeros_like(g), torch.zeros_like(g)
    else:
        z = d(pre)
        dz = g * act_grad(z, activation)
        e, e16 = dz_error(g, act_grad(z, activation), z, dy.dtype)
    check_products([dz], [e16], x, [w], dx, [dw])
    if dbias is not None:
        check("dbias", dbias, dz.sum(0), gamma(dz.shape[0]) * dz.abs().sum(0) + e.sum(0))


# -- gated linear ------------------------------------------------------------------


def check_gated(x, wg, wu, y, bias_gate=None, bias_up=None, activation="silu", gate=None, up=None):
    g, eg = product(x, wg, bias_gate)
    u, eu = product(x, wu, bias_up)
    if gate is not None:
        check("gate", gate, g, eg)
        check("up", up, u, eu)
    f = act(g, activation)
    ef = SLOPE * eg + ACT_ERROR * g.abs()
    check("y", y, f * u, ef * u.abs() + f.abs() * eu + ef * eu + 2.0 ** -23 * (f * u).abs())


def check_gated_backward(dy, x, wg, wu, gate, up, dx=None, dw_gate=None, dw_up=None, dbias_gate=None, dbias_up=None,
                         activation="silu"):
    t, g, u = d(dy), d(gate), d(up)
    dg, du = t * u * act_grad(g, activation), t * act(g, activation)
    eg, eg16 = dz_error(t * u, act_grad(g, activation), g, dy.dtype)
    eu, eu16 = dz_error(t, act(g, activation), g, dy.dtype)
    check_products([dg, du], [eg16, eu16], x, [wg, wu], dx, [dw_gate, dw_up])
    for dz, e, db in ((dg, eg, dbias_gate), (du, eu, dbias_up)):
        if db is not None:
            check("dbias", db, dz.sum(0), gamma(dz.shape[0]) * dz.abs().sum(0) + e.sum(0))
