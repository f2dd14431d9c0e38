"""The operators around 8-bit operands from their definitions in 64 bits, and how far a kernel may be from them.

Bounds as in ops_reference: a sum of K terms kept in 32 bits is off by at most (K + 8) 2^-23 of the sum of
their magnitudes, a result rounded to its type by half a unit.
"""

from __future__ import annotations

import torch

from ops_reference import ACT_ERROR, SLOPE, act, check, d, gamma

E4M3 = torch.float8_e4m3fn
BLOCK = 128
LEAST = 2.0 ** -126


def blocks(n: int, b: int = BLOCK) -> int:
    return -(-n // b)


def spread(scale: torch.Tensor, shape, block) -> torch.Tensor:
    """Each element's scale."""
    return scale.repeat_interleave(block[0], 0)[: shape[0]].repeat_interleave(block[1], 1)[:, : shape[1]]


def amax(v: torch.Tensor, block) -> torch.Tensor:
    """The largest finite magnitude of each block."""
    m, n = v.shape
    a, b = block
    p = torch.zeros(blocks(m, a) * a, blocks(n, b) * b, dtype=v.dtype, device=v.device)
    p[:m, :n] = torch.where(v.isfinite(), v.abs(), torch.zeros_like(v))
    return p.view(blocks(m, a), a, blocks(n, b), b).amax((1, 3))


def to_e4m3(v: torch.Tensor) -> torch.Tensor:
    """Values in 64 bits to the nearest e4m3 value, ties to even: four significant bits, multiples of 2^-9 at least."""
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp(min=2.0 ** -6))[1] - 4)
    q = (torch.round(v / step) * step).clamp(-448, 448)
    return torch.where(v.isfinite(), q, torch.full_like(q, float("nan")))


def make(v: torch.Tensor, block) -> tuple[torch.Tensor, torch.Tensor]:
    """An operand in 8 bits and its scales, on v's device, for a product's test."""
    f = v.double()
    scale = (amax(f, block) / 448).clamp(min=LEAST).float()
    return to_e4m3(f / spread(scale.double(), f.shape, block)).float().to(E4M3), scale


def check_fp8(name: str, v: torch.Tensor, slack: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, block) -> None:
    """q and scale against v in 64 bits, which the kernel has within `slack`.

    The scale is the largest magnitude's, as far off as any value of the block and two roundings.  An element is the
    nearest e4m3 value of its quotient by the kernel's own scale, within the quotient's own error: v's, and 2^-22 of
    itself for the division.  The two ends of that interval round to the only values it may have."""
    s, g = scale.detach().cpu().double(), q.detach().cpu().float().double()
    finite = torch.where(v.isfinite(), slack, torch.zeros_like(slack))
    want = (amax(v, block) / 448).clamp(min=LEAST)
    off = amax(finite, block) / 448 + 2.0 ** -22 * want
    assert s.shape == want.shape, (name, s.shape, want.shape)
    assert bool(((s - want).abs() <= off).all()), f"{name}: scale off by {((s - want).abs() / want).max().item():.3g}"
    each = spread(s, v.shape, block)
    t = v / each
    e = slack / each + 2.0 ** -22 * t.abs()
    low, high = to_e4m3(t - e), to_e4m3(t + e)
    fine = torch.where(v.isfinite(), (g >= low) & (g <= high), g.isnan())
    if not bool(fine.all()):
        at = tuple(int(i) for i in (~fine).nonzero()[0])
        raise AssertionError(f"{name}{list(at)}: got {g[at].item()!r}, want {low[at].item()!r}..{high[at].item()!r} of {t[at].item()!r} "
                             f"({int((~fine).sum())} of {fine.numel()} off)")


# -- root-mean-square norm --------------------------------------------------------------


def check_rms(x, w, eps, residual=None, total=None, y=None, rstd=None, q=None, q_scale=None):
    h = d(x) + (0 if residual is None else d(residual))
    n = x.shape[1]
    r = (h.square().mean(1) + eps) ** -0.5
    # h is rounded to 32 bits, its squares' sum is positive, and a square root halves what it carries
    e_h = 2.0 ** -24 * h.abs()
    e_r = r * (gamma(n) + 2.0 ** -21)
    if total is not None:
        check("total", total, h, e_h)
    if rstd is not None:
        check("rstd", rstd, r, e_r)
    want = h * r[:, None] * (1 if w is None else d(w))
    slack = want.abs() * ((e_r / r)[:, None] + 2.0 ** -21)
    if y is not None:
        check("y", y, want, slack)
    if q is not None:
        check_fp8("q", want, slack, q, q_scale, (1, BLOCK))


def check_rms_backward(dy, h, w, rstd, dx=None, dw=None, dtotal=None):
    t, h_, r = d(dy), d(h), d(rstd)
    m, n = h_.shape
    g = t * (1 if w is None else d(w))
    if dx is not None:
        b = r[:, None] ** 3 * (g * h_).mean(1, keepdim=True)
        big = r[:, None] ** 3 * (g * h_).abs().mean(1, keepdim=True)
        norm = g * r[:, None] - h_ * b
        add = 0 if dtotal is None else d(dtotal)
        slack = h_.abs() * big * (gamma(n) + 2.0 ** -20) + 2.0 ** -21 * ((g * r[:, None]).abs() + (norm + add).abs())
        check("dx", dx, norm + add, slack)
    if dw is not None:
        each = t * h_ * r[:, None]
        check("dweight", dw, each.sum(0), (gamma(m) + 2.0 ** -21) * each.abs().sum(0))


# -- conversion ---------------------------------------------------------------------------


def check_quantize(x, q, scale, block, gate=None, activation="none"):
    v = d(x)
    if gate is None:
        a = act(v, activation)
        slack = torch.zeros_like(v) if activation == "none" else ACT_ERROR * v.abs()
    else:
        z = d(gate)
        a = act(z, activation) * v
        slack = (torch.zeros_like(v) if activation == "none" else ACT_ERROR * (z * v).abs()) + 2.0 ** -23 * a.abs()
    slack = torch.where(a.isfinite(), slack, torch.zeros_like(slack))
    check_fp8("q", a, slack, q, scale, block)


# -- product --------------------------------------------------------------------------------


def values(q, scale, block):
    """What an 8-bit matrix stands for."""
    return q.detach().cpu().float().double() * spread(scale.detach().cpu().double(), q.shape, block)


def eights(x, w):
    """The largest magnitude of the products of each eight along k, summed over those."""
    m, k = x.shape
    out = torch.zeros(m, w.shape[1], dtype=x.dtype)
    for a in range(0, k, 8):
        most = torch.zeros_like(out)
        for i in range(a, min(a + 8, k)):
            most = torch.maximum(most, x[:, i, None].abs() * w[None, i].abs())
        out += most
    return out


def check_linear_fp8(x, w, y, bias=None, residual=None, activation="none", pre=None):
    """x, w: what the operands stand for, in 64 bits.  Products of 8-bit values are exact; each of the sums' terms meets
    two roundings of the scales' products besides those of the sum.  Where y is 16 bits, the matrix cores cut the products
    of each eight along k off at 2^-14 of the largest one's power of two, which is at most its magnitude."""
    k = x.shape[1]
    z = x @ w + (0 if bias is None else d(bias))
    e = (gamma(k) + 2.0 ** -21) * (x.abs() @ w.abs() + (0 if bias is None else d(bias).abs()))
    if y.dtype != torch.float32 and k:
        e = e + 8 * 2.0 ** -14 * eights(x, w)
    if pre is not None:
        check("pre", pre, z, e)
    want = act(z, activation)
    slack = e if activation == "none" else SLOPE * e + ACT_ERROR * z.abs()
    if residual is not None:
        want = want + d(residual)
        slack = slack + 2.0 ** -23 * want.abs()
    check("y", y, want, slack)
