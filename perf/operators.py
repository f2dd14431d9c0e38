"""The feed-forward operators' calls, for timing: layer norm, the matrix product with its
epilogue and the gated pair of projections, forward and backward.

A case is one call of a user's program on torch GPU tensors, with the outputs that the program
keeps from step to step.  ``op`` names the operator, ``rows`` is the number of tokens, ``k`` and
``n`` are the lengths of an input and an output row (``k`` alone for the norm), ``dtype`` the
operands' type; ``wt`` says that weights lie as [n, k] and are passed as their transposed view.

``run`` calls the framework's operators where ``own`` is true; elsewhere it computes the same in
elementary torch operations in 32 bits, each output rounded once.  ``listed()`` holds the standing
cases, ``draw(rng)`` gives another one of the same ranges.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # one token of a decoding step through the norm before a feed-forward block: latency
        {"name": "norm 1x4096 f16", "op": "norm", "rows": 1, "k": 4096, "dtype": "f16", "stats": False},
        # a long prompt or a training batch through the same norm, its statistics kept for the backward pass
        {"name": "norm 8192x4096 bf16", "op": "norm", "rows": 8192, "k": 4096, "dtype": "bf16", "stats": True},
        # the norm's backward pass in a training step: dx and the reductions for weight and bias
        {"name": "norm bwd 8192x4096 bf16", "op": "norm_bwd", "rows": 8192, "k": 4096, "dtype": "bf16"},
        # the same in fp32, on a ragged batch whose rows end off every alignment
        {"name": "norm bwd 1031x4099 f32", "op": "norm_bwd", "rows": 1031, "k": 4099, "dtype": "f32"},
        # one token through a block's down projection, added to its residual stream: the weights are all the bytes
        {"name": "linear 1x14336x4096 f16", "op": "linear", "rows": 1, "k": 14336, "n": 4096, "dtype": "f16",
         "wt": False, "bias": False, "residual": True, "act": "none", "pre": False},
        # a prompt's tokens through a projection with bias and gelu, the pre-activation kept for training
        {"name": "linear 4096x4096x4096 bf16", "op": "linear", "rows": 4096, "k": 4096, "n": 4096, "dtype": "bf16",
         "wt": False, "bias": True, "residual": False, "act": "gelu", "pre": True},
        # that projection's backward pass on a training batch: the input's, the weights' and the bias's gradients
        {"name": "linear bwd 4096x4096x4096 bf16", "op": "linear_bwd", "rows": 4096, "k": 4096, "n": 4096,
         "dtype": "bf16", "wt": False, "bias": True, "act": "gelu"},
        # a small model's backward pass with odd widths and a ragged batch, weights kept as [n, k]
        {"name": "linear bwd 517x1023x2047 f16", "op": "linear_bwd", "rows": 517, "k": 1023, "n": 2047,
         "dtype": "f16", "wt": True, "bias": True, "act": "gelu_tanh"},
        # a decoding step of sixteen sequences through the gated projections
        {"name": "gated 16x4096x14336 f16", "op": "gated", "rows": 16, "k": 4096, "n": 14336, "dtype": "f16",
         "wt": False, "bias": False, "act": "silu", "save": False},
        # a training batch through them, both pre-activations kept
        {"name": "gated 2048x4096x14336 bf16", "op": "gated", "rows": 2048, "k": 4096, "n": 14336, "dtype": "bf16",
         "wt": False, "bias": False, "act": "silu", "save": True},
        # and its backward pass: the most work of a block's training step
        {"name": "gated bwd 2048x4096x14336 bf16", "op": "gated_bwd", "rows": 2048, "k": 4096, "n": 14336,
         "dtype": "bf16", "wt": False, "bias": False, "act": "silu"},
        # a small fp32 model checked in full precision, odd sizes, with biases
        {"name": "gated bwd 300x512x1031 f32", "op": "gated_bwd", "rows": 300, "k": 512, "n": 1031,
         "dtype": "f32", "wt": False, "bias": True, "act": "gelu"},
    ]


def _size(rng, lo, hi):
    """A size of [lo, hi], even in its logarithm: half of them as they fall, half on a multiple of 8."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 8:
        v = v // 8 * 8
    v = min(hi, max(lo, v))
    return v + 1 if v == 3072 else v


def _cost(case):
    """Rough microseconds of a pass at this card's rates, to keep draws within the listed range."""
    w = work(case)
    return w["flops"] / (1e8 if case["dtype"] == "f32" else 1e9) + w["bytes"] / 5e6


def draw(rng):
    op = rng.choice(["norm", "norm_bwd", "linear", "linear_bwd", "gated", "gated_bwd"])
    most = max(_cost(c) for c in listed() if c["op"] in (op, "gated_bwd"))
    while True:
        case = {"op": op, "rows": _size(rng, 1, 8192), "k": _size(rng, 64, 14336),
                "dtype": rng.choice(["f16", "bf16", "bf16", "f32"])}
        if op == "norm":
            case["stats"] = rng.random() < 0.5
        elif op != "norm_bwd":
            case["n"] = _size(rng, 64, 14336)
            case["wt"] = rng.random() < 0.3
            case["bias"] = rng.random() < 0.5
            case["act"] = rng.choice(["silu", "gelu", "gelu_tanh", "relu"] if op.startswith("gated")
                                     else ["none", "relu", "gelu", "gelu_tanh", "silu"])
            if op == "linear":
                case["residual"] = rng.random() < 0.5
                case["pre"] = case["act"] != "none" and rng.random() < 0.5
            elif op == "gated":
                case["save"] = rng.random() < 0.5
        if _cost(case) <= most:
            return case


def work(case):
    m, k, e = case["rows"], case["k"], BYTES[case["dtype"]]
    op = case["op"]
    if op == "norm":
        return {"bytes": 2 * m * k * e + 2 * k * e + (8 * m if case["stats"] else 0), "flops": 8 * m * k}
    if op == "norm_bwd":
        return {"bytes": 3 * m * k * e + 3 * k * e + 8 * m, "flops": 14 * m * k}
    n = case["n"]
    xs, ws, ys, bs = m * k * e, k * n * e, m * n * e, (n * e if case["bias"] else 0)
    if op == "linear":
        return {"bytes": xs + ws + ys * (1 + case["residual"] + case["pre"]) + bs, "flops": 2 * m * k * n}
    if op == "linear_bwd":
        return {"bytes": 2 * xs + 2 * ws + ys * (1 + (case["act"] != "none")) + bs, "flops": 4 * m * k * n}
    if op == "gated":
        return {"bytes": xs + 2 * ws + ys * (3 if case["save"] else 1) + 2 * bs, "flops": 4 * m * k * n}
    return {"bytes": 2 * xs + 4 * ws + 3 * ys + 2 * bs, "flops": 8 * m * k * n}


# -- inputs -------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, m, k, n, op = DTYPES[case["dtype"]], case["rows"], case["k"], case.get("n", 0), case["op"]

    def normal(*shape, scale=1.0, mean=0.0, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).add_(mean).to(dtype)

    def weights():
        w = normal(n, k, scale=k ** -0.5) if case["wt"] else normal(k, n, scale=k ** -0.5)
        return w.t() if case["wt"] else w

    def like(t):
        return torch.empty_strided(t.shape, t.stride(), device=t.device, dtype=t.dtype)

    s = {"case": case}
    if op in ("norm", "norm_bwd"):
        # a residual stream: a mean that is not zero, and a few columns much larger than the others
        x = normal(m, k, scale=1.5, mean=0.2, dtype=torch.float32)
        x[:, :: max(1, k // 8)] *= 12.0
        s["x"] = x.to(dt)
        s["w"], s["b"] = normal(k, scale=0.1, mean=1.0), normal(k, scale=0.1)
        if op == "norm":
            s["y"] = torch.empty_like(s["x"])
            if case["stats"]:
                s["mean"], s["rstd"] = (torch.empty(m, device="cuda", dtype=torch.float32) for _ in range(2))
        else:
            xf = s["x"].float()
            s["mean"] = xf.mean(1)
            s["rstd"] = torch.rsqrt((xf - s["mean"][:, None]).square().mean(1) + EPS)
            s["dy"], s["dx"], s["dw"], s["db"] = normal(m, k), torch.empty_like(s["x"]), torch.empty_like(s["w"]), torch.empty_like(s["b"])
        return s
    s["x"] = normal(m, k)  # what a norm leaves
    if op in ("linear", "linear_bwd"):
        s["w"] = weights()
        s["b"] = normal(n, scale=0.1) if case["bias"] else None
        if op == "linear":
            s["res"] = normal(m, n) if case["residual"] else None
            s["y"] = torch.empty(m, n, device="cuda", dtype=dt)
            s["pre"] = torch.empty_like(s["y"]) if case["pre"] else None
        else:
            s["dy"] = normal(m, n)
            s["pre"] = normal(m, n) if case["act"] != "none" else None
            s["dx"], s["dw"] = torch.empty_like(s["x"]), like(s["w"])
            s["db"] = torch.empty(n, device="cuda", dtype=dt) if case["bias"] else None
        return s
    s["wg"], s["wu"] = weights(), weights()
    s["bg"], s["bu"] = (normal(n, scale=0.1), normal(n, scale=0.1)) if case["bias"] else (None, None)
    if op == "gated":
        s["y"] = torch.empty(m, n, device="cuda", dtype=dt)
        s["gate"], s["up"] = (torch.empty_like(s["y"]), torch.empty_like(s["y"])) if case["save"] else (None, None)
    else:
        s["dy"], s["gate"], s["up"] = normal(m, n), normal(m, n), normal(m, n)
        s["dx"], s["dwg"], s["dwu"] = torch.empty_like(s["x"]), like(s["wg"]), like(s["wu"])
        s["dbg"], s["dbu"] = (torch.empty(n, device="cuda", dtype=dt) for _ in range(2)) if case["bias"] else (None, None)
    return s


# -- the plain forms ----------------------------------------------------------------


def _act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_grad(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain(s):
    case = s["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    x = s["x"].float()
    if op == "norm":
        mean = x.mean(1, keepdim=True)
        d = x - mean
        rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
        out = {"y": (d * rstd * s["w"].float() + s["b"].float()).to(dt)}
        if case["stats"]:
            out["mean"], out["rstd"] = mean[:, 0], rstd[:, 0]
        return out
    if op == "norm_bwd":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        xhat = (x - s["mean"][:, None]) * rstd
        g = dy * s["w"].float()
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        return {"dx": dx.to(dt), "dw": (dy * xhat).sum(0).to(dt), "db": dy.sum(0).to(dt)}
    if op == "linear":
        z = x @ s["w"].float()
        if s["b"] is not None:
            z = z + s["b"].float()
        y = _act(z, case["act"])
        if s["res"] is not None:
            y = y + s["res"].float()
        return {"y": y.to(dt), **({"pre": z.to(dt)} if case["pre"] else {})}
    if op == "linear_bwd":
        dz = s["dy"].float()
        if case["act"] != "none":
            dz = dz * _act_grad(s["pre"].float(), case["act"])
        out = {"dx": (dz @ s["w"].float().t()).to(dt), "dw": (x.t() @ dz).to(dt)}
        if case["bias"]:
            out["db"] = dz.sum(0).to(dt)
        return out
    if op == "gated":
        a, b = x @ s["wg"].float(), x @ s["wu"].float()
        if case["bias"]:
            a, b = a + s["bg"].float(), b + s["bu"].float()
        return {"y": (_act(a, case["act"]) * b).to(dt), **({"gate": a.to(dt), "up": b.to(dt)} if case["save"] else {})}
    dy, a, b = s["dy"].float(), s["gate"].float(), s["up"].float()
    da, db = dy * b * _act_grad(a, case["act"]), dy * _act(a, case["act"])
    out = {"dx": (da @ s["wg"].float().t() + db @ s["wu"].float().t()).to(dt),
           "dwg": (x.t() @ da).to(dt), "dwu": (x.t() @ db).to(dt)}
    if case["bias"]:
        out["dbg"], out["dbu"] = da.sum(0).to(dt), db.sum(0).to(dt)
    return out


# -- the framework's operators --------------------------------------------------------


def _own(s):
    from easy_as_amd import ops

    case = s["case"]
    op = case["op"]
    if op == "norm":
        if case["stats"]:
            ops.layer_norm(s["x"], s["w"], s["b"], s["y"], s["mean"], s["rstd"], eps=EPS, _sync=False)
            return {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}
        ops.layer_norm(s["x"], s["w"], s["b"], s["y"], eps=EPS, _sync=False)
        return {"y": s["y"]}
    if op == "norm_bwd":
        ops.layer_norm_backward(s["dy"], s["x"], s["w"], s["mean"], s["rstd"], s["dx"], s["dw"], s["db"], _sync=False)
        return {"dx": s["dx"], "dw": s["dw"], "db": s["db"]}
    if op == "linear":
        ops.linear(s["x"], s["w"], s["y"], bias=s["b"], residual=s["res"], activation=case["act"], pre=s["pre"],
                   _sync=False)
        return {"y": s["y"], **({"pre": s["pre"]} if case["pre"] else {})}
    if op == "linear_bwd":
        ops.linear_backward(s["dy"], s["x"], s["w"], dx=s["dx"], dw=s["dw"], dbias=s["db"], activation=case["act"],
                            pre=s["pre"], _sync=False)
        return {"dx": s["dx"], "dw": s["dw"], **({"db": s["db"]} if case["bias"] else {})}
    if op == "gated":
        ops.gated_linear(s["x"], s["wg"], s["wu"], s["y"], bias_gate=s["bg"], bias_up=s["bu"],
                         activation=case["act"], gate=s["gate"], up=s["up"], _sync=False)
        return {"y": s["y"], **({"gate": s["gate"], "up": s["up"]} if case["save"] else {})}
    ops.gated_linear_backward(s["dy"], s["x"], s["wg"], s["wu"], s["gate"], s["up"], dx=s["dx"], dw_gate=s["dwg"],
                              dw_up=s["dwu"], dbias_gate=s["dbg"], dbias_up=s["dbu"], activation=case["act"],
                              _sync=False)
    return {"dx": s["dx"], "dwg": s["dwg"], "dwu": s["dwu"],
            **({"dbg": s["dbg"], "dbu": s["dbu"]} if case["bias"] else {})}


def run(state):
    return _own(state) if own else _plain(state)


# -- 64 bits --------------------------------------------------------------------------


def _phi(z):
    """The normal distribution's integral, and its density."""
    return torch.special.ndtr(z), torch.exp(z * z / -2) / math.sqrt(math.tau)


def _exact_act(z, name):
    """An activation and its derivative in 64 bits."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    if name == "gelu":
        p, d = _phi(z)
        return z * p, p + z * d
    # the tanh form is z sigmoid(2 u), u = sqrt(2/pi) (z + 0.044715 z^3)
    c = math.sqrt(8 / math.pi)
    s = torch.sigmoid(c * (z + 0.044715 * z ** 3))
    return z * s, s + z * s * (1 - s) * c * (1 + 0.134145 * z ** 2)


def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    op, x = case["op"], s["x"]
    if op == "norm":
        var, mean = torch.var_mean(x, dim=1, unbiased=False)
        rstd = (var + EPS) ** -0.5
        out = {"y": torch.addcmul(s["b"], (x - mean[:, None]) * rstd[:, None], s["w"])}
        return {**out, "mean": mean, "rstd": rstd} if case["stats"] else out
    if op == "norm_bwd":
        xh = (x - s["mean"][:, None]) * s["rstd"][:, None]
        h = s["w"] * s["dy"]
        a, b = h.sum(1) / case["k"], (h * xh).sum(1) / case["k"]
        return {"dx": (h - a[:, None] - b[:, None] * xh) * s["rstd"][:, None],
                "dw": torch.einsum("mk,mk->k", s["dy"], xh), "db": s["dy"].sum(0)}
    if op == "linear":
        z = torch.mm(x, s["w"]) if s["b"] is None else torch.addmm(s["b"], x, s["w"])
        y = _exact_act(z, case["act"])[0]
        y = y if s["res"] is None else s["res"] + y
        return {"y": y, "pre": z} if case["pre"] else {"y": y}
    if op == "linear_bwd":
        dz = s["dy"] if s["pre"] is None else s["dy"] * _exact_act(s["pre"], case["act"])[1]
        out = {"dx": torch.mm(dz, s["w"].t()), "dw": torch.mm(x.t(), dz)}
        return {**out, "db": dz.sum(0)} if case["bias"] else out
    if op == "gated":
        p = [torch.mm(x, s[w]) if s[b] is None else torch.addmm(s[b], x, s[w]) for w, b in (("wg", "bg"), ("wu", "bu"))]
        y = _exact_act(p[0], case["act"])[0] * p[1]
        return {"y": y, "gate": p[0], "up": p[1]} if case["save"] else {"y": y}
    f, d = _exact_act(s["gate"], case["act"])
    dg, du = s["dy"] * s["up"] * d, s["dy"] * f
    out = {"dx": torch.addmm(torch.mm(du, s["wu"].t()), dg, s["wg"].t()), "dwg": torch.mm(x.t(), dg), "dwu": torch.mm(x.t(), du)}
    return {**out, "dbg": dg.sum(0), "dbu": du.sum(0)} if case["bias"] else out
