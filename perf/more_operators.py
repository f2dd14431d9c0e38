"""The 8-bit feed-forward operators' calls, for timing: the root-mean-square norm with the residual's
addition and its gradient, the conversion to 8 bits with a scale for each block of 128, and the matrix
product of 8-bit operands so scaled.

A case is one call of a user's program on torch GPU tensors, with the outputs that the program keeps from
step to step.  ``op`` names the operator, ``dtype`` the type of its 16- or 32-bit tensors; 8-bit ones are
e4m3.  ``rms`` and ``rms_bwd`` take ``rows`` rows of ``n``, ``quantize`` a matrix [rows, n] and ``linear_fp8``
the product of [rows, k] and [k, n].  Its ``use`` is what the product is for, which says how its operands
lie and are scaled: ``y`` a layer's outputs (both along k, weights in blocks of 128 x 128), ``dx`` its
input's gradient (the same weights, now across the sum), ``dw`` its weights' (both operands across the
sum, a scale for each column and 128 tokens).

``run`` calls the framework's operators where ``own`` is true; elsewhere it computes the same in elementary
torch operations in 32 bits, each output rounded once.  ``listed()`` holds the standing cases,
``draw(rng)`` gives another one of the same ranges.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
BLOCK = 128
E4M3 = torch.float8_e4m3fn
LARGEST = 448.0      # of e4m3
LEAST = 2.0 ** -126  # of a scale
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # one token of a decoding step: added to its residual stream, normalised, and in 8 bits for the next product
        {"name": "rms 1x4096 f16", "op": "rms", "rows": 1, "n": 4096, "dtype": "f16", "residual": True, "total": True,
         "y": False, "q": True, "rstd": False},
        # a long prompt's tokens through the same
        {"name": "rms 8192x4096 bf16", "op": "rms", "rows": 8192, "n": 4096, "dtype": "bf16", "residual": True,
         "total": True, "y": False, "q": True, "rstd": False},
        # training in fp32 on a ragged batch whose rows end off every alignment: y, the sum and the statistics kept
        {"name": "rms 1031x4099 f32", "op": "rms", "rows": 1031, "n": 4099, "dtype": "f32", "residual": True,
         "total": True, "y": True, "q": False, "rstd": True},
        # the norm's backward pass on a training batch, the residual stream's own gradient added on the way
        {"name": "rms bwd 8192x4096 bf16", "op": "rms_bwd", "rows": 8192, "n": 4096, "dtype": "bf16", "dtotal": True},
        # the same for a small model of odd width
        {"name": "rms bwd 517x1023 f16", "op": "rms_bwd", "rows": 517, "n": 1023, "dtype": "f16", "dtotal": False},
        # between a gated block's two products: silu(gate) * up of a prompt, in 8 bits for the down projection
        {"name": "quantize gated 2048x14336 bf16", "op": "quantize", "rows": 2048, "n": 14336, "dtype": "bf16",
         "blocks": "rows", "act": "silu", "gate": True},
        # a training batch's gradient with a scale for each column and 128 tokens, as the weights' gradient reads it
        {"name": "quantize columns 4099x4096 bf16", "op": "quantize", "rows": 4099, "n": 4096, "dtype": "bf16",
         "blocks": "columns", "act": "none", "gate": False},
        # one token through a block's down projection, added to its residual stream: the weights are all the bytes
        {"name": "linear fp8 1x14336x4096 f16", "op": "linear_fp8", "use": "y", "rows": 1, "k": 14336, "n": 4096,
         "dtype": "f16", "bias": False, "residual": True, "act": "none", "pre": False},
        # a decoding step of sixteen sequences through the up projection
        {"name": "linear fp8 16x4096x14336 bf16", "op": "linear_fp8", "use": "y", "rows": 16, "k": 4096, "n": 14336,
         "dtype": "bf16", "bias": False, "residual": False, "act": "none", "pre": False},
        # a long prompt through a projection with bias and gelu, its input kept for training
        {"name": "linear fp8 8192x4096x14336 bf16", "op": "linear_fp8", "use": "y", "rows": 8192, "k": 4096, "n": 14336,
         "dtype": "bf16", "bias": True, "residual": False, "act": "gelu", "pre": True},
        # its input's gradient on a training batch: the weights as they are stored, read across the sum
        {"name": "linear fp8 dx 4096x14336x4096 bf16", "op": "linear_fp8", "use": "dx", "rows": 4096, "k": 14336,
         "n": 4096, "dtype": "bf16", "bias": False, "residual": False, "act": "none", "pre": False},
        # the weights' gradient of a small model with odd widths on a ragged batch, in fp32
        {"name": "linear fp8 dw 1023x517x2047 f32", "op": "linear_fp8", "use": "dw", "rows": 1023, "k": 517, "n": 2047,
         "dtype": "f32", "bias": False, "residual": False, "act": "none", "pre": False},
    ]


def _size(rng, lo, hi):
    """A size of [lo, hi], even in its logarithm: half of them as they fall, half on a multiple of 16."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 16:
        v = v // 16 * 16
    return min(hi, max(lo, v))


def _cost(case):
    """Rough microseconds of a pass at this card's rates, to keep draws within the listed range."""
    w = work(case)
    return w["flops"] / 2e9 + w["bytes"] / 5e6


def draw(rng):
    op = rng.choice(["rms", "rms_bwd", "quantize", "linear_fp8", "linear_fp8"])
    most = max(_cost(c) for c in listed())
    while True:
        case = {"op": op, "rows": _size(rng, 1, 8192), "n": _size(rng, 64, 14336),
                "dtype": rng.choice(["f16", "bf16", "bf16", "f32"])}
        if op == "rms":
            case["residual"] = rng.random() < 0.7
            case["total"] = case["residual"] and rng.random() < 0.8
            case["q"] = rng.random() < 0.6
            case["y"] = not case["q"] or rng.random() < 0.3
            case["rstd"] = rng.random() < 0.5
        elif op == "rms_bwd":
            case["dtotal"] = rng.random() < 0.5
        elif op == "quantize":
            case["blocks"] = rng.choice(["rows", "columns", "squares"])
            case["gate"] = case["blocks"] == "rows" and rng.random() < 0.6
            case["act"] = rng.choice(["silu", "gelu", "gelu_tanh"]) if case["gate"] else "none"
        else:
            case["k"] = _size(rng, 64, 14336)
            case["use"] = rng.choice(["y", "y", "dx", "dw"])
            forward = case["use"] == "y"
            case["bias"] = forward and rng.random() < 0.5
            case["residual"] = forward and rng.random() < 0.5
            case["act"] = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]) if forward else "none"
            case["pre"] = case["act"] != "none" and rng.random() < 0.5
        if _cost(case) <= most:
            return case


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    m, n, e = case["rows"], case["n"], BYTES[case["dtype"]]
    op = case["op"]
    if op == "rms":
        moved = m * n * e * (1 + case["residual"] + case["total"] + case["y"]) + n * e + 4 * m * case["rstd"]
        return {"bytes": moved + case["q"] * (m * n + 4 * m * _blocks(n)), "flops": m * n * (5 + 3 * case["q"])}
    if op == "rms_bwd":
        return {"bytes": m * n * e * (3 + case["dtotal"]) + 2 * n * e + 4 * m, "flops": 10 * m * n}
    if op == "quantize":
        scales = {"rows": m * _blocks(n), "columns": _blocks(m) * n, "squares": _blocks(m) * _blocks(n)}[case["blocks"]]
        return {"bytes": m * n * (e * (1 + case["gate"]) + 1) + 4 * scales, "flops": m * n * (3 + 8 * case["gate"])}
    k = case["k"]
    scales = _blocks(k) * (m + (n if case["use"] == "dw" else _blocks(n)))
    outs = m * n * e * (1 + case["residual"] + case["pre"]) + (n * e if case["bias"] else 0)
    return {"bytes": m * k + k * n + 4 * scales + outs, "flops": 2 * m * k * n}


# -- 8 bits ---------------------------------------------------------------------------


def _spread(scale, shape, blocks):
    """One scale for each element of `shape` from those of its blocks of blocks[0] x blocks[1]."""
    return scale.repeat_interleave(blocks[0], 0)[: shape[0]].repeat_interleave(blocks[1], 1)[:, : shape[1]]


def _amax(v, blocks):
    """The largest magnitude of each block; v's edges end where they end."""
    (m, n), (a, b) = v.shape, blocks
    p = torch.zeros(-(-m // a) * a, -(-n // b) * b, device=v.device, dtype=v.dtype)
    p[:m, :n] = v.abs()
    return p.view(-(-m // a), a, -(-n // b), b).amax((1, 3))


def _to_fp8(v, blocks):
    scale = (_amax(v, blocks) / LARGEST).clamp(min=LEAST)
    return (v / _spread(scale, v.shape, blocks)).to(E4M3), scale


SHAPES = {"rows": (1, BLOCK), "columns": (BLOCK, 1), "squares": (BLOCK, BLOCK)}


# -- inputs -------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, m, n, op = DTYPES[case["dtype"]], case["rows"], case["n"], case["op"]

    def normal(*shape, scale=1.0, mean=0.0, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).add_(mean).to(dtype)

    def empty(*shape, dtype=dt):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    def stream(rows, cols):
        # a residual stream: a few columns much larger than the others
        x = normal(rows, cols, scale=1.5, mean=0.2, dtype=torch.float32)
        x[:, :: max(1, cols // 8)] *= 12.0
        return x.to(dt)

    s = {"case": case}
    if op == "rms":
        s["x"], s["w"] = normal(m, n), normal(n, scale=0.1, mean=1.0)
        s["res"] = stream(m, n) if case["residual"] else None
        s["total"] = empty(m, n) if case["total"] else None
        s["y"] = empty(m, n) if case["y"] else None
        s["rstd"] = empty(m, dtype=torch.float32) if case["rstd"] else None
        s["q"] = empty(m, n, dtype=E4M3) if case["q"] else None
        s["scale"] = empty(m, _blocks(n), dtype=torch.float32) if case["q"] else None
    elif op == "rms_bwd":
        s["h"], s["w"], s["dy"] = stream(m, n), normal(n, scale=0.1, mean=1.0), normal(m, n)
        s["rstd"] = torch.rsqrt(s["h"].float().square().mean(1) + EPS)
        s["dtotal"] = normal(m, n) if case["dtotal"] else None
        s["dx"], s["dw"] = empty(m, n), empty(n)
    elif op == "quantize":
        s["x"] = normal(m, n)
        s["gate"] = normal(m, n) if case["gate"] else None
        a, b = SHAPES[case["blocks"]]
        s["q"], s["scale"] = empty(m, n, dtype=E4M3), empty(-(-m // a), -(-n // b), dtype=torch.float32)
    else:
        k, use = case["k"], case["use"]
        if use == "dw":  # tokens along k: each operand as it was made, [tokens, columns]
            x, xs = _to_fp8(normal(k, m, dtype=torch.float32), SHAPES["columns"])
            s["x"], s["xs"] = x.t(), xs.t()
            s["w"], s["ws"] = _to_fp8(normal(k, n, dtype=torch.float32), SHAPES["columns"])
        else:
            s["x"], s["xs"] = _to_fp8(normal(m, k, dtype=torch.float32), SHAPES["rows"])
            if use == "y":  # weights as a layer keeps them, [outputs, inputs]
                w, ws = _to_fp8(normal(n, k, scale=k ** -0.5, dtype=torch.float32), SHAPES["squares"])
                s["w"], s["ws"] = w.t(), ws.t()
            else:
                s["w"], s["ws"] = _to_fp8(normal(k, n, scale=k ** -0.5, dtype=torch.float32), SHAPES["squares"])
        s["b"] = normal(n, scale=0.1) if case["bias"] else None
        s["res"] = normal(m, n) if case["residual"] else None
        s["y"] = empty(m, n)
        s["pre"] = empty(m, n) if case["pre"] else None
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


def _plain(s):
    case = s["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "rms":
        h = s["x"].float()
        if case["residual"]:
            h = h + s["res"].float()
        rstd = torch.rsqrt((h * h).mean(1) + EPS)
        y = h * rstd[:, None] * s["w"].float()
        out = {"y": y.to(dt)} if case["y"] else {}
        if case["total"]:
            out["total"] = h.to(dt)
        if case["rstd"]:
            out["rstd"] = rstd
        if case["q"]:
            out["q"], out["scale"] = _to_fp8(y, SHAPES["rows"])
        return out
    if op == "rms_bwd":
        h, dy, rstd = s["h"].float(), s["dy"].float(), s["rstd"][:, None]
        xhat = h * rstd
        g = dy * s["w"].float()
        dx = rstd * (g - xhat * (g * xhat).mean(1, keepdim=True))
        if case["dtotal"]:
            dx = dx + s["dtotal"].float()
        return {"dx": dx.to(dt), "dw": (dy * xhat).sum(0).to(dt)}
    if op == "quantize":
        v = s["x"].float()
        if case["gate"]:
            v = _act(s["gate"].float(), case["act"]) * v
        q, scale = _to_fp8(v, SHAPES[case["blocks"]])
        return {"q": q, "scale": scale}
    x, w = s["x"], s["w"]
    z = ((x.float() * _spread(s["xs"], x.shape, (1, BLOCK)))
         @ (w.float() * _spread(s["ws"], w.shape, (BLOCK, 1 if case["use"] == "dw" else BLOCK))))
    if case["bias"]:
        z = z + s["b"].float()
    y = _act(z, case["act"])
    if case["residual"]:
        y = y + s["res"].float()
    return {"y": y.to(dt), **({"pre": z.to(dt)} if case["pre"] else {})}


# -- the framework's operators --------------------------------------------------------


def _own(s):
    from easy_as_amd import ops

    case = s["case"]
    op = case["op"]
    if op == "rms":
        ops.rms_norm(s["x"], s["w"], s["y"], s["rstd"], residual=s["res"], total=s["total"], q=s["q"],
                     q_scale=s["scale"], eps=EPS, _sync=False)
        return {k: s[k] for k in ("y", "total", "rstd", "q", "scale") if s[k] is not None}
    if op == "rms_bwd":
        ops.rms_norm_backward(s["dy"], s["h"], s["w"], s["rstd"], s["dx"], s["dw"], dtotal=s["dtotal"], _sync=False)
        return {"dx": s["dx"], "dw": s["dw"]}
    if op == "quantize":
        ops.quantize(s["x"], s["q"], s["scale"], gate=s["gate"], activation=case["act"], _sync=False)
        return {"q": s["q"], "scale": s["scale"]}
    ops.linear_fp8(s["x"], s["xs"], s["w"], s["ws"], s["y"], bias=s["b"], residual=s["res"], activation=case["act"],
                   pre=s["pre"], _sync=False)
    return {"y": s["y"], **({"pre": s["pre"]} if case["pre"] else {})}


def run(state):
    return _own(state) if own else _plain(state)


# -- 64 bits --------------------------------------------------------------------------


def _exact_act(z, name):
    if name == "none":
        return z
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    # the tanh form is z sigmoid(2 u), u = sqrt(2/pi) (z + 0.044715 z^3)
    return z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))


def _exact_scales(v, rows, cols):
    """Scales of blocks of rows x cols, and each element's own."""
    m, n = v.shape
    i = (torch.arange(m, device=v.device) // rows)[:, None] * _count(n, cols) + (torch.arange(n, device=v.device) // cols)[None]
    most = torch.zeros(_count(m, rows) * _count(n, cols), device=v.device, dtype=v.dtype)
    most.scatter_reduce_(0, i.reshape(-1), v.abs().reshape(-1), "amax")
    scale = torch.maximum(most / LARGEST, torch.tensor(LEAST, device=v.device, dtype=v.dtype))
    return scale.view(_count(m, rows), _count(n, cols)), scale[i]


def _count(n, block):
    return (n + block - 1) // block


def _exact_e4m3(v):
    """v to the nearest e4m3 value, ties to even: four significant bits, down to multiples of 2^-9."""
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp(min=2.0 ** -6))[1] - 4)
    return (torch.round(v / step) * step).clamp(-LARGEST, LARGEST)


def _exact_to_fp8(v, kind):
    rows, cols = SHAPES[kind]
    scale, each = _exact_scales(v, rows, cols)
    return _exact_e4m3(v / each), scale


def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    op = case["op"]
    if op == "rms":
        h = s["x"] if s["res"] is None else torch.add(s["x"], s["res"])
        rstd = (torch.linalg.vector_norm(h, dim=1) ** 2 / case["n"] + EPS) ** -0.5
        y = torch.einsum("mn,m,n->mn", h, rstd, s["w"])
        out = {"y": y} if case["y"] else {}
        if case["q"]:
            out["q"], out["scale"] = _exact_to_fp8(y, "rows")
        return {**out, **({"total": h} if case["total"] else {}), **({"rstd": rstd} if case["rstd"] else {})}
    if op == "rms_bwd":
        r = s["rstd"]
        g = s["dy"] * s["w"]
        dx = g * r[:, None] - s["h"] * ((g * s["h"]).sum(1) * r ** 3 / case["n"])[:, None]
        return {"dx": dx if s["dtotal"] is None else s["dtotal"] + dx, "dw": torch.einsum("mn,mn,m->n", s["dy"], s["h"], r)}
    if op == "quantize":
        v = s["x"] if s["gate"] is None else torch.mul(s["x"], _exact_act(s["gate"], case["act"]))
        q, scale = _exact_to_fp8(v, case["blocks"])
        return {"q": q, "scale": scale}
    m, k, n = case["rows"], case["k"], case["n"]
    i = torch.arange(k, device="cuda") // BLOCK
    x = s["x"] * s["xs"][:, i]
    w = s["w"] * (s["ws"][i] if case["use"] == "dw" else s["ws"][i][:, torch.arange(n, device="cuda") // BLOCK])
    z = torch.mm(x, w) if s["b"] is None else torch.addmm(s["b"], x, w)
    y = _exact_act(z, case["act"])
    y = y if s["res"] is None else s["res"] + y
    return {"y": y, "pre": z} if case["pre"] else {"y": y}
