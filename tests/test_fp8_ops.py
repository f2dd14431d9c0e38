"""The operators around 8-bit operands without a GPU: their C structures, refusals and scratch sizes."""

from __future__ import annotations

import ctypes
import re
import struct

import numpy as np
import pytest

import fp8_reference as ref
from easy_as_amd import ops
from test_ops import P, ROOT, fake, fields, mod, packed  # noqa: F401

torch = pytest.importorskip("torch")
E4M3 = torch.float8_e4m3fn
KINDS = {"rms_norm": 7, "rms_norm_backward": 8, "quantize": 9, "linear_fp8": 10}
RMS, RMS_BACKWARD, QUANTIZE, PRODUCT = KINDS.values()


@pytest.mark.parametrize("name,kind", KINDS.items())
def test_packed_arguments_match_the_header(name, kind):
    codes = "".join(c for _, c in fields(name))
    assert struct.Struct("@" + codes).size == ops._STRUCTS[kind].size
    assert ops._STRUCTS[kind].format.replace("@", "") == "".join(
        f"{len(g)}{g[0]}" if len(g) > 1 else g[0] for g in re.findall(r"P+|Q+|q+|i+|f+", codes))


def rms(**kw) -> bytes:
    v = dict(x=P, y=2 * P, m=8, n=300, x_ld=300, y_ld=300, q_scale_row=3, q_scale_block=1, eps=1e-5)
    return packed("rms_norm", **{**v, **kw})


def rms_q(**kw) -> bytes:
    return rms(**{**dict(q=4 * P, q_ld=300, q_scale=5 * P), **kw})


def rms_backward(**kw) -> bytes:
    v = dict(dy=P, h=2 * P, rstd=3 * P, dx=4 * P, dweight=5 * P, m=8, n=300, dy_ld=300, h_ld=300, dx_ld=300)
    return packed("rms_norm_backward", **{**v, **kw})


def quantize(**kw) -> bytes:
    v = dict(x=P, q=2 * P, scale=3 * P, m=200, n=300, x_ld=300, q_ld=300, scale_row=3, scale_col=1, block_m=1, block_n=128)
    return packed("quantize", **{**v, **kw})


def product(**kw) -> bytes:
    v = dict(x=P, x_scale=2 * P, w=3 * P, w_scale=4 * P, y=5 * P, m=100, k=256, n=64, x_ld=256, w_ld=64, x_scale_row=2, x_scale_block=1,
             w_scale_block=64, w_scale_col=1, y_ld=64)
    return packed("linear_fp8", **{**v, **kw})


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(str(ROOT / "easy_as_amd" / "libeas_hip.so"))


def refused(lib, name: str, args: bytes) -> str:
    """What the entry that enqueues says of `args`; their addresses are never read, so only refusals may come here."""
    buffer = ctypes.create_string_buffer(args, len(args))
    entry = getattr(lib, f"eas_hip_{name}")
    entry.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    lib.eas_hip_last_error.restype = ctypes.c_char_p
    assert entry(buffer, len(args), None) == -1
    return lib.eas_hip_last_error().decode()


@pytest.mark.parametrize("name,args,message", [
    ("rms_norm", rms(dtype=3), "dtype"), ("rms_norm", rms(hdtype=1), "dtype"), ("rms_norm", rms(wdtype=1), "dtype"),
    ("rms_norm", rms(n=0), "element"), ("rms_norm", rms(m=-1), "sizes"), ("rms_norm", rms(x_ld=299), "stride"),
    ("rms_norm", rms(residual=3 * P, residual_ld=299), "stride"), ("rms_norm", rms(eps=-1.0), "eps"),
    ("rms_norm", rms(eps=float("nan")), "eps"), ("rms_norm", rms(y=0), "NULL"), ("rms_norm", rms(x=0), "NULL"),
    ("rms_norm", rms(q=4 * P, q_ld=300), "together"), ("rms_norm", rms_q(q_ld=299), "stride"),
    ("rms_norm", rms_q(q_scale_row=2), "lines"), ("rms_norm", rms_q(q_scale_block=2), "lines"),
    ("rms_norm", rms_q(q_scale_row=1, q_scale_block=7), "lines"), ("rms_norm", rms_q(q_scale_row=-3), "lines"),
    ("rms_norm", rms_q(q_scale_row=1 << 41), "lines"),
    ("rms_norm", rms(y=P + 2), "shares"), ("rms_norm", rms(y=P, y_ld=301), "shares"), ("rms_norm", rms(weight=2 * P), "shares"),
    ("rms_norm", rms(total=2 * P, total_ld=300), "share"), ("rms_norm", rms(rstd=P), "shares"), ("rms_norm", rms_q(q=P), "shares"),
    ("rms_norm", rms(residual=2 * P, residual_ld=300, hdtype=2), "shares"), ("rms_norm", rms_q(q_scale=4 * P + 8), "share"),
    ("rms_norm_backward", rms_backward(h=0), "NULL"), ("rms_norm_backward", rms_backward(rstd=0), "NULL"),
    ("rms_norm_backward", rms_backward(dtotal=6 * P, dtotal_ld=299), "stride"), ("rms_norm_backward", rms_backward(n=0), "element"),
    ("rms_norm_backward", rms_backward(dx=2 * P + 2), "shares"), ("rms_norm_backward", rms_backward(dx=P, hdtype=2), "shares"),
    ("rms_norm_backward", rms_backward(dweight=2 * P), "shares"), ("rms_norm_backward", rms_backward(dx=3 * P), "shares"),
    ("rms_norm_backward", rms_backward(m=8192, dy=1 << 40, h=1 << 41, rstd=1 << 42, dx=1 << 43), "workspace"),
    ("quantize", quantize(dtype=3), "dtype"), ("quantize", quantize(activation=5), "activation"),
    ("quantize", quantize(block_m=64), "blocks"), ("quantize", quantize(block_n=1), "blocks"), ("quantize", quantize(scale=0), "NULL"),
    ("quantize", quantize(scale_row=2), "lines"), ("quantize", quantize(block_m=128, block_n=1, scale_row=299), "lines"),
    ("quantize", quantize(gate=4 * P, gate_ld=299), "stride"), ("quantize", quantize(q_ld=299), "stride"),
    ("quantize", quantize(q=P), "shares"), ("quantize", quantize(scale=P + 4), "shares"), ("quantize", quantize(gate=2 * P, gate_ld=300), "shares"),
    ("quantize", quantize(scale=2 * P), "share"),
    ("linear_fp8", product(ydtype=3), "dtype"), ("linear_fp8", product(activation=-1), "activation"),
    ("linear_fp8", product(x_trans=2), "x_trans"), ("linear_fp8", product(w_blocks=-1), "w_blocks"),
    ("linear_fp8", product(k=-1), "sizes"), ("linear_fp8", product(x_ld=255), "stride"), ("linear_fp8", product(x_trans=1, x_ld=99), "stride"),
    ("linear_fp8", product(w_ld=63), "stride"), ("linear_fp8", product(w_trans=1), "stride"), ("linear_fp8", product(y_ld=63), "stride"),
    ("linear_fp8", product(x_scale_row=-1), "negative"), ("linear_fp8", product(w_scale_col=1 << 22), "far"),
    ("linear_fp8", product(x_scale_row=1 << 22), "far"), ("linear_fp8", product(x_scale_block=1 << 41), "far"),
    ("linear_fp8", product(x=0), "NULL"), ("linear_fp8", product(w_scale=0), "NULL"), ("linear_fp8", product(y=0), "NULL"),
    ("linear_fp8", product(y=P), "shares"), ("linear_fp8", product(y=4 * P), "shares"), ("linear_fp8", product(pre=5 * P, pre_ld=64), "share"),
    ("linear_fp8", product(residual=5 * P + 2, residual_ld=64), "shares"), ("linear_fp8", product(bias=5 * P), "shares"),
    ("linear_fp8", product(x=P + 1), "workspace"),
])
def test_the_c_entries_refuse(lib, name, args, message):
    assert message in refused(lib, name, args)


def test_scales_whose_area_passes_64_bits_share_memory(lib):
    far = product(m=1, k=(1 << 30) + 128, n=1, x=1 << 50, x_ld=1 << 31, w=1 << 51, w_ld=64, x_scale_block=1 << 40, w_scale=1 << 52,
                  w_scale_block=1)
    assert "shares" in refused(lib, "linear_fp8", far)


def test_the_c_entries_refuse_other_arguments(lib):
    for name in KINDS:
        entry = getattr(lib, f"eas_hip_{name}")
        assert entry(None, ctypes.c_size_t(0), None) == -1
        assert "args_size" in refused(lib, name, bytes(8))


def test_scratch(mod):  # noqa: F811
    assert mod.op_workspace(RMS, rms()) == 0 and mod.op_workspace(QUANTIZE, quantize()) == 0
    assert mod.op_workspace(RMS_BACKWARD, rms_backward(dweight=0)) == 0
    assert mod.op_workspace(RMS_BACKWARD, rms_backward()) == 0                     # few elements: no partial sums
    assert mod.op_workspace(RMS_BACKWARD, rms_backward(dx=2 * P)) == 0             # in place too
    big = dict(dy=1 << 40, h=1 << 41, rstd=1 << 42, dx=1 << 43)
    assert mod.op_workspace(RMS_BACKWARD, rms_backward(m=8192, **big)) == 256 * 300 * 4  # four rows of 300 at a time
    assert mod.op_workspace(RMS_BACKWARD, rms_backward(**{**big, "dx": 0})) == 2 * 300 * 4
    assert mod.op_workspace(RMS_BACKWARD, rms_backward(m=0)) == 0
    assert mod.op_workspace(RMS_BACKWARD, rms_backward(m=100000, n=16384, dy_ld=16384, h_ld=16384, dx_ld=16384, **big)) == 256 * 16384 * 4
    assert mod.op_workspace(PRODUCT, product()) == 0
    # rows off 4 bytes, and rows along k that end within 16, are copied to rows of whole 16-byte units
    assert mod.op_workspace(PRODUCT, product(x=P + 1)) == 100 * 256
    assert mod.op_workspace(PRODUCT, product(k=250)) == 100 * 256
    assert mod.op_workspace(PRODUCT, product(n=63, w_ld=63)) == 256 * 64
    assert mod.op_workspace(PRODUCT, product(w=3 * P + 4, x_trans=1, x_ld=100)) == 0
    assert mod.op_workspace(PRODUCT, product(x_ld=8 << 20, w=1 << 40, x_scale=1 << 41, w_scale=1 << 42, y=1 << 43)) == 100 * 256


@pytest.mark.parametrize("args", [
    product(m=300, k=40000000, x_ld=40000000, x=1 << 40, w=1 << 44, y=1 << 45, w_scale=1 << 46, x_scale=1 << 47),
    product(n=40000000, w_ld=40000000, x=1 << 40, w=1 << 44, y=1 << 45, y_ld=40000000, w_scale=1 << 46, x_scale=1 << 47),
], ids=["x", "w"])
def test_rows_beyond_a_tiles_offsets_are_refused(mod, args):  # noqa: F811
    with pytest.raises(ValueError, match="too long"):
        mod.op_workspace(PRODUCT, args)


def f(*shape, dtype=np.float32):
    return np.zeros(shape, dtype)


def b(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(E4M3)


@pytest.mark.parametrize("call,error,message", [
    (lambda: ops.rms_norm(f(2, 0), None, f(2, 0)), ValueError, "at least one element"),
    (lambda: ops.rms_norm(f(2, 3), None), TypeError, "'y' or 'q'"),
    (lambda: ops.rms_norm(f(2, 3), None, q=b(2, 3)), TypeError, "go together"),
    (lambda: ops.rms_norm(f(2, 3), None, q=f(2, 3), q_scale=f(2, 1)), TypeError, "'q' must be a torch tensor of float8_e4m3fn"),
    (lambda: ops.rms_norm(f(2, 3), None, q=torch.zeros(2, 3), q_scale=f(2, 1)), TypeError, "'q' must be torch.float8_e4m3fn"),
    (lambda: ops.rms_norm(b(2, 3), None, f(2, 3)), TypeError, "'x' must be f16, bf16 or f32"),
    (lambda: ops.rms_norm(f(2, 3), None, q=b(2, 3), q_scale=f(2, 2)), ValueError, "'q_scale' must be"),
    (lambda: ops.rms_norm(f(2, 3), None, q=b(2, 3), q_scale=f(2, 1, dtype=np.float16)), TypeError, "'q_scale' must be f32"),
    (lambda: ops.rms_norm(f(2, 3), f(4), f(2, 3)), ValueError, "'weight' must hold 3"),
    (lambda: ops.rms_norm(f(2, 3), None, f(2, 4)), ValueError, "'y' must hold 2 rows of 3"),
    (lambda: ops.rms_norm(f(2, 3, dtype=np.float16), None, f(2, 3, dtype=np.float16), residual=f(2, 3), total=f(2, 3, dtype=np.float16)),
     TypeError, "'total' must be f32"),
    (lambda: ops.rms_norm(f(2, 3), None, f(2, 3), f(3)), ValueError, "'rstd' must hold 2"),
    (lambda: ops.rms_norm(f(2, 3), None, f(2, 3), eps=-1.0), ValueError, "eps"),
    (lambda: ops.rms_norm(f(2, 3), None, f(2, 3), _sync=0), TypeError, "_sync"),
    (lambda: ops.rms_norm_backward(f(2, 3), f(2, 4), None, f(2)), ValueError, "'h' must hold"),
    (lambda: ops.rms_norm_backward(f(2, 3), f(2, 3), None, None), TypeError, "'rstd'"),
    (lambda: ops.rms_norm_backward(f(2, 3, dtype=np.float16), f(2, 3), None, f(2), f(2, 3, dtype=np.float16)), TypeError, "'dx' must be f32"),
    (lambda: ops.quantize(f(2, 300), b(2, 299), f(2, 3)), ValueError, "'q' must hold"),
    (lambda: ops.quantize(f(2, 300), b(2, 300), f(2, 2)), ValueError, r"'scale' must be \[2, 3\] or \[1, 300\] or \[1, 3\]"),
    (lambda: ops.quantize(f(2, 300), b(2, 300), f(2, 3), gate=f(2, 3)), ValueError, "'gate' must hold"),
    (lambda: ops.quantize(f(2, 300), b(2, 300), f(2, 3), activation="tanh"), ValueError, "activation must be one of"),
    (lambda: ops.linear_fp8(b(2, 200), f(2, 1), b(200, 5), f(2, 5), f(2, 5)), ValueError, "'x_scale' must be"),
    (lambda: ops.linear_fp8(b(2, 200), f(2, 2), b(200, 5), f(2, 2), f(2, 5)), ValueError, "'w_scale' must be"),
    (lambda: ops.linear_fp8(b(2, 200), f(2, 2), b(201, 5), f(2, 5), f(2, 5)), ValueError, "'w' must be"),
    (lambda: ops.linear_fp8(f(2, 200), f(2, 2), b(200, 5), f(2, 5), f(2, 5)), TypeError, "'x' must be a torch tensor"),
    (lambda: ops.linear_fp8(b(2, 200), f(2, 2), f(200, 5), f(2, 5), f(2, 5)), TypeError, "'w' must be a torch tensor"),
    (lambda: ops.linear_fp8(b(2, 200), f(2, 2), b(200, 5), f(2, 5), b(2, 5)), TypeError, "'y' must be f16"),
    (lambda: ops.linear_fp8(b(2, 200), f(2, 2), b(200, 5), f(2, 5), f(2, 5), bias=f(5, dtype=np.float16)), TypeError, "'bias' must be f32"),
    (lambda: ops.linear(b(2, 200), b(200, 5), f(2, 5)), TypeError, "'x' must be f16"),
])
def test_the_python_layer_refuses(fake, call, error, message):  # noqa: F811
    with pytest.raises(error, match=message):
        call()
    assert not fake.ran


def fields_of(fake, kind: int) -> dict:
    name = {v: k for k, v in KINDS.items()}[kind]
    ran = [a for a in fake.ran if a[0] == kind][-1][1]
    return dict(zip((n for n, _ in fields(name)), ops._STRUCTS[kind].unpack(ran)))


def test_how_operands_lie(fake):  # noqa: F811
    c = ops._Call("linear_fp8", True)
    c.bytes8 = lambda name, v, write=False: (0, 3, tuple(v.shape), v.stride())
    x = b(40, 30)
    assert c.either("x", x)[1:] == (30, 40, 30, False)
    assert c.either("x", x.t())[1:] == (30, 30, 40, True)
    assert c.either("x", x[:, 5:25].t())[1:] == (30, 20, 40, True)
    assert c.either("x", x[:, :1])[1:] == (30, 40, 1, False)
    assert c.either("x", x[:, :1].t())[1:] == (30, 1, 40, True)   # one row, its elements 30 apart
    assert c.either("x", x[:1])[1:] == (30, 1, 30, False)
    assert c.either("x", x[:1].t())[1:4] == (30, 30, 1) or c.either("x", x[:1].t())[1:] == (1, 30, 1, False)
    assert c.either("x", b(2, 3, 5))[1:] == (5, 6, 5, False)
    for bad in (x[:, ::2], x[:1].expand(40, 30), x[::2].t()[::2], b(2, 3, 5).transpose(0, 1)):
        with pytest.raises(ValueError):
            c.either("x", bad)


def test_scales_shapes_and_strides(fake):  # noqa: F811
    c = ops._Call("linear_fp8", True)
    c.array = lambda name, v, write=False: (0, 2, tuple(v.shape), v.stride())
    s = torch.zeros(40, 30)
    shapes = ((40, 30), (20, 30), (30, 40))
    assert c.scales("s", s, shapes)[1:] == (30, 1, (40, 30))
    assert c.scales("s", s.t(), shapes)[1:] == (1, 30, (30, 40))
    assert c.scales("s", torch.zeros(1, 1).expand(40, 30), shapes)[1:] == (0, 0, (40, 30))
    assert c.scales("s", s[::2], shapes)[1:] == (60, 1, (20, 30))
    assert c.scales("s", torch.zeros(4, 10, 30), shapes)[1:] == (30, 1, (40, 30))
    assert c.scales("s", s, shapes, True)[1:3] == (30, 1)
    assert c.scales("s", torch.zeros(1, 7), ((1, 7),), True)[1:3] == (7, 1)
    assert c.scales("s", torch.zeros(7, 1), ((7, 1),), True)[1:3] == (1, 1)
    for bad in (torch.zeros(1, 1).expand(40, 30), torch.zeros(40, 60)[:, ::2], torch.zeros(40, 1).expand(40, 30)):
        with pytest.raises(ValueError, match="contiguous along one axis"):
            c.scales("s", bad, shapes, True)
    with pytest.raises(ValueError, match="must be"):
        c.scales("s", torch.zeros(30, 20), shapes)


@pytest.mark.parametrize("shape,dims,block", [((300, 200), (300, 2), (1, 128)), ((300, 200), (3, 200), (128, 1)), ((300, 200), (3, 2), (128, 128)),
                                              ((1, 200), (1, 2), (1, 128)), ((1, 200), (1, 200), (128, 1)), ((300, 1), (3, 1), (128, 1))])
def test_a_scales_shape_says_its_blocks(fake, shape, dims, block):  # noqa: F811
    ops.quantize(f(*shape), b(*shape), f(*dims))
    got = fields_of(fake, QUANTIZE)
    assert (got["block_m"], got["block_n"]) == block
    a, c = block
    assert dims == (-(-shape[0] // a), -(-shape[1] // c))


def test_calls_on_host_arrays_reach_the_entry(fake):  # noqa: F811
    ops.rms_norm(f(2, 300), f(300), f(2, 300), f(2), residual=f(2, 300), total=f(2, 300), q=b(2, 300), q_scale=f(2, 3), eps=0.5)
    got = fields_of(fake, RMS)
    assert (got["m"], got["n"], got["q_scale_row"], got["q_scale_block"], got["eps"], got["hdtype"]) == (2, 300, 3, 1, 0.5, 2)
    ops.linear_fp8(b(2, 300), f(2, 3), b(300, 200), f(3, 2), f(2, 200))
    got = fields_of(fake, PRODUCT)
    assert (got["w_blocks"], got["x_trans"], got["w_trans"], got["ydtype"], got["w_scale_block"]) == (1, 0, 0, 2, 2)
    ops.linear_fp8(b(2, 300), f(2, 3), b(300, 200), f(3, 200), f(2, 200))
    assert fields_of(fake, PRODUCT)["w_blocks"] == 0
    ops.rms_norm_backward(f(2, 300), f(2, 300), None, f(2), f(2, 300), f(300), dtotal=f(2, 300))
    assert fields_of(fake, RMS_BACKWARD)["hdtype"] == 2


def test_the_oracles_8_bit_values():
    """Against torch's conversion, which rounds to nearest, ties to even, from f32."""
    v = torch.cat([torch.randn(20000).double() * 2.0 ** e for e in range(-12, 9)]).float()
    v = v[v.abs() <= 448]
    assert torch.equal(ref.to_e4m3(v.double()).float(), v.to(E4M3).float())
    codes = torch.arange(256, dtype=torch.uint8).view(E4M3).float()
    codes = codes[codes.isfinite()].unique()
    ties = (codes[1:] + codes[:-1]) / 2
    assert torch.equal(ref.to_e4m3(ties.double()).float(), ties.to(E4M3).float())


def test_a_line_of_scales_lies_at_any_stride(fake):  # noqa: F811
    """One token's scales, kept as [blocks, tokens], and one column's."""
    c = ops._Call("rms_norm", True)
    c.array = lambda name, v, write=False: (0, 2, tuple(v.shape), v.stride())
    kept = torch.zeros(7, 40)
    for one in (kept.t()[:1], kept[:, 3:4].t(), torch.zeros(7, 40, 2)[:, 0, :1].t()):
        s0, s1 = c.scales("s", one, ((1, 7),), True)[1:3]
        assert s1 == one.stride(1) and s0 >= 1
        assert "NULL" in refused(ctypes.CDLL(str(ROOT / "easy_as_amd" / "libeas_hip.so")), "rms_norm",
                                 rms_q(m=1, n=900, x=0, x_ld=900, y_ld=900, q_ld=900, q_scale_row=s0, q_scale_block=s1))  # and not "lines"
    assert c.scales("s", kept[:, 3:4], ((7, 1),), True)[1:3] == (40, 1)
    assert c.scales("s", kept[:1], ((1, 40),), True)[1:3] == (40, 1)
    for bad in (torch.zeros(1, 1).expand(1, 7), torch.zeros(1, 1).expand(7, 1)):
        with pytest.raises(ValueError, match="contiguous along one axis"):
            c.scales("s", bad, (tuple(bad.shape),), True)


def test_how_far_the_products_offsets_reach(mod):  # noqa: F811
    far = dict(x=1 << 40, w=1 << 44, y=1 << 45, w_scale=1 << 46, x_scale=1 << 47)
    long, longer = (1 << 23) - 16, 1 << 23
    assert mod.op_workspace(PRODUCT, product(m=300, k=long, x_ld=long, **far)) >= 0
    assert mod.op_workspace(PRODUCT, product(n=long, w_ld=long, y_ld=long, **far)) >= 0
    for args in (product(m=300, k=longer, x_ld=longer, **far), product(m=17, k=longer, x_ld=longer, w_trans=1, w_ld=longer, **far)):
        with pytest.raises(ValueError, match="too long"):
            mod.op_workspace(PRODUCT, args)
    # up to 16 rows along k are read at 64-bit offsets, and not copied
    assert mod.op_workspace(PRODUCT, product(m=16, k=longer, x_ld=longer, w_trans=1, w_ld=longer, n=4096, y_ld=4096, **far)) >= 0
    for name in ("x_scale_row", "w_scale_col"):
        assert mod.op_workspace(PRODUCT, product(**far, **{name: 2105376})) == 0
        with pytest.raises(ValueError, match="too far apart"):
            mod.op_workspace(PRODUCT, product(**far, **{name: 2105377}))
    for name in ("x_scale_block", "w_scale_block"):
        assert mod.op_workspace(PRODUCT, product(**{**far, "x_scale": 1 << 50, "w_scale": 1 << 54}, **{name: 1 << 40})) == 0
        with pytest.raises(ValueError, match="too far apart"):
            mod.op_workspace(PRODUCT, product(**far, **{name: (1 << 40) + 1}))


def test_more_columns_than_a_grid_holds_are_refused(mod):  # noqa: F811
    """Before a column's number, rounded up to a workgroup's scales, leaves 31 bits."""
    far = dict(m=1, k=16, x_ld=16, w_ld=16, w_trans=1, w_blocks=1, w_scale_block=1 << 25, x=1 << 40, w=1 << 44, y=1 << 46, x_scale=1 << 47,
               w_scale=1 << 48)
    most = ((1 << 32) // 512 - 1) * 64
    assert mod.op_workspace(PRODUCT, product(n=most, y_ld=most, **far)) == 0 and most + 64 * 128 < 1 << 31
    for n in (1 << 30, (1 << 31) - 8000):
        with pytest.raises(ValueError, match="too many tiles"):
            mod.op_workspace(PRODUCT, product(n=n, y_ld=n, **far))
