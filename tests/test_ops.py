"""The feed-forward operators without a GPU: their C structures, refusals and scratch sizes."""

from __future__ import annotations

import ctypes
import re
import struct
from pathlib import Path

import numpy as np
import pytest

from easy_as_amd import ops
from easy_as_amd.runtime.hip_ext import load_hip_ext

ROOT = Path(__file__).resolve().parents[1]
HEADER = (ROOT / "include" / "eas_hip.h").read_text()
CTYPES = {"int64_t": "q", "int32_t": "i", "uint64_t": "Q", "float": "f"}
NAMES = ["layer_norm", "layer_norm_backward", "linear", "linear_backward", "gated_linear", "gated_linear_backward"]


def fields(name: str) -> list[tuple[str, str]]:
    body = re.search(r"typedef struct eas_hip_%s_args \{(.*?)\} eas_hip_%s_args;" % (name, name), HEADER, re.S).group(1)
    out = []
    for line in body.split(";"):
        line = line.strip()
        if not line:
            continue
        pointer = re.match(r"(?:const )?(?:void|float)\* (\w+)$", line)
        if pointer:
            out.append((pointer.group(1), "P"))
            continue
        kind, names = line.split(None, 1)
        out += [(n.strip(), CTYPES[kind]) for n in names.split(",")]
    return out


@pytest.mark.parametrize("kind,name", list(enumerate(NAMES)))
def test_packed_arguments_match_the_header(kind, name):
    assert struct.Struct("@" + "".join(c for _, c in fields(name))).size == ops._STRUCTS[kind].size
    assert ops._STRUCTS[kind].format.replace("@", "") == "".join(
        f"{len(g)}{g[0]}" if len(g) > 1 else g[0] for g in re.findall(r"P+|Q+|q+|i+|f+", "".join(c for _, c in fields(name))))


@pytest.fixture(scope="module")
def mod():
    return load_hip_ext(require=True)


def packed(name: str, **values) -> bytes:
    fs = fields(name)
    assert not set(values) - {n for n, _ in fs}
    return struct.pack("@" + "".join(c for _, c in fs), *(values.get(n, 0) for n, _ in fs))


P = 1 << 20  # addresses that are only compared, never read


def linear(**kw) -> bytes:
    v = dict(x=P, w=2 * P, y=3 * P, m=8, k=16, n=32, x_ld=16, w_ld=32, y_ld=32)
    return packed("linear", **{**v, **kw})


def backward(**kw) -> bytes:
    v = dict(dy=P, x=2 * P, w=3 * P, dx=4 * P, dw=5 * P, dbias=6 * P, m=8, k=16, n=32, dy_ld=32, x_ld=16, w_ld=32, dx_ld=16, dw_ld=32)
    return packed("linear_backward", **{**v, **kw})


def gated(**kw) -> bytes:
    v = dict(x=P, w_gate=2 * P, w_up=3 * P, y=4 * P, m=8, k=16, n=32, x_ld=16, w_gate_ld=32, w_up_ld=32, y_ld=32)
    return packed("gated_linear", **{**v, **kw})


@pytest.mark.parametrize("kind,args,message", [
    (2, linear(dtype=3), "dtype"), (2, linear(dtype=2, ydtype=0), "dtype"), (2, linear(activation=5), "activation"),
    (2, linear(w_trans=2), "w_trans"), (2, linear(m=-1), "sizes"), (2, linear(n=1 << 31, y_ld=1 << 31, w_ld=1 << 31), "sizes"),
    (2, linear(x_ld=15), "stride"), (2, linear(w_ld=31), "stride"), (2, linear(w_trans=1, w_ld=15), "stride"),
    (2, linear(y_ld=31), "stride"), (2, linear(pre=4 * P, pre_ld=31), "stride"), (2, linear(residual=4 * P), "stride"),
    (2, linear(x=0), "NULL"), (2, linear(w=0), "NULL"), (2, linear(y=0), "NULL"),
    (2, linear(y=P), "shares"), (2, linear(y=P + 200), "shares"), (2, linear(pre=3 * P + 32, pre_ld=32), "share"),
    (2, linear(residual=3 * P + 2, residual_ld=32), "shares"), (2, linear(residual=3 * P, residual_ld=40), "shares"),
    (3, backward(dw=2 * P), "shares"), (3, backward(activation=1, pre_ld=32), "NULL"), (3, backward(activation=1, pre=7 * P), "stride"),
    (3, backward(x=0), "NULL"), (3, backward(w=0), "NULL"), (3, backward(dy=0), "NULL"), (3, backward(dx_ld=15), "stride"),
    (3, backward(dw_ld=31), "stride"), (3, backward(wdtype=1), "dtype"), (3, backward(dbias=5 * P), "share"),
    (4, gated(gate=5 * P, gate_ld=32), "stride"), (4, gated(gate=5 * P, gate_ld=32, up_ld=32), "together"),
    (4, gated(w_up=0), "NULL"), (4, gated(y=3 * P), "shares"),
    (1, packed("layer_norm_backward", dy=P, x=P, mean=P, rstd=P, m=4, n=0), "element"),
    (1, packed("layer_norm_backward", dy=P, x=2 * P, mean=3 * P, m=4, n=8, dy_ld=8, x_ld=8), "NULL"),
])
def test_the_c_entries_refuse(mod, kind, args, message):
    with pytest.raises(ValueError, match=message):
        mod.op_workspace(kind, args)


def test_the_c_entries_take(mod):
    assert mod.op_workspace(2, linear()) == 0
    assert mod.op_workspace(2, linear(residual=3 * P, residual_ld=32)) == 0      # in place
    assert mod.op_workspace(2, linear(y_ld=64, pre=3 * P + 64, pre_ld=64)) == 0  # halves of one array
    assert mod.op_workspace(2, linear(m=0, x=0, y=0)) == 0
    # rows off 4 bytes, and rows along k that end within 16, are copied to rows of whole 16-byte units
    assert mod.op_workspace(2, linear(m=100, x=P + 2)) == 3328
    assert mod.op_workspace(2, linear(m=100, k=15)) == 3328
    assert mod.op_workspace(2, linear(m=100, x=P + 4, w=2 * P + 4, w_ld=34)) == 0
    assert mod.op_workspace(2, linear(x=P + 2, k=15)) == 0  # few rows go through registers
    assert mod.op_workspace(2, linear(x=P + 2, dtype=2, ydtype=2)) == 256 * 2
    # the rows of dz, and its sums
    assert mod.op_workspace(3, backward(dbias=0)) == 0
    assert mod.op_workspace(3, backward(activation=2, pre=7 * P, pre_ld=32, dbias=0)) == 8 * 32 * 2
    assert mod.op_workspace(3, backward(dx=0, dw=0)) == 0  # few rows: the sums in one stage
    assert mod.op_workspace(3, backward(dx=0, dw=0, x=0, dy=1 << 40, m=1 << 20)) == 1024 * 32 * 4


def test_sizes_beyond_32_bits_of_elements(mod):
    # 70000 x 70000 elements: every offset and scratch size in 64 bits
    n = 70001
    args = linear(m=n, k=n, n=n, x_ld=n, w_ld=n, y_ld=n, w=1 << 40, y=1 << 44)
    assert mod.op_workspace(2, args) == 2 * ((n * 70008 * 2 + 255) // 256 * 256)


def test_argument_bytes_of_another_operator_are_refused(mod):
    with pytest.raises(ValueError, match="args_size"):
        mod.op_workspace(2, bytes(8))
    with pytest.raises(ValueError, match="unknown operator"):
        mod.op_workspace(6, linear())
    with pytest.raises(TypeError):
        mod.op_workspace(2, "x")
    with pytest.raises(TypeError):
        mod.op_run(2, linear(), None)
    lib = ctypes.CDLL(str(ROOT / "easy_as_amd" / "libeas_hip.so"))
    assert lib.eas_hip_linear(None, 0, None) == -1
    assert lib.eas_hip_linear_workspace(None, 0, None) == -1
    assert lib.eas_hip_layer_norm(None, 0, None) == -1


# -- the Python layer's refusals, on a runtime that allocates nothing -----------------


class _Module:
    """Buffers that are numbers, and no launches."""

    def __init__(self):
        self.ran = []

    def alloc_buffer(self, nbytes, storage):
        return ["buffer", (1 << 30) + 4096 * (len(self.ran) + 1)]

    def buffer_info(self, buf):
        return buf[1], 0, 0

    def copy_from_host(self, buf, arr):
        pass

    def copy_to_host(self, buf, arr):
        pass

    def op_workspace(self, kind, args):
        return 0

    def op_run(self, *args):
        self.ran.append(args)


@pytest.fixture
def fake(monkeypatch):
    from easy_as_amd.runtime.hip import HipRuntime

    m = _Module()
    rt = HipRuntime(ext=m)
    monkeypatch.setattr(ops, "get_runtime", lambda: rt)
    return m


def f(*shape, dtype=np.float32):
    return np.zeros(shape, dtype)


@pytest.mark.parametrize("call,error,message", [
    (lambda: ops.linear(f(2, 3), f(4, 5), f(2, 5)), ValueError, "'w' must be"),
    (lambda: ops.linear(f(2, 3), f(3, 5), f(2, 4)), ValueError, "'y' must hold 2 rows of 5"),
    (lambda: ops.linear(f(2, 3), f(3, 5, dtype=np.float16), f(2, 5)), TypeError, "'w' must be f32"),
    (lambda: ops.linear(f(2, 3, dtype=np.int32), f(3, 5), f(2, 5)), TypeError, "float16 or float32"),
    (lambda: ops.linear([1.0], f(3, 5), f(2, 5)), TypeError, "expected numpy.ndarray"),
    (lambda: ops.linear(f(2, 3), f(3, 5), f(2, 5), activation="tanh"), ValueError, "activation must be one of"),
    (lambda: ops.linear(f(2, 3), f(3, 5), f(2, 5), activation=["relu"]), ValueError, "activation must be one of"),
    (lambda: ops.linear(f(2, 3), f(3, 5), f(2, 5), bias=f(4)), ValueError, "'bias' must hold 5"),
    (lambda: ops.linear(f(2, 3), f(3, 5), f(2, 5), residual=f(2, 5, dtype=np.float16)), TypeError, "'residual' must be f32"),
    (lambda: ops.linear(f(2, 3), f(3, 5), f(2, 5), _sync=1), TypeError, "_sync must be bool"),
    (lambda: ops.linear(f(3, 2).T, f(3, 5), f(2, 5)), ValueError, "C-contiguous"),
    (lambda: ops.linear(f(), f(3, 5), f(2, 5)), ValueError, "at least one axis"),
    (lambda: ops.linear_backward(f(2, 5), None, f(3, 5), dw=f(3, 5)), TypeError, "'x' must be given"),
    (lambda: ops.linear_backward(f(2, 5), f(2, 3), None, dx=f(2, 3)), TypeError, "'w' must be given"),
    (lambda: ops.linear_backward(f(2, 5), f(2, 3), f(3, 5), dx=f(2, 3), activation="silu"), TypeError, "'pre' must be given"),
    (lambda: ops.linear_backward(f(2, 5), f(3, 3), f(3, 5), dw=f(3, 5)), ValueError, "'x' must hold 2 rows"),
    (lambda: ops.linear_backward(f(2, 5), f(2, 3), f(3, 5), dx=f(2, 4)), ValueError, "'dx' must hold"),
    (lambda: ops.linear_backward(f(2, 5), f(2, 3), f(3, 5), dw=f(5, 3)), ValueError, "'dw' must be"),
    (lambda: ops.gated_linear(f(2, 3), f(3, 5), f(3, 6), f(2, 5)), ValueError, "'w_up' must be"),
    (lambda: ops.gated_linear(f(2, 3), f(3, 5), f(3, 5), f(2, 5), gate=f(2, 5)), TypeError, "go together"),
    (lambda: ops.gated_linear_backward(f(2, 5), f(2, 3), f(3, 5), f(3, 5), f(2, 5), f(2, 5), dw_up=f(3, 5)), TypeError, "go together"),
    (lambda: ops.layer_norm(f(2, 0), None, None, f(2, 0)), ValueError, "at least one element"),
    (lambda: ops.layer_norm(f(2, 3), f(3), f(2), f(2, 3)), ValueError, "'bias' must hold 3"),
    (lambda: ops.layer_norm(f(2, 3), None, None, f(2, 3), f(3)), ValueError, "'mean' must hold 2"),
    (lambda: ops.layer_norm(f(2, 3), None, None, f(2, 3), eps=-1.0), ValueError, "eps"),
    (lambda: ops.layer_norm(f(2, 3), None, None, f(2, 3), eps=float("nan")), ValueError, "eps"),
    (lambda: ops.layer_norm(f(2, 3, dtype=np.float16), f(3), f(3, dtype=np.float16), f(2, 3, dtype=np.float16)), TypeError, "'bias' must be f32"),
    (lambda: ops.layer_norm_backward(f(2, 3), f(2, 3), None, None, f(2), f(2, 3)), TypeError, "'mean' and 'rstd'"),
])
def test_the_python_layer_refuses(fake, call, error, message):
    with pytest.raises(error, match=message):
        call()
    assert not fake.ran


def test_weight_layouts(fake):
    torch = pytest.importorskip("torch")
    c = ops._Call("linear", True)
    c.array = lambda name, v, write=False: (0, 2, tuple(v.shape), v.stride())
    w = torch.zeros(40, 30)
    assert c.weights("w", w, 40, 2)[1:4] == (30, 30, False)
    assert c.weights("w", w.t(), 30, 2)[1:4] == (30, 40, True)
    assert c.weights("w", w[:, 5:25], 40, 2)[1:4] == (30, 20, False)
    assert c.weights("w", w[:, :20].t(), 20, 2)[1:4] == (30, 40, True)
    assert c.weights("w", w[:1], 1, 2)[1:4] == (30, 30, False)
    assert c.weights("w", w[:, :1], 40, 2)[1:4] == (30, 1, False)
    for bad in (w[:, ::2], w[:1].expand(40, 30), w.as_strided((40, 30), (1, 1))):
        with pytest.raises(ValueError, match="contiguous along one axis"):
            c.weights("w", bad, 40, 2)
    m = torch.zeros(4, 6, 10)
    assert c.matrix("x", m, None, None)[1:4] == (10, 24, 10)
    assert c.matrix("x", m[:, :, :7], None, None)[1:4] == (10, 24, 7)
    assert c.matrix("x", m[:, :1], None, None)[1:4] == (60, 4, 10)
    for bad in (m[:, :5], m[:, :, ::2], m.transpose(0, 1)):
        with pytest.raises(ValueError):
            c.matrix("x", bad, None, None)
    with pytest.raises(ValueError, match="overlap"):
        c.matrix("x", torch.zeros(10).expand(3, 10), None, None)


# -- calls again: what the native table takes for an earlier call -------------------------


class _Tensor:
    """What op_learn and op_again ask of a torch tensor."""

    def __init__(self, address, rows, cols, ld):
        self.dtype, self.address, self.shape, self.strides = "16 bits", address, (rows, cols), (ld, 1)

    def get_device(self):
        return 0

    def stride(self):
        return self.strides

    def data_ptr(self):
        return self.address


@pytest.fixture
def table(mod, monkeypatch):
    mod.op_setup(_Tensor, lambda device: 0, lambda nbytes, device: None)
    yield mod
    ops._table = None  # set up for torch again by the next call


@pytest.mark.parametrize("kind,args,shift", [
    (2, dict(m=100, k=64, n=64), "x"), (2, dict(m=100, k=64, n=64), "w"), (2, dict(m=100, k=64, n=64), "y"),
    (3, dict(m=100, k=64, n=64), "dy"), (3, dict(m=100, k=64, n=64), "x"), (3, dict(m=100, k=64, n=64), "w"),
    (4, dict(m=100, k=64, n=64), "x"), (4, dict(m=100, k=64, n=64), "w_up"),
    (5, dict(m=100, k=64, n=64), "x"), (5, dict(m=100, k=64, n=64), "w_gate"),
    (2, dict(m=16, k=64, n=64), "w"), (3, dict(m=16, k=64, n=64), "x"),
])
def test_a_call_again_has_the_scratch_of_the_earlier_one(table, kind, args, shift):
    """Of one shape at two addresses, the second call is the first again only where both need the same scratch."""
    mod, name = table, NAMES[kind]
    m, k, n = args["m"], args["k"], args["n"]
    sizes = {"x": (m, k), "dx": (m, k), **{w: (k, n) for w in ("w", "w_gate", "w_up", "dw", "dw_gate", "dw_up")}}
    pointers = [f for f, c in fields(name) if c == "P"][:-1]  # the last is the workspace

    def call(offset):
        values, tensors = dict(args), []
        for i, p in enumerate(pointers):
            if "bias" in p or p == "residual":
                tensors.append(None)
                continue
            rows, cols = sizes.get(p, (m, n))
            values[p] = (i + 1) * P + (offset if p == shift else 0)
            if any(f == p + "_ld" for f, _ in fields(name)):
                values[p + "_ld"] = cols
            tensors.append(_Tensor(values[p], rows, cols, cols))
        packed_args = packed(name, **values)
        return packed_args, tuple(tensors), mod.op_workspace(kind, packed_args)

    def known(tensors, option):
        try:  # no batch of 0 launches: the recipe's own check comes after it was found
            found = mod.op_again(kind, tensors, option, False, 0)
        except ValueError as e:
            assert "batch" in str(e)
            return True
        assert found is NotImplemented
        return False

    for option, (first, second) in enumerate((a, b) for a in range(0, 18, 2) for b in range(0, 18, 2)):
        learnt, tensors, need = call(first)
        mod.op_learn(kind, tensors, option, learnt, need)  # a new option: a new call
        assert known(tensors, option)
        _, again, wanted = call(second)
        assert not known(again, option) or wanted == need, (first, second)


# -- rows so long that 32-bit offsets within a tile of the product end before the tile does -----------


@pytest.mark.parametrize("kind,args", [
    (2, linear(m=65, k=20000008, n=64, x_ld=20000008, w=1 << 40, y=1 << 44, w_ld=64, y_ld=64)),
    (2, linear(m=65, k=20000008, n=64, x_ld=20000009, w=1 << 40, y=1 << 44, w_ld=64, y_ld=64)),  # and off 4 bytes
    (2, linear(m=3, k=16, n=300000000, w=1 << 40, w_ld=300000000, y=1 << 44, y_ld=300000000, dtype=2, ydtype=2)),
    (2, linear(m=300, k=40000008, n=300, x=1 << 40, x_ld=40000008, w_trans=1, w=1 << 44, w_ld=40000008, y=1 << 45, y_ld=300)),
    (3, backward(m=600, n=40000008, k=64, dy=1 << 40, dy_ld=40000008, x_ld=64, w=1 << 44, w_ld=40000008, dw=0, dbias=0, dx=1 << 45, dx_ld=64)),
    (3, backward(m=600, n=40000008, k=64, dy=1 << 40, dy_ld=40000008, x_ld=64, w=1 << 44, w_ld=40000008, dw=0, dbias=0, dx=1 << 45, dx_ld=64,
                 activation=1, pre=1 << 46, pre_ld=40000008)),
    (3, backward(m=600, n=64, k=40000008, dy_ld=64, x=1 << 40, x_ld=40000008, w=0, dx=0, dbias=0, dw=1 << 44, dw_ld=64)),
    (4, gated(m=65, k=20000008, n=64, x_ld=20000008, w_gate=1 << 40, w_up=1 << 41, y=1 << 44, w_gate_ld=64, w_up_ld=64, y_ld=64)),
], ids=["x", "x copied", "w across k", "x and w", "dy", "dz", "x of dw", "gated x"])
def test_rows_beyond_a_tiles_offsets_are_refused(mod, kind, args):
    with pytest.raises(ValueError, match="too long"):
        mod.op_workspace(kind, args)


def test_rows_within_a_tiles_offsets_are_taken(mod, monkeypatch):
    # one row reaches any k, 64 rows of 32 MB reach 2^31 - 2^25 bytes, 256 rows of 8 MB as far
    mod.op_workspace(2, linear(m=1, k=600000000, n=8, x_ld=600000000, w=1 << 40, w_ld=8, y=1 << 44, y_ld=8, dtype=2, ydtype=2))
    mod.op_workspace(2, linear(m=65, k=1 << 24, n=64, x_ld=1 << 24, w=1 << 40, y=1 << 44, w_ld=64, y_ld=64))
    # a long stride over short rows is copied, long rows at their own length are not
    assert mod.op_workspace(2, linear(m=100, x_ld=1 << 24, w=1 << 40, y=1 << 44)) == 100 * 16 * 2 + 128
    monkeypatch.setenv("EAS_HIP_OPS_GEMM", "tile256")
    long = dict(m=300, n=64, w=1 << 40, w_ld=64, y=1 << 44, y_ld=64)
    assert mod.op_workspace(2, linear(k=1 << 22, x_ld=1 << 22, **long)) == 0
    with pytest.raises(ValueError, match="too long"):
        mod.op_workspace(2, linear(k=1 << 23, x_ld=1 << 23, **long))
    monkeypatch.setenv("EAS_HIP_OPS_GEMM", "tile64")
    assert mod.op_workspace(2, linear(k=1 << 23, x_ld=1 << 23, **long)) == 0


# -- host arrays that overlap -------------------------------------------------------------


def halves(first: int, second: int, n: int = 160):
    a = np.zeros(400, np.float32)
    return a[first:first + n].reshape(4, -1), a[second:second + n].reshape(4, -1)


@pytest.mark.parametrize("call", [
    lambda: (lambda y, pre: ops.linear(f(4, 8), f(8, 40), y, pre=pre))(*halves(0, 40)),             # two outputs
    lambda: (lambda y, pre: ops.linear(f(4, 8), f(8, 40), y, pre=pre))(*halves(40, 0)),
    lambda: (lambda x, y: ops.linear(x, f(40, 40), y))(*halves(0, 100)),                             # an output over an input
    lambda: (lambda r, y: ops.linear(f(4, 8), f(8, 40), y, residual=r))(*halves(0, 1)),              # not quite in place
    lambda: (lambda y, b: ops.linear(f(4, 8), f(8, 40), y, bias=b.reshape(-1)[:40]))(*halves(0, 80)),
    lambda: (lambda w, y: ops.linear(f(4, 8), f(8, 40), y, bias=w.reshape(-1)[:40]))(*halves(0, 0)),  # a shorter one from the same place
    lambda: (lambda x: ops.layer_norm(x, None, None, f(4, 10), x.reshape(-1)[3:7]))(halves(0, 0, 40)[0]),  # mean over x
], ids=["two outputs", "the other way", "over an input", "one element on", "over a bias", "from the same place", "over a norm's x"])
def test_overlapping_host_arrays_are_refused(fake, call):
    with pytest.raises(ValueError, match="overlap"):
        call()
    assert not fake.ran


def test_host_arrays_side_by_side_in_place_and_shared_inputs(fake):
    y, pre = halves(0, 160)
    ops.linear(f(4, 8), f(8, 40), y, pre=pre)
    ops.linear(f(4, 8), f(8, 40), y, residual=y)
    x, w = halves(0, 0)
    ops.gated_linear(x, np.zeros((40, 40), np.float32), np.zeros((40, 40), np.float32), f(4, 40), bias_gate=x.reshape(-1)[:40], bias_up=x.reshape(-1)[20:60])
    a = np.zeros(160, np.float32)
    ops.linear(a[40:40].reshape(0, 8), f(8, 40), a[40:40].reshape(0, 40), bias=a[20:60])  # nothing lies nowhere
    assert len(fake.ran) == 4


def test_products_of_more_tiles_than_a_grid_has_threads_for(mod):
    few = dict(m=1, k=8, x_ld=8, w_trans=1, w=1 << 40, w_ld=8, y=1 << 44)
    assert mod.op_workspace(2, linear(n=1 << 29, y_ld=1 << 29, **few)) == 0
    with pytest.raises(ValueError, match="too many tiles"):  # 2^24 workgroups of 256 threads
        mod.op_workspace(2, linear(n=1 << 30, y_ld=1 << 30, **few))
    with pytest.raises(ValueError, match="too many tiles"):  # 2^26 tiles of 512
        mod.op_workspace(2, linear(m=1 << 21, n=1 << 21, k=8, x=1 << 40, x_ld=8, w=1 << 41, w_ld=1 << 21, y=1 << 44, y_ld=1 << 21))


def test_few_rows_of_any_length_are_taken(mod):
    """Up to 64 rows of 16-bit operands go through registers where offsets within a tile end: by 64-bit addresses."""
    k = 40000008
    mod.op_workspace(2, linear(m=64, k=k, n=64, x_ld=k, w=1 << 40, y=1 << 44, w_ld=64, y_ld=64))
    mod.op_workspace(2, linear(m=2, k=k, n=640, x_ld=k, w_trans=1, w=1 << 40, w_ld=k, y=1 << 44, y_ld=640))
    mod.op_workspace(2, linear(m=2, k=64, n=100000008, x_ld=64, w=1 << 40, w_ld=100000008, y=1 << 44, y_ld=100000008))
    mod.op_workspace(4, gated(m=64, k=k, n=64, x_ld=k, w_gate=1 << 40, w_up=1 << 41, y=1 << 44, w_gate_ld=64, w_up_ld=64, y_ld=64))
    dx = dict(m=64, n=k, k=640, dy=1 << 40, dy_ld=k, x=0, x_ld=640, w=1 << 44, w_ld=k, dw=0, dbias=0, dx=1 << 45, dx_ld=640)
    mod.op_workspace(3, backward(**dx))
    mod.op_workspace(3, backward(activation=1, pre=1 << 46, pre_ld=k, **dx))
