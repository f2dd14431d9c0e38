"""The feed-forward operators: layer norm, root-mean-square norm, linear and gated linear, with their gradients, and
the conversion to 8 bits with the product of 8-bit operands.

These are calls like an ``@eas.kernel``'s: outputs are arguments, every array is a torch GPU tensor,
an ``eas.Tensor`` or a NumPy array (staged through the GPU and copied back, which waits), the work
goes on torch's current stream when a torch GPU tensor is among them, and ``_sync=False`` returns
without waiting, within ``EAS_MAX_IN_FLIGHT`` (``get_runtime().synchronize()`` waits for all).
Under a HIP graph's capture ``_sync=False`` is required and records the work.

Arrays are matrices over their last axis: the axes before it are rows, which must lie at one
stride.  A torch tensor's rows may have any stride of at least their length and any alignment.
Weights are [k, n] as an eas matmul's, or any [k, n] view of rows along k, such as the
transpose of a torch ``nn.Linear``'s weight: ``linear(x, layer.weight.t(), y)``.

Operands are f16, bf16 (torch only) or f32, all of one type.  Sums and statistics are held in 32
bits and results rounded once.  ``activation``: ``"none"``, ``"relu"``, ``"gelu"`` (with erf),
``"gelu_tanh"`` or ``"silu"``.  Wrong types raise TypeError, wrong shapes, strides and overlaps
ValueError, and so do products over rows too long for the kernels' offsets (from about 32 MB on; of
``linear_fp8`` from 8 MB on, unless x has at most 16 rows and both operands lie along k), before
anything is launched.

8-bit operands are torch tensors of ``torch.float8_e4m3fn`` with f32 scales: an element stands for its own
value times the scale of its block, which is 128 elements of a row, of a column, or 128 x 128, and ends where
the matrix ends.  A block's scale is its largest finite magnitude over 448, at least 2^-126; an element is its
value in 32 bits over the scale, rounded once, ties to even, and NaN where the value is infinite or NaN.

The kernels are in ``csrc/ops``; there is no counterpart in the reference.
"""

from __future__ import annotations

import struct
from typing import Any

import numpy as np

from .runtime import get_runtime

__all__ = ["gated_linear", "gated_linear_backward", "layer_norm", "layer_norm_backward", "linear", "linear_backward",
           "linear_fp8", "quantize", "rms_norm", "rms_norm_backward"]

_F16, _BF16, _F32, _E4M3 = 0, 1, 2, 3
_NP_CODES = {np.dtype(np.float16): _F16, np.dtype(np.float32): _F32}
_NAMES = {_F16: "f16", _BF16: "bf16", _F32: "f32", _E4M3: "e4m3"}
_SIZES = {_F16: 2, _BF16: 2, _F32: 4}
_ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_MAX_BATCH = 16

# positions in the native operator table, and the C structures of include/eas_hip.h
_NORM, _NORM_BACKWARD, _LINEAR, _LINEAR_BACKWARD, _GATED, _GATED_BACKWARD = range(6)
_RMS, _RMS_BACKWARD, _QUANTIZE, _LINEAR_FP8 = range(7, 11)
_BLOCK = 128
_STRUCTS = {
    _NORM: struct.Struct("@6P4q2ifi"),
    _NORM_BACKWARD: struct.Struct("@9PQ5q2i"),
    _LINEAR: struct.Struct("@7PQ8q4i"),
    _LINEAR_BACKWARD: struct.Struct("@8PQ9q4i"),
    _GATED: struct.Struct("@9PQ9q4i"),
    _GATED_BACKWARD: struct.Struct("@12PQ12q4i"),
    _RMS: struct.Struct("@8P9q3if"),
    _RMS_BACKWARD: struct.Struct("@8PQ6q4i"),
    _QUANTIZE: struct.Struct("@4P7q4i"),
    _LINEAR_FP8: struct.Struct("@9PQ12q6i"),
}


class _Call:
    """The arguments of one call: their addresses, what has to stay alive and what is copied back."""

    def __init__(self, op: str, sync: Any) -> None:
        if type(sync) is not bool:
            raise TypeError(f"_sync must be bool, got {type(sync)!r}")
        self.op = op
        self.sync = sync
        self.rt = get_runtime()
        self.mod = self.rt._mod()
        torch = self.rt._torch_mod()
        self.tensor = torch.Tensor if torch is not None else ()
        self.codes = _torch_codes(torch)
        self.keep: list[Any] = []
        self.device: int | None = None
        self.staged: dict[tuple[int, int], tuple[Any, str, bool]] = {}
        self.back: list[tuple[Any, Any]] = []

    def array(self, name: str, v: Any, write: bool = False) -> tuple[int, int, tuple[int, ...], tuple[int, ...]]:
        """(address, type, shape, strides in elements) of an array of floats on the GPU."""
        return self._place(name, v, write, False)

    def bytes8(self, name: str, v: Any, write: bool = False) -> tuple[int, int, tuple[int, ...], tuple[int, ...]]:
        """The same of an 8-bit one."""
        return self._place(name, v, write, True)

    def _place(self, name: str, v: Any, write: bool, e4m3: bool) -> tuple[int, int, tuple[int, ...], tuple[int, ...]]:
        if isinstance(v, self.tensor):
            code = self.codes.get(v.dtype)
            if code is None or (code == _E4M3) != e4m3:
                raise TypeError(f"{name!r} must be {'torch.float8_e4m3fn' if e4m3 else 'f16, bf16 or f32'}, got {v.dtype}")
            if v.is_cuda:
                dev = v.get_device()
                if self.device is None:
                    self.device = dev
                elif self.device != dev:
                    raise ValueError(f"{name!r} is on GPU {dev}, the arguments before it on GPU {self.device}")
                self.keep.append(v)
                return v.data_ptr(), code, tuple(v.shape), v.stride()
            if v.device.type != "cpu":
                raise TypeError(f"unsupported torch device for {name!r}: {v.device}")
            if not v.is_contiguous():
                raise ValueError(f"{name!r} must be contiguous on the host")
            v = v.detach()
            torch = self.rt._torch_mod()
            host = (v.view(torch.int16) if code == _BF16 else v.view(torch.uint8) if code == _E4M3 else v).numpy()
            return self._stage(name, host, v.data_ptr(), write), code, tuple(v.shape), v.stride()
        if e4m3:
            raise TypeError(f"{name!r} must be a torch tensor of float8_e4m3fn, got {type(v)!r}")
        if getattr(v, "__eas_tensor__", False):
            if v.device == "hip":
                buf = v._hip_buffer()
                self.keep.append(v)
                return self.mod.buffer_info(buf)[0], _NP_CODES[v.dtype], v.shape, _dense(v.shape)
            v = v.numpy()
        if isinstance(v, np.ndarray):
            code = _NP_CODES.get(v.dtype)
            if code is None:
                raise TypeError(f"{name!r} must be float16 or float32, got {v.dtype}")
            if not v.flags.c_contiguous:
                raise ValueError(f"{name!r} must be C-contiguous")
            return self._stage(name, v, v.ctypes.data, write), code, v.shape, _dense(v.shape)
        raise TypeError(f"expected numpy.ndarray, eas.Tensor or torch.Tensor for {name!r}, got {type(v)!r}")

    def _stage(self, name: str, host: np.ndarray, start: int, write: bool) -> int:
        # By place: an array passed twice (in place) is one buffer, which the entry point judges as it does any.  Others
        # get one each, so that what is written must not lie over them.
        place = (start, int(host.nbytes))
        for (at, nbytes), (_, other, written) in self.staged.items():
            apart = not nbytes or not host.nbytes or start >= at + nbytes or at >= start + place[1]
            if (write or written) and not apart and (at, nbytes) != place:
                raise ValueError(f"{name!r} overlaps {other!r} on the host")
        buf, first, written = self.staged.get(place, (None, name, False))
        if buf is None:
            buf = self.mod.alloc_buffer(max(place[1], 1), "private")
            if host.nbytes:
                self.mod.copy_from_host(buf, host)
            self.keep.append(buf)
        self.staged[place] = (buf, first, written or write)
        if write and host.nbytes:
            self.back.append((buf, host))
        return self.mod.buffer_info(buf)[0]

    def matrix(self, name: str, v: Any, shape: tuple[int, int] | None, codes: tuple[int, ...] | None,
               write: bool = False) -> tuple[int, int, int, int, int]:
        """(address, row stride, rows, columns, type); `shape`: what it must be, -1 for any."""
        ptr, code, dims, strides = (self.bytes8 if codes == (_E4M3,) else self.array)(name, v, write)
        if codes is not None and code not in codes:
            raise TypeError(f"{name!r} must be {' or '.join(_NAMES[c] for c in codes)}, got {_NAMES[code]}")
        if len(dims) == 2:
            rows, cols = dims
            ld, step = strides
        elif not dims:
            raise ValueError(f"{name!r} must have at least one axis")
        else:
            cols, step = dims[-1], strides[-1]
            rows, ld = _one_stride(name, dims[:-1], strides[:-1])
        if shape is not None and (rows != shape[0] or cols != shape[1]):
            raise ValueError(f"{name!r} must hold {shape[0]} rows of {shape[1]}, got {tuple(dims)}")
        if cols > 1 and step != 1:
            raise ValueError(f"the last axis of {name!r} must be contiguous")
        if rows <= 1 or cols == 0:
            ld = max(cols, 1)
        elif ld < cols:
            raise ValueError(f"the rows of {name!r} overlap (a stride of {ld} for {cols} elements)")
        return ptr, ld, rows, cols, code

    def either(self, name: str, v: Any) -> tuple[int, int, int, int, bool]:
        """(address, row stride, rows, columns, whether memory's rows are v's columns) of an 8-bit matrix that is contiguous
        along either axis."""
        ptr, _, dims, strides = self.bytes8(name, v)
        if len(dims) == 2 and dims[1] > 1 and strides[1] != 1 and (strides[0] == 1 or dims[0] <= 1):
            if strides[1] < dims[0]:
                raise ValueError(f"the columns of {name!r} overlap (a stride of {strides[1]} for {dims[0]} elements)")
            return ptr, max(strides[1], 1), dims[0], dims[1], True
        ptr, ld, rows, cols, _ = self.matrix(name, v, None, (_E4M3,))
        return ptr, ld, rows, cols, False

    def weights(self, name: str, v: Any, k: int, code: int, n: int | None = None,
                codes: tuple[int, ...] | None = None, write: bool = False) -> tuple[int, int, int, bool, int]:
        """(address, row stride, n, rows along k, type) of a [k, n] array."""
        codes = codes or (code,)
        ptr, got, dims, strides = (self.bytes8 if codes == (_E4M3,) else self.array)(name, v, write)
        if got not in codes:
            raise TypeError(f"{name!r} must be {' or '.join(_NAMES[c] for c in codes)}, got {_NAMES[got]}")
        if len(dims) != 2 or dims[0] != k or (n is not None and dims[1] != n):
            raise ValueError(f"{name!r} must be [{k}, {'n' if n is None else n}], got {tuple(dims)}")
        n = dims[1]
        s0, s1 = strides
        if k == 0 or n == 0:
            return ptr, max(n, 1), n, False, got
        if (s1 == 1 or n == 1) and (s0 >= n or k == 1):
            return ptr, (s0 if k > 1 else n), n, False, got
        if (s0 == 1 or k == 1) and (s1 >= k or n == 1):
            return ptr, (s1 if n > 1 else k), n, True, got
        raise ValueError(f"{name!r} must be contiguous along one axis, its other stride at least that axis's length")

    def scales(self, name: str, v: Any, shapes: tuple[tuple[int, int], ...], write: bool = False) \
            -> tuple[int, int, int, tuple[int, int]]:
        """(address, strides, shape) of f32 scales of one of `shapes`."""
        ptr, code, dims, strides = self.array(name, v, write)
        if code != _F32:
            raise TypeError(f"{name!r} must be f32, got {_NAMES[code]}")
        if len(dims) > 2:
            rows, ld = _one_stride(name, dims[:-1], strides[:-1])
            dims, strides = (rows, dims[-1]), (ld, strides[-1])
        if tuple(dims) not in shapes:
            raise ValueError(f"{name!r} must be {' or '.join(str(list(s)) for s in dict.fromkeys(shapes))}, got {list(dims)}")
        s0, s1 = (s if d > 1 else 0 for d, s in zip(dims, strides))
        if write:  # each to a place of its own, in lines; one line by itself may lie at any stride
            s1 = s1 if dims[1] > 1 else 1
            s0 = s0 if dims[0] > 1 else 1 if s1 > 1 else max(dims[1], 1)
            if not ((s1 == 1 and s0 >= dims[1]) or (s0 == 1 and (s1 >= dims[0] or dims[1] <= 1)) or 0 in dims):
                raise ValueError(f"{name!r} must be contiguous along one axis, its other stride at least that axis's length")
        return ptr, s0, s1, (dims[0], dims[1])

    def vector(self, name: str, v: Any, n: int, codes: tuple[int, ...], write: bool = False) -> tuple[int, int]:
        """(address, type) of n contiguous elements; an absent one has address 0."""
        if v is None:
            return 0, -1
        ptr, code, dims, strides = self.array(name, v, write)
        if code not in codes:
            raise TypeError(f"{name!r} must be {' or '.join(_NAMES[c] for c in codes)}, got {_NAMES[code]}")
        if len(dims) == 0 or _numel(dims) != n:
            raise ValueError(f"{name!r} must hold {n} elements, got {tuple(dims)}")
        if n > 1 and tuple(strides) != _dense(dims):
            raise ValueError(f"{name!r} must be contiguous")
        return ptr, code

    def run(self, kind: int, at: int | None, tensors: tuple[Any, ...], option: Any, *fields: Any) -> None:
        """Launch operator `kind`; `at`: where in `fields` its scratch's address and size go.  `tensors` and `option`
        are what ``_again`` will see of a call like this one."""
        pack = _STRUCTS[kind].pack
        rt = self.rt
        stream = None if self.device is None else rt._current_stream(self.device)
        if self.device is not None and self.device != rt._torch_mod().cuda.current_device():
            with rt._torch_mod().cuda.device(self.device):
                return self._launch(kind, pack, at, fields, stream, tensors, option)
        return self._launch(kind, pack, at, fields, stream, tensors, option)

    def _launch(self, kind: int, pack: Any, at: int | None, fields: tuple[Any, ...], stream: int | None,
                tensors: tuple[Any, ...], option: Any) -> None:
        mod, rt = self.mod, self.rt
        need, scratch = 0, None
        if at is None:
            args = pack(*fields)
        else:
            head, tail = fields[:at], fields[at:]
            args = pack(*head, 0, 0, *tail)
            need = mod.op_workspace(kind, args)
            if need:
                if self.device is not None:  # torch's allocator orders its memory's reuse on the stream
                    torch = rt._torch_mod()
                    scratch = torch.empty(need, dtype=torch.uint8, device=f"cuda:{self.device}")
                    address = scratch.data_ptr()
                else:
                    scratch = mod.alloc_buffer(need, "private")
                    self.keep.append(scratch)
                    address = mod.buffer_info(scratch)[0]
                args = pack(*head, address, need, *tail)
        if self.sync or self.back or self.staged:
            mod.op_run(kind, args, stream, None, _MAX_BATCH)
            for buf, host in self.back:
                mod.copy_to_host(buf, host)
            if not self.staged:
                _learn(rt, kind, tensors, option, args, need)
            return
        limit = rt._max_pending()
        p = mod.op_run(kind, args, stream, tuple(self.keep), min(_MAX_BATCH, limit) if limit else _MAX_BATCH)
        _learn(rt, kind, tensors, option, args, need)
        if p is None:  # recorded in a graph
            return
        pending = rt._pending
        pending.append(p)
        while limit and len(pending) > limit:
            mod.synchronize(pending.popleft())


class _Again:
    """The native table of calls that ran: one differing from them in its addresses only is enqueued by it alone."""

    def __init__(self, rt: Any) -> None:
        torch = rt._torch_mod()
        uint8, empty = torch.uint8, torch.empty
        rt._mod().op_setup(torch.Tensor, rt._stream_getter(),
                           lambda nbytes, device: empty(nbytes, dtype=uint8, device=f"cuda:{device}"))
        self.rt = rt
        self.call, self.synchronize = rt._mod().op_again, rt._mod().synchronize
        self.pending, self.limit = rt._pending, rt._max_pending()
        self.batch = min(_MAX_BATCH, self.limit) if self.limit else _MAX_BATCH


_table: _Again | None = None


def _learn(rt: Any, kind: int, tensors: tuple[Any, ...], option: Any, args: bytes, need: int) -> None:
    global _table
    if rt._torch_mod() is None:
        return
    if _table is None or _table.rt is not rt:
        _table = _Again(rt)
    rt._mod().op_learn(kind, tensors, option, args, need)


def _again(kind: int, tensors: tuple[Any, ...], option: Any, sync: Any) -> bool:
    """Enqueue a call as an earlier one of its shape; False: not such a call, nothing done."""
    t = _table
    if t is None or type(sync) is not bool:
        return False
    p = t.call(kind, tensors, option, sync, t.batch)
    if p is None:
        return True
    if p is NotImplemented:
        return False
    pending = t.pending
    pending.append(p)
    while t.limit and len(pending) > t.limit:
        t.synchronize(pending.popleft())
    return True


_codes: dict[Any, int] = {}


def _torch_codes(torch: Any) -> dict[Any, int]:
    if not _codes and torch is not None:
        _codes.update({torch.float16: _F16, torch.bfloat16: _BF16, torch.float32: _F32, torch.float8_e4m3fn: _E4M3})
    return _codes


def _numel(dims: tuple[int, ...]) -> int:
    n = 1
    for d in dims:
        n *= d
    return n


def _one_stride(name: str, dims: tuple[int, ...], strides: tuple[int, ...]) -> tuple[int, int]:
    """How many rows the axes `dims` are, and the stride at which those lie."""
    rows, ld = 1, 0
    for d, s in zip(reversed(dims), reversed(strides)):
        if d != 1 and rows > 1 and s != ld * rows:
            raise ValueError(f"the rows of {name!r} must lie at one stride")
        if d != 1 and rows == 1:
            ld = s
        rows *= d
    return rows, ld


def _dense(dims: tuple[int, ...]) -> tuple[int, ...]:
    out, n = [], 1
    for d in reversed(dims):
        out.append(n)
        n *= d
    return tuple(reversed(out))


def _activation(name: Any) -> int:
    code = _ACTIVATIONS.get(name) if type(name) is str else None
    if code is None:
        raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}, got {name!r}")
    return code


def _wide(code: int) -> tuple[int, ...]:
    """An operand's type, or f32."""
    return (code,) if code == _F32 else (code, _F32)


def layer_norm(x: Any, weight: Any, bias: Any, y: Any, mean: Any = None, rstd: Any = None, *, eps: float = 1e-5,
               _sync: bool = True) -> None:
    """``y = (x - mean) * rstd * weight + bias`` over the last axis, ``rstd = (var + eps) ** -0.5``.

    The variance is the population's.  ``weight`` and ``bias`` hold one element per column, of x's
    type or f32 (both the same), or are None.  ``mean`` and ``rstd`` receive one f32 per row, for
    ``layer_norm_backward``.  ``y`` may be ``x``."""
    tensors = (x, weight, bias, y, mean, rstd)
    eps = float(eps)
    if _again(_NORM, tensors, eps, _sync):
        return
    c = _Call("layer_norm", _sync)
    xp, x_ld, m, n, code = c.matrix("x", x, None, None)
    if n == 0:
        raise ValueError("the rows of 'x' must hold at least one element")
    yp, y_ld, _, _, _ = c.matrix("y", y, (m, n), (code,), True)
    wp, wcode = c.vector("weight", weight, n, _wide(code))
    bp, bcode = c.vector("bias", bias, n, _wide(code) if wcode < 0 else (wcode,))
    mp, _ = c.vector("mean", mean, m, (_F32,), True)
    rp, _ = c.vector("rstd", rstd, m, (_F32,), True)
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    wcode = wcode if wcode >= 0 else bcode if bcode >= 0 else code
    c.run(_NORM, None, tensors, eps, xp, wp, bp, yp, mp, rp, m, n, x_ld, y_ld, code, wcode, eps, 0)


def layer_norm_backward(dy: Any, x: Any, weight: Any, mean: Any, rstd: Any, dx: Any = None, dweight: Any = None,
                        dbias: Any = None, *, _sync: bool = True) -> None:
    """The gradients of ``layer_norm`` from ``dy`` and what the forward pass saved.

    ``dx``, ``dweight`` and ``dbias`` are written where given; the last two are of weight's type (x's or
    f32 where weight is None), their sums over the rows added in the same order on every run.
    ``dx`` may be ``dy`` or ``x``."""
    tensors = (dy, x, weight, mean, rstd, dx, dweight, dbias)
    if _again(_NORM_BACKWARD, tensors, 0, _sync):
        return
    c = _Call("layer_norm_backward", _sync)
    xp, x_ld, m, n, code = c.matrix("x", x, None, None)
    if n == 0:
        raise ValueError("the rows of 'x' must hold at least one element")
    dyp, dy_ld, _, _, _ = c.matrix("dy", dy, (m, n), (code,))
    wp, wcode = c.vector("weight", weight, n, _wide(code))
    mp, _ = c.vector("mean", mean, m, (_F32,))
    rp, _ = c.vector("rstd", rstd, m, (_F32,))
    if mean is None or rstd is None:
        raise TypeError("'mean' and 'rstd' must be what layer_norm wrote")
    dxp, dx_ld = c.matrix("dx", dx, (m, n), (code,), True)[:2] if dx is not None else (0, n)
    dwp, dcode = c.vector("dweight", dweight, n, _wide(code) if wcode < 0 else (wcode,), True)
    wcode = wcode if wcode >= 0 else dcode
    dbp, dcode = c.vector("dbias", dbias, n, _wide(code) if wcode < 0 else (wcode,), True)
    wcode = wcode if wcode >= 0 else dcode if dcode >= 0 else code
    c.run(_NORM_BACKWARD, 8, tensors, 0, dyp, xp, wp, mp, rp, dxp, dwp, dbp, m, n, dy_ld, x_ld, dx_ld, code, wcode)


def linear(x: Any, w: Any, y: Any, *, bias: Any = None, residual: Any = None, activation: str = "none",
           pre: Any = None, _sync: bool = True) -> None:
    """``y = act(x @ w + bias) + residual``, in one pass over the product's sums.

    ``y`` is of x's type or f32, ``residual`` and ``pre`` are of y's; ``pre`` receives the activation's
    input, for ``linear_backward``.  ``y`` may be ``residual``."""
    act = _activation(activation)
    tensors = (x, w, bias, residual, y, pre)
    if _again(_LINEAR, tensors, act, _sync):
        return
    c = _Call("linear", _sync)
    xp, x_ld, m, k, code = c.matrix("x", x, None, None)
    wp, w_ld, n, trans, _ = c.weights("w", w, k, code)
    yp, y_ld, _, _, ycode = c.matrix("y", y, (m, n), _wide(code), True)
    bp, _ = c.vector("bias", bias, n, (code,))
    rp, r_ld = c.matrix("residual", residual, (m, n), (ycode,))[:2] if residual is not None else (0, n)
    pp, p_ld = c.matrix("pre", pre, (m, n), (ycode,), True)[:2] if pre is not None else (0, n)
    c.run(_LINEAR, 6, tensors, act, xp, wp, bp, rp, yp, pp, m, k, n, x_ld, w_ld, r_ld, y_ld, p_ld, code, ycode, act, trans)


def linear_backward(dy: Any, x: Any, w: Any, *, dx: Any = None, dw: Any = None, dbias: Any = None,
                    activation: str = "none", pre: Any = None, _sync: bool = True) -> None:
    """The gradients of ``linear``: ``dz = dy * act'(pre)``, ``dx = dz @ w.T``, ``dw = x.T @ dz``, ``dbias``
    = dz summed over rows (residual's gradient is dy itself).

    Each is written where given.  ``dw`` is laid out as ``w`` is; ``dw`` and ``dbias`` are of x's type
    or f32 (both the same).  ``x`` may be None without ``dw``, ``w`` without ``dx``; ``pre`` is needed with
    an activation.  16-bit operands round dz to their type for the two products, as a tensor of gradients
    between two calls would be: f16 needs a scaled loss where dz leaves [6e-5, 65504]."""
    act = _activation(activation)
    tensors = (dy, x, w, pre, dx, dw, dbias)
    if _again(_LINEAR_BACKWARD, tensors, act, _sync):
        return
    c = _Call("linear_backward", _sync)
    dyp, dy_ld, m, n, code = c.matrix("dy", dy, None, None)
    b = _Backward(c, m, n, code, x, (("w", w),), dx, (("dw", dw),), (("dbias", dbias),))
    pp, p_ld = 0, n
    if act:
        if pre is None:
            raise TypeError("'pre' must be given with an activation")
        pp, p_ld = c.matrix("pre", pre, (m, n), (code,))[:2]
    c.run(_LINEAR_BACKWARD, 7, tensors, act, dyp, b.x, b.w[0], pp, b.dx, b.dw[0], b.dbias[0], m, b.k, n, dy_ld, b.x_ld, b.w_ld[0],
          p_ld, b.dx_ld, b.dw_ld[0], code, b.wcode, act, b.trans)


def gated_linear(x: Any, w_gate: Any, w_up: Any, y: Any, *, bias_gate: Any = None, bias_up: Any = None,
                 activation: str = "silu", gate: Any = None, up: Any = None, _sync: bool = True) -> None:
    """``y = act(x @ w_gate + bias_gate) * (x @ w_up + bias_up)``: both products, the activation and their
    product in one kernel.

    ``y`` is of x's type or f32; ``gate`` and ``up`` (both or neither, of y's type) receive the two
    products, for ``gated_linear_backward``.  The weights lie alike."""
    act = _activation(activation)
    tensors = (x, w_gate, w_up, bias_gate, bias_up, y, gate, up)
    if _again(_GATED, tensors, act, _sync):
        return
    c = _Call("gated_linear", _sync)
    xp, x_ld, m, k, code = c.matrix("x", x, None, None)
    gp, g_ld, n, trans, _ = c.weights("w_gate", w_gate, k, code)
    up_, u_ld, _, trans_u, _ = c.weights("w_up", w_up, k, code, n)
    trans = _alike("w_gate", trans, "w_up", trans_u)
    yp, y_ld, _, _, ycode = c.matrix("y", y, (m, n), _wide(code), True)
    if (gate is None) != (up is None):
        raise TypeError("'gate' and 'up' go together")
    bg, _ = c.vector("bias_gate", bias_gate, n, (code,))
    bu, _ = c.vector("bias_up", bias_up, n, (code,))
    sg, sg_ld = c.matrix("gate", gate, (m, n), (ycode,), True)[:2] if gate is not None else (0, n)
    su, su_ld = c.matrix("up", up, (m, n), (ycode,), True)[:2] if up is not None else (0, n)
    c.run(_GATED, 8, tensors, act, xp, gp, up_, bg, bu, yp, sg, su, m, k, n, x_ld, g_ld, u_ld, y_ld, sg_ld, su_ld, code, ycode, act,
          trans)


def gated_linear_backward(dy: Any, x: Any, w_gate: Any, w_up: Any, gate: Any, up: Any, *, dx: Any = None,
                          dw_gate: Any = None, dw_up: Any = None, dbias_gate: Any = None, dbias_up: Any = None,
                          activation: str = "silu", _sync: bool = True) -> None:
    """The gradients of ``gated_linear`` from ``dy`` and the saved ``gate`` and ``up``: ``dg = dy * up * act'(gate)``,
    ``du = dy * act(gate)``, ``dx = dg @ w_gate.T + du @ w_up.T``, ``dw_* = x.T @ d*``, ``dbias_*`` their sums.

    Each is written where given (the two ``dw`` and the two ``dbias`` both or neither); types and layouts
    as in ``linear_backward``."""
    act = _activation(activation)
    tensors = (dy, x, w_gate, w_up, gate, up, dx, dw_gate, dw_up, dbias_gate, dbias_up)
    if _again(_GATED_BACKWARD, tensors, act, _sync):
        return
    c = _Call("gated_linear_backward", _sync)
    dyp, dy_ld, m, n, code = c.matrix("dy", dy, None, None)
    if (dw_gate is None) != (dw_up is None) or (dbias_gate is None) != (dbias_up is None):
        raise TypeError("the gradients of gate and up go together")
    b = _Backward(c, m, n, code, x, (("w_gate", w_gate), ("w_up", w_up)), dx, (("dw_gate", dw_gate), ("dw_up", dw_up)),
                  (("dbias_gate", dbias_gate), ("dbias_up", dbias_up)))
    gp, g_ld = c.matrix("gate", gate, (m, n), (code,))[:2]
    up_, u_ld = c.matrix("up", up, (m, n), (code,))[:2]
    c.run(_GATED_BACKWARD, 11, tensors, act, dyp, b.x, *b.w, gp, up_, b.dx, *b.dw, *b.dbias, m, b.k, n, dy_ld, b.x_ld, *b.w_ld, g_ld,
          u_ld, b.dx_ld, *b.dw_ld, code, b.wcode, act, b.trans)


def rms_norm(x: Any, weight: Any, y: Any = None, rstd: Any = None, *, residual: Any = None, total: Any = None,
             q: Any = None, q_scale: Any = None, eps: float = 1e-5, _sync: bool = True) -> None:
    """``h = x + residual``, ``y = h * rstd * weight`` over the last axis, ``rstd = (mean(h * h) + eps) ** -0.5``.

    ``y`` is of x's type; ``q`` (e4m3) receives y in 8 bits, made from y in 32 bits, and ``q_scale`` [rows,
    blocks of 128 columns] its scales, as ``linear_fp8`` reads them: y or q must be given, the two may both be.
    ``total`` receives h, for the next residual and for ``rms_norm_backward``; residual and total are of x's type or f32
    (both the same).  ``weight`` holds one element per column, of x's type or f32, or is None.  ``rstd`` receives one f32
    per row.  h is held in 32 bits, and so is its mean square: magnitudes beyond 1e19 leave its range.  ``y`` and
    ``total`` may each be ``x`` or ``residual``."""
    tensors = (x, weight, y, rstd, residual, total, q, q_scale)
    eps = float(eps)
    if _again(_RMS, tensors, eps, _sync):
        return
    c = _Call("rms_norm", _sync)
    xp, x_ld, m, n, code = c.matrix("x", x, None, None)
    if n == 0:
        raise ValueError("the rows of 'x' must hold at least one element")
    if y is None and q is None:
        raise TypeError("'y' or 'q' must be given")
    if (q is None) != (q_scale is None):
        raise TypeError("'q' and 'q_scale' go together")
    yp, y_ld = c.matrix("y", y, (m, n), (code,), True)[:2] if y is not None else (0, n)
    rp, r_ld, _, _, hcode = c.matrix("residual", residual, (m, n), _wide(code)) if residual is not None else (0, n, m, n, None)
    tp, t_ld, _, _, tcode = c.matrix("total", total, (m, n), _wide(code) if hcode is None else (hcode,), True) \
        if total is not None else (0, n, m, n, None)
    hcode = hcode if hcode is not None else tcode if tcode is not None else code
    wp, wcode = c.vector("weight", weight, n, _wide(code))
    sp, _ = c.vector("rstd", rstd, m, (_F32,), True)
    qp, q_ld = c.matrix("q", q, (m, n), (_E4M3,), True)[:2] if q is not None else (0, n)
    qs, s0, s1, _ = c.scales("q_scale", q_scale, ((m, -(-n // _BLOCK)),), True) if q_scale is not None else (0, 0, 0, None)
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    c.run(_RMS, None, tensors, eps, xp, wp, yp, sp, rp, tp, qp, qs, m, n, x_ld, y_ld, r_ld, t_ld, q_ld, s0, s1, code,
          wcode if wcode >= 0 else code, hcode, eps)


def rms_norm_backward(dy: Any, h: Any, weight: Any, rstd: Any, dx: Any = None, dweight: Any = None, *, dtotal: Any = None,
                      _sync: bool = True) -> None:
    """The gradients of ``rms_norm`` from ``dy``, what its norm was taken of (``h``: its x, or ``total``) and ``rstd``.

    ``dx`` is the gradient of x as of residual: the norm's, and ``dtotal``, what reaches h by other ways, added to it.
    ``dx`` and ``dweight`` are written where given; h, dtotal and dx are of dy's type or f32 (all the same), dweight is
    of weight's type (dy's or f32 where weight is None), its sums over the rows added in the same order on every run.
    ``dx`` may be ``dy``, ``h`` or ``dtotal``."""
    tensors = (dy, h, weight, rstd, dx, dweight, dtotal)
    if _again(_RMS_BACKWARD, tensors, 0, _sync):
        return
    c = _Call("rms_norm_backward", _sync)
    dyp, dy_ld, m, n, code = c.matrix("dy", dy, None, None)
    if n == 0:
        raise ValueError("the rows of 'dy' must hold at least one element")
    hp, h_ld, _, _, hcode = c.matrix("h", h, (m, n), _wide(code))
    wp, wcode = c.vector("weight", weight, n, _wide(code))
    if rstd is None:
        raise TypeError("'rstd' must be what rms_norm wrote")
    rp, _ = c.vector("rstd", rstd, m, (_F32,))
    dxp, dx_ld = c.matrix("dx", dx, (m, n), (hcode,), True)[:2] if dx is not None else (0, n)
    dwp, dcode = c.vector("dweight", dweight, n, _wide(code) if wcode < 0 else (wcode,), True)
    wcode = wcode if wcode >= 0 else dcode if dcode >= 0 else code
    dtp, dt_ld = c.matrix("dtotal", dtotal, (m, n), (hcode,))[:2] if dtotal is not None else (0, n)
    c.run(_RMS_BACKWARD, 7, tensors, 0, dyp, hp, wp, rp, dxp, dwp, dtp, m, n, dy_ld, h_ld, dx_ld, dt_ld, code, wcode, hcode, 0)


def quantize(x: Any, q: Any, scale: Any, *, gate: Any = None, activation: str = "none", _sync: bool = True) -> None:
    """``q`` (e4m3) = ``act(x)`` in 8 bits, or ``act(gate) * x`` where gate is given, in one pass.

    The shape of ``scale`` says what a block of x [m, n] is: [m, n / 128] 128 elements of a row, as a product over n
    reads its operand; [m / 128, n] of a column, as one over m does; [m / 128, n / 128] a square, as weights are kept
    (each count rounded up).  It may lie either way, and ``gate`` is of x's type.  The activation is made in 32 bits,
    within 2^-20 of itself, whatever that type is."""
    act = _activation(activation)
    tensors = (x, q, scale, gate)
    if _again(_QUANTIZE, tensors, act, _sync):
        return
    c = _Call("quantize", _sync)
    xp, x_ld, m, n, code = c.matrix("x", x, None, None)
    qp, q_ld = c.matrix("q", q, (m, n), (_E4M3,), True)[:2]
    mb, nb = -(-m // _BLOCK), -(-n // _BLOCK)
    sp, s0, s1, dims = c.scales("scale", scale, ((m, nb), (mb, n), (mb, nb)), True)
    # where two of the shapes are the same, so are their blocks
    block = (1, _BLOCK) if dims == (m, nb) else (_BLOCK, 1) if dims == (mb, n) else (_BLOCK, _BLOCK)
    gp, g_ld = c.matrix("gate", gate, (m, n), (code,))[:2] if gate is not None else (0, n)
    c.run(_QUANTIZE, None, tensors, act, xp, qp, sp, gp, m, n, x_ld, q_ld, g_ld, s0, s1, code, act, *block)


def linear_fp8(x: Any, x_scale: Any, w: Any, w_scale: Any, y: Any, *, bias: Any = None, residual: Any = None,
               activation: str = "none", pre: Any = None, _sync: bool = True) -> None:
    """``y = act(x @ w + bias) + residual`` of what the 8-bit ``x`` [m, k] and ``w`` [k, n] stand for.

    Each is contiguous along either axis, so a weight kept as [n, k] is passed as ``weight.t()``, and the gradients are
    products of the same kind: ``linear_fp8(dy, dy_scale, weight, weight_scale, dx)`` with dy [m, n] in blocks of its rows,
    and ``linear_fp8(dy.t(), dy_scale.t(), x, x_scale, dweight)`` with both in blocks of their columns.  ``x_scale``
    [m, k / 128] has a scale for each row and block of k, ``w_scale`` [k / 128, n / 128] one for each square, or
    [k / 128, n] one for each column (counts rounded up), at any strides (of x_scale's rows and w_scale's columns up to
    2105376 elements): one scale for all is an expanded one.
    The product of two blocks' scales is taken in 32 bits and has to be within their range.
    ``y`` is f16, bf16 or f32; bias, residual and pre, which receives the activation's input, are of y's type.  Sums
    are held in 32 bits, for an f32 y throughout; for 16 bits the matrix cores keep each eight products along k to 14
    bits below the largest of them (1.4e-5 of y in the 2-norm, at twice the rate).  ``y`` may be ``residual``."""
    act = _activation(activation)
    tensors = (x, x_scale, w, w_scale, bias, residual, y, pre)
    if _again(_LINEAR_FP8, tensors, act, _sync):
        return
    c = _Call("linear_fp8", _sync)
    xp, x_ld, m, k, x_trans = c.either("x", x)
    wp, w_ld, n, w_trans, _ = c.weights("w", w, k, _E4M3)
    kb, nb = -(-k // _BLOCK), -(-n // _BLOCK)
    xs, xs_row, xs_block, _ = c.scales("x_scale", x_scale, ((m, kb),))
    ws, ws_block, ws_col, dims = c.scales("w_scale", w_scale, ((kb, n), (kb, nb)))
    yp, y_ld, _, _, code = c.matrix("y", y, (m, n), None, True)
    bp, _ = c.vector("bias", bias, n, (code,))
    rp, r_ld = c.matrix("residual", residual, (m, n), (code,))[:2] if residual is not None else (0, n)
    pp, p_ld = c.matrix("pre", pre, (m, n), (code,), True)[:2] if pre is not None else (0, n)
    c.run(_LINEAR_FP8, 8, tensors, act, xp, xs, wp, ws, bp, rp, yp, pp, m, k, n, x_ld, w_ld, xs_row, xs_block, ws_block, ws_col,
          r_ld, y_ld, p_ld, code, act, x_trans, w_trans, dims != (kb, n), 0)


def _alike(a: str, trans_a: bool, b: str, trans_b: bool) -> bool:
    if trans_a != trans_b:
        raise ValueError(f"{a!r} and {b!r} must lie alike (both rows along k or both along n)")
    return trans_a


class _Backward:
    """What the two products' gradients share: x, the weights and the outputs."""

    def __init__(self, c: _Call, m: int, n: int, code: int, x: Any, ws: tuple, dx: Any, dws: tuple, dbs: tuple) -> None:
        self.x = self.dx = 0
        k: int | None = None
        self.x_ld = self.dx_ld = 0
        if x is not None:
            self.x, self.x_ld, rows, k, _ = c.matrix("x", x, None, (code,))
            if rows != m:
                raise ValueError(f"'x' must hold {m} rows, got {rows}")
        elif dws[0][1] is not None:
            raise TypeError("'x' must be given for the weights' gradient")
        if dx is not None:
            self.dx, self.dx_ld, rows, cols, _ = c.matrix("dx", dx, None, (code,), True)
            if rows != m or (k is not None and cols != k):
                raise ValueError(f"'dx' must hold {m} rows of {'k' if k is None else k}, got {rows} of {cols}")
            k = cols
            if ws[0][1] is None or ws[-1][1] is None:
                raise TypeError(f"{ws[0][0]!r} must be given for the input's gradient")
        if k is None:
            k = 0
        self.k = k
        self.w, self.w_ld, self.dw, self.dw_ld, self.dbias = [], [], [], [], []
        layout: tuple[str, bool] | None = None
        self.wcode = code
        got = None
        for (name, w), (dname, dw) in zip(ws, dws):
            for label, v, write, ptrs, lds in ((name, w if dx is not None else None, False, self.w, self.w_ld),
                                               (dname, dw, True, self.dw, self.dw_ld)):
                if v is None:
                    ptrs.append(0)
                    lds.append(0)
                    continue
                ptr, ld, _, trans, t = c.weights(label, v, k, code, n, _wide(code) if write else None, write)
                ptrs.append(ptr)
                lds.append(ld)
                if write:
                    if got is not None and got != t:
                        raise TypeError(f"{label!r} must be {_NAMES[got]}, got {_NAMES[t]}")
                    got = t
                if layout is None:
                    layout = (label, trans)
                else:
                    _alike(layout[0], layout[1], label, trans)
        self.trans = bool(layout and layout[1])
        for name, db in dbs:
            ptr, t = c.vector(name, db, n, _wide(code) if got is None else (got,), True)
            self.dbias.append(ptr)
            if t >= 0:
                got = t
        if got is not None:
            self.wcode = got
