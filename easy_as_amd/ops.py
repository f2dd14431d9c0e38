"""The feed-forward operators: layer norm, linear and gated linear, with their gradients.

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
ValueError, and so do products over rows too long for the kernels' offsets (from about 32 MB on),
before anything is launched.

The kernels are in ``csrc/ops``; there is no counterpart in the reference.
"""

from __future__ import annotations

import struct
from typing import Any

import numpy as np

from .runtime import get_runtime

__all__ = ["gated_linear", "gated_linear_backward", "layer_norm", "layer_norm_backward", "linear", "linear_backward"]

_F16, _BF16, _F32 = 0, 1, 2
_NP_CODES = {np.dtype(np.float16): _F16, np.dtype(np.float32): _F32}
_NAMES = {_F16: "f16", _BF16: "bf16", _F32: "f32"}
_SIZES = {_F16: 2, _BF16: 2, _F32: 4}
_ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_MAX_BATCH = 16

# positions in the native operator table, and the C structures of include/eas_hip.h
_NORM, _NORM_BACKWARD, _LINEAR, _LINEAR_BACKWARD, _GATED, _GATED_BACKWARD = range(6)
_STRUCTS = {
    _NORM: struct.Struct("@6P4q2ifi"),
    _NORM_BACKWARD: struct.Struct("@9PQ5q2i"),
    _LINEAR: struct.Struct("@7PQ8q4i"),
    _LINEAR_BACKWARD: struct.Struct("@8PQ9q4i"),
    _GATED: struct.Struct("@9PQ9q4i"),
    _GATED_BACKWARD: struct.Struct("@12PQ12q4i"),
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
        """(address, type, shape, strides in elements) of an array on the GPU."""
        if isinstance(v, self.tensor):
            code = self.codes.get(v.dtype)
            if code is None:
                raise TypeError(f"{name!r} must be f16, bf16 or f32, got {v.dtype}")
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
            host = (v.view(self.rt._torch_mod().int16) if code == _BF16 else v).numpy()
            return self._stage(name, host, v.data_ptr(), write), code, tuple(v.shape), v.stride()
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
        ptr, code, dims, strides = self.array(name, v, write)
        if codes is not None and code not in codes:
            raise TypeError(f"{name!r} must be {' or '.join(_NAMES[c] for c in codes)}, got {_NAMES[code]}")
        if len(dims) == 2:
            rows, cols = dims
            ld, step = strides
        elif not dims:
            raise ValueError(f"{name!r} must have at least one axis")
        else:
            cols, step = dims[-1], strides[-1]
            rows, ld = 1, 0
            for d, s in zip(reversed(dims[:-1]), reversed(strides[:-1])):
                if d != 1 and rows > 1 and s != ld * rows:
                    raise ValueError(f"the rows of {name!r} must lie at one stride")
                if d != 1 and rows == 1:
                    ld = s
                rows *= d
        if shape is not None and (rows != shape[0] or cols != shape[1]):
            raise ValueError(f"{name!r} must hold {shape[0]} rows of {shape[1]}, got {tuple(dims)}")
        if cols > 1 and step != 1:
            raise ValueError(f"the last axis of {name!r} must be contiguous")
        if rows <= 1 or cols == 0:
            ld = max(cols, 1)
        elif ld < cols:
            raise ValueError(f"the rows of {name!r} overlap (a stride of {ld} for {cols} elements)")
        return ptr, ld, rows, cols, code

    def weights(self, name: str, v: Any, k: int, code: int, n: int | None = None,
                codes: tuple[int, ...] | None = None, write: bool = False) -> tuple[int, int, int, bool, int]:
        """(address, row stride, n, rows along k, type) of a [k, n] array."""
        ptr, got, dims, strides = self.array(name, v, write)
        codes = codes or (code,)
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
        _codes.update({torch.float16: _F16, torch.bfloat16: _BF16, torch.float32: _F32})
    return _codes


def _numel(dims: tuple[int, ...]) -> int:
    n = 1
    for d in dims:
        n *= d
    return n


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
