"""ctypes / PyTorch loader of the training-step operator package
(``include/loom/b200_train.h``).

``TrainPackage(out_dir)[name]`` is an operator with the two forms of a
compiled entry (``loader.Entry``):

* ``op(stream=None, **arguments)`` runs it.  Without a stream the call runs on
  the legacy default stream and waits for it; with one (a torch.cuda.Stream or
  a raw handle) it is asynchronous on that stream.  Outputs and workspaces are
  allocated for the call, on its stream, so calls never share one.
* ``op.bind(stream=None, **arguments)`` checks and converts the arguments once
  and returns ``(call, out)``: ``call()`` launches on that stream (the legacy
  default stream when None) without waiting, as often as wanted, for launch
  loops and stream capture.  The binding owns its workspace: keep it as long
  as a graph that captured it is replayed, and let only one launch of it be in
  flight at a time.

Bad arguments raise TypeError or ValueError before anything runs; a status
other than OK raises ``loader.LoomError``.  There is no CPU fallback.
"""

from __future__ import annotations

import ctypes
import json
import os
from collections import namedtuple
from typing import Dict, List, Optional, Sequence, Tuple

from .loader import LoomError, _torch

BLOCK = 256          # values of an 8-bit state that share one top (a value is code * top / 256)
MAX_WIDTH = 32768    # widest row of block_norm

BlockNormResult = namedtuple("BlockNormResult", "y z post_rstd pre_rstd")
BlockNormGrads = namedtuple("BlockNormGrads", "dx dh dgate dpost_weight dpre_weight")

_P, _I64, _INT = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
_F, _D, _SIZE, _U64 = ctypes.c_float, ctypes.c_double, ctypes.c_size_t, ctypes.c_uint64

_ADAM = [_P] * 5 + [_P, _P, _INT, _INT, _P, _D, _D, _D, _P, _P]
_ADAM8 = [_P] * 7 + [_P, _P, _INT, _INT, _P, _D, _D, _D, _P, _P, _U64]
# argument types after the leading count, before the stream
_ARGTYPES = {
    "grad_norm": [_I64, _P, _P, _INT, _F, _P, _P, _SIZE],
    "adamw": [_I64] + _ADAM + [_P, _SIZE],
    "adamw8": [_I64] + _ADAM8 + [_P, _SIZE],
    "block_norm": [_P, _I64, _P, _I64, _P, _I64, _I64, _P, _P, _I64, _I64, _INT, _INT, _INT, _INT,
                   _F, _F, _F, _F, _P, _P, _P, _P],
    "block_norm_backward": [_P, _I64, _P, _I64, _P, _I64, _I64, _P, _P, _P, _P, _P, _I64, _P,
                            _I64, _I64, _I64, _INT, _INT, _INT, _INT, _F, _F, _F, _P, _P, _P, _P,
                            _P, _P, _SIZE],
}


# the same as the structure of a packed call
_PACKED = {name: type("Args_" + name, (ctypes.Structure,),
                      {"_fields_": [(f"a{i}", t) for i, t in enumerate(types)]})
           for name, types in _ARGTYPES.items()}


def _dtype_code(dtype) -> Optional[int]:
    torch = _torch()
    return {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}.get(dtype)


def _need(cond: bool, exc, text: str) -> None:
    if not cond:
        raise exc(text)


def _f32(v) -> float:
    """A number as the C entries get it where they take a float."""
    return ctypes.c_float(float(v)).value


def _tensor(op: str, name: str, t, dtype=None):
    """A CUDA tensor of the given type (or of an operator's three)."""
    torch = _torch()
    _need(isinstance(t, torch.Tensor) and t.is_cuda, TypeError,
          f"{op}: {name} must be a CUDA tensor")
    if dtype is None:
        _need(_dtype_code(t.dtype) is not None, TypeError,
              f"{op}: {name} is {t.dtype}; expected float32, bfloat16 or float16")
    else:
        _need(t.dtype == dtype, TypeError, f"{op}: {name} is {t.dtype}, expected {dtype}")
    return t


def _list(op: str, name: str, tensors, sizes=None, dtype=None) -> List:
    """A list of contiguous CUDA tensors of one type, with the sizes of
    another list where given."""
    torch = _torch()
    _need(not isinstance(tensors, torch.Tensor), TypeError, f"{op}: {name} must be a list of "
                                                            "tensors")
    out = list(tensors)
    if out and dtype is None:
        dtype = _tensor(op, f"{name}[0]", out[0]).dtype
    for i, t in enumerate(out):
        _tensor(op, f"{name}[{i}]", t, dtype)
        _need(t.is_contiguous(), TypeError, f"{op}: {name}[{i}] must be contiguous")
    if sizes is not None:
        _need(len(out) == len(sizes), ValueError,
              f"{op}: {name} has {len(out)} tensors, expected {len(sizes)}")
        for i, (t, n) in enumerate(zip(out, sizes)):
            _need(t.numel() == n, ValueError,
                  f"{op}: {name}[{i}] has {t.numel()} elements, expected {n}")
    return out


def _one_device(op: str, tensors):
    devices = {t.device for t in tensors if t is not None}
    _need(len(devices) == 1, ValueError,
          f"{op}: tensors must be on one CUDA device, got {sorted(str(d) for d in devices)}")
    return devices.pop()


def _disjoint(op: str, written, read) -> None:
    """No tensor that is written may overlap another one of the call."""
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), w)
             for ts, w in ((written, True), (read, False)) for t in ts if t.numel()]
    spans.sort()
    end, write_end = 0, 0    # furthest ends seen, of any tensor and of written ones
    for lo, hi, w in spans:
        _need(lo >= (end if w else write_end), ValueError,
              f"{op}: a tensor that is written overlaps another tensor of the call (or is "
              "given twice)")
        end = max(end, hi)
        if w:
            write_end = max(write_end, hi)


def _span(t):
    """(first, last + 1) address of a strided tensor's elements."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _rows_disjoint(op: str, written, read) -> None:
    """No output may overlap another tensor of the call, or be given twice."""
    outs = [_span(w) for w in written if w is not None and w.numel()]
    others = [_span(r) for r in read if r is not None and r.numel()]
    for i, (a, b) in enumerate(outs):
        for c, d in others + outs[:i]:
            _need(b <= c or d <= a, ValueError,
                  f"{op}: an output overlaps another tensor of the call (or is given twice)")


def _pointers(tensors) -> ctypes.Array:
    return (ctypes.c_void_p * max(1, len(tensors)))(*[t.data_ptr() for t in tensors])


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


class _Call:
    """The converted arguments of one call: everything but the stream."""

    __slots__ = ("args", "out", "keep", "device")

    def __init__(self, args, out, keep, device):
        self.args, self.out, self.keep, self.device = args, out, keep, device


class Operator:
    """One operator of the package."""

    name = ""

    def __init__(self, lib: ctypes.CDLL, meta: dict, package: "TrainPackage"):
        self.meta = meta
        self.package = package
        self.symbol = meta["symbol_name"]
        types = _ARGTYPES[self.name]
        self.fn = getattr(lib, self.symbol)
        self.fn.argtypes, self.fn.restype = types, _INT
        self.stream_fn = getattr(lib, meta["stream_symbol"])
        self.stream_fn.argtypes, self.stream_fn.restype = types + [_P], _INT
        self.packed_fn = getattr(lib, meta["packed_symbol"])
        self.packed_fn.argtypes, self.packed_fn.restype = [_P, _P], _INT
        self.ws_fn = None
        if meta.get("workspace_symbol"):
            self.ws_fn = getattr(lib, meta["workspace_symbol"])
            self.ws_fn.restype = _SIZE
            self.ws_fn.argtypes = [_I64] * (3 if self.name == "block_norm_backward" else 1)

    def workspace_size(self, *sizes: int) -> int:
        return int(self.ws_fn(*sizes)) if self.ws_fn is not None else 0

    def _workspace(self, device, *sizes: int):
        return _torch().empty(self.workspace_size(*sizes), dtype=_torch().uint8, device=device)

    def _prepare(self, **kwargs) -> _Call:
        raise NotImplementedError

    def _on(self, stream, kwargs) -> Tuple[_Call, int]:
        """The call with what it allocates allocated on its stream, and the
        stream's handle (the legacy default stream's for None)."""
        torch = _torch()
        if stream is not None and not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(int(stream)) if int(stream) else None
        with torch.cuda.stream(stream if stream is not None else torch.cuda.default_stream()):
            call = self._prepare(**kwargs)
        return call, (stream.cuda_stream if stream is not None else 0)

    def __call__(self, stream=None, **kwargs):
        torch = _torch()
        device = self._device_of(kwargs)
        with torch.cuda.device(device):
            call, handle = self._on(stream, kwargs)
            if stream is None:
                status = self.fn(*call.args)
            else:
                status = self.stream_fn(*call.args, handle)
                self._used_on(handle, stream, call)
        if status != 0:
            raise LoomError(self.symbol, status)
        return call.out

    def bind(self, stream=None, **kwargs):
        """``(call, out)``: see the module's text.  Bind with the tensors'
        device current."""
        torch = _torch()
        device = self._device_of(kwargs)
        if device.index != torch.cuda.current_device():
            raise ValueError(f"{self.name}: bind with the tensors' device ({device}) current")
        prepared, handle = self._on(stream, kwargs)
        self._used_on(handle, stream, prepared)   # should the binding go while a launch runs
        # one structure instead of up to 31 arguments: converting these took half of
        # a call of one row
        packed = _PACKED[self.name](*prepared.args)
        prepared.keep.append(packed)
        args = (ctypes.c_void_p(ctypes.addressof(packed)), ctypes.c_void_p(handle))
        fn, symbol, index = self.packed_fn, self.symbol, device.index
        current = torch._C._cuda_getDevice    # current_device() without its checks

        def call():
            if current() == index:
                status = fn(*args)
            else:
                with torch.cuda.device(index):
                    status = fn(*args)
            if status != 0:
                raise LoomError(symbol, status)

        call.keep = prepared     # tensors, pointer arrays and workspace live with the call
        return call, prepared.out

    def _used_on(self, handle: int, stream, call: _Call) -> None:
        """Tell the allocator of tensors that a stream other than the current
        one is still using."""
        torch = _torch()
        if torch.cuda.current_stream().cuda_stream == handle:
            return
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(handle) if handle else torch.cuda.default_stream()
        with torch.cuda.stream(stream):
            if torch.cuda.is_current_stream_capturing():
                return
        for t in call.keep:
            if isinstance(t, torch.Tensor):
                t.record_stream(stream)

    def _device_of(self, kwargs):
        """The device of the call's first tensor."""
        torch = _torch()
        for v in kwargs.values():
            items = v if isinstance(v, (list, tuple)) else [v]
            for t in items:
                if isinstance(t, torch.Tensor):
                    if not t.is_cuda:
                        raise TypeError(f"{self.name}: tensors must be CUDA tensors")
                    return t.device
        raise ValueError(f"{self.name}: no tensor given")


class GradNorm(Operator):
    """``grad_norm(grads, max_norm, out=None)``: float32 ``[norm, factor]``,
    the 2-norm of a list of tensors and the factor that brings it down to
    `max_norm` (NaN where the norm is not finite: a step given that factor as
    its ``grad_scale`` changes nothing)."""

    name = "grad_norm"

    def _prepare(self, grads, max_norm, out=None) -> _Call:
        torch = _torch()
        grads = _list(self.name, "grads", grads)
        _need(bool(grads), ValueError, f"{self.name}: no gradients")
        _need(_f32(max_norm) > 0, ValueError,
              f"{self.name}: max_norm must be above zero (as a float32)")
        if out is None:
            out = torch.empty(2, dtype=torch.float32, device=grads[0].device)
        _tensor(self.name, "out", out, torch.float32)
        _need(out.is_contiguous() and out.numel() >= 2, ValueError,
              f"{self.name}: out must be two contiguous float32")
        device = _one_device(self.name, grads + [out])
        _disjoint(self.name, [out], grads)
        ws = self._workspace(device, len(grads))
        ptrs = _pointers(grads)
        sizes = (ctypes.c_int64 * len(grads))(*[g.numel() for g in grads])
        args = (len(grads), ctypes.addressof(ptrs), ctypes.addressof(sizes),
                _dtype_code(grads[0].dtype), float(max_norm), out.data_ptr(), ws.data_ptr(),
                ws.numel())
        return _Call(args, out, grads + [out, ws, ptrs, sizes], device)


class AdamW(Operator):
    """``adamw(params, grads, exp_avg, exp_avg_sq, step, lr, betas=(0.9, 0.999),
    eps=1e-8, weight_decay=0, master=None, grad_scale=None)``: one step of a list
    of tensors, in place; returns `params`.

    params, grads: contiguous, each list of one type (float32, bfloat16 or
    float16); exp_avg, exp_avg_sq (and master, the fp32 copies beside 16-bit
    parameters): float32 of the same sizes.  step: one int64, advanced by every
    call: lists that make up one step in several calls (parameters of two
    types, two learning rates) each need a step of their own.  lr: one float32, or a number, which a bound call then keeps.
    weight_decay: a number, or one per tensor.  grad_scale: one float32 that
    the gradients are multiplied by; where it is not finite the step is
    skipped."""

    name = "adamw"
    state_dtype = "float32"
    default_betas = (0.9, 0.999)

    def _prepare(self, params, grads, exp_avg, exp_avg_sq, step, lr, betas=None, eps=1e-8,
                 weight_decay=0.0, master=None, grad_scale=None, exp_avg_top=None,
                 exp_avg_sq_top=None, seed=None) -> _Call:
        torch = _torch()
        op = self.name
        eight = op == "adamw8"
        params = _list(op, "params", params)
        _need(bool(params), ValueError, f"{op}: no parameters")
        sizes = [p.numel() for p in params]
        grads = _list(op, "grads", grads, sizes)
        state = getattr(torch, self.state_dtype)
        lists: Dict[str, List] = {
            "exp_avg": _list(op, "exp_avg", exp_avg, sizes, state),
            "exp_avg_sq": _list(op, "exp_avg_sq", exp_avg_sq, sizes, state)}
        if eight:
            blocks = [-(-n // BLOCK) for n in sizes]
            lists["exp_avg_top"] = _list(op, "exp_avg_top", exp_avg_top, blocks, torch.float32)
            lists["exp_avg_sq_top"] = _list(op, "exp_avg_sq_top", exp_avg_sq_top, blocks,
                                            torch.float32)
            _need(isinstance(seed, int) and 0 <= seed < 1 << 64, ValueError,
                  f"{op}: seed must be an integer of 64 bits")
        if master is not None:
            _need(params[0].dtype != torch.float32, ValueError,
                  f"{op}: float32 parameters take no master copies")
            lists["master"] = _list(op, "master", master, sizes, torch.float32)
        _tensor(op, "step", step, torch.int64)
        _need(step.numel() == 1, ValueError, f"{op}: step must be one int64")
        if not isinstance(lr, torch.Tensor):
            lr = torch.full((1,), float(lr), dtype=torch.float32, device=params[0].device)
        _tensor(op, "lr", lr, torch.float32)
        _need(lr.numel() == 1, ValueError, f"{op}: lr must be one float32")
        if grad_scale is not None:
            _tensor(op, "grad_scale", grad_scale, torch.float32)
            _need(grad_scale.numel() == 1, ValueError, f"{op}: grad_scale must be one float32")
        decay = [float(w) for w in weight_decay] if isinstance(weight_decay, (list, tuple)) \
            else [float(weight_decay)] * len(params)
        _need(len(decay) == len(params), ValueError,
              f"{op}: weight_decay has {len(decay)} values, expected {len(params)}")
        _need(all(abs(w) < float("inf") for w in decay), ValueError,
              f"{op}: weight_decay must be finite")
        beta1, beta2 = (float(b) for b in (self.default_betas if betas is None else betas))
        _need(0 <= beta1 < 1 and 0 <= beta2 < 1, ValueError, f"{op}: betas must be in [0, 1)")
        least = torch.finfo(torch.float32).tiny if eight else 0.0
        _need(least <= eps < float("inf"), ValueError, f"{op}: eps must be at least {least}")
        scalars = [t for t in (lr, grad_scale) if t is not None]
        written = params + [t for ts in lists.values() for t in ts] + [step]
        device = _one_device(op, written + grads + scalars)
        _disjoint(op, written, grads + scalars)
        ws = self._workspace(device, len(params))
        arrays = {k: _pointers(v) for k, v in lists.items()}
        arrays["params"], arrays["grads"] = _pointers(params), _pointers(grads)
        arrays["sizes"] = (ctypes.c_int64 * len(sizes))(*sizes)
        arrays["decay"] = (ctypes.c_double * len(decay))(*decay)
        at = {k: ctypes.addressof(v) for k, v in arrays.items()}
        args = [len(params), at["params"], at["grads"], at["exp_avg"], at["exp_avg_sq"]]
        if eight:
            args += [at["exp_avg_top"], at["exp_avg_sq_top"]]
        args += [at.get("master"), at["sizes"], at["decay"], _dtype_code(params[0].dtype),
                 _dtype_code(grads[0].dtype), lr.data_ptr(), beta1, beta2, float(eps),
                 _ptr(grad_scale), step.data_ptr()]
        if eight:
            args.append(seed)
        args += [ws.data_ptr(), ws.numel()]
        keep = written + grads + scalars + [ws] + list(arrays.values())
        return _Call(tuple(args), params, keep, device)


class AdamW8(AdamW):
    """``adamw8(..., betas=(0.9, 0.95), exp_avg_top, exp_avg_sq_top, seed)``: the
    same step with both moments as float8_e4m3fn codes, blocks of 256 values
    sharing one float32 top (a value is code * top / 256).  New moments are rounded up or
    down by random bits of `seed`, the step's number and the value's place,
    so that small changes are kept on average; the noise this adds to the
    second moment grows with 1 / (1 - beta2): it is about 12% (one standard
    deviation) at beta2 = 0.95, the default here, and 26% at 0.99, which is as
    far as 8 bits are meant to be used."""

    name = "adamw8"
    state_dtype = "float8_e4m3fn"
    default_betas = (0.9, 0.95)


def _rows(op: str, name: str, t, width: int, dtype=None):
    """A tensor as (tensor, rows, row stride): its last dimension has `width`
    consecutive elements, and its rows lie at one distance."""
    _tensor(op, name, t, dtype)
    _need(t.dim() >= 1 and t.shape[-1] == width, ValueError,
          f"{op}: {name} has shape {tuple(t.shape)}; its last dimension must be {width}")
    if t.dim() == 2 and (t.stride(1) == 1 or width == 1):
        rows, stride = t.shape[0], t.stride(0)
    elif t.is_contiguous():
        rows, stride = t.numel() // width, width
    else:
        try:
            v = t.view(-1, width)
        except RuntimeError:
            raise ValueError(f"{op}: the rows of {name} must lie at one distance") from None
        _need(v.stride(1) == 1 or width == 1, ValueError,
              f"{op}: the last dimension of {name} must be contiguous")
        rows, stride = v.shape[0], v.stride(0)
    stride = stride if rows > 1 else width
    _need(rows < 1 << 31 and stride < 1 << 31, ValueError,
          f"{op}: {name} has {rows} rows at a distance of {stride}; both must be below 2^31")
    return rows, stride


class _Norms(Operator):
    """What both directions check: types, shapes and which parts are there."""

    def _common(self, x_name, x, h, gate, post_weight, pre_weight, post_norm, pre_norm):
        torch = _torch()
        op = self.name
        _tensor(op, x_name, x)
        _need(x.dim() >= 1 and 1 <= x.shape[-1] <= MAX_WIDTH, ValueError,
              f"{op}: {x_name} must have rows of 1 to {MAX_WIDTH} elements")
        width = x.shape[-1]
        rows, x_stride = _rows(op, x_name, x, width)
        branch = next((t.dtype for t in (h, pre_weight) if isinstance(t, torch.Tensor)), x.dtype)
        _need(branch == x.dtype or x.dtype == torch.float32, TypeError,
              f"{op}: a {x.dtype} residual stream takes a branch of its own type, not {branch}")
        if h is None:
            _need(gate is None and post_weight is None and pre_norm, ValueError,
                  f"{op}: without h there is only the pre norm")
            post_norm = False
        _need(post_norm or post_weight is None, ValueError, f"{op}: post_weight without post norm")
        _need(pre_norm or pre_weight is None, ValueError, f"{op}: pre_weight without pre norm")
        h_stride = gate_stride = gate_rows = 0
        if h is not None:
            h_rows, h_stride = _rows(op, "h", h, width, branch)
            _need(h_rows == rows, ValueError, f"{op}: h has {h_rows} rows, {x_name} {rows}")
        if gate is not None:
            gate_rows, gate_stride = _rows(op, "gate", gate, width, branch)
            _need(gate_rows > 0 and rows % gate_rows == 0, ValueError,
                  f"{op}: {rows} rows do not divide over {gate_rows} rows of gate")
        for name, w in (("post_weight", post_weight), ("pre_weight", pre_weight)):
            if w is not None:
                _tensor(op, name, w, branch)
                _need(w.shape == (width,) and w.is_contiguous(), ValueError,
                      f"{op}: {name} must be {width} contiguous elements")
        return (width, rows, x_stride, h_stride, gate_stride, gate_rows, branch, bool(post_norm),
                bool(pre_norm))

    def _scales(self, *values):
        for v in values:
            _need(abs(_f32(v)) < float("inf"), ValueError,
                  f"{self.name}: scales and offsets must be finite (as float32)")
        return tuple(float(v) for v in values)


class BlockNorm(_Norms):
    """``block_norm(x, h=None, gate=None, post_weight=None, pre_weight=None,
    post_norm=True, pre_norm=True, eps=1e-6, weight_offset=0, residual_scale=1,
    branch_scale=1, out=None)``: ``BlockNormResult(y, z, post_rstd, pre_rstd)``

        u = rms_norm(h) * (post_weight + weight_offset)
        y = residual_scale * x + branch_scale * gate * u
        z = rms_norm(y) * (pre_weight + weight_offset)

    over the last dimension (at most 32768 wide).  x: the residual stream; h:
    the block's output, of x's type, or 16-bit beside a float32 x; gate: of
    h's type, its rows each serving an equal run of x's rows (as many rows as
    x, one a sequence, or one for all).  Without h, y is x, whatever
    residual_scale is; a missing weight is all ones; post_norm or pre_norm False
    leaves that norm out.  Rows may be strided; outputs are contiguous.  `out`
    (a BlockNormResult) takes the place of new outputs; what is not made is
    None."""

    name = "block_norm"

    def _prepare(self, x, h=None, gate=None, post_weight=None, pre_weight=None, post_norm=True,
                 pre_norm=True, eps=1e-6, weight_offset=0.0, residual_scale=1.0, branch_scale=1.0,
                 out=None) -> _Call:
        torch = _torch()
        op = self.name
        (width, rows, x_stride, h_stride, gate_stride, gate_rows, branch, post_norm,
         pre_norm) = self._common("x", x, h, gate, post_weight, pre_weight, post_norm, pre_norm)
        _need(0 <= _f32(eps) < float("inf"), ValueError,
              f"{op}: eps must be at least zero and finite (as a float32)")
        scales = self._scales(weight_offset, residual_scale, branch_scale)
        device = _one_device(op, [x, h, gate, post_weight, pre_weight])
        if out is None:
            new = lambda dtype, *shape: torch.empty(*shape, dtype=dtype, device=device)  # noqa: E731
            out = BlockNormResult(
                new(x.dtype, x.shape) if h is not None else x,
                new(branch, x.shape) if pre_norm else None,
                new(torch.float32, rows) if post_norm else None,
                new(torch.float32, rows) if pre_norm else None)
        else:
            out = BlockNormResult(*out)
            _need((out.y is x) if h is None else True, ValueError,
                  f"{op}: without h, out.y must be x")
            self._check_out("y", out.y if h is not None else None, x.shape, x.dtype,
                            h is not None, device)
            self._check_out("z", out.z, x.shape, branch, pre_norm, device)
            self._check_out("post_rstd", out.post_rstd, (rows,), torch.float32, post_norm, device)
            self._check_out("pre_rstd", out.pre_rstd, (rows,), torch.float32, pre_norm, device)
            _rows_disjoint(op, [out.y if h is not None else None] + list(out[1:]),
                           [x, h, gate, post_weight, pre_weight])
        y = out.y if h is not None else None
        args = (x.data_ptr(), x_stride, _ptr(h), h_stride, _ptr(gate), gate_stride, gate_rows,
                _ptr(post_weight), _ptr(pre_weight), rows, width, _dtype_code(x.dtype),
                _dtype_code(branch), int(post_norm), int(pre_norm), float(eps), *scales, _ptr(y),
                _ptr(out.z), _ptr(out.post_rstd), _ptr(out.pre_rstd))
        return _Call(args, out, [x, h, gate, post_weight, pre_weight, *out], device)

    def _check_out(self, name, t, shape, dtype, made, device) -> None:
        if not made:
            _need(t is None, ValueError, f"{self.name}: out.{name} is not made by this call")
            return
        _tensor(self.name, f"out.{name}", t, dtype)
        _need(tuple(t.shape) == tuple(shape) and t.is_contiguous() and t.device == device,
              ValueError, f"{self.name}: out.{name} must be contiguous, of shape {tuple(shape)}, "
                          f"on {device}")


class BlockNormBackward(_Norms):
    """``block_norm_backward(y, h=None, gate=None, post_weight=None,
    pre_weight=None, post_rstd=None, pre_rstd=None, dy=None, dz=None,
    post_norm=True, pre_norm=True, weight_offset=0, residual_scale=1,
    branch_scale=1)``: ``BlockNormGrads(dx, dh, dgate, dpost_weight,
    dpre_weight)``.

    y (x where there is no h), the statistics and the other arguments are
    those of block_norm; dy and dz the gradients of y and z (dy None: zero).
    Each gradient has the shape and type of what it is the gradient of, rounded
    once; what is not there is None."""

    name = "block_norm_backward"

    def _prepare(self, y, h=None, gate=None, post_weight=None, pre_weight=None, post_rstd=None,
                 pre_rstd=None, dy=None, dz=None, post_norm=True, pre_norm=True,
                 weight_offset=0.0, residual_scale=1.0, branch_scale=1.0) -> _Call:
        torch = _torch()
        op = self.name
        (width, rows, y_stride, h_stride, gate_stride, gate_rows, branch, post_norm,
         pre_norm) = self._common("y", y, h, gate, post_weight, pre_weight, post_norm, pre_norm)
        scales = self._scales(weight_offset, residual_scale, branch_scale)
        dy_stride = dz_stride = 0
        if dy is not None:
            dy_rows, dy_stride = _rows(op, "dy", dy, width, y.dtype)
            _need(dy_rows == rows, ValueError, f"{op}: dy has {dy_rows} rows, y {rows}")
        _need((dz is not None) == pre_norm, ValueError,
              f"{op}: dz goes with the pre norm")
        if dz is not None:
            dz_rows, dz_stride = _rows(op, "dz", dz, width, branch)
            _need(dz_rows == rows, ValueError, f"{op}: dz has {dz_rows} rows, y {rows}")
        for name, t, there in (("post_rstd", post_rstd, post_norm),
                               ("pre_rstd", pre_rstd, pre_norm)):
            _need((t is not None) == there, ValueError, f"{op}: {name} goes with its norm")
            if there:
                _tensor(op, name, t, torch.float32)
                _need(t.numel() == rows and t.is_contiguous(), ValueError,
                      f"{op}: {name} must be {rows} contiguous float32")
        device = _one_device(op, [y, h, gate, post_weight, pre_weight, post_rstd, pre_rstd, dy,
                                  dz])
        like = lambda t: None if t is None else torch.empty(  # noqa: E731
            t.shape, dtype=t.dtype, device=device)
        out = BlockNormGrads(like(y), like(h), like(gate), like(post_weight), like(pre_weight))
        ws = self._workspace(device, rows, width, gate_rows)
        args = (y.data_ptr(), y_stride, _ptr(h), h_stride, _ptr(gate), gate_stride, gate_rows,
                _ptr(post_weight), _ptr(pre_weight), _ptr(post_rstd), _ptr(pre_rstd), _ptr(dy),
                dy_stride, _ptr(dz), dz_stride, rows, width, _dtype_code(y.dtype),
                _dtype_code(branch), int(post_norm), int(pre_norm), *scales, _ptr(out.dx),
                _ptr(out.dh), _ptr(out.dgate), _ptr(out.dpost_weight), _ptr(out.dpre_weight),
                ws.data_ptr(), ws.numel())
        keep = [y, h, gate, post_weight, pre_weight, post_rstd, pre_rstd, dy, dz, *out, ws]
        return _Call(args, out, keep, device)


OPERATORS = {cls.name: cls for cls in (GradNorm, AdamW, AdamW8, BlockNorm, BlockNormBackward)}


class TrainPackage:
    """The built operator package: ``TrainPackage(out_dir)`` or
    ``TrainPackage(manifest_path)``."""

    def __init__(self, path: str):
        manifest = path if path.endswith(".json") else os.path.join(path, "manifest.json")
        with open(manifest, "r", encoding="utf-8") as fh:
            self.manifest = json.load(fh)
        self.name = self.manifest["package_name"]
        artifact = self.manifest["artifact_path"]
        if not os.path.exists(artifact):
            artifact = os.path.join(os.path.dirname(manifest), os.path.basename(artifact))
        self.path = artifact
        self.lib = ctypes.CDLL(artifact)
        self.entries = {e["entry_name"]: OPERATORS[e["entry_name"]](self.lib, e, self)
                        for e in self.manifest["entries"]}

    def __getitem__(self, name: str) -> Operator:
        return self.entries[name]

    def __getattr__(self, name: str) -> Operator:
        entries = self.__dict__.get("entries", {})
        if name in entries:
            return entries[name]
        raise AttributeError(name)
