"""Operators of a recurrent policy or dynamics model on the device: the linear
layer with its epilogue, the gated recurrence over the steps of a rollout, and
the Muon update of the layers' matrices, each with the gradients that training
it needs. Torch CUDA tensors in and out, over the C ABI's phyzb_linear,
phyzb_gated_scan and phyzb_muon_update families (include/phyzb.h); no autograd.

Tensors may have any strides (the policy history's [step][feature][world] is a
view), and a call runs on the current stream of its tensors' device, without
waiting for it. Scratch comes from torch's allocator on that stream.
"""
from __future__ import annotations

import ctypes as C
import math
import struct

import torch

from . import _lib

_DT = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}
_ACT = {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "tanh": _lib.ACT_TANH, "silu": _lib.ACT_SILU,
        "gelu": _lib.ACT_GELU}

# phyzb_linear_args and its siblings, field for field (native alignment)
_LINEAR = struct.Struct("3i3qP2qP2qPP2qP2qP2q")
_LINEAR_GRAD = struct.Struct("3i3qP2qP2qP2qP2qP2qP2qP")
_SCAN = struct.Struct("2i3qP3qP3qP2qP3qP3qP")
_SCAN_GRAD = struct.Struct("2i3qP3qP3qP3qP3qP2qP3qP2qP3qP3qP")
_MUON = struct.Struct("4i3qP3qP3qP3q2iP3q4d")
_ORTH = struct.Struct("4i3qP3qP3q")

_NO2, _NO3 = (0, (0, 0)), (0, (0, 0, 0))


def _need(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _dtype(t: torch.Tensor, name: str) -> int:
    d = _DT.get(t.dtype)
    if d is None:
        raise ValueError(f"{name} is {t.dtype}: float32, bfloat16 or float16 is wanted")
    return d


def _arr(t, name: str, shape, dtype, dev: int, none=None) -> tuple:
    """(address, strides) of a tensor that must have this shape, type and device."""
    if t is None:
        _need(none is not None, f"{name} is missing")
        return none
    if t.shape != shape or t.dtype is not dtype or t.get_device() != dev:
        raise ValueError(f"{name} is {tuple(t.shape)} {t.dtype} on {t.device}: {tuple(shape)} {dtype} on cuda:{dev} "
                         "is wanted")
    return t.data_ptr(), t.stride()


def _device(t: torch.Tensor, name: str) -> int:
    dev = t.get_device()
    if dev < 0:
        raise ValueError(f"{name} is on {t.device}: a CUDA device is wanted")
    return dev


def _activation(name: str) -> int:
    a = _ACT.get(name)
    _need(a is not None, f"activation {name!r} is none of {', '.join(_ACT)}")
    return a


class _Op:
    """One operator of the library: asks for its workspace, then runs on the current stream of a device."""

    def __init__(self, run: str, query: str):
        self._names, self._fns = (run, query), None

    def __call__(self, args: bytes, dev: int) -> None:
        if self._fns is None:
            lib = _lib.load()
            self._fns = tuple(getattr(lib, n) for n in self._names)
        run, query = self._fns
        need = C.c_int64()
        code = query(args, C.byref(need))
        if code:
            _lib.check(code)
        n = need.value
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        code = run(args, ws.data_ptr() if n else None, n, torch._C._cuda_getCurrentRawStream(dev))
        if code:
            _lib.check(code)


_linear = _Op("phyzb_linear", "phyzb_linear_workspace")
_linear_grad = _Op("phyzb_linear_grad", "phyzb_linear_grad_workspace")
_scan = _Op("phyzb_gated_scan", "phyzb_gated_scan_workspace")
_scan_grad = _Op("phyzb_gated_scan_grad", "phyzb_gated_scan_grad_workspace")
_muon = _Op("phyzb_muon_update", "phyzb_muon_workspace")
_orth = _Op("phyzb_orthogonalize", "phyzb_orthogonalize_workspace")


def _like(x: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """An [rows, cols] output in x's order: feature-major where x is."""
    if x.stride(0) == 1 and x.stride(1) != 1 and x.shape[0] > 1:
        return torch.empty((cols, rows), dtype=x.dtype, device=x.device).t()
    return torch.empty((rows, cols), dtype=x.dtype, device=x.device)


def linear(x, weight, bias=None, *, activation: str = "none", residual=None, save_pre: bool = False, out=None):
    """act(x @ weight.T + bias) + residual for x [m, k], weight [n, k] of one type, bias [n] float32 and residual
    [m, n] as x. The output takes x's order (feature-major in, feature-major out) unless `out` is given (which may be
    the residual). With `save_pre` also returns x @ weight.T + bias, which the backward pass reads."""
    _need(x.dim() == 2 and weight.dim() == 2, "x and weight must be matrices")
    m, k = x.shape
    n = weight.shape[0]
    dt, dev, act = _dtype(x, "x"), _device(x, "x"), _activation(activation)
    y = _like(x, m, n) if out is None else out
    pre = _like(x, m, n) if save_pre else None
    t = x.dtype
    pw, sw = _arr(weight, "weight", (n, k), t, dev)
    py, sy = (y.data_ptr(), y.stride()) if out is None else _arr(out, "out", (m, n), t, dev)
    pr, sr = _arr(residual, "residual", (m, n), t, dev, _NO2)
    pp, sp = (pre.data_ptr(), pre.stride()) if save_pre else _NO2
    pb = 0
    if bias is not None:
        pb, sb = _arr(bias, "bias", (n,), torch.float32, dev)
        _need(sb[0] == 1 or n == 1, "bias must be contiguous")
    args = _LINEAR.pack(dt, act, dev, m, k, n, x.data_ptr(), *x.stride(), pw, *sw, pb, pr, *sr, py, *sy, pp, *sp)
    _linear(args, dev)
    return (y, pre) if save_pre else y


def linear_backward(dy, x, weight, pre=None, *, activation: str = "none", bias: bool = True, need_dx: bool = True,
                    need_dw: bool = True):
    """Gradients (dx, dweight, dbias) of `linear` from dy [m, n], with the forward's x, weight and pre-activations
    (not needed without an activation). dx and dweight have the inputs' type, dbias is float32; what is not wanted is
    None. The residual's gradient is dy itself."""
    _need(x.dim() == 2 and weight.dim() == 2, "x and weight must be matrices")
    m, k = x.shape
    n = weight.shape[0]
    dt, dev, act = _dtype(x, "x"), _device(x, "x"), _activation(activation)
    t = x.dtype
    pw, sw = _arr(weight, "weight", (n, k), t, dev)
    pd, sd = _arr(dy, "dy", (m, n), t, dev)
    pp, sp = _arr(pre, "pre", (m, n), t, dev, _NO2 if act == 0 else None)
    dx = _like(x, m, k) if need_dx else None
    dw = torch.empty((n, k), dtype=t, device=x.device) if need_dw else None
    db = torch.empty(n, dtype=torch.float32, device=x.device) if bias else None
    px, sx = (dx.data_ptr(), dx.stride()) if need_dx else _NO2
    pg, sg = (dw.data_ptr(), dw.stride()) if need_dw else _NO2
    args = _LINEAR_GRAD.pack(dt, act, dev, m, k, n, pd, *sd, pp, *sp, x.data_ptr(), *x.stride(), pw, *sw, px, *sx,
                             pg, *sg, db.data_ptr() if bias else 0)
    _linear_grad(args, dev)
    return dx, dw, db


def _reset(reset, shape, dev: int) -> tuple:
    if reset is None:
        return _NO3
    if reset.dtype is not torch.uint8 and reset.dtype is not torch.bool or reset.get_device() != dev:
        raise ValueError(f"reset is {reset.dtype} on {reset.device}: uint8 or bool on cuda:{dev} is wanted")
    if reset.shape == shape:
        return reset.data_ptr(), reset.stride()
    if reset.dim() == 2:
        reset = reset.unsqueeze(2)
    return reset.data_ptr(), reset.expand(shape).stride()


def gated_scan(x, gate, h0=None, reset=None, *, out=None):
    """h_t = a_t h_{t-1} + (1 - a_t) x_t along dim 1 of x, gate [b, t, c], a = sigmoid(gate), from h0 [b, c] (float32;
    zeros without). Where reset ([b, t], or [b, t, c] with broadcasting) is not 0 the state before that step is
    dropped. Returns (h in x's type and order, the last state [b, c] in float32)."""
    _need(x.dim() == 3, "x must be [b, t, c]")
    b, t, c = shape = x.shape
    dt, dev = _dtype(x, "x"), _device(x, "x")
    h = torch.empty_like(x) if out is None else out
    last = torch.empty((b, c), dtype=torch.float32, device=x.device)
    pg, sg = _arr(gate, "gate", shape, x.dtype, dev)
    p0, s0 = _arr(h0, "h0", (b, c), torch.float32, dev, _NO2)
    pr, sr = _reset(reset, shape, dev)
    ph, sh = (h.data_ptr(), h.stride()) if out is None else _arr(out, "out", shape, x.dtype, dev)
    args = _SCAN.pack(dt, dev, b, t, c, x.data_ptr(), *x.stride(), pg, *sg, p0, *s0, pr, *sr, ph, *sh,
                      last.data_ptr())
    _scan(args, dev)
    return h, last


def gated_scan_backward(dh, x, gate, h, h0=None, reset=None, dh_last=None, *, out=None):
    """Gradients (dx, dgate, dh0) of `gated_scan` from dh [b, t, c] and dh_last [b, c] (float32), with the forward's
    inputs and its h. `out`: the tensors (dx, dgate) to write, such as the halves of one projection's gradient."""
    _need(x.dim() == 3, "x must be [b, t, c]")
    b, t, c = shape = x.shape
    dt, dev = _dtype(x, "x"), _device(x, "x")
    pd, sd = _arr(dh, "dh", shape, x.dtype, dev)
    pg, sg = _arr(gate, "gate", shape, x.dtype, dev)
    ph, sh = _arr(h, "h", shape, x.dtype, dev)
    p0, s0 = _arr(h0, "h0", (b, c), torch.float32, dev, _NO2)
    pr, sr = _reset(reset, shape, dev)
    pl, sl = _arr(dh_last, "dh_last", (b, c), torch.float32, dev, _NO2)
    dx, dg = (torch.empty_like(x), torch.empty_like(gate)) if out is None else out
    px, sx = _arr(dx, "dx", shape, x.dtype, dev)
    pq, sq = _arr(dg, "dgate", shape, x.dtype, dev)
    dh0 = torch.empty((b, c), dtype=torch.float32, device=x.device)
    args = _SCAN_GRAD.pack(dt, dev, b, t, c, pd, *sd, x.data_ptr(), *x.stride(), pg, *sg, ph, *sh, p0, *s0, pr, *sr,
                           pl, *sl, px, *sx, pq, *sq, dh0.data_ptr())
    _scan_grad(args, dev)
    return dx, dg, dh0


def _matrices(t, name: str, shape=None):
    _need(t.dim() in (2, 3), f"{name} must be [rows, cols] or [batch, rows, cols]")
    t = t if t.dim() == 3 else t.unsqueeze(0)
    if shape is not None:
        _need(t.shape == shape, f"{name} is {tuple(t.shape)}: {tuple(shape)} is wanted")
    return t


def muon_update(weight, grad, momentum, *, lr: float, mu: float = 0.95, nesterov: bool = True,
                weight_decay: float = 0.0, steps: int = 5, scale: float | None = None, copy=None) -> None:
    """Muon step of one matrix [rows, cols] or a stack [batch, rows, cols], in place: momentum <- mu momentum + grad,
    weight <- (1 - lr weight_decay) weight - lr scale NewtonSchulz(grad + mu momentum). weight and momentum are
    float32, grad any type, scale sqrt(max(1, rows / cols)) unless given; `copy` (bfloat16 or float16) gets the new
    weights too."""
    w = _matrices(weight, "weight")
    shape = w.shape
    g = _matrices(grad, "grad", shape)
    dt, dev = _dtype(g, "grad"), _device(w, "weight")
    b, r, c = shape
    pw, sw = _arr(w, "weight", shape, torch.float32, dev)
    pg, sg = _arr(g, "grad", shape, g.dtype, dev)
    pm, sm = _arr(_matrices(momentum, "momentum", shape), "momentum", shape, torch.float32, dev)
    pc, sc, cdt = 0, (0, 0, 0), 0
    if copy is not None:
        _need(copy.dtype in (torch.bfloat16, torch.float16), f"copy is {copy.dtype}: bfloat16 or float16 is wanted")
        pc, sc = _arr(_matrices(copy, "copy", shape), "copy", shape, copy.dtype, dev)
        cdt = _DT[copy.dtype]
    scale = math.sqrt(max(1.0, r / c)) if scale is None else scale
    args = _MUON.pack(dt, dev, int(bool(nesterov)), steps, b, r, c, pg, *sg, pm, *sm, pw, *sw, cdt, 0, pc, *sc,
                      lr, mu, weight_decay, scale)
    _muon(args, dev)


def orthogonalize(x, *, steps: int = 5):
    """The Newton-Schulz iterate of one matrix or a stack of them, X = x / |x|_F first: singular values towards 1 (the
    Muon coefficients leave them within about 0.7 .. 1.2). In x's type."""
    v = _matrices(x, "x")
    dt, dev = _dtype(v, "x"), _device(v, "x")
    out = torch.empty_like(v, memory_format=torch.contiguous_format)
    args = _ORTH.pack(dt, dev, steps, 0, *v.shape, v.data_ptr(), *v.stride(), out.data_ptr(), *out.stride())
    _orth(args, dev)
    return out if x.dim() == 3 else out[0]


def status(device: int = 0) -> None:
    """Raises PhyzbError if a wait inside an operator's kernel on `device` ever ran out (phyzb_nn_status). Waits for the
    device."""
    _lib.check(_lib.load().phyzb_nn_status(int(device)))
