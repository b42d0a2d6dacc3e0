"""Dense layers on the HIP kernels: linear with its epilogue and its backward, and activations kept in 8 bits ("mx8").

Tensor-level calls and autograd nodes over the `lt_mx8_*`, `lt_linear_*` and `lt_rms_norm_*` entry points of include/latte_hip.h; the public
names are re-exported by latte_amd.functional, the modules are latte_amd.sparse_modules.Linear / RMSNorm.  Types: fp32,
bfloat16, float16 (all operands of a call share one); sums are fp32.  GPU tensors only: there is no CPU fallback."""
from __future__ import annotations

import torch
from torch.autograd import Function

from . import _lib
from .ops import _ws_bytes

__all__ = ["Mx8", "quantize_mx8", "linear", "rms_norm"]

_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACT = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
_BITS, _BYTE, _FULL = 1, 2, 3     # LT_DERIV_*


def _dt(t: torch.Tensor, name: str) -> int:
    if not t.is_cuda:
        raise _lib.LatteHipError(f"{name}: tensor must be on the GPU (no CPU fallback in the product path)")
    d = _DT.get(t.dtype)
    if d is None:
        raise TypeError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    return d


def _like(t, ref: torch.Tensor, shape, name: str):
    """`t` checked against the operand it goes with: type, device, shape (a torch.Size)"""
    if t.dtype != ref.dtype:
        raise TypeError(f"{name}: expected {ref.dtype}, got {t.dtype}")
    if t.device != ref.device:
        raise ValueError(f"{name}: on {t.device}, the other operands on {ref.device}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _rows(t: torch.Tensor, cols: int):
    """-> (2-D tensor with neighbouring columns, its row stride): a view wherever the strides allow one"""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    ld, c = t.stride()
    if c != 1 and cols > 1:
        t = t.contiguous()
        ld = cols
    return t, (ld if t.shape[0] > 1 else cols)   # a single row's stride means nothing


_raw_stream = torch._C._cuda_getCurrentRawStream


def _stream_of(t: torch.Tensor) -> int:
    """the current stream of the tensor's own device, whatever device is current"""
    return _raw_stream(t.device.index)


def _p(t):
    return None if t is None else t.data_ptr()


_LIB = None


def _call(name: str, *args) -> None:
    """_lib.call with plain integers for pointers: a call costs 4 us of host time here, of which 1 is spent in ctypes"""
    global _LIB
    if _LIB is None:
        _LIB = _lib.load()
    rc = getattr(_LIB, name)(*args)
    if rc != 0:
        raise _lib.LatteHipError(f"{name} failed (rc={rc}): {(_LIB.lt_last_error() or b'').decode()}")


def _no_second(name: str) -> None:
    """a backward pass runs with gradients enabled only where its own graph is asked for, which these kernels do not build"""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{name}: gradients of gradients are not implemented (create_graph=True)")


def _buf(nbytes: int, device) -> torch.Tensor:
    """workspace of one call: torch's allocator (and a graph's private pool) keeps it from any other stream or graph"""
    return torch.empty(nbytes if nbytes > 256 else 256, dtype=torch.uint8, device=device)


# ------------------------------------------------------------------ mx8
class Mx8:
    """A matrix held in 8 bits: `values` float8_e4m3fn [M, K] and `scales` uint8 [M, ceil(K / 32)] -- element (i, j) stands for
    values[i, j] * 2^(scales[i, j // 32] - 127)."""

    __slots__ = ("values", "scales")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if values.dtype != torch.float8_e4m3fn or values.dim() != 2:
            raise TypeError(f"Mx8: values must be a float8_e4m3fn matrix, got {values.dtype} {tuple(values.shape)}")
        if scales.dtype != torch.uint8 or tuple(scales.shape) != (values.shape[0], (values.shape[1] + 31) // 32):
            raise ValueError(f"Mx8: scales must be uint8 [M, ceil(K / 32)], got {scales.dtype} {tuple(scales.shape)} "
                             f"for values {tuple(values.shape)}")
        if values.device != scales.device:
            raise ValueError(f"Mx8: values on {values.device}, scales on {scales.device}")
        self.values = values.contiguous()
        self.scales = scales.contiguous()

    @property
    def shape(self):
        return self.values.shape

    @property
    def device(self):
        return self.values.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """the values it stands for (exact in float32 and bfloat16)"""
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        dt = _dt(out, "Mx8.dequantize")
        M, K = self.shape
        _call("lt_mx8_dequantize", _p(self.values), _p(self.scales), M, K, dt, _p(out), _stream_of(out))
        return out

    @staticmethod
    def empty(M: int, K: int, device) -> "Mx8":
        return Mx8(torch.empty((M, K), dtype=torch.float8_e4m3fn, device=device),
                   torch.empty((M, (K + 31) // 32), dtype=torch.uint8, device=device))


def quantize_mx8(x: torch.Tensor) -> Mx8:
    """x [..., K] -> Mx8 [rows, K]: 32 neighbours share the smallest power of two that brings their largest finite magnitude
    to at most 448; nearest even e4m3.  Infinities and NaN are held as NaN."""
    dt = _dt(x, "quantize_mx8")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"quantize_mx8: expected rows of at least one element, got shape {tuple(x.shape)}")
    K = x.shape[-1]
    x2, ld = _rows(x.detach(), K)
    q = Mx8.empty(x2.shape[0], K, x.device)
    _call("lt_mx8_quantize", _p(x2), ld, x2.shape[0], K, dt, _p(q.values), _p(q.scales), _stream_of(x2))
    return q


# ------------------------------------------------------------------ linear
def _linear_fwd(x2, ldx, w, ldw, bias, res, act: str, deriv_kind: int):
    """-> (y [M, N], deriv | None)"""
    M, K = x2.shape
    N = w.shape[0]
    dt = _DT[x2.dtype]
    dev = x2.device
    y = torch.empty((M, N), dtype=x2.dtype, device=dev)
    deriv = None
    if deriv_kind == _BITS:
        deriv = torch.empty((M, (N + 15) // 16), dtype=torch.int16, device=dev)
    elif deriv_kind == _BYTE:
        deriv = torch.empty((M, N), dtype=torch.uint8, device=dev)
    elif deriv_kind == _FULL:
        deriv = torch.empty((M, N), dtype=torch.float32 if dt == 0 else torch.int16, device=dev)
    nb = _ws_bytes("lt_linear_workspace_bytes", M, K, N, dt)
    ws = _buf(nb, dev) if nb > 0 else None
    r2, ldr = _rows(res, N) if res is not None else (None, 0)
    _call("lt_linear_fwd", _p(x2), ldx, _p(w), ldw, _p(bias), _p(r2), ldr, _ACT[act], M, K, N, dt, _p(y), _p(deriv),
              deriv_kind, _p(ws), nb, _stream_of(x2))
    return y, deriv


class _Linear(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, checkpoint):
        N, K = weight.shape
        x2, ldx = _rows(x, K)
        w2, ldw = _rows(weight, K)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        kind = 0
        if act != "none" and (need_x or need_w or need_b):
            kind = _BITS if act == "relu" else (_BYTE if checkpoint == "mx8" else _FULL)
        if bias is not None and not bias.is_contiguous():
            bias = bias.contiguous()
        y, deriv = _linear_fwd(x2, ldx, w2, ldw, bias, residual, act, kind)
        keep_x = x_scales = None
        if need_w:
            if checkpoint == "mx8":
                q = quantize_mx8(x2)
                keep_x, x_scales, ldx = q.values, q.scales, K
            else:
                keep_x = x2
        ctx.save_for_backward(keep_x, x_scales, w2 if need_x else None, deriv)
        ctx.meta = (K, N, x.dtype, kind, ldx, ldw, x.shape)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], N)

    @staticmethod
    def backward(ctx, dy):
        _no_second("linear")
        x2, xs, w2, deriv = ctx.saved_tensors
        K, N, dtype, kind, ldx, ldw, x_shape = ctx.meta
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            dev = dy.device
            dy2, lddy = _rows(dy, N)
            M = dy2.shape[0]
            if need_x:
                dx = torch.empty((M, K), dtype=dtype, device=dev)
            if need_w:
                dw = torch.empty((N, K), dtype=dtype, device=dev)
            if need_b:
                db = torch.empty((N,), dtype=dtype, device=dev)
            dt = _DT[dtype]
            ws = _buf(_ws_bytes("lt_linear_bwd_workspace_bytes", M, K, N, dt, int(xs is not None)), dev)
            _call("lt_linear_bwd", dy2.data_ptr(), lddy, _p(x2), ldx, _p(xs), _p(w2), ldw, _p(deriv), kind, M, K, N, dt, _p(dx), _p(dw),
                  _p(db), ws.data_ptr(), ws.numel(), _stream_of(dy2))
            if need_x and len(x_shape) != 2:
                dx = dx.view(x_shape)
        return dx, dw, db, (dy if need_r else None), None, None


def _linear_mx8(x: Mx8, weight: Mx8, bias, act: str, residual, dtype):
    M, K = x.shape
    N = weight.shape[0]
    given = [t for t in (bias, residual) if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        raise RuntimeError("linear: mx8 operands carry no gradient; call it under torch.no_grad()")
    dtype = dtype or (given[0].dtype if given else torch.bfloat16)
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"linear: results of mx8 operands are bfloat16 or float16, not {dtype}")
    if weight.shape[1] != K or min(M + 1, K, N) < 1:
        raise ValueError(f"linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not go together")
    if not x.values.is_cuda:
        raise _lib.LatteHipError("linear: tensor must be on the GPU (no CPU fallback in the product path)")
    if weight.device != x.device:
        raise ValueError(f"linear weight: on {weight.device}, the other operands on {x.device}")
    y = torch.empty((M, N), dtype=dtype, device=x.device)
    if bias is not None:
        bias = _like(bias, y, y.shape[1:], "linear bias").contiguous()
    r2, ldr = (None, 0) if residual is None else _rows(_like(residual, y, y.shape, "linear residual"), N)
    nb = _ws_bytes("lt_linear_mx8_workspace_bytes", M, K, N)
    ws = _buf(nb, x.device) if nb > 0 else None
    _call("lt_linear_mx8_fwd", _p(x.values), _p(x.scales), _p(weight.values), _p(weight.scales), _p(bias), _p(r2), ldr, _ACT[act],
              M, K, N, _DT[dtype], _p(y), _p(ws), nb, _stream_of(y))
    return y


def linear(x, weight, bias=None, act: str = "none", residual=None, checkpoint: str | None = None, dtype: torch.dtype | None = None):
    """act(x @ weight.T + bias) + residual as one kernel; act: "none" | "relu" | "gelu" (exact) | "silu".

    x [..., K], weight [N, K], bias [N], residual [..., N] -> [..., N], all of one type (float32, bfloat16, float16), sums in
    fp32.  Differentiable in all four; the backward pass reads x, weight and act'.  checkpoint="mx8" keeps what it reads of x
    in 8 bits (quantize_mx8: relative error at most 2^-4 an element) and act' of GELU / SiLU on a uniform 8-bit grid
    (error at most 1/384); the ReLU's act' is one bit either way.  The output does not depend on `checkpoint`.

    x and weight both Mx8 (serving, no gradient): the product of the held values on the 8-bit matrix instructions; bias,
    residual and the result are bfloat16 or float16 (`dtype`; bias' or the residual's, else bfloat16)."""
    if act not in _ACT:
        raise ValueError(f"linear: act must be one of {sorted(_ACT)}, got {act!r}")
    if checkpoint not in (None, "mx8"):
        raise ValueError(f"linear: checkpoint must be None or 'mx8', got {checkpoint!r}")
    if isinstance(x, Mx8) or isinstance(weight, Mx8):
        if not (isinstance(x, Mx8) and isinstance(weight, Mx8)):
            raise TypeError("linear: x and weight are both Mx8 or neither is (quantize_mx8, Mx8.dequantize)")
        return _linear_mx8(x, weight, bias, act, residual, dtype)
    if dtype is not None and dtype != x.dtype:
        raise TypeError(f"linear: results have the operands' type {x.dtype}, not {dtype}")
    _dt(x, "linear x")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or min(weight.shape) < 1:
        raise ValueError(f"linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not go together")
    N, K = weight.shape
    _like(weight, x, weight.shape, "linear weight")
    if bias is not None:
        _like(bias, x, weight.shape[:1], "linear bias")
    if residual is not None:
        _like(residual, x, x.shape[:-1] + weight.shape[:1], "linear residual")
    return _Linear.apply(x, weight, bias, residual, act, checkpoint)


# ------------------------------------------------------------------ rms_norm
def _rms_fwd(x, w, residual, eps, want_h, want_y, want_y8, want_h8, want_rstd):
    """-> (h, y, y8, h8, rstd), None where not asked for"""
    C = x.shape[-1]
    x2, ldx = _rows(x, C)
    M, dev = x2.shape[0], x.device
    r2, ldr = (None, 0) if residual is None else _rows(residual, C)
    h = torch.empty((M, C), dtype=x.dtype, device=dev) if want_h else None
    y = torch.empty((M, C), dtype=x.dtype, device=dev) if want_y else None
    y8 = Mx8.empty(M, C, dev) if want_y8 else None
    h8 = Mx8.empty(M, C, dev) if want_h8 else None
    rstd = torch.empty((M,), dtype=torch.float32, device=dev) if want_rstd else None
    p8 = lambda q: (None, None) if q is None else (_p(q.values), _p(q.scales))  # noqa: E731
    _call("lt_rms_norm_fwd", _p(x2), ldx, _p(r2), ldr, _p(w), float(eps), M, C, _DT[x.dtype], _p(h), _p(y), *p8(y8), *p8(h8),
              _p(rstd), _stream_of(x2))
    return h, y, y8, h8, rstd


class _RmsNorm(Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, checkpoint):
        C = x.shape[-1]
        w = weight.contiguous()
        need = any(ctx.needs_input_grad)
        ck = need and checkpoint == "mx8"
        h, y, _, h8, rstd = _rms_fwd(x, w, residual, eps, residual is not None, True, False, ck, need)
        if need:
            if ck:
                ctx.save_for_backward(None, h8.values, h8.scales, w, rstd)
            else:   # without a residual h is x itself
                ctx.save_for_backward(h if residual is not None else _rows(x, C)[0], None, None, w, rstd)
        ctx.set_materialize_grads(False)   # a sum that nothing reads costs no zeros
        ctx.x_shape = x.shape
        if x.dim() != 2:
            y, h = y.view(x.shape), (h.view(x.shape) if h is not None else None)
        return y if residual is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        _no_second("rms_norm")
        h, q, sc, w, rstd = ctx.saved_tensors
        C, M = w.shape[0], rstd.shape[0]
        need = ctx.needs_input_grad
        if dy is None and dh is None:
            return None, None, None, None, None
        if dy is None:   # only the sum was used: its gradient passes through
            return (dh if need[0] else None), (torch.zeros_like(w) if need[1] else None), (dh if need[2] else None), None, None
        dy2, lddy = _rows(dy, C)
        dh2, lddh = (None, 0) if dh is None else _rows(dh, C)
        dx = torch.empty((M, C), dtype=w.dtype, device=w.device) if (need[0] or need[2]) else None
        dw = torch.empty((C,), dtype=w.dtype, device=w.device) if need[1] else None
        nb = _ws_bytes("lt_rms_norm_bwd_workspace_bytes", M, C) if dw is not None else 0
        ws = _buf(nb, w.device) if dw is not None else None
        ldh = 0 if h is None else _rows(h, C)[1]
        _call("lt_rms_norm_bwd", _p(dy2), lddy, _p(dh2), lddh, _p(h), ldh, _p(q), _p(sc), _p(w), _p(rstd), M, C, _DT[w.dtype],
                  _p(dx), _p(dw), _p(ws), 0 if ws is None else ws.numel(), _stream_of(dy2))
        if dx is not None and len(ctx.x_shape) != 2:
            dx = dx.view(ctx.x_shape)
        return (dx if need[0] else None), dw, (dx if need[2] else None), None, None


def rms_norm(x, weight, residual=None, eps: float = 1e-6, checkpoint: str | None = None, out: str | None = None):
    """h = x + residual (h = x without one);  y = h / sqrt(mean over the row of h^2 + eps) * weight.  -> y, or (y, h) with a
    residual.

    x [..., C], residual the same shape, weight [C], all float32, bfloat16 or float16, C <= 16384; the sum of squares and the
    row's scale are fp32, h enters the norm unrounded.  Differentiable in all three; checkpoint="mx8": the backward pass
    reads h from 8 bits.  out="mx8" (serving, no gradient): y comes as Mx8 [rows, C], for linear() with an Mx8 weight."""
    if checkpoint not in (None, "mx8"):
        raise ValueError(f"rms_norm: checkpoint must be None or 'mx8', got {checkpoint!r}")
    if out not in (None, "mx8"):
        raise ValueError(f"rms_norm: out must be None or 'mx8', got {out!r}")
    _dt(x, "rms_norm x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 16384:
        raise ValueError(f"rms_norm: expected rows of 1 to 16384 elements, got shape {tuple(x.shape)}")
    _like(weight, x, x.shape[-1:], "rms_norm weight")
    if residual is not None:
        _like(residual, x, x.shape, "rms_norm residual")
    if out == "mx8":
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
            raise RuntimeError("rms_norm: out='mx8' carries no gradient; call it under torch.no_grad()")
        h, _, y8, _, _ = _rms_fwd(x, weight.contiguous(), residual, eps, residual is not None, False, True, False, False)
        return y8 if residual is None else (y8, h.view(x.shape))
    return _RmsNorm.apply(x, weight, residual, float(eps), checkpoint)
