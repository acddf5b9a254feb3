"""RMS norms around a block: the one in front of it, and the junction behind it -- norm of the block's output, gate,
residual with its scale, and the norm in front of the next block -- forward and backward, one pass over memory each.

No counterpart in the reference, whose layer begins at the router and ends at the experts.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional

import torch

from . import cpu_ref
from ._common import ELEM, Entry, declare, on_device, refuse_tangents, require, require_device, rows_view, stream_ptr, use_native
from .expert import sm_count

GATE_NONE, GATE_CHANNEL, GATE_ROW, GATE_FULL = 0, 1, 2, 3
MAX_COLUMNS = 16384


class NormArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("y", "res", "w", "gate", "w2", "h", "n", "r1", "r2", "dh", "dn", "dy", "dres",
                                          "dgate", "dw", "dw2", "partial")] \
        + [(n, C.c_longlong) for n in ("ld_y", "ld_res", "ld_gate", "ld_dh", "ld_dn")] \
        + [(n, C.c_int) for n in ("T", "H", "elem", "w_f32", "w2_f32", "gate_f32", "norm", "gate_kind", "aligned", "parts")] \
        + [("scale", C.c_float), ("eps", C.c_float)]


_FORWARD = Entry("b200_norm_forward", C.POINTER(NormArgs), C.c_int, C.c_void_p)
_BACKWARD = Entry("b200_norm_backward", C.POINTER(NormArgs), C.c_int, C.c_void_p)
_F32 = torch.float32


def _gate_kind(gate: torch.Tensor, shape) -> int:
    if gate.shape == shape[-1:]:
        return GATE_CHANNEL
    if gate.shape == shape and shape[-1] > 1:     # of a single column, a gate per element is one per row
        return GATE_FULL
    if gate.shape != shape[:-1] + (1,):
        raise ValueError(f"gate must be one value per column {tuple(shape[-1:])}, per row {tuple(shape[:-1] + (1,))} or per "
                         f"element {tuple(shape)} (got {tuple(gate.shape)})")
    return GATE_ROW


def _check(y, residual, weight, gate, next_weight) -> int:
    """Refuses what does not fit together; the kind of gate."""
    shape = y.shape
    require(len(shape) >= 1 and shape[-1] >= 1, "y must have at least one dimension, and columns in the last one")
    H, dt = shape[-1], y.dtype
    require(residual is None or residual.shape == shape, "residual must have y's shape")
    require(weight is None or weight.shape == shape[-1:], "weight must have one value per column")
    require(next_weight is None or next_weight.shape == shape[-1:], "next_weight must have one value per column")
    kind = GATE_NONE if gate is None else _gate_kind(gate, shape)
    if not y.is_cuda:
        return kind
    if H > MAX_COLUMNS or y.numel() > H << 30:
        raise ValueError(f"at most {MAX_COLUMNS} columns (got {H}) and 2^30 rows")
    if dt not in ELEM:
        raise ValueError(f"y must be float32, bfloat16 or float16 (got {dt})")
    require(residual is None or residual.dtype == dt, "residual must have y's dtype")
    require(weight is None or weight.dtype == dt or weight.dtype == _F32, "weight must have y's dtype or be float32")
    require(next_weight is None or next_weight.dtype == dt or next_weight.dtype == _F32,
            "next_weight must have y's dtype or be float32")
    require(kind == GATE_NONE or gate.dtype == dt or (gate.dtype == _F32 and kind != GATE_FULL),
            "gate must have y's dtype, or be float32 where it is one value per column or row")
    require_device(y.device, residual=residual, weight=weight, gate=gate, next_weight=next_weight)
    return kind


def _fill(y, residual, weight, gate, kind, norm, scale, next_weight, eps, keep):
    """Argument block of one call; ``keep`` holds what has to outlive the launch."""
    a = NormArgs()
    H, size = y.shape[-1], y.element_size()
    a.H, a.elem, a.norm, a.gate_kind, a.scale, a.eps = H, ELEM[y.dtype], norm, kind, scale, eps
    y = rows_view(y)
    T = a.T = y.shape[0]
    ld = H if T == 1 else y.stride(0)
    p = y.data_ptr()
    a.y, a.ld_y, bits, lds = p, ld, p, H | ld
    keep.append(y)
    if residual is not None:
        residual = rows_view(residual)
        ld = H if T == 1 else residual.stride(0)
        p = residual.data_ptr()
        a.res, a.ld_res, bits, lds = p, ld, bits | p, lds | ld
        keep.append(residual)
    if weight is not None:
        weight = weight.contiguous()
        a.w = p = weight.data_ptr()
        a.w_f32, bits = weight.dtype == _F32, bits | p
        keep.append(weight)
    if next_weight is not None:
        next_weight = next_weight.contiguous()
        a.w2 = p = next_weight.data_ptr()
        a.w2_f32, bits = next_weight.dtype == _F32, bits | p
        keep.append(next_weight)
    if kind != GATE_NONE:
        a.gate_f32 = gate.dtype == _F32
        if kind == GATE_CHANNEL:
            gate = gate.contiguous()
            bits |= gate.data_ptr()
        else:
            gate = rows_view(gate)
            a.ld_gate = ld = gate.shape[1] if T == 1 else gate.stride(0)
            if kind == GATE_FULL:
                bits, lds = bits | gate.data_ptr(), lds | ld
        a.gate = gate.data_ptr()
        keep.append(gate)
    # whole 16-byte packs are moved where every row of every tensor starts on one
    a.aligned = bits % 16 == 0 and lds * size % 16 == 0
    return a


def _new(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


@functools.lru_cache(maxsize=256)
def _parts(T: int, H: int, elem: int, aligned: int, sms: int) -> int:
    return declare("b200_norm_parts", [C.c_int] * 5)(T, H, elem, aligned, sms)


def _forward(y, residual, weight, gate, kind, norm, scale, next_weight, eps, save):
    h = _new(y)
    n = None if next_weight is None else torch.empty_like(h)
    T = y.numel() // y.shape[-1]
    stats = torch.empty((2, T), dtype=_F32, device=y.device) if save else None
    if T == 0:
        return h, n, stats
    keep = []
    a = _fill(y, residual, weight, gate, kind, norm, scale, next_weight, eps, keep)
    a.h = h.data_ptr()
    if n is not None:
        a.n = n.data_ptr()
    if save:
        a.r1 = p = stats.data_ptr()
        a.r2 = p + 4 * T
    with on_device(y):
        _FORWARD(a, sm_count(y.device), stream_ptr(y))
    return h, n, stats


def _backward(saved, kind, norm, scale, eps, need, dh, dn):
    """Gradients of (y, residual, weight, gate, next_weight), None where ``need`` says so."""
    y, residual, weight, gate, next_weight, stats = saved
    like = (y, residual, weight, gate, next_weight)
    grads = [_new(t) if n and t is not None else None for t, n in zip(like, need)]
    T = y.numel() // y.shape[-1]
    if T == 0 or (dh is None and dn is None):
        return [None if g is None else g.zero_() for g in grads]
    keep = []
    a = _fill(y, residual, weight, gate, kind, norm, scale, next_weight, eps, keep)
    bits = lds = 0
    if dh is not None:
        dh = rows_view(dh)
        a.dh, a.ld_dh = bits, lds = dh.data_ptr(), dh.stride(0) if T > 1 else dh.shape[1]
    if dn is not None:
        dn = rows_view(dn)
        p, ld = dn.data_ptr(), dn.stride(0) if T > 1 else dn.shape[1]
        a.dn, a.ld_dn, bits, lds = p, ld, bits | p, lds | ld
    elif grads[4] is not None:                    # the second output has no gradient
        grads[4].zero_()
    a.aligned = a.aligned and bits % 16 == 0 and lds * y.element_size() % 16 == 0
    a.dy, a.dres, a.dw, a.dgate = (None if g is None else g.data_ptr() for g in grads[:4])
    if grads[4] is not None and dn is not None:
        a.dw2 = grads[4].data_ptr()
    a.r1 = p = stats.data_ptr()
    a.r2 = p + 4 * T
    sms = sm_count(y.device)
    if a.dw or a.dw2 or (a.dgate and kind == GATE_CHANNEL):
        partial = torch.empty(2 * _parts(T, a.H, a.elem, a.aligned, sms) * a.H, dtype=_F32, device=y.device)
        a.partial = partial.data_ptr()
    with on_device(y):
        _BACKWARD(a, sms, stream_ptr(y))
    return grads


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, weight, gate, next_weight, kind, norm, scale, eps):
        h, n, stats = _forward(y, residual, weight, gate, kind, norm, scale, next_weight, eps, True)
        ctx.save_for_backward(y, residual, weight, gate, next_weight, stats)
        ctx.how = (kind, norm, scale, eps)
        ctx.set_materialize_grads(False)
        return h if n is None else (h, n)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dn=None):
        refuse_tangents(dh=dh, dn=dn)
        return (*_backward(ctx.saved_tensors, *ctx.how, ctx.needs_input_grad[:5], dh, dn), None, None, None, None)


def _apply(y, residual, weight, gate, next_weight, kind, norm, scale, eps):
    refuse_tangents(y=y, residual=residual, weight=weight, gate=gate, next_weight=next_weight)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (y, residual, weight, gate, next_weight)):
        return _Norm.apply(y, residual, weight, gate, next_weight, kind, norm, scale, eps)
    h, n, _ = _forward(y, residual, weight, gate, kind, norm, scale, next_weight, eps, False)
    return h if n is None else (h, n)


def pre_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, in x's dtype; differentiable.

    x       [..., H] float32, bfloat16 or float16, H <= 16384; rows may be strided
    weight  [H] in x's dtype or float32, or None

    Statistics and products are fp32, rounded once.  Derivatives are reverse mode, of first order.  CPU tensors take plain
    PyTorch."""
    _check(x, None, weight, None, None)
    if not use_native(x):
        return cpu_ref.rms_norm_ref(x, weight, eps).to(x.dtype)
    return _apply(x, None, weight, None, None, GATE_NONE, True, 1.0, float(eps))


def post_norm(y: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None,
              gate: Optional[torch.Tensor] = None, *, norm: bool = True, residual_scale: float = 1.0,
              next_weight: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """``h = residual_scale * residual + gate * norm(y)``, and with ``next_weight`` also ``n = norm(h) * next_weight``:
    returns ``h`` or ``(h, n)`` in y's dtype; differentiable.

    y, residual  [..., H] of one dtype (float32, bfloat16, float16), H <= 16384; rows may be strided
    weight       [H] of the norm of y in y's dtype or float32, or None; ``norm=False`` leaves y as it is
    gate         None, [H] (one value per column), [..., 1] (one per row) or [..., H]; the first two also as float32
    next_weight  [H]: weight of the norm in front of the next block, in y's dtype or float32

    n is the norm of h before h is rounded.  Gradients of weight, gate and next_weight are summed in fp32 in a fixed
    order: the same inputs give the same bits.  Derivatives are reverse mode, of first order.  CPU tensors take plain PyTorch."""
    require(norm or weight is None, "weight belongs to the norm of y: norm=False takes none")
    require(residual is not None, "post_norm needs the residual (pre_norm is the norm alone)")
    kind = _check(y, residual, weight, gate, next_weight)
    if not use_native(y):
        h, n = cpu_ref.post_norm_ref(y, residual, weight, gate, norm, residual_scale, next_weight, eps)
        return h.to(y.dtype) if n is None else (h.to(y.dtype), n.to(y.dtype))
    return _apply(y, residual, weight, gate, next_weight, kind, bool(norm), float(residual_scale), float(eps))
