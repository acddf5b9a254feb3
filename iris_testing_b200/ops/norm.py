"""RMS norms around a block: the one in front of it, and the junction behind it -- norm of the block's output, gate,
residual with its scale, and the norm in front of the next block -- forward and backward, one pass over memory each.

No counterpart in the reference, whose layer begins at the router and ends at the experts.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from .. import _native as nv
from . import cpu_ref
from ._common import (ELEM, declare, on_device, ptr, require, require_device, require_elem, rows_view, stream_ptr,
                      use_native)
from .expert import sm_count

GATE_NONE, GATE_CHANNEL, GATE_ROW, GATE_FULL = 0, 1, 2, 3
MAX_COLUMNS = 16384


class NormArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("y", "res", "w", "gate", "w2", "h", "n", "r1", "r2", "dh", "dn", "dy", "dres",
                                          "dgate", "dw", "dw2", "partial")] \
        + [(n, C.c_longlong) for n in ("ld_y", "ld_res", "ld_gate", "ld_dh", "ld_dn")] \
        + [(n, C.c_int) for n in ("T", "H", "elem", "w_f32", "w2_f32", "gate_f32", "norm", "gate_kind", "aligned", "parts")] \
        + [("scale", C.c_float), ("eps", C.c_float)]


def _gate_kind(gate: Optional[torch.Tensor], shape) -> int:
    if gate is None:
        return GATE_NONE
    if gate.shape == shape[-1:]:
        return GATE_CHANNEL
    if gate.shape == shape and shape[-1] > 1:     # of a single column, a gate per element is one per row
        return GATE_FULL
    require(gate.shape == shape[:-1] + (1,),
            f"gate must be one value per column {tuple(shape[-1:])}, per row {tuple(shape[:-1] + (1,))} or per element "
            f"{tuple(shape)} (got {tuple(gate.shape)})")
    return GATE_ROW


def _check(y, residual, weight, gate, next_weight):
    require(y.dim() >= 1 and y.shape[-1] >= 1, "y must have at least one dimension, and columns in the last one")
    H = y.shape[-1]
    require(residual is None or residual.shape == y.shape, "residual must have y's shape")
    for name, w in (("weight", weight), ("next_weight", next_weight)):
        require(w is None or w.shape == (H,), f"{name} must have one value per column ({H})")
    kind = _gate_kind(gate, y.shape)
    if not use_native(y):
        return kind
    require(H <= MAX_COLUMNS, f"at most {MAX_COLUMNS} columns (got {H})")
    require(y.numel() // H <= 2 ** 30, "too many rows")
    require_elem(y, "y")
    require(residual is None or residual.dtype == y.dtype, "residual must have y's dtype")
    for name, w in (("weight", weight), ("next_weight", next_weight), ("gate", gate if kind != GATE_FULL else None)):
        require(w is None or w.dtype in (y.dtype, torch.float32), f"{name} must have y's dtype or be float32")
    require(kind != GATE_FULL or gate.dtype == y.dtype, "a gate per element must have y's dtype")
    require_device(y.device, residual=residual, weight=weight, gate=gate, next_weight=next_weight)
    return kind


def _fill(y, residual, weight, gate, kind, norm, scale, next_weight, eps, keep):
    """Argument block of one call and the number of rows; ``keep`` holds what has to outlive the launch."""
    a = NormArgs()
    a.H, a.elem, a.norm, a.gate_kind, a.scale, a.eps = y.shape[-1], ELEM[y.dtype], int(norm), kind, scale, eps

    def rows(t):
        v = rows_view(t)
        keep.append(v)
        return v, v.data_ptr(), (v.stride(0) if v.shape[0] > 1 else v.shape[1])

    def vector(t):
        v = t if t.is_contiguous() else t.contiguous()
        keep.append(v)
        return v.data_ptr(), int(t.dtype == torch.float32)

    y2, a.y, a.ld_y = rows(y)
    a.T = y2.shape[0]
    if residual is not None:
        _, a.res, a.ld_res = rows(residual)
    if weight is not None:
        a.w, a.w_f32 = vector(weight)
    if next_weight is not None:
        a.w2, a.w2_f32 = vector(next_weight)
    if kind == GATE_CHANNEL:
        a.gate, a.gate_f32 = vector(gate)
    elif kind != GATE_NONE:
        _, a.gate, a.ld_gate = rows(gate)
        a.gate_f32 = int(gate.dtype == torch.float32)
    return a


def _align(a: NormArgs, size: int) -> None:
    """Whole 16-byte packs are moved where every row of every tensor starts on one."""
    bits = (a.y or 0) | (a.res or 0) | (a.w or 0) | (a.w2 or 0) | (a.dh or 0) | (a.dn or 0)
    lds = a.H | a.ld_y | a.ld_res | a.ld_dh | a.ld_dn
    if a.gate_kind in (GATE_CHANNEL, GATE_FULL):
        bits |= a.gate
    if a.gate_kind == GATE_FULL:
        lds |= a.ld_gate
    a.aligned = int(bits % 16 == 0 and lds * size % 16 == 0)


def _call(name, a, t):
    fn = declare(name, [C.POINTER(NormArgs), C.c_int, C.c_void_p])
    with on_device(t):
        nv.check(fn(C.byref(a), sm_count(t.device), stream_ptr(t)), name.replace("b200_", "").replace("_", " ") + " launch")


def _forward(y, residual, weight, gate, kind, norm, scale, next_weight, eps, save):
    h = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    n = None if next_weight is None else torch.empty_like(h)
    T = y.numel() // y.shape[-1]
    stats = torch.empty((2, T), dtype=torch.float32, device=y.device) if save else None
    if T == 0:
        return h, n, stats
    keep = []
    a = _fill(y, residual, weight, gate, kind, norm, scale, next_weight, eps, keep)
    a.h, a.n = h.data_ptr(), None if n is None else n.data_ptr()
    if save:
        a.r1 = stats.data_ptr()
        a.r2 = a.r1 + 4 * T
    _align(a, y.element_size())
    _call("b200_norm_forward", a, y)
    return h, n, stats


def _backward(saved, kind, norm, scale, eps, need, dh, dn):
    """Gradients of (y, residual, weight, gate, next_weight), None where ``need`` says so."""
    y, residual, weight, gate, next_weight, stats = saved
    like = (y, residual, weight, gate, next_weight)
    grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None and n else None for t, n in zip(like, need)]
    T = y.numel() // y.shape[-1]
    if T == 0 or (dh is None and dn is None):
        return [None if g is None else g.zero_() for g in grads]
    keep = []
    a = _fill(y, residual, weight, gate, kind, norm, scale, next_weight, eps, keep)
    for name, t in (("dh", dh), ("dn", dn)):
        if t is not None:
            v = rows_view(t)
            keep.append(v)
            setattr(a, name, v.data_ptr())
            setattr(a, "ld_" + name, v.stride(0) if T > 1 else v.shape[1])
    if dn is None and grads[4] is not None:       # the second output has no gradient
        grads[4].zero_()
    a.dy, a.dres, a.dw, a.dgate = (None if g is None else g.data_ptr() for g in grads[:4])
    a.dw2 = None if grads[4] is None or dn is None else grads[4].data_ptr()
    a.r1 = stats.data_ptr()
    a.r2 = a.r1 + 4 * T
    _align(a, y.element_size())
    if a.dw or a.dw2 or (a.dgate and kind == GATE_CHANNEL):
        parts = declare("b200_norm_parts", [C.c_int] * 5)(T, a.H, a.elem, a.aligned, sm_count(y.device))
        partial = torch.empty((2, parts, a.H), dtype=torch.float32, device=y.device)
        a.partial = partial.data_ptr()
    _call("b200_norm_backward", a, y)
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
        return (*_backward(ctx.saved_tensors, *ctx.how, ctx.needs_input_grad[:5], dh, dn), None, None, None, None)


def _apply(y, residual, weight, gate, next_weight, kind, norm, scale, eps):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (y, residual, weight, gate, next_weight)):
        return _Norm.apply(y, residual, weight, gate, next_weight, kind, norm, scale, eps)
    h, n, _ = _forward(y, residual, weight, gate, kind, norm, scale, next_weight, eps, False)
    return h if n is None else (h, n)


def pre_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, in x's dtype; differentiable.

    x       [..., H] float32, bfloat16 or float16, H <= 16384; rows may be strided
    weight  [H] in x's dtype or float32, or None

    Statistics and products are fp32, rounded once.  CPU tensors take plain PyTorch."""
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
    order: the same inputs give the same bits.  CPU tensors take plain PyTorch."""
    require(norm or weight is None, "weight belongs to the norm of y: norm=False takes none")
    require(residual is not None, "post_norm needs the residual (pre_norm is the norm alone)")
    kind = _check(y, residual, weight, gate, next_weight)
    if not use_native(y):
        h, n = cpu_ref.post_norm_ref(y, residual, weight, gate, norm, residual_scale, next_weight, eps)
        return h.to(y.dtype) if n is None else (h.to(y.dtype), n.to(y.dtype))
    return _apply(y, residual, weight, gate, next_weight, kind, bool(norm), float(residual_scale), float(eps))
