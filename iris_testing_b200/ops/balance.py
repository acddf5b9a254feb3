"""The router's auxiliary losses -- balance over the experts and z loss -- with per-expert counts, and their gradient.

No counterpart in the reference, which draws its router at random and never trains it (utils.py:201-202).
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from .. import _native as nv
from . import cpu_ref
from ._common import (ELEM, declare, launch_status, on_device, ptr, require, require_device, require_elem, rows_view,
                      stream_ptr, use_native)
from .expert import sm_count

MAX_BALANCE_EXPERTS = 1024


class BalanceArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("logits", "idx", "seq_rows", "mask", "loss", "counts", "kept", "record", "seq_loss",
                                          "seq_z", "seq_tokens", "total", "ticket", "grad_loss", "grad", "status")] \
        + [("ld", C.c_longlong)] + [(n, C.c_int) for n in ("T", "E", "k", "S", "elem", "runs", "run_tokens")] \
        + [("coef", C.c_float), ("z", C.c_float)]


def _fill(logits, k, seq_rows, mask, coef, z, S):
    a = BalanceArgs()
    a.T, a.E = logits.shape
    a.k, a.S, a.elem, a.coef, a.z = k, S, ELEM[logits.dtype], coef, z
    a.logits, a.ld = logits.data_ptr(), logits.stride(0)
    a.seq_rows = None if seq_rows is None else seq_rows.data_ptr()
    a.mask = None if mask is None else mask.data_ptr()
    runs = declare("b200_balance_runs", [C.c_int] * 4)(a.T, a.E, a.elem, sm_count(logits.device))
    a.run_tokens = -(-a.T // runs)
    a.runs = -(-a.T // a.run_tokens)
    if seq_rows is not None:
        a.status = launch_status(logits.device).data_ptr()
    return a


def _call(name, a, t):
    fn = declare(name, [C.POINTER(BalanceArgs), C.c_void_p])
    with on_device(t):
        nv.check(fn(C.byref(a), stream_ptr(t)), name.replace("b200_", "").replace("_", " ") + " launch")


def _forward(logits, idx, seq_rows, mask, coef, z):
    """(loss, counts [S, E], what the backward pass reads)."""
    T, E = logits.shape
    S = 1 if seq_rows is None else seq_rows.numel()
    dev = logits.device
    loss = torch.empty((), dtype=torch.float32, device=dev)
    counts = torch.empty((S, E), dtype=torch.int32, device=dev)
    if T == 0 or S == 0:
        return loss.zero_(), counts.zero_(), None
    a = _fill(logits, idx.shape[1], seq_rows, mask, coef, z, S)
    keep = torch.empty(S * E + S + 2, dtype=torch.int32, device=dev)          # counts, tokens per sequence, two fp32 words
    parts = S * -(-E // 32)
    work = torch.empty((a.runs + S) * (2 * E + 2) + parts + S + 1, dtype=torch.float32, device=dev)
    a.idx, a.loss, a.counts = idx.data_ptr(), loss.data_ptr(), counts.data_ptr()
    a.record = work.data_ptr()
    a.seq_loss = a.record + 4 * (a.runs + S) * (2 * E + 2)
    a.seq_z = a.seq_loss + 4 * parts
    a.ticket = a.seq_z + 4 * S
    _keep(a, keep, S, E)
    _call("b200_balance_forward", a, logits)
    return loss, counts, keep


def _keep(a, keep, S, E):
    a.kept = keep.data_ptr()
    a.seq_tokens = a.kept + 4 * S * E
    a.total = a.seq_tokens + 4 * S


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, idx, seq_rows, mask, coef, z):
        loss, counts, keep = _forward(logits, idx, seq_rows, mask, coef, z)
        ctx.save_for_backward(logits, seq_rows, mask, keep)
        ctx.how = (idx.shape[1], coef, z)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss, _):
        logits, seq_rows, mask, keep = ctx.saved_tensors
        if dloss is None:
            return (None,) * 6
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if keep is None:
            return (grad.zero_(),) + (None,) * 5
        k, coef, z = ctx.how
        S = 1 if seq_rows is None else seq_rows.numel()
        a = _fill(logits, k, seq_rows, mask, coef, z, S)
        _keep(a, keep, S, logits.shape[1])
        dloss = dloss.float().contiguous()
        a.grad_loss, a.grad = dloss.data_ptr(), grad.data_ptr()
        _call("b200_balance_backward", a, logits)
        return (grad,) + (None,) * 5


def balance_loss(logits: torch.Tensor, topk_idx: torch.Tensor, *, balance_coef: float = 0.01, z_coef: float = 0.0,
                 seq_rows: Optional[torch.Tensor] = None, token_mask: Optional[torch.Tensor] = None
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss fp32 [], counts int32): the auxiliary losses of a softmax router; differentiable by the logits.

    ``loss = balance_coef * mean over sequences of E * sum_e f_e P_e + z_coef * mean over tokens of logsumexp(logits)^2``
    with f_e the share of a sequence's routed copies that went to expert e and P_e the mean of its probability.

    logits      [T, E] float32, bfloat16 or float16 (E <= 1024), rows may be strided
    topk_idx    int32 [T, k]: the experts the router chose; values outside [0, E) count for none
    seq_rows    int32 [S] on the logits' device: lengths of the sequences packed one after another; tokens behind the last
                one take no part.  None: all tokens are one sequence.  Lengths that add up to more than T are cut off
                there and reported (:func:`check_default_status`).
    token_mask  bool [T]: False for padding, which takes no part

    A token also takes no part where its logits hold a NaN or +infinity, or nothing above their type's lowest value (all
    experts masked).  Such tokens get a zero gradient, sequences without any token are left out of the mean, and
    without any token at all the loss is zero.  ``counts`` is [E], or [S, E] with ``seq_rows``; it may be changed by the
    caller.  The same inputs give the same bits.  CPU tensors take plain PyTorch."""
    require(logits.dim() == 2 and logits.shape[1] >= 1, "logits must be [T, E]")
    T, E = logits.shape
    require(topk_idx.dim() == 2 and topk_idx.shape[0] == T and topk_idx.shape[1] >= 1, "topk_idx must be [T, k]")
    require(topk_idx.dtype == torch.int32, "topk_idx must be int32")
    require(seq_rows is None or (seq_rows.dim() == 1 and seq_rows.dtype == torch.int32), "seq_rows must be int32 [S]")
    require(token_mask is None or (token_mask.shape == (T,) and token_mask.dtype == torch.bool), "token_mask must be bool [T]")
    if not use_native(logits):
        loss, counts = cpu_ref.balance_loss_ref(logits, topk_idx, balance_coef, z_coef, seq_rows, token_mask)
        return loss, counts if seq_rows is not None else counts[0]
    require_elem(logits, "logits")
    require(E <= MAX_BALANCE_EXPERTS, f"at most {MAX_BALANCE_EXPERTS} experts (got {E})")
    require_device(logits.device, topk_idx=topk_idx, seq_rows=seq_rows, token_mask=token_mask)
    logits = rows_view(logits)
    idx = topk_idx.contiguous()
    rows = None if seq_rows is None else seq_rows.contiguous()
    mask = None if token_mask is None else token_mask.contiguous()
    how = (float(balance_coef), float(z_coef))
    if torch.is_grad_enabled() and logits.requires_grad:
        loss, counts = _Balance.apply(logits, idx, rows, mask, *how)
    else:
        loss, counts, _ = _forward(logits, idx, rows, mask, *how)
    return loss, counts if seq_rows is not None else counts[0]
