"""The router's auxiliary losses -- balance over the experts and z loss -- with per-expert counts, and their gradient.

No counterpart in the reference, which draws its router at random and never trains it (utils.py:201-202).
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional, Tuple

import torch

from . import cpu_ref
from ._common import (ELEM, Entry, declare, launch_status, on_device, refuse_tangents, require, require_device, rows_view,
                      stream_ptr, use_native)
from .expert import sm_count

MAX_BALANCE_EXPERTS = 1024
MAX_TOKENS = 2 ** 31 - 2 ** 20      # also of the blocks of 32 experts of all sequences


class BalanceArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("logits", "idx", "seq_rows", "mask", "loss", "counts", "kept", "record", "seq_loss",
                                          "seq_z", "seq_tokens", "total", "ticket", "grad_loss", "grad", "status")] \
        + [("ld", C.c_longlong)] + [(n, C.c_int) for n in ("T", "E", "k", "S", "elem", "runs", "run_tokens")] \
        + [("coef", C.c_float), ("z", C.c_float)]


_FORWARD = Entry("b200_balance_forward", C.POINTER(BalanceArgs), C.c_void_p)
_BACKWARD = Entry("b200_balance_backward", C.POINTER(BalanceArgs), C.c_void_p)
_I32, _F32 = torch.int32, torch.float32


@functools.lru_cache(maxsize=256)
def _runs(T: int, E: int, elem: int, backward: bool, sms: int) -> Tuple[int, int]:
    """(blocks, tokens of each)."""
    tokens = -(-T // declare("b200_balance_runs", [C.c_int] * 5)(T, E, elem, backward, sms))
    return -(-T // tokens), tokens


def _fill(logits, k, seq_rows, mask, coef, z, S, backward=False):
    a = BalanceArgs()
    T, E = logits.shape
    elem = ELEM[logits.dtype]
    a.T, a.E, a.k, a.S, a.elem, a.coef, a.z = T, E, k, S, elem, coef, z
    a.logits, a.ld = logits.data_ptr(), logits.stride(0)
    if seq_rows is not None:
        a.seq_rows, a.status = seq_rows.data_ptr(), launch_status(logits.device).data_ptr()
    if mask is not None:
        a.mask = mask.data_ptr()
    a.runs, a.run_tokens = _runs(T, E, elem, backward, sm_count(logits.device))
    return a


def _forward(logits, idx, seq_rows, mask, coef, z):
    """(loss, counts [E] or [S, E], scratch that holds what the backward pass reads, or None)."""
    T, E = logits.shape
    dev = logits.device
    S = 1 if seq_rows is None else seq_rows.numel()
    loss = torch.empty((), dtype=_F32, device=dev)
    counts = torch.empty((E,) if seq_rows is None else (S, E), dtype=_I32, device=dev)
    if T == 0 or S == 0:
        return loss.zero_(), counts.zero_(), None
    a = _fill(logits, idx.shape[1], seq_rows, mask, coef, z, S)
    # kept counts, tokens per sequence, two fp32 words; then the records, parts of the terms, z sums and a ticket
    parts, kept, records = S * -(-E // 32), S * E + S + 2, (a.runs + S) * (2 * E + 2)
    work = torch.empty(kept + records + parts + S + 1, dtype=_I32, device=dev)
    a.idx, a.loss, a.counts = idx.data_ptr(), loss.data_ptr(), counts.data_ptr()
    base = work.data_ptr()
    _keep(a, base, S, E)
    a.record = p = base + 4 * kept
    a.seq_loss = p = p + 4 * records
    a.seq_z = p = p + 4 * parts
    a.ticket = p + 4 * S
    with on_device(logits):
        _FORWARD(a, stream_ptr(logits))
    return loss, counts, work


def _keep(a, base, S, E):
    a.kept = base
    a.seq_tokens = base + 4 * S * E
    a.total = base + 4 * S * (E + 1)


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
        refuse_tangents(dloss=dloss)
        logits, seq_rows, mask, keep = ctx.saved_tensors
        if dloss is None:
            return (None,) * 6
        grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
        if keep is None:
            return (grad.zero_(),) + (None,) * 5
        k, coef, z = ctx.how
        S = 1 if seq_rows is None else seq_rows.numel()
        a = _fill(logits, k, seq_rows, mask, coef, z, S, True)
        _keep(a, keep.data_ptr(), S, logits.shape[1])
        if dloss.dtype != _F32:
            dloss = dloss.float()
        a.grad_loss, a.grad = dloss.data_ptr(), grad.data_ptr()
        with on_device(logits):
            _BACKWARD(a, stream_ptr(logits))
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
    without any token at all the loss is zero.  ``counts`` is [E], or [S, E] with ``seq_rows``, of the copies of tokens that
    take part; it may be changed by the caller.  They are not sizes of groups of packed rows, where the copies of the other
    tokens may lie too: ``make_plan(topk_idx, E).counts`` are.  The same inputs give the same bits.  Derivatives are reverse
    mode, of first order.  CPU tensors take plain PyTorch."""
    require(logits.dim() == 2 and logits.shape[1] >= 1, "logits must be [T, E]")
    T, E = logits.shape
    require(topk_idx.dim() == 2 and topk_idx.shape[0] == T and topk_idx.shape[1] >= 1, "topk_idx must be [T, k]")
    require(topk_idx.dtype == torch.int32, "topk_idx must be int32")
    require(seq_rows is None or (seq_rows.dim() == 1 and seq_rows.dtype == torch.int32), "seq_rows must be int32 [S]")
    require(token_mask is None or (token_mask.shape == (T,) and token_mask.dtype == torch.bool), "token_mask must be bool [T]")
    if not use_native(logits):
        loss, counts = cpu_ref.balance_loss_ref(logits, topk_idx, balance_coef, z_coef, seq_rows, token_mask)
        return loss, counts if seq_rows is not None else counts[0]
    if logits.dtype not in ELEM:
        raise ValueError(f"logits must be float32, bfloat16 or float16 (got {logits.dtype})")
    if E > MAX_BALANCE_EXPERTS:
        raise ValueError(f"at most {MAX_BALANCE_EXPERTS} experts (got {E})")
    if T > MAX_TOKENS or (seq_rows is not None and seq_rows.numel() * -(-E // 32) > MAX_TOKENS):
        raise ValueError(f"at most {MAX_TOKENS} tokens, and blocks of 32 experts of all sequences")
    if topk_idx.shape[1] > MAX_TOKENS:
        raise ValueError(f"at most {MAX_TOKENS} experts of a token")
    require_device(logits.device, topk_idx=topk_idx, seq_rows=seq_rows, token_mask=token_mask)
    refuse_tangents(logits=logits)
    logits, idx = rows_view(logits), topk_idx.contiguous()
    if seq_rows is not None:
        seq_rows = seq_rows.contiguous()
    if token_mask is not None:
        token_mask = token_mask.contiguous()
    how = (float(balance_coef), float(z_coef))
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Balance.apply(logits, idx, seq_rows, token_mask, *how)
    return _forward(logits, idx, seq_rows, token_mask, *how)[:2]
