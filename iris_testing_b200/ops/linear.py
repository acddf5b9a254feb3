"""Matrix product with bias, activation and residual in its epilogue, dense (a shared expert, a projection) or with one
weight per expert over packed ragged rows, with its gradients.

``grouped_gemm`` is the plain product of the expert path, forward only; the reference's expert is forward only too
(layers/expert.py:6-65).
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional

import torch

from .. import _native as nv
from . import cpu_ref
from ._common import ELEM, Entry, declare, launch_status, on_device, refuse_tangents, require, require_device, stream_ptr, use_native
from .expert import pairs_pay, sm_count

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "silu_gate": 4}
_FORWARD, _DX, _DW = 0, 1, 2
MAX_GRAD_COLUMNS = 65535 * 1024  # blocks side by side in the activation's gradient, of 1024 columns each
MAX_ROWS = 2 ** 31 - 1024        # a last tile that is partly empty still has row numbers of 32 bits


def _run_rows(M: int, n_out: int) -> int:
    """Rows that a thread of the activation's gradient goes down: as many as leave 16 blocks for every SM, so that enough
    loads are under way.  64 / 32 / 16 rows, us, with cold caches, alone: 1000 x 4096 59 / 33 / 23, 8192 x 4096 76 / 53 / 53,
    4000 x 14336 88 / 90 / 80, gated 65536 x 2816 196 / 176 / 176; with the bias' gradient, whose records shorter runs make
    more of: 60 / 36 / 24, 79 / 58 / 69, 91 / 95 / 91, 255 / 226 / 241."""
    blocks = -(-n_out // 1024)
    return 64 if M * blocks >= 64 * 2368 else 32 if M * blocks >= 32 * 2368 else 16


class LinearArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("a", "b", "out", "z", "zexp", "bias", "res", "group_rows", "status")] \
        + [("wait_budget_ns", C.c_ulonglong)] \
        + [(n, C.c_int) for n in ("mode", "G", "M", "N", "K", "n_out", "elem", "act", "pair", "group_m")] \
        + [("record", C.c_void_p)]


class ActGradArgs(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("dy", "z", "zexp", "dz", "dres", "dbias", "record", "group_rows", "peak")] \
        + [(n, C.c_int) for n in ("G", "M", "N", "n_out", "elem", "act", "chunks", "chunk_rows")]


_PRODUCT = Entry("b200_linear", C.POINTER(LinearArgs), C.c_int, C.c_void_p)
_ACT_GRAD = Entry("b200_act_grad", C.POINTER(ActGradArgs), C.c_void_p)


def _plain(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Contiguous and starting on 16 bytes, by a copy where it is not."""
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _pairs(mode: int, M: int, N: int, K: int, G: int) -> bool:
    """Whether a tile is shared by two CTAs: by the rows per group (:func:`pairs_pay`); of dW, whose tiles are all full, from as many
    tiles on as there are pairs (single / pair, us, over 2048 rows: 2048 x 2048, 64 tiles, 28.0 / 29.1; 4096 x 1280, 80 tiles,
    40.7 / 40.4)."""
    if mode == _DW:
        return G * -(-N // 256) * -(-K // 256) >= 74
    return pairs_pay(M / G)


def _splits(mode: int, M: int, N: int, K: int, G: int, grouped: bool, sms: int) -> bool:
    """Whether the contracted dimension is split over the SMs: where whole tiles would leave most of them without work for
    long, or have a few of them read all the weights for a few tokens.

    Measured on one B200 (split / whole tiles, us, launches included), bf16, x [M, K], w [N, K]: forward of 4096 x 4096 40 / 44
    at 256 rows (32 SMs have a tile, 64 blocks each) and 50 / 46 at 512; of 4096 x 14336 (224 blocks) 97 / 101 at 512 rows;
    of 256 x 2048 (32 blocks) 25 / 26 at 2048 rows and 31 / 26 at 4096; dW of 768 x 768 34 / 49 over 4096 rows and 29 / 24 over
    1024.  One token of 28672 x 4096 (112 SMs) 51 / 67, 64 tokens 66 / 60.  Groups' dW ends inside a block as a
    rule and is not split."""
    if mode == _DW and grouped:
        return False
    pair = _pairs(mode, M, N, K, G)
    rows, cols, blocks = (N, K, M) if mode == _DW else (-(-M // G), N if mode == _FORWARD else K, K if mode == _FORWARD else N)
    blocks = -(-blocks // 64)
    busy = G * -(-rows // (256 if pair else 128)) * -(-cols // 256) * (2 if pair else 1)
    return busy <= min(64, blocks // 2) or (mode != _DW and busy < sms and blocks >= 16 and M <= 16 * G)


@functools.lru_cache(maxsize=256)
def _record_floats(mode: int, M: int, N: int, K: int, G: int, sms: int) -> int:
    return declare("b200_linear_record_floats", [C.c_int] * 6, C.c_longlong)(mode, M, N, K, G, sms)


def _product(mode, a, b, out, M, N, K, G, group_rows, act=0, z=None, bias=None, res=None, peak=None):
    la = LinearArgs()
    la.a, la.b, la.out = a.data_ptr(), b.data_ptr(), out.data_ptr()
    if z is not None:
        la.z, la.zexp = z[0].data_ptr(), z[1].data_ptr()
    if bias is not None:
        la.bias = bias.data_ptr()
    if res is not None:
        la.res = res.data_ptr()
    if group_rows is not None:
        la.group_rows = group_rows.data_ptr()
    if peak is not None:
        la.res = peak.data_ptr()             # in the residual's place
    la.status = launch_status(a.device).data_ptr()
    la.wait_budget_ns = 2_000_000_000
    la.mode, la.G, la.M, la.N, la.K, la.n_out = mode, G, M, N, K, out.shape[-1]
    la.elem, la.act = ELEM[a.dtype], act
    sms = sm_count(a.device)
    if _splits(mode, M, N, K, G, group_rows is not None, sms):
        record = torch.empty(_record_floats(mode, M, N, K, G, sms), dtype=torch.float32, device=a.device)
        la.record = record.data_ptr()
    else:
        la.pair = _pairs(mode, M, N, K, G)
    _PRODUCT(la, sms, stream_ptr(a))


def _forward(x, w, bias, residual, group_rows, act, save):
    """(y [M, n_out], z or None): x [M, K], w [N, K] or [G, N, K], all plain.  z, for bf16: [M, N] of fp16 under a power of two, or of
    bf16, and a byte for every 32 columns of a row that says which; for fp16: the upper 16 bits of fp32, and a byte with the next 8."""
    M, K = x.shape
    G, N = (1, w.shape[0]) if w.dim() == 2 else w.shape[:2]
    n_out = N // 2 if act == 4 else N
    y = torch.empty((M, n_out), dtype=x.dtype, device=x.device)
    z = None
    if save and act:
        z = (torch.empty((M, N), dtype=torch.float16, device=x.device),
             torch.empty((M, -(-N // 256) * (256 if x.dtype == torch.float16 else 8)), dtype=torch.uint8, device=x.device))
    if M > 0:
        with on_device(x):
            _product(_FORWARD, x, w, y, M, N, K, G, group_rows, act, z, bias, residual)
    return y, z


def _backward(x, w, z, has_bias, has_res, group_rows, act, need, dy):
    M, K = x.shape
    G, N = (1, w.shape[0]) if w.dim() == 2 else w.shape[:2]
    dev, dt = x.device, x.dtype
    dx = torch.empty_like(x) if need[0] else None
    dw = torch.empty_like(w) if need[1] else None
    db = torch.empty((G, N) if w.dim() == 3 else (N,), dtype=dt, device=dev) if has_bias and need[2] else None
    dres = None
    if has_res and need[3]:                  # without groups every row of dy is the residual's gradient as it is
        dres = dy if group_rows is None else torch.empty_like(dy)
    if M == 0:
        return dx, None if dw is None else dw.zero_(), None if db is None else db.zero_(), dres
    own_dres = dres is not None and dres is not dy
    slope = act and (db is not None or dx is not None or dw is not None)      # act'(z) has a part in what is asked for
    with on_device(x):
        dz, peak = dy, None
        if db is not None or own_dres or slope:
            a = ActGradArgs()
            if slope:
                dz = torch.empty((M, N), dtype=dt, device=dev)
                a.z, a.zexp, a.dz, a.act = z[0].data_ptr(), z[1].data_ptr(), dz.data_ptr(), act
                if dt == torch.float16:
                    peak = torch.empty(1, dtype=torch.int32, device=dev)
                    a.peak = peak.data_ptr()
            a.dy = dy.data_ptr()
            a.dres = dres.data_ptr() if own_dres else None
            a.G, a.M, a.N, a.n_out, a.elem = G, M, dz.shape[1], dy.shape[1], ELEM[dt]
            a.group_rows = None if group_rows is None else group_rows.data_ptr()
            a.chunk_rows = run = _run_rows(M, dy.shape[1])
            a.chunks = -(-M // run)
            if db is not None:
                record = torch.empty((a.chunks + G, N), dtype=torch.float32, device=dev)
                a.dbias, a.record = db.data_ptr(), record.data_ptr()
            _ACT_GRAD(a, stream_ptr(x))
        if dx is not None:
            _product(_DX, dz, w, dx, M, N, K, G, group_rows, peak=peak)
        if dw is not None:
            _product(_DW, dz, x, dw, M, N, K, G, group_rows, peak=peak)
    return dx, dw, db, dres


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, group_rows, act):
        y, z = _forward(x, w, bias, residual, group_rows, act, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, w, *(z or (None, None)), group_rows)
        ctx.how = (bias is not None, residual is not None, act)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        refuse_tangents(dy=dy)
        x, w, z, exponents, group_rows = ctx.saved_tensors
        has_bias, has_res, act = ctx.how
        return (*_backward(x, w, (z, exponents), has_bias, has_res, group_rows, act, ctx.needs_input_grad[:4], _plain(dy)), None, None)


def linear(x: torch.Tensor, w_kmajor: torch.Tensor, bias: Optional[torch.Tensor] = None,
           residual: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
           group_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ w.T + bias) + residual`` in x's dtype; differentiable by x, w, bias and residual.

    x           [..., K] bfloat16 or float16 (with ``group_rows``: [M, K], the groups' rows packed one after another)
    w_kmajor    [N, K], or with ``group_rows`` [G, N, K] (:func:`to_kmajor`), G <= 128
    bias        [N] or [G, N];  residual [..., n_out]: what is added after the activation
    activation  None, "relu", "silu", "gelu" (tanh form), or "silu_gate": every 256 rows of w hold 128 gate rows and
                then 128 up rows, the result is silu(gate) * up and n_out = N / 2
    group_rows  int32 [G] on x's device: rows of each group, none allowed (of copies packed by expert: ``make_plan``'s
                counts; those of a balance loss leave some out).  Rows of x behind the last group are not read; the result
                and the gradients of x and residual are zero there.

    All of one dtype; K and N are multiples of 8.  Sums are fp32, results are rounded once; for the backward pass
    the pre-activation is kept to 16 bits (fp16), or to 11 bits and to 2^-30 (bf16; to 8 bits where 32 neighbouring ones hold
    both a value of 1024 or more and one 2^31 times smaller), and its gradient dz in x's dtype.  fp16 dz are divided by one
    power of two, 2^10 at most, where the call's largest is above 65504, and multiplied with one where it is below 2^-10.
    A relu's slope is 0 or 1 where its pre-activation is nothing but the sum's rounding.
    Groups that hold more rows than x has, and device-side timeouts, are reported to :func:`check_default_status`; what the
    call returns is then undefined.  The same inputs give the same bits.  Derivatives are reverse mode, of first order.  CPU
    tensors take plain PyTorch."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)} (got {activation!r})")
    grouped = group_rows is not None
    require(w_kmajor.dim() == (3 if grouped else 2), "w_kmajor must be [N, K], or [G, N, K] with group_rows")
    N, K = w_kmajor.shape[-2:]
    require(x.dim() >= 1 and x.shape[-1] == K and (x.dim() == 2 or not grouped),
            "x must be [..., K], or [M, K] with group_rows")
    require(N >= 1 and K >= 1, "w_kmajor must have rows and columns")
    act = ACTIVATIONS[activation]
    require(act != 4 or N % 256 == 0, "silu_gate needs N (= 2 * n_out) to be a multiple of 256")
    n_out = N // 2 if act == 4 else N
    G = w_kmajor.shape[0] if grouped else 1
    require(bias is None or bias.shape == ((G, N) if grouped else (N,)), "bias must have one value per row of w_kmajor")
    require(residual is None or residual.shape == x.shape[:-1] + (n_out,), "residual must have the result's shape")
    require(not grouped or (group_rows.dtype == torch.int32 and group_rows.shape == (G,)),
            "group_rows must be int32 with one entry per group")
    require(not grouped or 1 <= G <= nv.MAX_GROUPS, "too many groups (128 at most), or none")
    shape = x.shape[:-1] + (n_out,)
    if not use_native(x):
        require(not grouped or int(group_rows.clamp(min=0).sum()) <= x.shape[0], "the groups hold more rows than x")
        r = None if residual is None else residual.reshape(-1, n_out)
        return cpu_ref.linear_ref(x.reshape(-1, K), w_kmajor, bias, r, activation, group_rows).to(x.dtype).view(shape)
    dt = x.dtype
    if dt != torch.bfloat16 and dt != torch.float16:
        raise ValueError(f"x must be bfloat16 or float16 (got {dt})")
    require(w_kmajor.dtype == dt and (bias is None or bias.dtype == dt) and (residual is None or residual.dtype == dt),
            "w_kmajor, bias and residual must have x's dtype")
    require(K % 8 == 0 and N % 8 == 0, "K and N must be multiples of 8")
    if x.numel() // K > MAX_ROWS or G * N > MAX_ROWS or K > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows of x and of the weights of all groups, and columns")
    require_device(x.device, w_kmajor=w_kmajor, bias=bias, residual=residual, group_rows=group_rows)
    refuse_tangents(x=x, w_kmajor=w_kmajor, bias=bias, residual=residual)
    flat = len(shape) == 2                   # no views, which autograd would have to pass through
    x2 = _plain(x if flat else x.reshape(-1, K))
    r2 = residual if residual is None or flat else residual.reshape(-1, n_out)
    w, b, r2 = _plain(w_kmajor), _plain(bias), _plain(r2)
    rows = None if group_rows is None else group_rows.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w_kmajor, bias, residual)):
        if n_out > MAX_GRAD_COLUMNS and (act or b is not None or (grouped and r2 is not None)):
            raise ValueError(f"at most {MAX_GRAD_COLUMNS} columns of the result with gradients")
        y = _Linear.apply(x2, w, b, r2, rows, act)
    else:
        y, _ = _forward(x2, w, b, r2, rows, act, False)
    return y if flat else y.view(shape)
