"""Helpers shared by the op wrappers: stream handles, pointer casts, dispatch rule."""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad

from .. import _native as nv


def use_native(t: torch.Tensor) -> bool:
    """CUDA tensors always take the native kernels (a missing library raises);
    CPU tensors take the PyTorch restatement."""
    return t.is_cuda


# The raw handle of a device's current stream without building a Stream object, where torch has it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_ptr(t: torch.Tensor) -> C.c_void_p:
    idx = t.get_device()
    if _raw_stream is None or idx < 0:
        return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)
    return C.c_void_p(_raw_stream(idx))


def ptr(t) -> C.c_void_p:
    return C.c_void_p(0 if t is None else t.data_ptr())


def require(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def contiguous_bf16(t: torch.Tensor, name: str) -> torch.Tensor:
    require(t.dtype == torch.bfloat16, f"{name} must be bfloat16 on the CUDA path (got {t.dtype})")
    return t if t.is_contiguous() else t.contiguous()


# Element types as the kernels name them (ElemType in csrc/elementwise.cuh).
ELEM = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def require_device(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} must be on {device} (got {t.device})")


def refuse_tangents(**tensors) -> None:
    """Refuses tensors that carry a forward-mode tangent: a kernel works on the values alone, and a result without a tangent
    would read as a derivative of zero.  Outside of a dual level, which is where nearly all calls are, nothing is looked at."""
    if getattr(forward_ad, "_current_level", 0) < 0:
        return
    for name, t in tensors.items():
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name} carries a tangent: forward-mode derivatives are only there for CPU tensors")


class _Here:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def on_device(t: torch.Tensor):
    """Context in which ``t``'s device is the current one: a kernel can only be launched there, and on its streams."""
    return _HERE if t.get_device() == torch.cuda.current_device() else torch.cuda.device(t.device)


def rows_view(t: torch.Tensor) -> torch.Tensor:
    """``t`` as [rows, last dim] with unit stride along a row; a copy only where no such view exists."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


class Entry:
    """One exported function, looked up and declared at its first call; a non-zero code raises."""

    def __init__(self, name: str, *argtypes):
        self.name, self.argtypes, self.fn = name, argtypes, None

    def __call__(self, *args) -> None:
        fn = self.fn
        if fn is None:
            fn = self.fn = declare(self.name, list(self.argtypes))
        code = fn(*args)
        if code != 0:
            nv.check(code, self.name.replace("b200_", "").replace("_", " ") + " launch")


_declared = set()


def declare(name: str, argtypes, restype=C.c_int):
    if name not in _declared:
        nv.declare(name, argtypes, restype)
        _declared.add(name)
    return getattr(nv.lib(), name)


_DEFAULT_STATUS = {}


def default_status(device) -> torch.Tensor:
    """The device's default status word (int32 [4], zero = ok): where a kernel launched
    without a caller-owned status tensor records timeouts, overflows and bad indices, so that
    such a report is never dropped.  Read it with :func:`check_default_status`."""
    device = torch.device(device)
    idx = device.index if device.index is not None else torch.cuda.current_device()
    t = _DEFAULT_STATUS.get(idx)
    if t is None:
        t = torch.zeros(4, dtype=torch.int32, device=torch.device("cuda", idx))
        with torch.cuda.device(idx):
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream().synchronize()      # once: kernels on other streams report to it next
        _DEFAULT_STATUS[idx] = t
    return t


def launch_status(device) -> torch.Tensor:
    """:func:`default_status` for a launch that may be under capture into a graph.  The word itself cannot be made there: it
    would live in that graph's memory and be zeroed by every replay."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx not in _DEFAULT_STATUS and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("first call on this device is under graph capture: call the op, or default_status(device), once before")
    return default_status(device)


def check_default_status(device=None, reset: bool = True) -> None:
    """Raise if a kernel that was launched without a caller-owned status tensor has reported
    an error on ``device`` (default: the current device).  Synchronises."""
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    st = default_status(device).tolist()
    if st[0] != 0:
        if reset:
            default_status(device).zero_()
        extra = f" (rows needed: {st[1]})" if st[0] == 10 and st[1] > 0 else ""
        raise nv.NativeError(f"device status {st[0]}: {nv.status_message(st[0])}{extra}")
