"""The ctypes mirrors of the argument blocks of the norms, the balance loss and the linear products, byte for byte."""
import ctypes as C

import pytest


def test_argument_block_sizes_match():
    from iris_testing_b200 import _native
    from iris_testing_b200.ops.balance import MAX_BALANCE_EXPERTS, BalanceArgs
    from iris_testing_b200.ops.norm import MAX_COLUMNS, NormArgs
    import importlib
    linear = importlib.import_module("iris_testing_b200.ops.linear")
    try:
        lib = _native.lib()
    except Exception as exc:        # no nvcc and no prebuilt library on this machine
        pytest.skip(f"native library unavailable: {exc}")
    assert lib.b200_abi_size_norm_args() == C.sizeof(NormArgs)
    assert lib.b200_abi_size_balance_args() == C.sizeof(BalanceArgs)
    sizes = (C.c_int * 2)()
    lib.b200_abi_sizes_linear(sizes)
    assert list(sizes) == [C.sizeof(linear.LinearArgs), C.sizeof(linear.ActGradArgs)]
    assert lib.b200_norm_max_columns() == MAX_COLUMNS
    assert lib.b200_balance_max_experts() == MAX_BALANCE_EXPERTS


def _split_args(linear):
    la = linear.LinearArgs()
    la.G, la.M, la.N, la.K, la.n_out, la.elem, la.mode = 1, 16, 64, 64, 64, 1, 0
    return la


def test_entries_refuse_bad_arguments_without_a_gpu():
    """Every check below comes before the first CUDA call."""
    from iris_testing_b200 import _native
    from iris_testing_b200.ops.balance import BalanceArgs
    from iris_testing_b200.ops.norm import NormArgs
    import importlib
    linear = importlib.import_module("iris_testing_b200.ops.linear")
    try:
        lib = _native.lib()
    except Exception as exc:
        pytest.skip(f"native library unavailable: {exc}")
    assert lib.b200_norm_forward(None, 148, None) < 0
    n = NormArgs()
    n.T, n.H, n.y, n.h = 1, 16385, 16, 16
    assert lib.b200_norm_forward(C.byref(n), 148, None) < 0
    n.H, n.gate_kind = 64, 1                       # a gate without a residual
    assert lib.b200_norm_forward(C.byref(n), 148, None) < 0
    n.H, n.gate_kind, n.T = 64, 0, (1 << 30) + 1
    assert lib.b200_norm_forward(C.byref(n), 148, None) < 0
    b = BalanceArgs()
    b.T, b.E, b.k, b.S, b.runs, b.run_tokens = 10, 8, 2, 1, 2, 4       # runs that do not cover the tokens
    assert lib.b200_balance_forward(C.byref(b), None) < 0
    b.T, b.runs, b.run_tokens = 2 ** 31 - 1000, 1, 2 ** 31 - 1000
    assert lib.b200_balance_forward(C.byref(b), None) < 0
    b.T, b.runs, b.run_tokens, b.S = 10, 2, 5, 2 ** 31 - 1000
    assert lib.b200_balance_forward(C.byref(b), None) < 0
    b.S, b.E = 1, 1025
    assert lib.b200_balance_forward(C.byref(b), None) < 0
    for field, value in (("N", 60), ("K", 4), ("G", 129), ("G", 2), ("M", 0), ("M", 2 ** 31 - 1000), ("n_out", 128), ("elem", 0), ("mode", 3)):
        la = _split_args(linear)
        setattr(la, field, value)
        assert lib.b200_linear(C.byref(la), 148, None) < 0, field
    la = _split_args(linear)
    la.mode, la.record, la.group_rows = 2, 16, 16        # a grouped dW is not split
    assert lib.b200_linear(C.byref(la), 148, None) < 0
    a = linear.ActGradArgs()
    a.G, a.M, a.N, a.n_out, a.elem, a.act, a.chunks, a.chunk_rows = 1, 16, 64, 64, 1, 1, 1, 16
    assert lib.b200_act_grad(C.byref(a), None) < 0       # an activation without its z
