"""What the C entries of ``linear`` refuse of the scratch that its backward pass uses, before the first CUDA call."""
import ctypes as C
import importlib

import pytest


def test_scratch_that_does_not_fit_together():
    from iris_testing_b200 import _native
    linear = importlib.import_module("iris_testing_b200.ops.linear")
    try:
        lib = _native.lib()
    except Exception as exc:        # no nvcc and no prebuilt library on this machine
        pytest.skip(f"native library unavailable: {exc}")

    def product(**how):
        la = linear.LinearArgs()
        la.G, la.M, la.N, la.K, la.n_out, la.elem, la.mode = 1, 16, 64, 64, 64, 2, 0
        for k, v in how.items():
            setattr(la, k, v)
        return lib.b200_linear(C.byref(la), 148, None)
    assert product(z=16) == -17 and product(zexp=16) == -17          # one without the other
    assert product(z=16, zexp=24) == -17                             # not on 16 bytes
    assert product(mode=1, elem=1, res=16) == -18                    # a power of two of bf16 dz

    def gradient(**how):
        a = linear.ActGradArgs()
        a.G, a.M, a.N, a.n_out, a.elem, a.act, a.chunks, a.chunk_rows = 1, 16, 64, 64, 2, 1, 1, 16
        a.z, a.zexp, a.dz = 16, 16, 16
        for k, v in how.items():
            setattr(a, k, v)
        return lib.b200_act_grad(C.byref(a), None)
    assert gradient() == -15                                         # fp16 without a word for the largest |dz|
    assert gradient(elem=1, peak=16) == -15                          # bf16 with one
    assert gradient(act=0, z=None, zexp=None, dz=None, peak=16) == -15
    assert gradient(zexp=None) == -14
