"""Sizes above 32 bits are refused before anything is copied or launched: the argument blocks hold them as C ints, which take the
lower 32 bits without a word.  All tensors are views of one element; the ops take the kernels' path for CPU tensors here, with a
stand-in for the first copy that they make."""
import importlib

import pytest
import torch


class Reached(Exception):
    pass


def reached(*args, **kwargs):
    raise Reached


def one(*shape, dtype=torch.bfloat16):
    return torch.zeros((1,) * len(shape), dtype=dtype).expand(*shape)


@pytest.mark.parametrize("K", [2 ** 31, 2 ** 32 + 8])
@pytest.mark.parametrize("grouped", [False, True])
def test_contracted_length(K, grouped, monkeypatch):
    mod = importlib.import_module("iris_testing_b200.ops.linear")
    monkeypatch.setattr(mod, "use_native", lambda t: True)
    monkeypatch.setattr(mod, "_plain", reached)
    rows = torch.ones(1, dtype=torch.int32) if grouped else None

    def call(k):
        return mod.linear(one(1, k), one(1, 8, k) if grouped else one(8, k), group_rows=rows)
    with pytest.raises(ValueError, match="columns"):
        call(K)
    with pytest.raises(Reached):
        call(4096)


@pytest.mark.parametrize("k", [2 ** 31, 2 ** 32 + 2])
def test_copies_of_a_token(k, monkeypatch):
    mod = importlib.import_module("iris_testing_b200.ops.balance")
    monkeypatch.setattr(mod, "use_native", lambda t: True)
    monkeypatch.setattr(mod, "rows_view", reached)
    with pytest.raises(ValueError, match="experts of a token"):
        mod.balance_loss(one(1, 8, dtype=torch.float32), one(1, k, dtype=torch.int32))
    with pytest.raises(Reached):
        mod.balance_loss(one(1, 8, dtype=torch.float32), one(1, 8, dtype=torch.int32))


def test_columns_of_a_result_with_gradients(monkeypatch):
    """The gradient of an activation, a bias or a grouped residual takes 1024 columns a block, 65535 blocks side by side."""
    mod = importlib.import_module("iris_testing_b200.ops.linear")
    monkeypatch.setattr(mod, "use_native", lambda t: True)
    monkeypatch.setattr(mod._Linear, "apply", reached)
    monkeypatch.setattr(mod, "_plain", lambda t: t)
    monkeypatch.setattr(mod, "_forward", reached)
    N = 65535 * 1024

    def call(n, grad=True, **how):
        return mod.linear(one(1, 8).requires_grad_(grad), one(n, 8), **how)
    for how in (dict(activation="relu"), dict(bias=one(N + 8))):
        with pytest.raises(ValueError, match="columns"):
            call(N + 8, **how)
        with pytest.raises(Reached):
            call(N + 8, False, **how)
    for n, how in ((N, dict(activation="relu")), (N + 8, dict(residual=one(1, N + 8))), (N + 256, {}),
                   (2 * N, dict(activation="silu_gate"))):
        with pytest.raises(Reached):
            call(n, **how)
    with pytest.raises(ValueError, match="columns"):
        mod.linear(one(1, 8).requires_grad_(), one(1, N + 8, 8), residual=one(1, N + 8), group_rows=torch.ones(1, dtype=torch.int32))
