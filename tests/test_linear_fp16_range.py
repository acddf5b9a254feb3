"""fp16 products with an activation whose gradient dz leaves fp16's range while the results do not.

dz is kept in fp16, off by 2^-11 |dz| and 2^-25 in absolute terms.  Where a call's largest |dz| would round to infinity (from 65520
on), or is below 2^-10, all of its dz are kept under a power of two that takes the largest into [2^14, 2^15): off by 2^-25 of that power of
two, which is below 2^-39 of the largest.  The power of two stays below 2^11; above that dz is infinite, as fp16 has it.  All other bounds are
those of test_linear_kept_z.py."""
import importlib

import pytest
import torch

import test_linear_kept_z as kept
from test_linear import ACTS, act_and_slope, halves, inputs, joined, within


def largest(x, w, b, act, rows, dy):
    """Largest |dz|."""
    top, start = 0.0, 0
    for g, n in enumerate(rows):
        s = slice(start, start + n)
        start += n
        if n:
            z, d = x[s].double() @ w[g].double().t() + b[g].double(), dy[s].double()
            if act == "silu_gate":
                (zg, zu), (a, sl) = halves(z), act_and_slope(halves(z)[0], "silu")
                dz = joined(d * zu * sl, d * a)
            else:
                dz = d * act_and_slope(z, act)[1]
            top = max(top, float(dz.abs().max()))
    return top


def check(x, w, b, dy, act, rows, dense):
    from iris_testing_b200 import ops
    leaves = [t.detach().requires_grad_() for t in ((x, w[0], b[0]) if dense else (x, w, b))]
    gr = None if dense else torch.tensor(rows, dtype=torch.int32, device=x.device)
    grads = torch.autograd.grad(ops.linear(*leaves, activation=act, group_rows=gr), leaves, dy)
    top = largest(x, w, b, act, rows, dy)
    # the bounds there hold 2^-25 for dz's absolute error: as much more as the power of two is
    power = top * 2.0 ** -14 if top >= 65000 else 1.0
    want = reference_under(x, w, b, act, rows, dy, power)
    for got, t, pair, name in zip(grads, (x, w, b), want, ("dx", "dw", "dbias")):
        within(got.view(t.shape), pair, name)
        assert torch.isfinite(got).all() and bool(got.any()), name
    ops.check_default_status()
    return top


def reference_under(x, w, b, act, rows, dy, power):
    """The bounds of ``kept.reference`` with dz's absolute error 2^-25 times ``power`` (of small dz: 2^-38 of the largest)."""
    top = largest(x, w, b, act, rows, dy)
    extra = 2.0 ** -25 * power if top >= 2.0 ** -10 else 2.0 ** -38 * top
    plain = kept.reference(x, w, b, act, rows, dy)
    # what 2^-25 adds to each result there is taken off, and what ``extra`` adds is put on; both without the results' own half step
    start, out = 0, []
    (dx, ex), (dw, ew), (db, eb) = plain
    ex, ew = ex.clone(), ew.clone()
    for g, n in enumerate(rows):
        s = slice(start, start + n)
        start += n
        if n:
            ex[s] += (extra - 2.0 ** -25) * w[g].double().abs().sum(0)
            ew[g] += (extra - 2.0 ** -25) * x[s].double().abs().sum(0)
    return [(dx, ex), (dw, ew), (db, eb)]


SHAPES = [([37], 256, 64), ([333], 512, 264), ([40, 0, 129, 1], 256, 72), ([200, 300], 768, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("rows,N,K", SHAPES)
def test_small_gradients(rows, N, K, act, split, monkeypatch):
    """Output gradients next to fp16's smallest numbers under large weights and inputs: dz is below them, its products are not."""
    mod = importlib.import_module("iris_testing_b200.ops.linear")
    monkeypatch.setattr(mod, "_splits", lambda mode, M, N, K, G, grouped, sms: split and not (grouped and mode == 2))
    x, w, b, _, dy = inputs(rows, N, K, torch.float16, act, True, False, "cuda")
    w, x, dy = w * 64, x / 64, dy * 2.0 ** -18
    if act == "silu_gate":                                           # small up halves, which dz of the gate half is a multiple of
        half = w.view(len(rows), N // 256, 2, 128, K)
        half[:, :, 1] /= 64
        b.view(len(rows), N // 256, 2, 128)[:, :, 1] /= 64
    x, w = x * 1024, w / 1024 * 16                                   # z of about 16; x large enough for dw to be within the type
    assert check(x, w, b, dy, act, rows, len(rows) == 1) < 2.0 ** -10


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("rows,N,K", SHAPES)
def test_large_gradients(rows, N, K, split, monkeypatch):
    """Output gradients under a loss scale times a large half of the gated form: dz passes 65504, its products with small weights
    and inputs do not."""
    mod = importlib.import_module("iris_testing_b200.ops.linear")
    monkeypatch.setattr(mod, "_splits", lambda mode, M, N, K, G, grouped, sms: split and not (grouped and mode == 2))
    x, w, b, _, dy = inputs(rows, N, K, torch.float16, "silu_gate", False, False, "cuda")
    x, w, dy = x * 2.0 ** -11, w * 2.0 ** -9, dy * 2000
    b = torch.zeros(len(rows), N, device="cuda", dtype=torch.float16)
    b.view(len(rows), N // 256, 2, 128)[:, :, 0] = 1.5
    b.view(len(rows), N // 256, 2, 128)[:, :, 1] = 300
    leaves = [x.requires_grad_(), (w[0] if len(rows) == 1 else w).requires_grad_()]
    from iris_testing_b200 import ops
    gr = None if len(rows) == 1 else torch.tensor(rows, dtype=torch.int32, device="cuda")
    grads = torch.autograd.grad(ops.linear(leaves[0], leaves[1], b[0] if gr is None else b, activation="silu_gate", group_rows=gr), leaves, dy)
    x, w = x.detach(), w.detach()
    top = largest(x, w, b, "silu_gate", rows, dy)
    assert 2.0 ** 17 < top < 2.0 ** 24
    for got, t, pair, name in zip(grads, (x, w), reference_under(x, w, b, "silu_gate", rows, dy, top * 2.0 ** -14), ("dx", "dw")):
        assert torch.isfinite(pair[0]).all() and float(pair[0].abs().max()) < 6e4, "the results are meant to fit"
        within(got.view(t.shape), pair, name)
    ops.check_default_status()
