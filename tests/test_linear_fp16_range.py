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
    start = 0
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


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [[3, 9, 0, 20], [300, 170, 0, 500]])
def test_the_power_of_two_goes_with_the_inputs_of_a_replay(rows):
    """Captured with ordinary gradients, replayed with ones that need a power of two, then with smaller ones and with ordinary
    ones again; two graphs, and another stream, get the same bits as calls without a graph."""
    from iris_testing_b200 import ops
    x, w, b, _, dy = inputs(rows, 512, 256, torch.float16, "silu_gate", True, False, "cuda", slack=11)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    gr = torch.tensor(rows, dtype=torch.int32, device="cuda")

    def step():
        y = ops.linear(*leaves, activation="silu_gate", group_rows=gr)
        return torch.autograd.grad(y, leaves, dy)
    first = step()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step())
    plain, bx, bw = dy.clone(), x.detach().clone(), w.detach().clone()
    seen = []
    for scale, small in ((1.0, 1.0), (2000.0, 2.0 ** -8), (2.0 ** -20, 1.0), (1.0, 1.0)):
        with torch.no_grad():
            dy.copy_(plain * scale)
            x.copy_(bx * small)
            b.copy_(torch.full_like(b, 100.0) if scale > 1 else torch.full_like(b, 0.25))
        for g in graphs:
            g.replay()
        want = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream().wait_stream(side)
        for out in (*outs, other):
            for p, q in zip(out, want):
                assert torch.equal(p, q)
        # of the second, dx sums 512 products of 2e5 and 1 / 16 and dw up to 500 of 2e5 and 2^-8, up to four times 17000: what is
        # beyond the type is infinite, and nothing is NaN
        assert not torch.isnan(want[0]).any() and not torch.isnan(want[1]).any()
        seen.append(largest(x.detach(), w.detach(), b.detach(), "silu_gate", rows, dy))
    assert seen[0] == seen[3] and seen[1] > 65520 and seen[2] < 2.0 ** -10 < seen[0] < 65504
    assert all(t.shape == s.shape for t, s in zip(first, leaves))
    ops.check_default_status()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_an_infinite_gradient_stays_in_its_row(bad):
    """It has no part in the power of two, and reaches no other row or group."""
    from iris_testing_b200 import ops
    rows = [70, 33, 0, 100]
    x, w, b, _, dy = inputs(rows, 256, 128, torch.float16, "silu_gate", True, False, "cuda", slack=9)
    dy = dy * 2.0 ** -18                                             # small ones, under a power of two
    gr = torch.tensor(rows, dtype=torch.int32, device="cuda")

    def grads():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        return torch.autograd.grad(ops.linear(*leaves, activation="silu_gate", group_rows=gr), leaves, dy)
    want = grads()
    dy[80] = 0
    dy[203:] = bad                                                   # behind the last group
    clean = grads()
    dy[80] = bad
    got = grads()
    others, keep = [0, 2, 3], [i for i in range(212) if i != 80]
    assert torch.equal(want[0][:70], got[0][:70]) and torch.equal(clean[0][keep], got[0][keep])
    for i in (1, 2):
        assert torch.equal(got[i][others], want[i][others]) and not torch.isfinite(got[i][1]).all()
