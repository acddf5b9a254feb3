"""fp16 gradients behind an activation: as near to 64 bits as rounding dz and the result allows.

Rounding a result to 11 bits puts it r = 2e-4 off in the norm.  dz, an operand of the tensor cores, is rounded likewise, each value on its own,
so that products of many of them are off by r too: together sqrt(2) r = 1.42 r.  z kept to 16 bits (2^-15, r / 13 in the norm at most)
and fp32 sums add next to nothing.  11 bits of z would be off by r in slopes and, of the gated form, in both factors of dz."""
import importlib

import pytest
import torch

from test_linear import F64, act_and_slope, halves, inputs, joined


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("act", ["silu", "gelu", "silu_gate"])
@pytest.mark.parametrize("rows,N,K", [([700], 768, 520), ([300, 0, 257, 1], 1024, 264)])
def test_gradients_in_the_norm(rows, N, K, act, split, monkeypatch):
    from iris_testing_b200 import ops
    mod = importlib.import_module("iris_testing_b200.ops.linear")
    monkeypatch.setattr(mod, "_splits", lambda mode, M, N, K, G, grouped, sms: split and not (grouped and mode == 2))
    dense = len(rows) == 1
    x, w, b, _, dy = inputs(rows, N, K, torch.float16, act, True, False, "cuda")
    leaves = [t.detach().requires_grad_() for t in ((x, w[0]) if dense else (x, w))]
    gr = None if dense else torch.tensor(rows, dtype=torch.int32, device="cuda")
    got = torch.autograd.grad(ops.linear(*leaves, b[0] if dense else b, activation=act, group_rows=gr), leaves, dy)
    dx, dw, start = torch.zeros(x.shape, dtype=F64, device="cuda"), torch.zeros(w.shape, dtype=F64, device="cuda"), 0
    for g, n in enumerate(rows):
        s = slice(start, start + n)
        start += n
        z, d = x[s].double() @ w[g].double().t() + b[g].double(), dy[s].double()
        if act == "silu_gate":
            (zg, zu), (a, sl) = halves(z), act_and_slope(halves(z)[0], "silu")
            dz = joined(d * zu * sl, d * a)
        else:
            dz = d * act_and_slope(z, act)[1]
        dx[s], dw[g] = dz @ w[g].double(), dz.t() @ x[s].double()
    for a, want in zip(got, (dx, dw)):
        rounding = float((want.half().double() - want).norm() / want.norm())
        off = float((a.double().view(want.shape) - want).norm() / want.norm())
        assert off <= 1.5 * rounding, (off, rounding)
    ops.check_default_status()


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("act,N", [("silu", 136), ("silu_gate", 256)])
def test_what_is_kept(act, N, split, monkeypatch):
    """z as fp32 cut to its upper 24 bits: 16 in z, 8 in the bytes beside it."""
    mod = importlib.import_module("iris_testing_b200.ops.linear")
    monkeypatch.setattr(mod, "_splits", lambda *a: split)
    M, K = 96, N
    g = torch.Generator().manual_seed(6)
    x = (torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-20, 12, (M, 1), generator=g).float())).to("cuda", torch.float16)
    x[7], x[:, 40:42] = 0, 0
    w = torch.eye(K).to("cuda", torch.float16)
    b = (torch.randn(N, generator=g) * 2.0 ** -5).to("cuda", torch.float16)
    b[40], b[41], b[50] = float("inf"), float("nan"), 0
    x[:, 50] = 0
    _, (z, low) = mod._forward(x, w, b, None, None, mod.ACTIVATIONS[act], True)
    assert low.shape == (M, 256)
    bits = (z.view(torch.int16).int() << 16) | (low[:, :N].int() << 8)
    got, want = bits.view(torch.float32).double(), x.double() + b.double()
    assert torch.isinf(got[:, 40]).all() and torch.isnan(got[:, 41]).all() and not got[:, 50].any()
    got[:, 40:42] = want[:, 40:42] = 0
    assert bool(((got - want).abs() <= (2.0 ** -15 + 2.0 ** -23) * want.abs()).all())      # and one fp32 rounding of x + b
