"""The pre-activations that ``linear`` keeps for its backward pass, and gradients held to what they are kept to.

z is kept to 11 bits (of fp16 products to 16: see test_linear_fp16_precision.py), off by 2^-11 |z|, and in absolute terms by 2^-30; where 32 neighbouring columns of a row hold both a value of
1024 or more and one 2^31 times smaller than their largest, to 8 bits, off by 2^-8 |z| whatever the size.  Everything else is bounded
as in test_linear.py: sums of K products by (K / 16 + 16) 2^-23 of their magnitudes, the activations' slopes by 1.13 and their
curvatures by 1.2, 32 roundings for computing them, dz and the results rounded to the element type."""
import importlib

import pytest
import torch

from test_linear import ACTS, F64, act_and_slope, halves, inputs, joined, within

BF16_CHUNK = 255                                     # the exponent byte of 32 columns that are kept as bf16


def mod():
    return importlib.import_module("iris_testing_b200.ops.linear")


def kept_to(z):
    """How far what is kept may be from z [M, N].  The conditions leave some room: z itself is only known to its rounding."""
    M, N = z.shape
    chunks = torch.nn.functional.pad(z.abs(), (0, -N % 32)).view(M, -1, 32)
    most = chunks.amax(2)
    least = torch.where(chunks > 0, chunks, torch.full_like(chunks, float("inf"))).amin(2)
    wide, small = (most >= 1000) & (least < most * 2.0 ** -27), most < 1100

    def spread(per_chunk):
        return per_chunk.to(F64).repeat_interleave(32, 1)[:, :N]
    return (2.0 ** -11 + (2.0 ** -8 - 2.0 ** -11) * spread(wide)) * z.abs() + 2.0 ** -30 * spread(small)


def reference(x, w, bias, act, rows, dy):
    """[(value, bound)] of dx, dw, dbias in fp64."""
    u = torch.finfo(x.dtype).eps / 2
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 1e-38
    G, N, K = w.shape

    def acc(k):
        return (k / 16 + 16) * 2.0 ** -23
    zeros = dict(dtype=F64, device=x.device)
    dx, ex = torch.zeros(x.shape, **zeros), torch.zeros(x.shape, **zeros)
    dw, ew = torch.zeros(G, N, K, **zeros), torch.zeros(G, N, K, **zeros)
    db, eb = torch.zeros(G, N, **zeros), torch.zeros(G, N, **zeros)
    start, r32 = 0, 32 * 2.0 ** -24
    for g, n in enumerate(rows):
        s = slice(start, start + n)
        start += n
        if n == 0:
            continue
        xg, wg, d, bg = x[s].double(), w[g].double(), dy[s].double(), bias[g].double()
        z = xg @ wg.t() + bg
        ez = acc(K) * (xg.abs() @ wg.abs().t() + bg.abs()) + kept_to(z)
        if act == "silu_gate":
            (zg, zu), (eg, eu) = halves(z), halves(ez)
            a, sl = act_and_slope(zg, "silu")
            dz = joined(d * zu * sl, d * a)
            ed = joined(d.abs() * (1.2 * eg * (zu.abs() + eu) + 1.13 * eu), d.abs() * 1.13 * eg)
            ed = ed + r32 * joined(d.abs() * zu.abs() * 1.2, d.abs() * zg.abs())
        else:
            _, sl = act_and_slope(z, act)
            dz = d * sl
            ed = d.abs() * ((z.abs() <= ez).to(F64) if act == "relu" else 1.2 * ez) + r32 * 1.2 * d.abs()
        edz = ed + u * (dz.abs() + ed) + tiny
        dx[s], ex[s] = dz @ wg, edz @ wg.abs() + acc(N) * (dz.abs() @ wg.abs())
        dw[g], ew[g] = dz.t() @ xg, edz.t() @ xg.abs() + acc(n) * (dz.abs().t() @ xg.abs())
        db[g], eb[g] = dz.sum(0), ed.sum(0) + 256 * 2.0 ** -24 * dz.abs().sum(0)
    return [(v, b + u * v.abs() + tiny) for v, b in ((dx, ex), (dw, ew), (db, eb))]


def as_type(got, pair):
    """``got`` in 64 bits, with an infinity read as the result itself where that rounds to one: from half a step above the type's
    largest number on, (2 - 2^-11) 2^15 = 65504 and 16 more for fp16, all values are rounded to infinity; the result may be off by its bound
    before it is rounded."""
    ref, bound = pair
    top = torch.finfo(got.dtype)
    over = ref.abs() + bound >= top.max * (1 + top.eps / 4)
    return torch.where(over & torch.isinf(got) & ((got > 0) == (ref > 0)), ref, got.double())


def check(x, w, b, dy, act, rows, dense):
    from iris_testing_b200 import ops
    leaves = [t.detach().requires_grad_() for t in ((x, w[0], b[0]) if dense else (x, w, b))]
    gr = None if dense else torch.tensor(rows, dtype=torch.int32, device=x.device)
    grads = torch.autograd.grad(ops.linear(*leaves, activation=act, group_rows=gr), leaves, dy)
    for got, t, want, name in zip(grads, (x, w, b), reference(x, w, b, act, rows, dy), ("dx", "dw", "dbias")):
        within(as_type(got.view(t.shape), want), want, name)
    ops.check_default_status()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("rows,N,K", [([1], 256, 64), ([333], 512, 264), ([40, 0, 129, 1], 256, 72), ([200, 300], 768, 1024)])
def test_gradients_to_11_bits_of_z(rows, N, K, act, dtype):
    x, w, b, _, dy = inputs(rows, N, K, dtype, act, True, False, "cuda", slack=70 if len(rows) > 1 else 0)
    check(x, w, b, dy, act, rows, len(rows) == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("size", [2.0 ** 9, 2.0 ** 12, 2.0 ** 27, 2.0 ** 31, 1e10, 1e12, 1e13, 1e20])
def test_gradients_next_to_a_large_value(size, act, dtype, split, monkeypatch):
    """One column of 32 holds a value that leaves ordinary ones far behind: their slopes and, of the gated form, the products with
    them are as right as without it."""
    monkeypatch.setattr(mod(), "_splits", lambda *a: split)
    M, K = 40, 128
    N = 2 * K if act == "silu_gate" else K
    g = torch.Generator().manual_seed(int(size) % 1000)
    x = torch.randn(M, K, generator=g)
    x[3, ::2] *= 2.0 ** -10
    w = torch.zeros(1, N, K)
    w[0, :K] = torch.eye(K)                          # each z has one x in it: sums add no error of other columns
    if act == "silu_gate":
        w[0, K:] = torch.eye(K).flip(0)
    root = size ** 0.5 if size > 6e4 else 1.0        # a value above fp16's range, as a product of two within it
    for c in (5, 64):
        x[::3, c] = size / root
        w[0, c, c] = root
    x, w = x.to("cuda", dtype), w.to("cuda", dtype)
    if not torch.isfinite(x).all() or not torch.isfinite(w).all():
        pytest.skip("beyond this type's range")
    b = (torch.randn(1, N, generator=g) * 0.1).to("cuda", dtype)
    dy = torch.randn(M, N // 2 if act == "silu_gate" else N, generator=g).to("cuda", dtype)
    dy[::3, [5, 64]] = 0                             # what the large values themselves get is not looked at here
    if act == "silu_gate":
        dy[::3, [K - 6, K - 65]] = 0
    check(x, w, b, dy, act, [M], True)


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("act,N", [("silu", 136), ("silu_gate", 256)])
def test_what_is_kept(act, N, split, monkeypatch):
    """Rows whose values lie up to 2^200 apart, next to an infinity, a NaN and zeros."""
    monkeypatch.setattr(mod(), "_splits", lambda *a: split)
    M, K = 96, N
    g = torch.Generator().manual_seed(5)
    apart = torch.linspace(0, 100, M).view(M, 1)
    x = torch.randn(M, K, generator=g) * torch.exp2((torch.rand(M, K, generator=g) * 2 - 1) * apart)
    x[7], x[:, 9], x[:, 40:42] = 0, 0, 0
    x, w = x.to("cuda", torch.bfloat16), torch.eye(K).to("cuda", torch.bfloat16)
    b = torch.zeros(N, device="cuda", dtype=torch.bfloat16)
    b[40], b[41] = float("inf"), float("nan")
    _, (z, e) = mod()._forward(x, w, b, None, None, mod().ACTIVATIONS[act], True)
    chunk = e.repeat_interleave(32, 1)[:, :N]
    got = torch.where(chunk == BF16_CHUNK, z.view(torch.bfloat16).double(), z.double() * torch.exp2(chunk.double() - 141))
    assert torch.isinf(got[:, 40]).all() and torch.isnan(got[:, 41]).all()
    got[:, 40:42] = 0
    off = (got - x.double()).abs() - kept_to(x.double())
    assert bool((off <= 0).all()), float(off.max())
    assert bool((chunk == BF16_CHUNK).any()) and bool((chunk != BF16_CHUNK).any())
