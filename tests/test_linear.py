"""``linear`` against its definition in 64 bits, forward and backward, dense and grouped.

Tolerances are bounds, not estimates; ``u`` is half a step of the element type.  The tensor cores add 16 products at a time
into an fp32 accumulator and may truncate, so a sum over K terms is off by at most (K / 16 + 16) 2^-23 of the sum of
magnitudes; joining split sums stays within the 16.  A result's own rounding adds u.  The activations here have slopes of at most 1.13 and curvatures of at most
1.2, and are computed to 32 roundings.  The backward pass reads z rounded to the element type (off by u |z| more) and
rounds dz (u |dz|); where a relu's z is within its error of zero the slope may be either.  Column sums of dz add up
to 64 terms and 64 records in order: 256 x 2^-24."""
import importlib

import pytest
import torch

F64 = torch.float64
ACTS = [None, "relu", "silu", "gelu", "silu_gate"]


def act_and_slope(z, act):
    if act is None:
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).to(F64)
    if act == "silu":
        q = torch.sigmoid(z)
        return z * q, q * (1 + z * (1 - q))
    a, b = (2 / torch.pi) ** 0.5, 0.044715
    t = torch.tanh(a * (z + b * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * b * z * z)


def halves(t):
    v = t.unflatten(1, (-1, 2, 128))
    return v[:, :, 0].flatten(1), v[:, :, 1].flatten(1)


def joined(a, b):
    return torch.stack((a.unflatten(1, (-1, 128)), b.unflatten(1, (-1, 128))), 2).flatten(1)


def reference(x, w, bias, res, act, rows, dy):
    """[(value, bound)] of y, dx, dw, dbias, dres in fp64; ``rows`` is a list, dense is one group."""
    u = torch.finfo(x.dtype).eps / 2
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 1e-38       # half a step below the smallest normal number
    G, N, K = w.shape
    M = x.shape[0]
    n_out = N // 2 if act == "silu_gate" else N

    def acc(k):
        return (k / 16 + 16) * 2.0 ** -23
    zeros = dict(dtype=F64, device=x.device)
    y, ey = torch.zeros(M, n_out, **zeros), torch.zeros(M, n_out, **zeros)
    dx, ex = torch.zeros(M, K, **zeros), torch.zeros(M, K, **zeros)
    dw, ew = torch.zeros(G, N, K, **zeros), torch.zeros(G, N, K, **zeros)
    db, eb = torch.zeros(G, N, **zeros), torch.zeros(G, N, **zeros)
    dr = torch.zeros(M, n_out, **zeros)
    start = 0
    for g, n in enumerate(rows):
        s = slice(start, start + n)
        start += n
        if n == 0:
            continue
        xg, wg, d = x[s].double(), w[g].double(), dy[s].double()
        bg = bias[g].double() if bias is not None else torch.zeros(N, **zeros)
        z = xg @ wg.t() + bg
        e = acc(K) * (xg.abs() @ wg.abs().t() + bg.abs())
        r32 = 32 * 2.0 ** -24
        ez = e + u * z.abs()                       # of the z that the backward pass reads
        if act == "silu_gate":
            (zg, zu), (eg, eu), (eg2, eu2) = halves(z), halves(e), halves(ez)
            a, sl = act_and_slope(zg, "silu")
            val = a * zu
            err = 1.13 * eg * (zu.abs() + eu) + eu * a.abs() + r32 * (zg * zu).abs()
            dz = joined(d * zu * sl, d * a)
            ed = joined(d.abs() * (1.2 * eg2 * (zu.abs() + eu2) + 1.13 * eu2), d.abs() * 1.13 * eg2)
            ed = ed + r32 * joined(d.abs() * zu.abs() * 1.2, d.abs() * zg.abs())
        else:
            val, sl = act_and_slope(z, act)
            err = 1.13 * e + r32 * z.abs()
            dz = d * sl
            flip = (z.abs() <= ez).to(F64) if act == "relu" else 1.2 * ez if act is not None else 0.0 * ez
            ed = d.abs() * flip + r32 * 1.2 * d.abs()
        if res is not None:
            val = val + res[s].double()
            err = err + 2.0 ** -23 * (val.abs() + res[s].double().abs())
        y[s], ey[s] = val, err + u * val.abs() + tiny
        round_dz = 0.0 if act is None else 1.0     # without an activation dz is dy itself
        if act is None:
            ed = torch.zeros_like(ed)
        edz = ed + round_dz * (u * (dz.abs() + ed) + tiny)
        dx[s] = dz @ wg
        ex[s] = edz @ wg.abs() + acc(N) * (dz.abs() @ wg.abs())
        dw[g] = dz.t() @ xg
        ew[g] = edz.t() @ xg.abs() + acc(n) * (dz.abs().t() @ xg.abs())
        db[g] = dz.sum(0)
        eb[g] = ed.sum(0) + 256 * 2.0 ** -24 * dz.abs().sum(0)
        dr[s] = d
    own = [(v, b + u * v.abs() + tiny) for v, b in ((dx, ex), (dw, ew), (db, eb))]
    return [(y, ey)] + own + [(dr, torch.zeros_like(dr))]


def inputs(rows, N, K, dtype, act, bias, res, dev, slack=0, seed=0, std=None):
    g = torch.Generator().manual_seed(seed + N + 7 * K + sum(rows))
    M, G = sum(rows) + slack, len(rows)
    n_out = N // 2 if act == "silu_gate" else N

    def rnd(*shape, std=1.0):
        return (torch.randn(*shape, generator=g) * std).to(dev, dtype)
    x, w, dy = rnd(M, K), rnd(G, N, K, std=std or K ** -0.5), rnd(M, n_out)
    return x, w, (rnd(G, N) if bias else None), (rnd(M, n_out) if res else None), dy


def within(got, pair, what):
    ref, bound = pair
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got.double() - ref).abs() - bound
    assert bool((off <= 0).all()), (what, float(off.max()), int((off > 0).sum()))


def check(x, w, bias, res, dy, act, rows, dense=False):
    from iris_testing_b200 import ops
    G, N, K = w.shape
    leaves = [t.detach().requires_grad_() for t in (x, w[0] if dense else w, None if bias is None else bias[0] if dense else bias, res)
              if t is not None]
    it = iter(leaves)
    xl, wl = next(it), next(it)
    bl = next(it) if bias is not None else None
    rl = next(it) if res is not None else None
    gr = None if dense else torch.tensor(rows, dtype=torch.int32, device=x.device)
    y = ops.linear(xl, wl, bl, rl, activation=act, group_rows=gr)
    grads = iter(torch.autograd.grad(y, leaves, dy))
    with torch.no_grad():
        assert torch.equal(y, ops.linear(xl, wl, bl, rl, activation=act, group_rows=gr))
    want = reference(x, w, bias, res, act, rows, dy)
    assert y.dtype == x.dtype
    within(y.detach(), want[0], "y")
    within(next(grads), want[1], "dx")
    within(next(grads).view(G, N, K), want[2], "dw")
    if bias is not None:
        within(next(grads).view(G, N), want[3], "dbias")
    if res is not None:
        within(next(grads), want[4], "dres")
    if x.is_cuda:
        ops.check_default_status()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,N,K", [([5], 256, 16), ([3, 0, 9], 256, 24)])
def test_definition_on_cpu(rows, N, K, act):
    x, w, b, r, dy = inputs(rows, N, K, torch.float16, act, True, True, "cpu", slack=0 if len(rows) == 1 else 2)
    check(x, w, b, r, dy, act, rows, dense=len(rows) == 1)


@pytest.mark.parametrize("act", ACTS)
def test_reference_slopes_against_differences(act):
    """Gradients of the reference in fp64 by central differences of its value."""
    x, w, b, r, dy = (t.double() for t in inputs([2, 3], 256, 8, torch.float64, act, True, True, "cpu"))
    want = reference(x, w, b, r, act, [2, 3], dy)
    g = torch.Generator().manual_seed(1)
    for t, (grad, _) in zip((x, w, b, r), want[1:]):
        step = torch.randn(t.shape, generator=g, dtype=F64) * 1e-5
        t += step
        up = (reference(x, w, b, r, act, [2, 3], dy)[0][0] * dy).sum()
        t -= 2 * step
        down = (reference(x, w, b, r, act, [2, 3], dy)[0][0] * dy).sum()
        t += step
        want_diff = 2 * (grad * step).sum()
        # a relu may be crossed: by at most |dy| |step| for the few values next to zero
        assert abs(float(up - down - want_diff)) < (2e-4 if act == "relu" else 1e-8) * max(1.0, float(grad.abs().sum() * 1e-3))


def test_refusals():
    from iris_testing_b200 import ops
    x, w = torch.ones(6, 16), torch.ones(256, 16)
    w3, rows = torch.ones(2, 256, 16), torch.tensor([3, 3], dtype=torch.int32)
    for bad in (lambda: ops.linear(x, torch.ones(256, 8)),
                lambda: ops.linear(x, w3),
                lambda: ops.linear(x, w, group_rows=rows),
                lambda: ops.linear(x, w, activation="tanh"),
                lambda: ops.linear(x, w[:128], activation="silu_gate"),
                lambda: ops.linear(x, w, torch.ones(255)),
                lambda: ops.linear(x, w3, torch.ones(256), group_rows=rows),
                lambda: ops.linear(x, w, residual=torch.ones(6, 255)),
                lambda: ops.linear(x, w3, group_rows=rows.long()),
                lambda: ops.linear(x, w3, group_rows=rows[:1]),
                lambda: ops.linear(x[None], w3, group_rows=rows),
                lambda: ops.linear(x, w3, group_rows=rows + 1)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("pair", [False, True, None])
@pytest.mark.parametrize("rows,N,K", [([64], 256, 64), ([128], 256, 128), ([1], 8, 8), ([300], 264, 136), ([1000], 512, 1024),
                                      ([63, 65, 1, 0, 200], 264, 136), ([0, 0, 5], 24, 40), ([0, 128, 64, 256, 0], 256, 512),
                                      ([37] * 16, 1408, 256), ([5000], 72, 200), ([700], 40, 4096)])
def test_plain_products(rows, N, K, pair, monkeypatch):
    """Each way to cut the work, whatever the rule would take (None: split along the contraction)."""
    mod = importlib.import_module("iris_testing_b200.ops.linear")
    monkeypatch.setattr(mod, "_pairs", lambda *a: bool(pair))
    monkeypatch.setattr(mod, "_splits", lambda mode, M, N, K, G, grouped, sms: pair is None and not (grouped and mode == 2))
    x, w, b, r, dy = inputs(rows, N, K, torch.bfloat16, None, False, False, "cuda", slack=9 if len(rows) > 1 else 0)
    check(x, w, b, r, dy, None, rows, dense=len(rows) == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,N,K", [([1], 256, 64), ([333], 512, 264), ([40, 0, 129, 1], 256, 72), ([200, 300], 768, 1024)])
def test_epilogues(rows, N, K, act, dtype):
    x, w, b, r, dy = inputs(rows, N, K, dtype, act, True, True, "cuda", slack=70 if len(rows) > 1 else 0)
    check(x, w, b, r, dy, act, rows, dense=len(rows) == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 64, 65, 100, 127, 129, 200, 255, 257, 513])
def test_every_small_number_of_rows(M):
    act = ACTS[M % 5]
    x, w, b, r, dy = inputs([M], 512, 520, torch.bfloat16, act, M % 2 == 0, M % 3 == 0, "cuda")
    check(x, w, b, r, dy, act, [M], dense=True)


@pytest.mark.gpu
@pytest.mark.parametrize("G,most", [(128, 3), (100, 40), (64, 130)])
def test_many_groups(G, most):
    g = torch.Generator().manual_seed(G)
    rows = torch.randint(0, most + 1, (G,), generator=g).tolist()
    x, w, b, r, dy = inputs(rows, 256, 136, torch.bfloat16, "silu_gate", True, True, "cuda", slack=33)
    check(x, w, b, r, dy, "silu_gate", rows)


@pytest.mark.gpu
def test_long_contraction_and_one_hot_group():
    x, w, b, r, dy = inputs([5, 3000, 0, 7], 512, 256, torch.bfloat16, "gelu", True, False, "cuda", slack=100)
    check(x, w, b, r, dy, "gelu", [5, 3000, 0, 7])
    x, w, b, r, dy = inputs([3], 256, 14336, torch.bfloat16, None, True, True, "cuda")
    check(x, w, b, r, dy, None, [3], dense=True)


@pytest.mark.gpu
def test_rows_behind_the_groups_and_other_groups_stay_apart():
    """NaN and infinities behind the last group reach nothing; those of one group stay in it."""
    from iris_testing_b200 import ops
    rows = [70, 33, 0, 100]
    x, w, b, r, dy = inputs(rows, 256, 128, torch.bfloat16, "silu_gate", True, True, "cuda", slack=60)
    clean = [t.clone() for t in (x, w, b, r, dy)]

    def grads(x, w, b, r, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = ops.linear(*leaves, activation="silu_gate", group_rows=torch.tensor(rows, dtype=torch.int32, device="cuda"))
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    want = grads(*clean)
    for t in (x, r, dy):
        t[203:] = float("nan")
        t[210] = float("inf")
    for a, b2 in zip(grads(x, w, b, r, dy), want):
        assert torch.equal(a, b2)
    for i in (0, 1, 4):
        assert not want[i][203:].any()
    x[80] = float("nan")             # a row of the second group
    dy[81] = float("inf")
    got = grads(x, w, b, r, dy)
    others = torch.tensor([0, 2, 3], device="cuda")
    for i in (2, 3):
        assert torch.equal(got[i][others], want[i][others])
        assert not torch.isfinite(got[i][1]).all()
    keep = torch.ones(263, dtype=torch.bool, device="cuda")
    keep[80:82] = False
    for i in (0, 1):
        assert torch.equal(got[i][keep], want[i][keep])


@pytest.mark.gpu
def test_too_many_rows_are_reported_and_nothing_is_written_out_of_place():
    from iris_testing_b200 import ops
    from iris_testing_b200._native import NativeError
    x, w, b, r, dy = inputs([10, 10], 256, 64, torch.bfloat16, None, False, False, "cuda")
    ops.check_default_status()
    for rows in ([10, 11], [2 ** 31 - 1, 2 ** 31 - 1]):
        leaves = [t.detach().requires_grad_() for t in (x, w)]
        y = ops.linear(*leaves, group_rows=torch.tensor(rows, dtype=torch.int32, device="cuda"))
        torch.autograd.grad(y, leaves, dy)
        with pytest.raises(NativeError, match="overflow"):
            ops.check_default_status()
    y = ops.linear(x, w, group_rows=torch.tensor([-5, 20], dtype=torch.int32, device="cuda"))      # a negative count is none
    within(y, reference(x, w, None, None, None, [0, 20], dy)[0], "y")


@pytest.mark.gpu
def test_empty_strided_shifted_and_leading_dimensions():
    from iris_testing_b200 import ops
    x, w, b, r, dy = inputs([24], 256, 64, torch.bfloat16, "gelu", True, True, "cuda")
    want = ops.linear(x, w[0], b[0], r, activation="gelu")
    assert torch.equal(ops.linear(x.view(2, 3, 4, 64), w[0], b[0], r.view(2, 3, 4, 256), activation="gelu").view(24, 256), want)
    wide = torch.cat((x, x), 1)[:, :64]
    shifted = torch.cat((x.new_zeros(3), x.reshape(-1)))[3:].view(24, 64)
    wt = w[0].t().contiguous().t()
    for xx in (wide, shifted):
        assert torch.equal(ops.linear(xx, wt, b[0], r, activation="gelu"), want)
    e = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    we = w[0].detach().requires_grad_()
    y = ops.linear(e, we, activation="silu")
    assert y.shape == (0, 256)
    ge, gw = torch.autograd.grad(y.sum(), [e, we])
    assert ge.shape == (0, 64) and not gw.any()
    # a gradient that is one number spread over the result
    xl = x.detach().requires_grad_()
    g1, = torch.autograd.grad(ops.linear(xl, w[0]).sum(), xl)
    g2, = torch.autograd.grad(ops.linear(xl, w[0]), xl, torch.ones(24, 256, device="cuda", dtype=torch.bfloat16))
    assert torch.equal(g1, g2)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu_gate", "gelu", None])
@pytest.mark.parametrize("grouped", [False, True])
def test_only_the_gradients_asked_for(grouped, act):
    from iris_testing_b200 import ops
    rows = [20, 0, 25] if grouped else [50]
    x, w, b, r, dy = inputs(rows, 256, 64, torch.bfloat16, act, True, True, "cuda", slack=5 if grouped else 0)
    gr = torch.tensor(rows, dtype=torch.int32, device="cuda") if grouped else None
    leaves = [t.detach().requires_grad_() for t in ((x, w, b, r) if grouped else (x, w[0], b[0], r))]
    full = torch.autograd.grad(ops.linear(*leaves, activation=act, group_rows=gr), leaves, dy)
    for i in range(4):
        args = [t if j == i else t.detach() for j, t in enumerate(leaves)]
        one, = torch.autograd.grad(ops.linear(*args, activation=act, group_rows=gr), leaves[i], dy)
        assert torch.equal(one, full[i]), i


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [[3, 9, 0, 20], [300, 170, 0, 500]])
def test_same_bits_twice_on_another_stream_and_in_two_graphs(rows):
    from iris_testing_b200 import ops
    x, w, b, r, dy = inputs(rows, 512, 256, torch.bfloat16, "silu_gate", True, True, "cuda", slack=11)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    gr = torch.tensor(rows, dtype=torch.int32, device="cuda")

    def step():
        y = ops.linear(*leaves, activation="silu_gate", group_rows=gr)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step())
    for a, b2 in zip(first, second):
        assert torch.equal(a, b2)
    with torch.no_grad():
        x.mul_(0.5)
        gr.copy_(torch.tensor(rows[::-1], dtype=torch.int32))       # the sizes are read on the device, at every replay
    graphs[0].replay()
    graphs[1].replay()
    want = step()
    for out in outs:
        for a, b2 in zip(out, want):
            assert torch.equal(a, b2)
    ops.check_default_status()


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    from iris_testing_b200 import ops
    x = torch.ones(6, 16, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(256, 16, device="cuda", dtype=torch.bfloat16)
    for bad in (lambda: ops.linear(x.float(), w.float()),
                lambda: ops.linear(x, w.half()),
                lambda: ops.linear(x, w.cpu()),
                lambda: ops.linear(x[:, :12], w[:, :12]),
                lambda: ops.linear(x, w[:252]),
                lambda: ops.linear(x, w, torch.ones(256, device="cuda")),
                lambda: ops.linear(x[:1].expand(2 ** 31 - 1000, 16), w),       # a view of one row
                lambda: ops.linear(x, torch.ones(129, 8, 16, device="cuda", dtype=torch.bfloat16),
                                   group_rows=torch.zeros(129, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("act,N", [("silu", 136), ("silu_gate", 256)])
def test_kept_pre_activations_have_11_bits(act, N, split, monkeypatch):
    """What the forward pass keeps for the backward one, in rows of very different sizes and next to an infinity and a NaN: off by
    half a step of 11 bits, or of the smallest normal number under the chunk's scale, 2^-24 2^-14 of its largest value's power of two."""
    mod = importlib.import_module("iris_testing_b200.ops.linear")
    monkeypatch.setattr(mod, "_splits", lambda *a: split)
    M, K = 160, N
    g = torch.Generator().manual_seed(3)
    size = torch.exp2(torch.randint(-100, 100, (M, 1), generator=g).float()) * torch.exp2(torch.randint(-8, 1, (1, K), generator=g).float())
    x = (torch.randn(M, K, generator=g) * size).to("cuda", torch.bfloat16)
    w = torch.eye(K).to("cuda", torch.bfloat16)                   # z is x + b, exact but for one fp32 rounding
    b = (torch.randn(N, generator=g) * 2.0 ** -9).to("cuda", torch.bfloat16)
    b[5], b[70] = float("inf"), float("nan")
    x[11] = 0
    x[12, 40:72] = 2.0 ** -126                                    # next to nothing, under a bias
    _, (z, e) = mod._forward(x, w, b, None, None, mod.ACTIVATIONS[act], True)
    want = x.double() + b.double()
    chunk = e.repeat_interleave(32, 1)[:, :N].double()
    got = z.double() * torch.exp2(chunk - 141)
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)) and torch.equal(torch.isnan(want), torch.isnan(got))
    tol = (2.0 ** -11 + 2.0 ** -23) * want.abs() + 2.0 ** -25 * torch.exp2(chunk - 141)
    assert bool(((got - want).abs() <= tol)[fine].all())
    assert bool((torch.exp2(chunk - 141) <= torch.maximum(want.abs()[fine].max(), want.new_tensor(2.0 ** -100)))[fine].all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS)
def test_saturated_activations(act, dtype):
    """Far from zero the slopes are 0, 1 or the other half's value; nothing overflows on the way.  At -60, the nearest, silu is
    60 e^-60 = 5.3e-25 off its limit and its slope 59 e^-60, twice that under an up half of 2: both below 2e-24."""
    from iris_testing_b200 import ops
    top = 3e38 if dtype == torch.bfloat16 else 6e4
    far = [v for v in (60.0, 3e4, 1e13, 1e15, 1e20, 1e30, 3e38) if v <= top]
    z = torch.tensor([s * v for v in far for s in (1, -1)], dtype=dtype, device="cuda")
    K = 128
    n = 2 * K if act == "silu_gate" else K
    w = torch.zeros(n, K, dtype=dtype, device="cuda")
    w[:K] = torch.eye(K)                     # each z reaches its own column; gated: up = 2 (through the bias)
    b = torch.zeros(n, dtype=dtype, device="cuda")
    if act == "silu_gate":
        b[K:] = 2.0
    x = torch.zeros(len(z), K, dtype=dtype, device="cuda")
    x[torch.arange(len(z)), torch.arange(len(z))] = z
    x.requires_grad_()
    w.requires_grad_()
    y = ops.linear(x, w, b, activation=act)
    dy = torch.zeros_like(y)
    i = torch.arange(len(z), device="cuda")
    dy[i, i] = 1.0
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    up = 2.0 if act == "silu_gate" else 1.0
    slope = torch.ones_like(z) if act is None else (z > 0).to(dtype)
    if act != "silu_gate":                   # twice the largest z is infinite
        assert bool(((y.detach()[i, i].double() - torch.where(slope > 0, z, torch.zeros_like(z)).double()).abs() <= 2e-24).all())
    assert bool(((dx[i, i].double() - up * slope.double()).abs() <= 2e-24).all()), dx[i, i]
    off = dx.clone()
    off[i, i] = 0
    assert not off.any() and torch.isfinite(dx).all()
