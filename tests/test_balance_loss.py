"""``balance_loss`` against its definition in 64 bits, with the gradient by differentiating that definition.

Tolerance: a token's softmax in fp32 is off by at most about 16 roundings (two ulp of expf, the argument's difference,
additions over the lanes, division) times 2^-24 relative; its logarithm adds 4.  A column sum adds up to 512 terms in a
thread and 64 records, so 600 roundings in all, and the few products of the loss are below that: 1024 x 2^-24 of the terms'
magnitudes, plus half a step of the gradient's type.  The argument logit - max is rounded at the logits' magnitude, which
is relative to p as |logit| 2^-24; |logit| < 32 here, within the same bound."""
import pytest
import torch

ULPS = 1024 * 2.0 ** -24
F64 = torch.float64


def reference(logits, idx, coef, z, rows, mask):
    """(loss, counts, gradient, the gradient's magnitude) in fp64, one sequence after another."""
    T, E = logits.shape
    k = idx.shape[1]
    lg = logits.double().cpu()
    low = torch.finfo(logits.dtype).min
    part = torch.tensor([bool(not torch.isnan(r).any() and low < r.max() < float("inf")) for r in lg], dtype=torch.bool)
    if mask is not None:
        part &= mask.cpu()
    lengths = [T] if rows is None else rows.tolist()
    grad, mag, terms, zs, counts, start, per = torch.zeros(T, E, dtype=F64), torch.zeros(T, E, dtype=F64), [], [], [], 0, []
    for n in lengths:
        t = [i for i in range(start, min(T, start + max(n, 0))) if part[i]]
        start += max(n, 0)
        c = torch.zeros(E, dtype=F64)
        for e in idx[t].reshape(-1).tolist():
            if 0 <= e < E:
                c[e] += 1
        counts.append(c)
        per.append((t, c))
        if t:
            p = torch.softmax(lg[t], 1)
            terms.append(E * (c / (k * len(t)) * p.mean(0)).sum())
            zs.append(torch.logsumexp(lg[t], 1) ** 2)
    total = sum(len(t) for t, _ in per)
    loss = (coef * torch.stack(terms).mean() + z * torch.cat(zs).mean()) if terms else torch.zeros((), dtype=F64)
    for t, c in per:
        if t:
            p = torch.softmax(lg[t], 1)
            a = coef / len(terms) * E * c / (k * len(t) ** 2)
            lse = torch.logsumexp(lg[t], 1)
            w = 2 * z / total * lse
            dot = (p * a).sum(1, keepdim=True)
            grad[t] = p * (a - dot) + w[:, None] * p
            mag[t] = p * (a + dot) + w.abs()[:, None] * p
    return loss, torch.stack(counts).to(torch.int32), grad, mag


def inputs(T, E, k, dtype, dev, seed=0, S=None, mask=False, tail=0):
    g = torch.Generator().manual_seed(seed + T + 31 * E)
    lg = (torch.randn(T, E, generator=g) * 2).to(dtype)
    idx = torch.rand(T, E, generator=g).topk(k, dim=1).indices.to(torch.int32)
    rows = None
    if S is not None:
        cuts = torch.sort(torch.randint(0, T - tail + 1, (S - 1,), generator=g)).values
        rows = torch.diff(torch.cat((torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([T - tail])))).to(torch.int32)
    m = torch.rand(T, generator=g) < 0.8 if mask else None
    return [x if x is None else x.to(dev) for x in (lg, idx, rows, m)]


def check(lg, idx, rows, mask, coef=0.01, z=1e-3, scale=1.0):
    from iris_testing_b200 import ops
    lg = lg.detach().requires_grad_()
    loss, counts = ops.balance_loss(lg, idx, balance_coef=coef, z_coef=z, seq_rows=rows, token_mask=mask)
    with torch.no_grad():
        l2, c2 = ops.balance_loss(lg, idx, balance_coef=coef, z_coef=z, seq_rows=rows, token_mask=mask)
    assert torch.equal(loss, l2) and torch.equal(counts, c2)
    counts_got = counts.clone()
    counts.zero_()                                           # the caller's to change
    grad, = torch.autograd.grad(loss * scale, lg)
    rl, rc, rg, rm = reference(lg.detach(), idx.cpu(), coef, z, rows if rows is None else rows.cpu(), mask)
    assert loss.dtype == torch.float32 and counts.dtype == torch.int32 and grad.dtype == lg.dtype
    assert torch.equal(counts_got.cpu(), rc if rows is not None else rc[0])
    assert abs(float(loss.detach()) - float(rl)) <= ULPS * abs(float(rl))
    tiny = 2.0 ** -25 if grad.dtype == torch.float16 else 1e-38
    tol = scale * (torch.finfo(grad.dtype).eps / 2 * rg.abs() + ULPS * rm) + tiny
    off = (grad.double().cpu() - scale * rg).abs() - tol
    assert bool((off <= 0).all()), float(off.max())
    assert not grad.cpu()[rm.sum(1) == 0].any()


@pytest.mark.parametrize("S,mask,tail", [(None, False, 0), (None, True, 0), (5, False, 0), (7, True, 9)])
def test_definition_on_cpu(S, mask, tail):
    check(*inputs(60, 8, 2, torch.float32, "cpu", S=S, mask=mask, tail=tail))


def test_reference_gradient_against_differences():
    lg, idx, rows, mask = inputs(9, 4, 2, F64, "cpu", S=3, mask=True, tail=1)
    _, _, grad, _ = reference(lg, idx, 0.5, 0.1, rows, mask)
    for i in range(9):
        for j in range(4):
            step = []
            for d in (1e-5, -1e-5):
                m = lg.clone()
                m[i, j] += d
                step.append(float(reference(m, idx, 0.5, 0.1, rows, mask)[0]))
            assert abs((step[0] - step[1]) / 2e-5 - float(grad[i, j])) < 1e-8


def test_refusals():
    from iris_testing_b200 import ops
    lg, idx = torch.randn(6, 4), torch.zeros(6, 2, dtype=torch.int32)
    for bad in (lambda: ops.balance_loss(lg[0], idx),
                lambda: ops.balance_loss(lg, idx[:5]),
                lambda: ops.balance_loss(lg, idx.long()),
                lambda: ops.balance_loss(lg, idx, seq_rows=torch.tensor([6])),
                lambda: ops.balance_loss(lg, idx, seq_rows=torch.tensor([[6]], dtype=torch.int32)),
                lambda: ops.balance_loss(lg, idx, token_mask=torch.ones(6)),
                lambda: ops.balance_loss(lg, idx, token_mask=torch.ones(5, dtype=torch.bool))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,S,mask,tail", [
    (1, 1, 1, None, False, 0), (1, 8, 2, None, False, 0), (64, 8, 2, None, False, 0), (333, 3, 1, 4, True, 10),
    (1000, 16, 4, 40, False, 0), (700, 32, 4, 3, True, 50), (2111, 64, 8, 33, True, 100), (900, 65, 8, None, True, 0),
    (600, 128, 8, 500, False, 17), (129, 200, 8, 5, False, 1), (50, 257, 3, 3, True, 0), (20, 1024, 8, 2, False, 0)])
def test_definition(T, E, k, S, mask, tail, dtype):
    check(*inputs(T, E, k, dtype, "cuda", S=S, mask=mask, tail=tail), scale=128.0)


@pytest.mark.gpu
def test_many_tokens_and_more_sequences_than_a_block_scans_at_once():
    check(*inputs(6000, 64, 8, torch.float32, "cuda", S=1500, mask=True, tail=300))
    check(*inputs(20000, 8, 2, torch.float32, "cuda", S=3, tail=5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_masked_experts_and_tokens_without_any(dtype):
    lg, idx, rows, mask = inputs(200, 40, 4, dtype, "cuda", S=6)
    low = torch.finfo(dtype).min
    lg[:, 7] = -float("inf")
    lg[:, 9] = low
    lg[3] = -float("inf")
    lg[4] = low
    lg[5, 2] = float("nan")
    lg[6, 39] = float("inf")
    idx[3:7] = -1                       # the router's answer for such tokens
    idx[20, 1] = 40
    check(lg, idx, rows, mask, scale=128.0)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_next_to_the_largest(dtype, dev):
    """Probabilities of exactly 0, 1 and 1 / 2: no z loss, whose square overflows."""
    g = torch.Generator().manual_seed(0)
    lg = torch.randn(12, 8, generator=g).to(dtype)
    lg[2, 3], lg[2, 4] = 3e38, -3e38
    lg[5] = -3e38
    lg[5, 1] = lg[5, 6] = -2.9e38
    idx = torch.rand(12, 8, generator=g).topk(2, dim=1).indices.to(torch.int32)
    check(lg.to(dev), idx.to(dev), None, None, z=0.0)


@pytest.mark.gpu
def test_nothing_left():
    from iris_testing_b200 import ops
    lg = torch.randn(30, 8, device="cuda", requires_grad=True)
    idx = torch.zeros(30, 2, dtype=torch.int32, device="cuda")
    for rows, mask in ((None, torch.zeros(30, dtype=torch.bool, device="cuda")),
                       (torch.zeros(4, dtype=torch.int32, device="cuda"), None),
                       (torch.empty(0, dtype=torch.int32, device="cuda"), None)):
        loss, counts = ops.balance_loss(lg, idx, z_coef=1.0, seq_rows=rows, token_mask=mask)
        assert float(loss.detach()) == 0.0 and not counts.any()
        assert counts.shape == ((8,) if rows is None else (rows.numel(), 8))
        assert not torch.autograd.grad(loss, lg)[0].any()
    empty = torch.empty(0, 8, device="cuda", requires_grad=True)
    loss, counts = ops.balance_loss(empty, idx[:0])
    assert float(loss.detach()) == 0.0 and torch.autograd.grad(loss, empty)[0].shape == (0, 8)
    # an infinite loss gradient stays out of the rows that take no part
    mask = torch.arange(30, device="cuda") % 2 == 0
    loss, _ = ops.balance_loss(lg, idx, token_mask=mask)
    assert not torch.autograd.grad(loss, lg, torch.tensor(float("inf"), device="cuda"))[0][~mask].any()


@pytest.mark.gpu
def test_lengths_beyond_the_tokens_are_cut_off_and_reported():
    from iris_testing_b200 import ops
    from iris_testing_b200._native import NativeError
    lg, idx, _, _ = inputs(100, 8, 2, torch.float32, "cuda")
    ops.check_default_status()
    loss, counts = ops.balance_loss(lg, idx, seq_rows=torch.tensor([60, -3, 50, 7], dtype=torch.int32, device="cuda"))
    with pytest.raises(NativeError, match="overflow"):
        ops.check_default_status()
    want, wc = ops.balance_loss(lg, idx, seq_rows=torch.tensor([60, 0, 40, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(loss, want) and torch.equal(counts, wc)


@pytest.mark.gpu
def test_strided_logits_graph_and_other_stream():
    from iris_testing_b200 import ops
    lg, idx, rows, mask = inputs(3000, 64, 8, torch.bfloat16, "cuda", S=11, mask=True, tail=40)
    wide = torch.full((3000, 80), float("nan"), device="cuda", dtype=torch.bfloat16)
    wide[:, 8:72] = lg
    check(wide[:, 8:72], idx, rows, mask)
    lg = lg.requires_grad_()

    def step():
        loss, counts = ops.balance_loss(lg, idx, seq_rows=rows, token_mask=mask, z_coef=1e-3)
        return loss.detach(), counts, torch.autograd.grad(loss, lg)[0]
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    for a, b in zip(first, second):
        assert torch.equal(a, b)
    with torch.no_grad():
        lg.mul_(0.5)
    graph.replay()
    for a, b in zip(third, step()):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_counts_agree_with_the_plan():
    from iris_testing_b200 import ops
    from iris_testing_b200.utils import gen_local_tokens, gen_router
    x = gen_local_tokens(1, 500, 256, torch.bfloat16, torch.device("cuda"), 0, 0, "normal")
    idx, _, logits = ops.router_topk(x, gen_router(256, 16, torch.bfloat16, torch.device("cuda"), 0, std=None), 4, return_logits=True)
    _, counts = ops.balance_loss(logits, idx)
    assert torch.equal(counts, ops.make_plan(idx, 16).counts)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    from iris_testing_b200 import ops
    lg, idx = torch.randn(6, 4, device="cuda"), torch.zeros(6, 2, dtype=torch.int32, device="cuda")
    for bad in (lambda: ops.balance_loss(lg.double(), idx),
                lambda: ops.balance_loss(lg, idx.cpu()),
                lambda: ops.balance_loss(lg, idx, seq_rows=torch.tensor([6], dtype=torch.int32)),
                lambda: ops.balance_loss(lg[:1].expand(2 ** 31 - 1000, 4), idx[:1].expand(2 ** 31 - 1000, 2)),
                lambda: ops.balance_loss(torch.randn(2, 1025, device="cuda"), idx[:2])):
        with pytest.raises(ValueError):
            bad()
