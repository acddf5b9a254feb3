"""``pre_norm`` and ``post_norm`` against the formulas in 64 bits, forward and backward.

Tolerance: the formulas are also run with every value replaced by its magnitude and every difference by a sum.  fp32
arithmetic is off by at most c 2^-24 of that, where c counts the roundings on the longest path: up to 64 sequential additions
of a thread, 10 of the tree, two for the inverse root and about 50 products and sums, in all below 128; a sum over
rows adds T / parts + parts / 8 + 8, below 128 at these sizes.  The result's own rounding adds half a step."""
import pytest
import torch

C_ROW, C_COL = 128, 256
EPS = 1e-5
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(t, scale, norm, mag=False):
    """(outputs, gradients) in fp64 of the dict of tensors ``t``; with ``mag`` the bound's magnitudes."""
    v = {n: x.double().abs() if mag else x.double() for n, x in t.items()}
    r = {n: x.double() for n, x in t.items()}
    sign = 1.0 if mag else -1.0

    def mean(x):
        return x.mean(-1, keepdim=True)
    H = r["y"].shape[-1]
    yr = r["y"]
    r1 = torch.rsqrt(mean(yr * yr) + EPS) if norm else torch.ones_like(yr[..., :1])
    w = v.get("weight", torch.ones(H, dtype=torch.float64, device=yr.device))
    yh = v["y"] * r1
    u = yh * w
    if "residual" not in t:
        dn = v["dn"]
        q = dn * w
        return {"h": u}, {"y": r1 * (q + sign * yh * mean(q * yh)), "weight": (dn * yh).reshape(-1, H).sum(0)}
    gate = v.get("gate", torch.ones(1, dtype=torch.float64, device=yr.device))
    s = abs(scale) if mag else scale
    h = s * v["residual"] + gate * u
    rw, rg = r.get("weight", torch.ones_like(w)), r.get("gate", torch.ones_like(gate))
    hr = scale * r["residual"] + rg * (yr * r1 * rw)
    outs, g = {"h": h}, {}
    gh = v.get("dh", torch.zeros_like(h))
    if "next_weight" in t:
        r2 = torch.rsqrt(mean(hr * hr) + EPS)
        hh = h * r2
        outs["n"] = hh * v["next_weight"]
        if "dn" in t:
            k = v["dn"] * v["next_weight"]
            gh = gh + r2 * (k + sign * hh * mean(k * hh))
            g["next_weight"] = (v["dn"] * hh).reshape(-1, H).sum(0)
        else:
            g["next_weight"] = torch.zeros_like(w)
    g["residual"] = s * gh
    p = gh * u
    if "gate" in t:
        shape = t["gate"].shape
        g["gate"] = p if shape == p.shape else p.reshape(-1, H).sum(0) if shape == (H,) else p.sum(-1, keepdim=True)
    du = gate * gh
    g["weight"] = (du * yh).reshape(-1, H).sum(0)
    q = du * w
    g["y"] = r1 * (q + sign * yh * mean(q * yh)) if norm else du
    return outs, g


def close(got, ref, mag, c, what):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + c * 2.0 ** -24 * mag + (2.0 ** -25 if got.dtype == torch.float16 else 1e-38)
    off = (got.double() - ref).abs() - tol
    assert bool((off <= 0).all()), (what, float(off.max()), float((got.double() - ref).abs().max()))


def make(T, H, dtype, kind, dev, seed=0, lead=None):
    g = torch.Generator().manual_seed(seed + 17 * T + H)
    shape = (T, H) if lead is None else lead + (H,)

    def rnd(s, dt=dtype, mean=0.0, std=1.0):
        return (torch.randn(s, generator=g) * std + mean).to(dev, dt)
    t = {"y": rnd(shape, std=1.5)}
    wt = torch.float32 if "w32" in kind else dtype
    if "nonorm" not in kind:
        t["weight"] = rnd((H,), wt, 1.0, 0.2)
    if "pre" not in kind:
        t["residual"] = rnd(shape, std=2.0)
        if "channel" in kind:
            t["gate"] = rnd((H,), wt, 0.5, 0.3)
        elif "row" in kind:
            t["gate"] = rnd(shape[:-1] + (1,), wt, 0.5, 0.3)
        elif "full" in kind:
            t["gate"] = rnd(shape, dtype, 0.5, 0.3)
        if "next" in kind:
            t["next_weight"] = rnd((H,), wt, 1.0, 0.2)
        t["dh"] = rnd(shape)
    if "next" in kind or "pre" in kind:
        t["dn"] = rnd(shape)
    return t


def call(t, scale, norm):
    from iris_testing_b200 import ops
    if "residual" not in t:
        return (ops.pre_norm(t["y"], t.get("weight"), eps=EPS),)
    out = ops.post_norm(t["y"], t["residual"], t.get("weight"), t.get("gate"), norm=norm, residual_scale=scale,
                        next_weight=t.get("next_weight"), eps=EPS)
    return out if isinstance(out, tuple) else (out,)


def check(t, scale, kind):
    norm = "nonorm" not in kind
    leaves = [n for n in ("y", "residual", "weight", "gate", "next_weight") if n in t]
    for n in leaves:
        t[n].requires_grad_()
    outs = call(t, scale, norm)
    with torch.no_grad():
        for a, b in zip(outs, call(t, scale, norm)):      # the form without saved statistics
            assert torch.equal(a, b)
    up = [t["dn"]] if "residual" not in t else [t.get("dh"), t.get("dn")][:len(outs)]
    pairs = [(o, d) for o, d in zip(outs, up) if d is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], [t[n] for n in leaves], [d for _, d in pairs])
    again = torch.autograd.grad(call(t, scale, norm)[0].float().sum(), [t["y"]])[0]
    assert torch.isfinite(again).all()
    plain = {n: x.detach() for n, x in t.items()}
    ro, rg = reference(plain, scale, norm)
    mo, mg = reference(plain, scale, norm, mag=True)
    for o, n in zip(outs, ("h", "n")):
        assert o.dtype == t["y"].dtype
        close(o.detach(), ro[n], mo[n], C_ROW, n)
    for g, n in zip(grads, leaves):
        assert g.dtype == t[n].dtype
        rows = t[n].dim() == 1 and n in ("weight", "next_weight", "gate")
        close(g, rg[n], mg[n], C_COL if rows else C_ROW, "d" + n)


KINDS = ["pre", "pre w32", "norm", "next", "nonorm next", "nonorm", "channel next w32", "row", "full next", "row next w32"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,H", [(1, 1), (3, 7), (2, 64)])
def test_formulas_on_cpu(T, H, kind):
    check(make(T, H, torch.float32, kind, "cpu"), 0.5, kind)


def test_reference_gradients_against_differences():
    """The formulas that everything here is held to, against central differences in fp64 (h^2 and 1e-16 / h errors)."""
    kind = "channel next"
    t = {n: x.double() for n, x in make(2, 5, torch.float32, kind, "cpu").items()}
    _, g = reference(t, 0.5, True)
    step = 1e-5
    for n in ("y", "residual", "weight", "gate", "next_weight"):
        flat = g[n].reshape(-1)
        for i in range(flat.numel()):
            total = []
            for d in (step, -step):
                m = {k: x.clone() for k, x in t.items()}
                m[n].view(-1)[i] += d
                o, _ = reference(m, 0.5, True)
                total.append(float((o["h"] * t["dh"]).sum() + (o["n"] * t["dn"]).sum()))
            assert abs((total[0] - total[1]) / (2 * step) - float(flat[i])) < 1e-6 * (1 + abs(float(flat[i])))


def test_refusals():
    from iris_testing_b200 import ops
    y, w = torch.ones(4, 8), torch.ones(8)
    for bad in (lambda: ops.pre_norm(y, torch.ones(7)),
                lambda: ops.pre_norm(torch.tensor(1.0)),
                lambda: ops.post_norm(y, torch.ones(4, 7)),
                lambda: ops.post_norm(y, None),
                lambda: ops.post_norm(y, y, w, norm=False),
                lambda: ops.post_norm(y, y, w, torch.ones(4)),
                lambda: ops.post_norm(y, y, w, next_weight=torch.ones(4, 8))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,H", [(1, 1), (1, 4096), (3, 7), (5, 769), (33, 256), (65, 264), (200, 1408), (9, 6144), (700, 520)])
def test_norms(T, H, kind, dtype):
    check(make(T, H, dtype, kind, "cuda"), 0.5, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H", [(3, 16384), (2, 16383), (1000, 8), (2000, 4096)])
def test_norms_at_the_ends_of_the_range(T, H, dtype):
    check(make(T, H, dtype, "channel next w32", "cuda"), -1.5, "channel next w32")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["full", "full next", "row", "channel next w32"])
@pytest.mark.parametrize("T,H", [(1301, 4104), (1000, 6144), (500, 8184), (400, 8200), (700, 4099)])
def test_several_wide_rows_per_block(T, H, kind, dtype):
    check(make(T, H, dtype, kind, "cuda"), 0.5, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["pre", "full next", "row next"])
@pytest.mark.parametrize("how", ["strided", "shifted", "expanded", "3d"])
def test_layouts(how, kind):
    t = make(24, 512, torch.bfloat16, kind, "cuda", lead=(2, 3, 4) if how == "3d" else None)

    def lay(x):
        if x.dim() < 2 or x.shape[-1] == 1:
            return x
        if how == "strided":
            return torch.cat((x, torch.full_like(x, float("nan"))), -1)[..., :512]
        if how == "shifted":                                    # rows that do not start on 16 bytes
            return torch.cat((torch.full_like(x[..., :3], float("nan")), x), -1)[..., 3:]
        if how == "expanded":
            return x[:1].expand(x.shape)
        return x.transpose(0, 1).contiguous().transpose(0, 1)   # no view as rows
    t = {n: lay(x).detach() for n, x in t.items()}
    check(t, 1.0, kind)


@pytest.mark.gpu
def test_zero_rows_zero_inputs_and_missing_gradients():
    from iris_testing_b200 import ops
    dev = "cuda"
    w = torch.ones(64, device=dev, requires_grad=True)
    y = torch.empty(0, 64, device=dev, requires_grad=True)
    h, n = ops.post_norm(y, y, w, next_weight=w)
    assert h.shape == n.shape == (0, 64)
    g = torch.autograd.grad(h.sum() + n.sum(), [y, w])
    assert g[0].shape == (0, 64) and not g[1].any()
    z = torch.zeros(3, 64, device=dev, requires_grad=True)     # a row of zeros: 1 / sqrt(eps) times nothing
    assert not ops.pre_norm(z, w).any()
    h, n = ops.post_norm(z, z, w, next_weight=w)
    gz, gw = torch.autograd.grad(n.sum(), [z, w])
    assert torch.isfinite(gz).all() and torch.isfinite(gw).all()
    # only the first output is used: the next weight gets zeros
    x = torch.randn(5, 64, device=dev, requires_grad=True)
    w2 = torch.ones(64, device=dev, requires_grad=True)
    h, n = ops.post_norm(x, x, w, next_weight=w2)
    assert not torch.autograd.grad(h.sum(), [w2])[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["channel next w32", "row next", "full next", "nonorm channel", "pre"])
@pytest.mark.parametrize("H", [128, 1000, 2049])
def test_only_the_gradients_asked_for(H, kind):
    t = make(37, H, torch.bfloat16, kind, "cuda")
    names = [n for n in ("y", "residual", "weight", "gate", "next_weight") if n in t]
    up = [t["dn"]] if "residual" not in t else [t.get("dh"), t.get("dn")]

    def grads(wanted):
        m = {n: x.detach().requires_grad_(n in wanted) for n, x in t.items()}
        outs = call(m, 0.5, "nonorm" not in kind)
        return torch.autograd.grad(outs, [m[n] for n in wanted], [d for d in up if d is not None])
    full = dict(zip(names, grads(names)))
    for n in names:
        assert torch.equal(grads([n])[0], full[n]), n


@pytest.mark.gpu
def test_infinities_stay_in_their_row():
    from iris_testing_b200 import ops
    y = torch.randn(6, 256, device="cuda")
    r = torch.randn(6, 256, device="cuda")
    w = torch.ones(256, device="cuda")
    want = ops.post_norm(y, r, w, next_weight=w)
    y[2, 5], y[4, 7] = float("inf"), float("nan")
    got = ops.post_norm(y, r, w, next_weight=w)
    for a, b in zip(got, want):
        assert torch.equal(a[[0, 1, 3, 5]], b[[0, 1, 3, 5]])
        assert torch.isnan(a[4]).all()


@pytest.mark.gpu
def test_same_bits_twice_and_on_another_stream_and_in_a_graph():
    from iris_testing_b200 import ops
    t = make(777, 1408, torch.bfloat16, "channel next w32", "cuda")
    leaves = [t[n].requires_grad_() for n in ("y", "residual", "weight", "gate", "next_weight")]

    def step():
        outs = ops.post_norm(t["y"], t["residual"], t["weight"], t["gate"], next_weight=t["next_weight"])
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, [t["dh"], t["dn"]]))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    with torch.no_grad():
        t["y"].mul_(2.0)
    graph.replay()
    fourth = step()
    for a, b in zip(first, second):
        assert torch.equal(a, b)
    for a, b in zip(third, fourth):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    from iris_testing_b200 import ops
    y = torch.ones(4, 8, device="cuda")
    for bad in (lambda: ops.pre_norm(y.double()),
                lambda: ops.pre_norm(y, torch.ones(8)),                                     # weight on the CPU
                lambda: ops.pre_norm(y, torch.ones(8, device="cuda", dtype=torch.float16)),
                lambda: ops.post_norm(y, y.half()),
                lambda: ops.post_norm(y.half(), y.half(), gate=y),                          # full gate of another type
                lambda: ops.pre_norm(torch.ones(1, 16385, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
