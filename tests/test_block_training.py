"""The norms, the balance loss and ``linear`` together, as one training step of an MoE block uses them: norm, router with its
auxiliary loss, routed experts, a shared expert that adds to them, gated residual and the next block's norm.

The same step is run in fp64 with the routing that the ops chose (every op takes plain PyTorch on fp64 CPU tensors; their
GPU forms are held to their formulas one by one elsewhere).  Tolerance, on the norm of each result: about twelve tensors on
the way are rounded to bf16, each by at most half a step, 2^-8 of its norm, and every stage passes a relative error on with a factor of
about one (norms take scale out, the products average), so 12 x 2^-8 = 0.047."""
import pytest
import torch

T, D, F, E, K = 300, 256, 256, 8, 2
NAMES = ["x", "router", "w13", "w2", "shared13", "shared2", "pre", "post", "gate", "nxt"]


def parameters(dtype, dev):
    g = torch.Generator().manual_seed(0)

    def rnd(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g) * std + mean).to(torch.bfloat16).to(dev, dtype)
    return {"x": rnd(T, D), "router": rnd(D, E, std=D ** -0.5), "w13": rnd(E, 2 * F, D, std=D ** -0.5),
            "w2": rnd(E, D, F, std=F ** -0.5), "shared13": rnd(2 * F, D, std=D ** -0.5), "shared2": rnd(D, F, std=F ** -0.5),
            "pre": rnd(D, std=0.1, mean=1.0), "post": rnd(D, std=0.1, mean=1.0), "gate": rnd(D, std=0.2, mean=0.5),
            "nxt": rnd(D, std=0.1, mean=1.0), "dh": rnd(T, D), "dn": rnd(T, D)}


def block(p, idx=None):
    """(h, n, loss, counts, idx): one block; ``idx`` fixes the routing."""
    from iris_testing_b200 import ops
    n = ops.pre_norm(p["x"], p["pre"])
    wide = torch.float64 if n.dtype == torch.float64 else torch.float32
    logits = n.to(wide) @ p["router"].to(wide)
    if idx is None:
        idx = torch.topk(logits, K, dim=1).indices.to(torch.int32)
    loss, counts = ops.balance_loss(logits, idx, z_coef=1e-3)
    weight = torch.softmax(logits, 1).gather(1, idx.long())
    order = torch.argsort(idx.reshape(-1), stable=True)               # rows of an expert one after another
    packed = n[order // K]
    hidden = ops.linear(packed, p["w13"], activation="silu_gate", group_rows=counts)
    out = ops.linear(hidden, p["w2"], group_rows=counts)
    scaled = out.to(wide) * weight.reshape(-1)[order].unsqueeze(1)
    routed = torch.zeros(T, D, dtype=wide, device=n.device).index_add(0, order // K, scaled).to(n.dtype)
    shared = ops.linear(n, p["shared13"], activation="silu_gate")
    y = ops.linear(shared, p["shared2"], residual=routed)
    h, nxt = ops.post_norm(y, p["x"], p["post"], p["gate"], residual_scale=0.5, next_weight=p["nxt"])
    return h, nxt, loss, counts, idx


def step(p, idx=None):
    h, n, loss, counts, idx = block(p, idx)
    grads = torch.autograd.grad([h, n, loss], [p[k] for k in NAMES], [p["dh"], p["dn"], torch.ones_like(loss)])
    return [h.detach(), n.detach(), loss.detach()] + list(grads), counts, idx


def leaves(p):
    for k in NAMES:
        p[k].requires_grad_()
    return p


def test_block_on_cpu_has_gradients_of_every_parameter():
    out, counts, _ = step(leaves(parameters(torch.float32, "cpu")))
    assert all(torch.isfinite(t).all() and t.abs().max() > 0 for t in out)
    assert int(counts.sum()) == T * K


@pytest.mark.gpu
def test_block_against_64_bits():
    from iris_testing_b200 import ops
    got, counts, idx = step(leaves(parameters(torch.bfloat16, "cuda")))
    want, wc, _ = step(leaves(parameters(torch.float64, "cpu")), idx.cpu())
    assert torch.equal(counts.cpu(), wc)
    for name, a, b in zip(["h", "n", "loss"] + NAMES, got, want):
        assert a.shape == b.shape
        rel = float((a.double().cpu() - b).norm() / b.norm())
        assert rel <= 12 * 2.0 ** -8, (name, rel)
    ops.check_default_status()


@pytest.mark.gpu
def test_block_step_replays_from_a_graph_with_new_inputs():
    from iris_testing_b200 import ops
    p = leaves(parameters(torch.bfloat16, "cuda"))
    idx = step(p)[2]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, counts, _ = step(p, idx)
    with torch.no_grad():
        p["x"].mul_(-1.0)
        idx.copy_((idx + 1) % E)                   # other group sizes
    graph.replay()
    want, wc, _ = step(p, idx)
    assert torch.equal(counts, wc)
    for name, a, b in zip(["h", "n", "loss"] + NAMES, out, want):
        # index_add and the products' row order leave nothing to chance but the additions of a token's two rows
        assert float((a.double() - b.double()).norm()) <= 2.0 ** -8 * float(b.double().norm()), name
    ops.check_default_status()


@pytest.mark.gpu
def test_first_call_under_capture_is_refused(monkeypatch):
    """The device's status word cannot be made inside a graph."""
    import importlib
    common = importlib.import_module("iris_testing_b200.ops._common")
    from iris_testing_b200 import ops
    x, w = torch.ones(4, 64, device="cuda", dtype=torch.bfloat16), torch.ones(64, 64, device="cuda", dtype=torch.bfloat16)
    ops.linear(x, w)
    torch.cuda.synchronize()
    monkeypatch.setattr(common, "_DEFAULT_STATUS", {})
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="under graph capture"):
        with torch.cuda.graph(graph):
            ops.linear(x, w)
