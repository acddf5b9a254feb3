"""The block of README's section "Around the experts", run as it is printed: packed sequences with padding and a tail, every
parameter trained, against a plain computation token by token in fp64 with the routing that the example chose.

Tolerance, on the norm of each result.  bf16: as for one block's training step, about twelve tensors on the way are rounded, each by at
most half a step, 12 x 2^-8.  fp64 on the CPU: only the logits are fp32, sums of 256 products of magnitudes that add up to less than 16
here, off by at most 258 x 16 x 2^-24 = 2.5e-4; a softmax weight by twice that, everything behind it in proportion, gradients (which
hold a weight and its slope) by twice that again: 1e-3."""
import re
from pathlib import Path

import pytest
import torch

T, D, F, E, K = 90, 256, 128, 8, 2
PARAMETERS = ["x", "w_pre", "router", "w13", "w2", "s13", "s2", "w_post", "gate", "w_next"]


def example() -> str:
    text = (Path(__file__).resolve().parents[1] / "README.md").read_text()
    section = text.split("## Around the experts", 1)[1].split("\n## ", 1)[0]
    return re.search(r"```python\n(.*?)```", section, re.S).group(1)


def names(dtype, dev):
    g = torch.Generator().manual_seed(0)

    def rnd(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g) * std + mean).to(torch.bfloat16).to(dev, dtype)
    mask = torch.rand(T, generator=g) < 0.8
    mask[:3] = False                                   # padding in front: the first rows of the batch belong to no expert
    return {"x": rnd(T, D), "w_pre": rnd(D, std=0.1, mean=1.0), "router": rnd(D, E, std=D ** -0.5),
            "w13": rnd(E, 2 * F, D, std=D ** -0.5), "w2": rnd(E, D, F, std=F ** -0.5), "s13": rnd(2 * F, D, std=D ** -0.5),
            "s2": rnd(D, F, std=F ** -0.5), "w_post": rnd(D, std=0.1, mean=1.0), "gate": rnd(D, std=0.2, mean=0.5),
            "w_next": rnd(D, std=0.1, mean=1.0), "k": K, "E": E, "mask": mask.to(dev),
            "lengths": torch.tensor([30, 0, 41, 12], dtype=torch.int32, device=dev)}      # 7 tokens behind the last


def plain(v, idx, mask):
    """(h, n, balance loss) in fp64; experts one token at a time."""
    def rms(t, w):
        return t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6) * w

    def mlp(t, w13, w2):
        z = t @ w13.t()
        return (torch.nn.functional.silu(z[..., :F]) * z[..., F:]) @ w2.t()       # F = 128: one block of gate, one of up rows
    n = rms(v["x"], v["w_pre"])
    logits = n @ v["router"]
    p = torch.softmax(logits, 1)
    routed = []
    for t in range(T):
        own = torch.zeros(D, dtype=torch.float64)
        for e in idx[t].tolist() if mask[t] else []:
            own = own + p[t, e] * mlp(n[t], v["w13"][e], v["w2"][e])
        routed.append(own)
    y = torch.stack(routed) + mlp(n, v["s13"], v["s2"])
    h = 0.5 * v["x"] + v["gate"] * rms(y, v["w_post"])
    terms, taken, start = [], [], 0
    for length in (30, 0, 41, 12):
        t = [i for i in range(start, start + length) if mask[i]]
        start += length
        if t:
            share = torch.bincount(idx[t].reshape(-1).long(), minlength=E).double() / (K * len(t))
            terms.append(E * (share * p[t].mean(0)).sum())
            taken += t
    loss = 0.01 * torch.stack(terms).mean() + 1e-3 * torch.logsumexp(logits[taken], 1).pow(2).mean()
    return h, rms(h, v["w_next"]), loss


def run(dtype, dev, tol):
    v = names(dtype, dev)
    for name in PARAMETERS:
        v[name].requires_grad_()
    g = torch.Generator().manual_seed(1)
    up = [torch.randn(T, D, generator=g).to(dev, dtype) for _ in range(2)]
    exec(example(), v)
    results = [v["h"], v["n"], v["loss"]]
    assert v["plan"].counts.sum() == int(v["mask"].sum()) * K       # a group per expert, with every copy that is packed
    got = [t.detach() for t in results] + list(
        torch.autograd.grad(results, [v[name] for name in PARAMETERS], up + [torch.ones_like(v["loss"])]))
    w = {name: v[name].detach().double().cpu().requires_grad_() for name in PARAMETERS}
    idx, mask = v["idx"].cpu(), v["mask"].cpu()
    want = plain(w, idx, mask)
    want = [t.detach() for t in want] + list(
        torch.autograd.grad(want, [w[name] for name in PARAMETERS],
                            [t.double().cpu() for t in up] + [torch.ones((), dtype=torch.float64)]))
    for name, a, b in zip(["h", "n", "loss"] + PARAMETERS, got, want):
        assert a.shape == b.shape
        rel = float((a.double().cpu() - b).norm() / b.norm())
        assert rel <= tol, (name, rel)


def test_example_on_cpu():
    run(torch.float64, "cpu", 1e-3)


@pytest.mark.gpu
def test_example():
    from iris_testing_b200 import ops
    run(torch.bfloat16, "cuda", 12 * 2.0 ** -8)
    ops.check_default_status()
