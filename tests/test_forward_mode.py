"""Forward-mode derivatives: the ops with gradients have none of them, and say so instead of returning a result without a tangent,
which would read as a derivative of zero.  CPU tensors take plain PyTorch, which has them.

On the CPU the refusals are reached by having the ops take the kernels' path for CPU tensors: it refuses before anything is
launched, or asked of a device."""
import importlib

import pytest
import torch
from torch.autograd import forward_ad


def cases(dev):
    """(name, call, arguments): every floating-point argument may carry a tangent."""
    from iris_testing_b200 import ops
    g = torch.Generator().manual_seed(0)

    def rnd(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g).to(dev, dtype)
    idx = torch.randint(0, 8, (6, 2), generator=g).to(dev, torch.int32)
    rows = torch.tensor([2, 4], dtype=torch.int32, device=dev)
    return [("pre_norm", lambda x, w: ops.pre_norm(x, w), [rnd(6, 16), rnd(16)]),
            ("post_norm", lambda y, r, w, gate, nxt: ops.post_norm(y, r, w, gate, next_weight=nxt)[1],
             [rnd(6, 16), rnd(6, 16), rnd(16), rnd(6, 1), rnd(16)]),
            ("balance_loss", lambda lg: ops.balance_loss(lg, idx)[0], [rnd(6, 8, dtype=torch.float32)]),
            ("linear", lambda x, w, b, r: ops.linear(x, w, b, r, activation="silu"), [rnd(6, 16), rnd(8, 16), rnd(8), rnd(6, 8)]),
            ("linear, grouped", lambda x, w, b, r: ops.linear(x, w, b, r, group_rows=rows),
             [rnd(6, 16), rnd(2, 8, 16), rnd(2, 8), rnd(6, 8)])]


def refused(call, args):
    for i in range(len(args)):
        for other in (False, True):                  # the other arguments may ask for gradients at the same time
            with forward_ad.dual_level():
                these = [forward_ad.make_dual(a, torch.ones_like(a)) if j == i else a.detach().requires_grad_(other)
                         for j, a in enumerate(args)]
                with pytest.raises(ValueError, match="forward-mode"):
                    call(*these)
                with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                    call(*these)


@pytest.mark.parametrize("which", range(5))
def test_a_tangent_is_refused_on_the_kernels_path(which, monkeypatch):
    for name in ("norm", "balance", "linear"):
        mod = importlib.import_module(f"iris_testing_b200.ops.{name}")
        monkeypatch.setattr(mod, "use_native", lambda t: True)
    _, call, args = cases("cpu")[which]
    refused(call, args)


@pytest.mark.parametrize("which", range(5))
def test_cpu_tensors_have_tangents(which):
    _, call, args = cases("cpu")[which]
    with forward_ad.dual_level():
        out = call(*(forward_ad.make_dual(a, torch.ones_like(a)) for a in args))
        assert forward_ad.unpack_dual(out).tangent is not None


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(5))
def test_a_tangent_is_refused(which):
    _, call, args = cases("cuda")[which]
    refused(call, args)
    with forward_ad.dual_level():                    # a level that no argument takes part in
        want = call(*args)
    assert torch.equal(want, call(*args))


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(5))
def test_a_tangent_of_the_results_gradient_is_refused(which):
    _, call, args = cases("cuda")[which]
    leaves = [a.requires_grad_() for a in args]
    out = call(*leaves)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(ValueError, match="forward-mode"):
            torch.autograd.grad(out, leaves, d, retain_graph=True)
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(out, leaves, torch.ones_like(out)))
