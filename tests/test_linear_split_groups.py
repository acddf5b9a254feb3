"""Split products of groups with everything that their joining kernel does per group: bias, activation, residual, kept
pre-activations, empty groups and rows behind the last; the rule that chooses them; and what lies around their results."""
import ctypes as C
import importlib

import pytest
import torch

from test_linear import ACTS, check, inputs, reference, within

linear = importlib.import_module("iris_testing_b200.ops.linear")
FORWARD, DX, DW = 0, 1, 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,N,K", [([40, 0, 129, 1], 256, 72), ([200, 300], 768, 1024), ([0, 3, 0, 16, 7, 0], 512, 200)])
def test_epilogues_of_split_groups(rows, N, K, act, dtype, monkeypatch):
    monkeypatch.setattr(linear, "_splits", lambda mode, M, N, K, G, grouped, sms: not (grouped and mode == DW))
    x, w, b, r, dy = inputs(rows, N, K, dtype, act, True, True, "cuda", slack=70)
    check(x, w, b, r, dy, act, rows)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu_gate", "gelu"])
def test_groups_that_the_rule_splits(act):
    rows = [3, 0, 16, 7, 1, 12, 0, 9]
    x, w, b, r, dy = inputs(rows, 512, 1536, torch.bfloat16, act, True, True, "cuda", slack=5)
    assert linear._splits(FORWARD, x.shape[0], 512, 1536, 8, True, 148)
    check(x, w, b, r, dy, act, rows)


def test_rule_on_both_sides_of_its_limits():
    """Grouped dW never; whole tiles for at most 64 SMs and half as many as there are blocks of the contraction; or for fewer than
    all SMs, over 16 blocks or more, with at most 16 rows a group."""
    def splits(mode, M, N, K, G=1, grouped=False, sms=148):
        return linear._splits(mode, M, N, K, G, grouped, sms)
    assert not splits(DW, 4096, 768, 768, 1, True) and splits(DW, 4096, 768, 768)       # 18 tiles, 64 blocks
    assert not splits(DW, 1024, 768, 768)                                               # 16 blocks: no more than 8 tiles
    assert splits(FORWARD, 256, 4096, 4096) and not splits(FORWARD, 512, 4096, 4096)    # 32 SMs; 64 SMs for 64 blocks
    assert splits(FORWARD, 512, 4096, 14336) and not splits(FORWARD, 1024, 4096, 14336)
    assert splits(FORWARD, 2048, 256, 2048) and not splits(FORWARD, 4096, 256, 2048)    # 16 SMs for 32 blocks; 32
    assert splits(DX, 256, 4096, 4096) and not splits(DX, 512, 4096, 4096)
    assert splits(FORWARD, 1, 28672, 4096) and splits(FORWARD, 16, 28672, 4096) and not splits(FORWARD, 17, 28672, 4096)
    assert splits(FORWARD, 1, 4096, 1024) and not splits(FORWARD, 1, 2304, 960)         # 15 blocks for 9 tiles
    assert not splits(FORWARD, 1, 148 * 256, 4096) and splits(FORWARD, 1, 147 * 256, 4096)
    assert splits(FORWARD, 8 * 16, 2816, 4096, 8, True) and not splits(FORWARD, 8 * 16 + 1, 2816, 4096, 8, True)
    assert not splits(FORWARD, 4096, 4096, 4096)


class Guarded:
    """Tensors as slices of larger ones whose other bytes must stay as they are."""

    def __init__(self):
        self.whole = []

    def __call__(self, like):
        size = like.numel() * like.element_size()
        buf = torch.full((4096 + (size + 255) // 256 * 256 + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
        self.whole.append((buf, size))
        return buf[4096:4096 + size].view(like.dtype).view(like.shape)

    def check(self):
        for buf, size in self.whole:
            assert bool((buf[:4096] == 0xA5).all()) and bool((buf[4096 + size:] == 0xA5).all())


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("act", ["silu_gate", "gelu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [[7, 0, 40, 13], [300, 171, 0, 200], [30, 31], [2 ** 31 - 1, 2 ** 31 - 1]])
def test_nothing_is_written_around_the_results(rows, dtype, act, split):
    """Products and activation gradients through the C entries, with sizes that fit and with more rows than there are."""
    from iris_testing_b200 import ops
    from iris_testing_b200._native import NativeError
    N, K, G = 512, 200, len(rows)
    M = 60 if sum(rows) != 671 else 671 + 5
    n_out = N // 2 if act == "silu_gate" else N
    g = torch.Generator().manual_seed(M)

    def rnd(*shape):
        return torch.randn(*shape, generator=g).to("cuda", dtype)
    x, w, b, r, dy = rnd(M, K), rnd(G, N, K), rnd(G, N), rnd(M, n_out), rnd(M, n_out)
    gr = torch.tensor(rows, dtype=torch.int32, device="cuda")
    code = linear.ACTIVATIONS[act]
    ops.check_default_status()
    guard = Guarded()
    y, z, zexp = guard(dy), guard(torch.empty(M, N, dtype=torch.float16)), guard(torch.empty(M, N if dtype == torch.float16 else N // 32, dtype=torch.uint8))
    dx, dw, dz, dres, db = guard(x), guard(w), guard(torch.empty(M, N, dtype=dtype)), guard(dy), guard(b)
    z.zero_()
    zexp.fill_(127)
    dz.zero_()
    sms = linear.sm_count(x.device)

    def product(mode, a, w_or_x, out, **how):
        # as ops.linear makes the call, but for the scratch of a split product, which is guarded here
        la = linear.LinearArgs()
        la.a, la.b, la.out, la.group_rows = a.data_ptr(), w_or_x.data_ptr(), out.data_ptr(), gr.data_ptr()
        for name, t in how.items():
            setattr(la, name, t if isinstance(t, int) else t.data_ptr())
        la.status, la.wait_budget_ns = ops.default_status(x.device).data_ptr(), 2_000_000_000
        la.mode, la.G, la.M, la.N, la.K, la.n_out, la.elem = mode, G, M, N, K, out.shape[-1], linear.ELEM[dtype]
        if split and mode != DW:
            la.record = guard(torch.empty(linear._record_floats(mode, M, N, K, G, sms))).data_ptr()
        linear._PRODUCT(la, sms, linear.stream_ptr(x))
    product(FORWARD, x, w, y, z=z, zexp=zexp, bias=b, res=r, act=code)
    a = linear.ActGradArgs()
    a.dy, a.z, a.zexp, a.dz, a.dres, a.dbias = (t.data_ptr() for t in (dy, z, zexp, dz, dres, db))
    a.G, a.M, a.N, a.n_out, a.elem, a.act, a.group_rows = G, M, N, n_out, linear.ELEM[dtype], code, gr.data_ptr()
    a.chunk_rows, a.chunks = 16, -(-M // 16)
    a.record = guard(torch.empty(a.chunks + G, N)).data_ptr()
    if dtype == torch.float16:
        a.peak = guard(torch.empty(1, dtype=torch.int32)).data_ptr()
    linear._ACT_GRAD(a, linear.stream_ptr(x))
    product(DX, dz, w, dx)
    product(DW, dz, x, dw)
    torch.cuda.synchronize()
    guard.check()
    if sum(rows) > M:
        with pytest.raises(NativeError, match="overflow"):
            ops.check_default_status()
    else:
        ops.check_default_status()
        for got, pair, name in zip((y, dx, dw, db, dres), reference(x, w, b, r, act, rows, dy), ("y", "dx", "dw", "dbias", "dres")):
            within(got, pair, name)
