"""The operators around the experts of an MoE block, as cases that can be timed and compared.

Three kinds of case:

``norm``     ``ops.pre_norm`` and ``ops.post_norm``: the RMS norm in front of a block, and the junction behind it
             (norm of the block's output, gate, residual with its scale, and the norm in front of the next block).
``balance``  ``ops.balance_loss``: the router's balance and z loss with per-expert counts.
``linear``   ``ops.linear``: matrix product with bias, activation and residual, dense (a shared expert) or with one
             weight per expert over packed ragged rows.

With ``train`` a pass is forward and backward and returns the gradients too.  Activations are N(0, 1), expert weights
N(0, 0.02), as in ``bench.py``; sizes are those of the layer presets, of their decode batches, and odd ones.
"""
import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


def _norm(name, T, H, dtype, pre=False, norm=True, gate=None, scale=1.0, nxt=False, weights="same", train=False):
    return dict(name=name, op="norm", T=T, H=H, dtype=dtype, pre=pre, norm=norm, gate=gate, scale=scale, next=nxt,
                weights=weights, train=train)


def _balance(name, T, E, k, dtype="fp32", S=0, mask=False, banned=False, z=0.0, train=True):
    return dict(name=name, op="balance", T=T, E=E, k=k, dtype=dtype, S=S, mask=mask, banned=banned, z=z, train=train)


def _linear(name, M, K, N, G=0, dtype="bf16", act="none", bias=False, residual=False, slack=0, train=False):
    return dict(name=name, op="linear", M=M, K=K, N=N, G=G, dtype=dtype, act=act, bias=bias, residual=residual, slack=slack,
                train=train)


def listed():
    return [
        # one token between two blocks of a decode step: latency alone
        _norm("junction-decode-1", 1, 4096, "bf16", nxt=True),
        # the junction of a training step of two sequences of 4096, LayerScale-like gate, fp32 master norm weights
        _norm("junction-train-8192", 8192, 4096, "bf16", gate="channel", nxt=True, weights="fp32", train=True),
        # the norm in front of a block over a long packed prefill, odd number of tokens, fp16
        _norm("norm-prefill-30001", 30001, 2048, "fp16", pre=True),
        # a block's output under a gate per token (a shared expert's), scaled residual, odd batch, the large preset's width
        _norm("gate-train-5003", 5003, 6144, "bf16", gate="token", scale=0.5, train=True),
        # the loss of a fine-tuning microbatch: latency alone
        _balance("balance-64", 64, 8, 2),
        # one training step of the fine-grained preset, with z loss
        _balance("balance-16384", 16384, 64, 8, z=1e-3),
        # packed sequences with padding and a banned expert, as many experts as the plan takes, bf16 logits
        _balance("balance-packed-250000", 250000, 128, 8, dtype="bf16", S=97, mask=True, banned=True, z=1e-3),
        # a shared expert's gated up projection for one token: 235 MB of weights streamed
        _linear("shared-decode-1", 1, 4096, 28672, act="silu_gate"),
        # a decode step of fine-grained experts, 25 rows each on average, one expert without any, buffer larger than the load
        _linear("experts-decode-1600", 1600, 2048, 2816, G=64, act="silu_gate", slack=400),
        # a down projection with bias and the residual stream, odd rows, fp16
        _linear("down-1000", 1000, 14336, 4096, dtype="fp16", bias=True, residual=True),
        # a dense up projection in training
        _linear("up-train-4000", 4000, 4096, 14336, act="gelu", bias=True, train=True),
        # the experts' gated up projections in training, every row of a step of 8192 tokens with 8 copies
        _linear("experts-train-65536", 65536, 2048, 2816, G=64, act="silu_gate", train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm", "balance", "balance", "linear", "linear", "linear", "linear"])
    train = rng.random() < 0.5
    if op == "norm":
        H = rng.choice([256, 768, 1408, 2048, 4096, 6144, 8 * rng.randint(1, 1000), rng.randint(1, 5000)])
        c = _norm("", _log_int(rng, 1, max(1, 70_000_000 // max(H, 1024))), H, rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                  pre=rng.random() < 0.3, norm=rng.random() < 0.7, gate=rng.choice([None, "channel", "token", "full"]),
                  scale=rng.choice([1.0, 0.5, 0.125]), nxt=rng.random() < 0.5, weights=rng.choice(["same", "fp32"]), train=train)
    elif op == "balance":
        E = rng.choice([4, 8, 16, 32, 64, 128, 256, rng.randint(2, 200)])
        T = _log_int(rng, 1, 250000)      # gradients shrink with T: no fp16, which would need a loss scale
        c = _balance("", T, E, rng.randint(1, min(8, E // 2)), dtype=rng.choice(["fp32", "fp32", "bf16"]),
                     S=0 if rng.random() < 0.4 else _log_int(rng, 1, min(T, 500)), mask=rng.random() < 0.4,
                     banned=E > 10 and rng.random() < 0.3, z=rng.choice([0.0, 1e-3]), train=train)
    else:
        act = rng.choice(["none", "relu", "silu", "gelu", "silu_gate", "silu_gate"])
        G = rng.choice([0, 0, 4, 8, 64, rng.randint(1, 100)])
        K = rng.choice([256, 768, 1408, 2048, 4096, 8 * rng.randint(4, 600)])
        N = 256 * rng.randint(1, 40) if act == "silu_gate" else rng.choice([256, 768, 2048, 4096, 8 * rng.randint(1, 600)])
        G = max(1, min(G, 370_000_000 // (K * N))) if G else 0
        cap = min(65536, 1_800_000_000_000 // (6 * K * N), 190_000_000 // max(K, N))
        c = _linear("", _log_int(rng, 1, cap), K, N, G=G, dtype=rng.choice(["bf16", "bf16", "fp16"]), act=act,
                    bias=rng.random() < 0.5, residual=rng.random() < 0.4, slack=rng.choice([0, 0, 100]) if G else 0, train=train)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------- inputs
def _randn(gen, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device=gen.device) * std + mean).to(dtype)


def _split(total, parts, seed):
    """Whole numbers that add up to ``total``, uneven, one of several parts without any."""
    g = torch.Generator().manual_seed(seed)
    p = torch.exp(0.6 * torch.randn(parts, generator=g))
    if parts > 2:
        p[parts // 3] = 0.0
    n = torch.floor(p / p.sum() * total).to(torch.int64)
    n[int(torch.argmax(p))] += total - int(n.sum())
    return n.tolist()


def _inputs(c, seed, dev):
    """The tensors of a case by name; those that a training step differentiates by are leaves."""
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = TYPES[c["dtype"]]
    s = dict(case=c)
    if c["op"] == "norm":
        T, H = c["T"], c["H"]
        wt = dt if c["weights"] == "same" else F32
        s["y"] = _randn(g, (T, H), dt, 1.5)
        if c["pre"] or c["norm"]:
            s["weight"] = _randn(g, (H,), wt, 0.1, 1.0)
        if not c["pre"]:
            s["residual"] = _randn(g, (T, H), dt, 2.0)
            if c["gate"]:
                s["gate"] = _randn(g, {"channel": (H,), "token": (T, 1), "full": (T, H)}[c["gate"]], dt, 0.3, 0.5)
            if c["next"]:
                s["next_weight"] = _randn(g, (H,), wt, 0.1, 1.0)
        leaves = [n for n in ("y", "residual", "weight", "gate", "next_weight") if n in s]
        s["dh"] = _randn(g, (T, H), dt)
        s["dn"] = _randn(g, (T, H), dt)
    elif c["op"] == "balance":
        T, E, k = c["T"], c["E"], c["k"]
        lg = _randn(g, (T, E), F32) + _randn(g, (E,), F32, 0.7)
        if c["banned"]:
            lg[:, E // 2] = -math.inf
        s["logits"] = lg.to(dt)
        s["idx"] = torch.topk(lg, k, dim=1).indices.to(torch.int32)
        s["rows"] = s["mask"] = None
        if c["S"]:
            s["rows"] = torch.tensor(_split(T - T // 50, c["S"], int(seed)), dtype=torch.int32, device=dev)
        if c["mask"]:
            s["mask"] = torch.rand(T, generator=g, device=dev) < 0.9
        s["dloss"] = torch.tensor(1.0, device=dev)
        leaves = ["logits"]
    else:
        M, K, N, G = c["M"] + c["slack"], c["K"], c["N"], c["G"]
        out = N // 2 if c["act"] == "silu_gate" else N
        s["x"] = _randn(g, (M, K), dt)
        s["w"] = _randn(g, (G, N, K) if G else (N, K), dt, 0.02)
        if c["bias"]:
            s["bias"] = _randn(g, (G, N) if G else (N,), dt, 0.1)
        if c["residual"]:
            s["residual"] = _randn(g, (M, out), dt)
        s["rows"], s["most"] = None, c["M"]
        if G:
            rows = _split(c["M"], G, int(seed))
            s["rows"], s["most"] = torch.tensor(rows, dtype=torch.int32, device=dev), max(rows)
        s["dy"] = _randn(g, (M, out), dt)
        leaves = [n for n in ("x", "w", "bias", "residual") if n in s]
    s["leaves"] = leaves
    return s


def prepare(case, seed):
    s = _inputs(case, seed, torch.device("cuda", torch.cuda.current_device()))
    if case["train"]:
        for n in s["leaves"]:
            s[n].requires_grad_()
    return s


# ------------------------------------------------------------------------------------- the framework's calls
def _own_norm(s):
    from iris_testing_b200 import ops
    c = s["case"]
    if c["pre"]:
        outs, grads = (ops.pre_norm(s["y"], s["weight"], eps=EPS),), (s["dn"],)
    else:
        outs = ops.post_norm(s["y"], s["residual"], s.get("weight"), s.get("gate"), norm=c["norm"], residual_scale=c["scale"],
                             next_weight=s.get("next_weight"), eps=EPS)
        outs, grads = (outs, (s["dh"], s["dn"])) if c["next"] else ((outs,), (s["dh"],))
    if not c["train"]:
        return tuple(outs)
    return tuple(o.detach() for o in outs) + torch.autograd.grad(outs, [s[n] for n in s["leaves"]], grads)


def _own_balance(s):
    from iris_testing_b200 import ops
    c = s["case"]
    loss, counts = ops.balance_loss(s["logits"], s["idx"], balance_coef=1e-2, z_coef=c["z"], seq_rows=s["rows"],
                                    token_mask=s["mask"])
    if not c["train"]:
        return loss, counts
    return loss.detach(), counts, torch.autograd.grad(loss, s["logits"], s["dloss"])[0]


def _own_linear(s):
    from iris_testing_b200 import ops
    c = s["case"]
    y = ops.linear(s["x"], s["w"], s.get("bias"), s.get("residual"), activation=None if c["act"] == "none" else c["act"],
                   group_rows=s["rows"])
    if not c["train"]:
        return (y,)
    return (y.detach(),) + torch.autograd.grad(y, [s[n] for n in s["leaves"]], s["dy"])


# ------------------------------------------------------------------------------------------- the plain forms
def _plain_norm(s):
    c, dt = s["case"], TYPES[s["case"]["dtype"]]
    f = {n: s[n].to(F32) for n in ("y", "weight", "residual", "gate", "next_weight", "dh", "dn") if n in s}
    y, w, gate = f["y"], f.get("weight"), f.get("gate")
    normed = c["pre"] or c["norm"]
    if normed:
        r1 = 1.0 / torch.sqrt((y * y).mean(1, keepdim=True) + EPS)
        yh = y * r1
        u = yh * w
    else:
        u = y
    if c["pre"]:
        outs, du = [u], f["dn"]
    else:
        h = c["scale"] * f["residual"] + (u if gate is None else gate * u)
        outs = [h]
        if c["next"]:
            r2 = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
            hh = h * r2
            outs.append(hh * f["next_weight"])
    outs = [o.to(dt) for o in outs]
    if not c["train"]:
        return tuple(outs)
    grads = {}
    if not c["pre"]:
        gh = f["dh"]
        if c["next"]:
            t = f["dn"] * f["next_weight"]
            gh = gh + r2 * (t - hh * (t * hh).mean(1, keepdim=True))
            grads["next_weight"] = (f["dn"] * hh).sum(0, dtype=F64)
        grads["residual"] = c["scale"] * gh
        du = gh
        if gate is not None:
            du = gate * gh
            p = gh * u
            grads["gate"] = p if c["gate"] == "full" else p.sum(0, dtype=F64) if c["gate"] == "channel" else p.sum(1, keepdim=True)
    if normed:
        grads["weight"] = (du * yh).sum(0, dtype=F64)
        t = du * w
        grads["y"] = r1 * (t - yh * (t * yh).mean(1, keepdim=True))
    else:
        grads["y"] = du
    return tuple(outs) + tuple(grads[n].to(s[n].dtype) for n in s["leaves"])


def _plain_balance(s):
    c = s["case"]
    T, E, k, S = c["T"], c["E"], c["k"], max(c["S"], 1)
    lg = s["logits"].to(F32)
    mx = lg.amax(1, keepdim=True)
    e = torch.exp(lg - mx)
    total = e.sum(1, keepdim=True)
    p, lse = e / total, mx + torch.log(total)
    t = torch.arange(T, device=lg.device)
    valid = torch.ones(T, dtype=torch.bool, device=lg.device)
    seq = torch.zeros(T, dtype=torch.int64, device=lg.device)
    if s["rows"] is not None:
        ends = torch.cumsum(s["rows"].to(torch.int64), 0)
        seq = (t[:, None] >= ends[None, :]).sum(1)
        valid = seq < S
        seq = torch.where(valid, seq, torch.zeros_like(seq))
    if s["mask"] is not None:
        valid = valid & s["mask"]
    v64 = valid.to(F64)
    n_s = torch.zeros(S, dtype=F64, device=lg.device).index_add_(0, seq, v64)
    where = (seq[:, None] * E + s["idx"].to(torch.int64)).reshape(-1)
    counts = torch.zeros(S * E, dtype=torch.int64, device=lg.device)
    counts.index_add_(0, where, valid[:, None].expand(T, k).reshape(-1).to(torch.int64))
    counts = counts.view(S, E)
    col = torch.zeros(S, E, dtype=F64, device=lg.device).index_add_(0, seq, p.to(F64) * v64[:, None])
    full = torch.clamp((n_s > 0).sum(), min=1)
    one = torch.clamp(n_s, min=1.0)[:, None]
    a = 1e-2 / full * E * counts.to(F64) / (k * one * one)
    n = torch.clamp(n_s.sum(), min=1.0)
    loss = (a * col).sum() + c["z"] / n * (v64 * lse[:, 0].to(F64) ** 2).sum()
    outs = (loss.to(F32), counts.to(torch.int32) if c["S"] else counts[0].to(torch.int32))
    if not c["train"]:
        return outs
    at = a.to(F32)[seq]
    d = p * (at - (p * at).sum(1, keepdim=True)) + (2.0 * c["z"] / n).to(F32) * lse * p
    return outs + ((s["dloss"] * torch.where(valid[:, None], d, torch.zeros_like(d))).to(s["logits"].dtype),)


def _act(z, act):
    """The activation and its derivative by z (of the gated form: what to multiply with, for gate and up)."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.clamp(z, min=0.0), (z > 0).to(z.dtype)
    if act == "silu":
        q = 1.0 / (1.0 + torch.exp(-z))
        return z * q, q * (1.0 + z * (1.0 - q))
    if act == "gelu":
        a = math.sqrt(2.0 / math.pi)
        q = 1.0 / (1.0 + torch.exp(-2.0 * a * (z + 0.044715 * z * z * z)))
        return z * q, q + z * q * (1.0 - q) * 2.0 * a * (1.0 + 3.0 * 0.044715 * z * z)
    v = z.view(z.shape[:-1] + (z.shape[-1] // 256, 2, 128))
    gate, up = v[..., 0, :], v[..., 1, :]
    q = 1.0 / (1.0 + torch.exp(-gate))
    both = torch.stack((q * (1.0 + gate * (1.0 - q)) * up, gate * q), -2)
    return (gate * q * up).reshape(z.shape[:-1] + (z.shape[-1] // 2,)), both.reshape(z.shape)


def _spread(d, act):
    """The output's gradient beside every pre-activation that it belongs to."""
    if act != "silu_gate":
        return d
    v = d.view(d.shape[:-1] + (d.shape[-1] // 128, 1, 128))
    return v.expand(v.shape[:-2] + (2, 128)).reshape(d.shape[:-1] + (2 * d.shape[-1],))


def _plain_linear(s):
    c = s["case"]
    x, w, act = s["x"].to(F32), s["w"].to(F32), c["act"]
    M = x.shape[0]
    if c["G"]:
        # rows of expert g side by side, short groups padded with zero rows
        rows = s["rows"].to(torch.int64)
        j = torch.arange(s["most"], device=x.device)
        at = (torch.cumsum(rows, 0) - rows)[:, None] + j[None, :]
        real = (j[None, :] < rows[:, None])
        at = torch.where(real, at, torch.full_like(at, M))

        def pack(t):
            return torch.cat((t, torch.zeros_like(t[:1])))[at]

        def unpack(t):
            return torch.zeros((M + 1, t.shape[-1]), dtype=t.dtype, device=t.device).index_copy_(
                0, at[real], t[real])[:M]
    else:
        x, w, real = x[None], w[None], None

        def pack(t):
            return t[None]

        def unpack(t):
            return t[0]
    xg = pack(x) if c["G"] else x
    z = xg @ w.transpose(1, 2)
    if c["bias"]:
        z = z + s["bias"].to(F32).view(w.shape[0], 1, -1)
    a, da = _act(z, act)
    y = unpack(a)
    if c["residual"]:
        res = s["residual"].to(F32)
        y = y + (unpack(pack(res)) if c["G"] else res)
    outs = (y.to(s["x"].dtype),)
    if not c["train"]:
        return outs
    dy = s["dy"].to(F32)
    dz = _spread(pack(dy), act) * da
    if real is not None:
        dz = dz * real[:, :, None]
    grads = {"x": unpack(dz @ w), "w": (dz.transpose(1, 2) @ xg).view(s["w"].shape)}
    if c["bias"]:
        grads["bias"] = dz.sum(1, dtype=F64).view(s["bias"].shape)
    if c["residual"]:
        grads["residual"] = unpack(pack(dy))
    return outs + tuple(grads[n].to(s[n].dtype) for n in s["leaves"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "balance": _own_balance, "linear": _own_linear}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "balance": _plain_balance, "linear": _plain_linear}[op](state)


# ---------------------------------------------------------------------------------- from the definitions, fp64
def _rms(t, w):
    return t / torch.sqrt(t.pow(2).sum(1, keepdim=True) / t.shape[1] + EPS) * w


def _exact_norm(c, s, v):
    y = _rms(v["y"], v["weight"]) if c["pre"] or c["norm"] else v["y"]
    if c["pre"]:
        return (y,), (v["dn"],)
    h = v["residual"] * c["scale"] + y * v.get("gate", 1.0)
    return ((h, _rms(h, v["next_weight"])), (v["dh"], v["dn"])) if c["next"] else ((h,), (v["dh"],))


def _exact_balance(c, s, v):
    T, E, k = c["T"], c["E"], c["k"]
    mask = torch.ones(T, dtype=torch.bool, device=s["idx"].device) if s["mask"] is None else s["mask"]
    lengths = [T] if s["rows"] is None else s["rows"].tolist()
    counts, terms, lse, start = [], [], [], 0
    for length in lengths:
        keep = mask[start:start + length]
        lg = v["logits"][start:start + length][keep]
        chosen = s["idx"][start:start + length][keep].reshape(-1).long()
        counts.append(torch.bincount(chosen, minlength=E))
        start += length
        if lg.shape[0]:
            share = counts[-1].to(F64) / (k * lg.shape[0])
            terms.append(E * (share * torch.softmax(lg, 1).mean(0)).sum())
            lse.append(torch.logsumexp(lg, 1))
    loss = 0.0 * v["logits"].nan_to_num(neginf=0.0).sum()
    if terms:
        loss = loss + 1e-2 * torch.stack(terms).mean() + c["z"] * torch.cat(lse).pow(2).mean()
    counts = torch.stack(counts).to(torch.int32)
    return (loss, counts if c["S"] else counts[0]), (torch.ones((), dtype=F64, device=loss.device),)


def _exact_linear(c, s, v):
    M, G = c["M"] + c["slack"], c["G"]
    lengths = s["rows"].tolist() if G else [M]
    parts, start = [], 0
    for g, length in enumerate(lengths):
        z = v["x"][start:start + length] @ (v["w"][g] if G else v["w"]).t()
        if c["bias"]:
            z = z + (v["bias"][g] if G else v["bias"])
        if c["act"] == "relu":
            z = torch.relu(z)
        elif c["act"] == "silu":
            z = torch.nn.functional.silu(z)
        elif c["act"] == "gelu":
            z = torch.nn.functional.gelu(z, approximate="tanh")
        elif c["act"] == "silu_gate":
            halves = z.unflatten(1, (-1, 2, 128))
            z = (torch.nn.functional.silu(halves[:, :, 0]) * halves[:, :, 1]).flatten(1)
        if c["residual"]:
            z = z + v["residual"][start:start + length]
        parts.append(z)
        start += length
    parts.append(torch.zeros((M - start, parts[0].shape[1]), dtype=F64, device=parts[0].device))
    return (torch.cat(parts),), (v["dy"],)


def exact(case, seed):
    """What ``run`` returns, by differentiating the definitions in fp64; rows behind the last group give zeros."""
    s = _inputs(case, seed, torch.device("cuda", torch.cuda.current_device()))
    v = {n: t.to(F64) for n, t in s.items() if torch.is_tensor(t) and t.is_floating_point()}
    leaves = [v[n].requires_grad_() for n in s["leaves"]] if case["train"] else []
    outs, grads = {"norm": _exact_norm, "balance": _exact_balance, "linear": _exact_linear}[case["op"]](case, s, v)
    done = tuple(o.detach() for o in outs)
    if case["train"]:
        done += torch.autograd.grad([o for o in outs if o.is_floating_point()], leaves, grads)
    return done


def work(case):
    c, b = case, BYTES[case["dtype"]]
    if c["op"] == "norm":
        n, wide = c["T"] * c["H"], c["gate"] == "full" and not c["pre"]
        reads, writes = (1, 1) if c["pre"] else (2 + wide, 1 + c["next"])
        if c["train"]:                      # the forward's inputs, the outputs' gradients, the inputs' gradients
            reads, writes = reads + (1 if c["pre"] else 1 + c["next"]), writes + (1 if c["pre"] else 2 + wide)
        return dict(bytes=n * b * (reads + writes), flops=n * (30 if c["train"] else 10))
    if c["op"] == "balance":
        n = c["T"] * c["E"]
        return dict(bytes=n * b * (2 if c["train"] else 1) + c["T"] * c["k"] * 4, flops=n * (12 if c["train"] else 6))
    rows, K, N, G = c["M"], c["K"], c["N"], max(c["G"], 1)
    out = N // 2 if c["act"] == "silu_gate" else N
    weights = min(G, rows) * N * K
    moved = rows * K + weights + rows * out * (2 if c["residual"] else 1)
    if c["train"]:
        moved += rows * out + rows * K + G * N * K
    return dict(bytes=moved * b, flops=2 * rows * N * K * (3 if c["train"] else 1))
