"""Cases over which the operators of ``moodist_b200.ops`` that a decoder's training step and its evaluation use are timed:
layer normalisation, rotary positions, distillation from a teacher's top logits, the gated projection.

``run`` computes a case in plain torch arithmetic (32 bits throughout, rounded once at the end), or, with ``own`` set, through
the framework's operators.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # eight sequences advance by one token: the norm of a 4096-wide decoder, latency only
        dict(name="norm_decode", op="layer_norm", rows=8, dim=4096, dtype="bf16", weights="same", train=False),
        # the norm of a training step of 8192 tokens at the width of the flagship model
        dict(name="norm_train", op="layer_norm", rows=8192, dim=4096, dtype="bf16", weights="same", train=True),
        # an odd width that no vector load fits, half precision with 32-bit weights
        dict(name="norm_odd_train", op="layer_norm", rows=5003, dim=1537, dtype="fp16", weights="fp32", train=True),
        # one token of each of 64 sequences at positions all over a 131072-token context
        dict(name="rotary_decode", op="rotary", batch=64, seq=1, heads=32, kv=8, dim=128, rot=128, length=131072,
             interleaved=False, dtype="bf16", positions="far", train=False),
        # q and k heads of a training step of 8192 tokens, positions in order
        dict(name="rotary_train", op="rotary", batch=1, seq=8192, heads=32, kv=8, dim=128, rot=128, length=8192,
             interleaved=False, dtype="bf16", positions="order", train=True),
        # a padded batch, adjacent pairs, 32 of 80 dimensions rotated
        dict(name="rotary_partial_train", op="rotary", batch=3, seq=1021, heads=20, kv=4, dim=80, rot=32, length=2048,
             interleaved=True, dtype="fp16", positions="padded", train=True),
        # a small student of the tests' size, in 32 bits, with hard targets
        dict(name="distill_small", op="distill", rows=37, vocab=1003, top=5, tau=1.0, hard=0.25, dtype="fp32", reduction="mean", train=True),
        # a distillation step at the flagship vocabulary
        dict(name="distill_train", op="distill", rows=4096, vocab=128256, top=64, tau=2.0, hard=0.0, dtype="bf16", reduction="mean", train=True),
        # an odd vocabulary in half precision, soft and hard terms at once
        dict(name="distill_odd_train", op="distill", rows=515, vocab=50257, top=128, tau=1.5, hard=0.5, dtype="fp16", reduction="sum", train=True),
        # one token through the flagship model's gate and up projections
        dict(name="gated_decode", op="gated", rows=1, dim=4096, ffn=14336, act="silu", train=False),
        # the same projections in a training step of 8192 tokens
        dict(name="gated_train", op="gated", rows=8192, dim=4096, ffn=14336, act="silu", train=True),
        # ragged sizes, another activation
        dict(name="gated_odd_train", op="gated", rows=301, dim=1016, ffn=2728, act="gelu_tanh", train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "rotary", "distill", "gated"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.6
    if op == "layer_norm":
        dim = _log_int(rng, 64, 16384)
        if rng.random() < 0.7:
            dim = -(-dim // 8) * 8
        rows = _log_int(rng, 1, max(2, min(32768, (1 << 25) // dim)))
        return dict(op=op, rows=rows, dim=dim, dtype=dtype, weights=rng.choice(["same", "fp32"]), train=train)
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 192, 256])
        heads = rng.choice([1, 4, 7, 8, 16, 32, 64])
        kv = max(1, heads // rng.choice([1, 2, 4, 8]))
        tokens = _log_int(rng, 1, max(2, (1 << 25) // (dim * heads)))
        batch = rng.choice([1, 2, 3, 8])
        seq = max(1, tokens // batch)
        return dict(op=op, batch=batch, seq=seq, heads=heads, kv=kv, dim=dim, rot=rng.choice([dim, dim, dim // 2, dim // 4 * 2]),
                    length=max(seq, _log_int(rng, 1024, 131072)), interleaved=rng.random() < 0.5, dtype=dtype,
                    positions=rng.choice(["order", "far", "padded"]), train=train)
    if op == "distill":
        vocab = _log_int(rng, 256, 160000)
        if rng.random() < 0.7:
            vocab = -(-vocab // 8) * 8
        rows = _log_int(rng, 1, max(2, min(16384, (1 << 28) // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, top=rng.choice([1, 4, 10, 32, 64, 100, 256]), tau=rng.choice([1.0, 1.5, 2.0, 4.0]),
                    hard=rng.choice([0.0, 0.0, 0.3, 0.5]), dtype=dtype, reduction="sum" if dtype == "fp16" else "mean", train=train)
    dim = 8 * _log_int(rng, 32, 1024)
    ffn = 8 * _log_int(rng, 32, 2048)
    rows = _log_int(rng, 1, max(2, min(8192, (1 << 38) // (dim * ffn))))
    return dict(op=op, rows=rows, dim=dim, ffn=ffn, act=rng.choice(["silu", "gelu", "gelu_tanh"]), train=train)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda")

    s = {"case": case}
    op, train = case["op"], case["train"]
    if op == "gated":
        t, d, f = case["rows"], case["dim"], case["ffn"]
        s["x"] = normal(t, d, dtype=torch.bfloat16).requires_grad_(train)
        s["w"] = normal(2 * f, d, dtype=torch.bfloat16, scale=d**-0.5).requires_grad_(train)
        s["dy"] = normal(t, f, dtype=torch.bfloat16, scale=0.01)
        return s
    dtype = DTYPES[case["dtype"]]
    if op == "layer_norm":
        t, d = case["rows"], case["dim"]
        wt = dtype if case["weights"] == "same" else torch.float32
        s["x"] = normal(t, d, dtype=dtype, scale=2.0, shift=0.5).requires_grad_(train)
        s["w"] = normal(d, dtype=wt, scale=0.1, shift=1.0).requires_grad_(train)
        s["b"] = normal(d, dtype=wt, scale=0.1).requires_grad_(train)
        s["dy"] = normal(t, d, dtype=dtype)
    elif op == "rotary":
        b, n, h, kv, d, r, length = (case[k] for k in ("batch", "seq", "heads", "kv", "dim", "rot", "length"))
        # q and k as they lie in the projection's output: side by side in each token's row
        qkv = normal(b, n, h + 2 * kv, d, dtype=dtype)
        s["q"] = qkv[:, :, :h].detach().requires_grad_(train)
        s["k"] = qkv[:, :, h : h + kv].detach().requires_grad_(train)
        s["dq"], s["dk"] = normal(b, n, h, d, dtype=dtype), normal(b, n, kv, d, dtype=dtype)
        inv = 500000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
        angle = torch.outer(torch.arange(length, device="cuda", dtype=torch.float64), inv)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["positions"] = None
        if case["positions"] == "far":
            s["positions"] = whole(0, length, b, n)
        elif case["positions"] == "padded":
            # sequences of different lengths, padded at their end with -1
            order = torch.arange(n, device="cuda").expand(b, n)
            s["positions"] = torch.where(order < whole(1, n + 1, b, 1), order, torch.full_like(order, -1))
    else:
        t, v, k = case["rows"], case["vocab"], case["top"]
        k = min(k, v)
        # the teacher's entries: distinct words of a row, best first, some rows shorter than others and some without any
        ids = (whole(0, v, t, 1) + torch.arange(k, device="cuda") * whole(1, max(2, v // k), t, 1)) % v
        top = normal(t, k, scale=2.0).sort(dim=-1, descending=True).values
        logits = normal(t, v, scale=2.0)
        logits.scatter_add_(1, ids, top * 0.5 + 4.0)
        s["logits"] = logits.to(dtype).requires_grad_(train)
        keep = torch.arange(k, device="cuda") < whole(0, 4 * k, t, 1)
        keep[0] = True
        s["ids"] = torch.where(keep, ids, torch.full_like(ids, -1))
        s["top"] = top.to(dtype)
        s["targets"] = None
        if case["hard"] > 0:
            targets = whole(0, v, t)
            targets[1:][whole(0, 10, t)[1:] == 0] = -100
            s["targets"] = targets
    return s


def _plain_layer_norm(s):
    x, w, b = s["x"].detach().float(), s["w"].detach().float(), s["b"].detach().float()
    c = x - x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5)
    h = c * r
    y = (h * w + b).to(s["x"].dtype)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": (dy * h).sum(0).to(s["w"].dtype), "db": dy.sum(0).to(s["b"].dtype)}


def _plain_turn(x, cos, sin, rot, interleaved):
    t = x.detach().float()
    head, rest = t[..., :rot], t[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., : rot // 2], head[..., rot // 2 :]
        head = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([head, rest], -1).to(x.dtype)


def _plain_rotary(s):
    case = s["case"]
    pos = s["positions"]
    if pos is None:
        pos = torch.arange(case["seq"], device="cuda").expand(case["batch"], case["seq"])
    at = pos.clamp(min=0)
    padded = (pos < 0)[..., None, None]
    cos = torch.where(padded, 1.0, s["cos"][at][:, :, None])
    sin = torch.where(padded, 0.0, s["sin"][at][:, :, None])
    rot, inter = case["rot"], case["interleaved"]
    out = {"q": _plain_turn(s["q"], cos, sin, rot, inter), "k": _plain_turn(s["k"], cos, sin, rot, inter)}
    if case["train"]:
        out["dq"], out["dk"] = _plain_turn(s["dq"], cos, -sin, rot, inter), _plain_turn(s["dk"], cos, -sin, rot, inter)
    return out


def _plain_distill(s):
    case = s["case"]
    tau, hard = case["tau"], case["hard"]
    z, ids, targets = s["logits"].detach().float(), s["ids"], s["targets"]
    valid = (ids >= 0) & (ids < z.shape[1])
    at = ids.clamp(0, z.shape[1] - 1)
    live = valid.any(-1)
    if targets is not None:
        live = live & (targets >= 0) & (targets < z.shape[1])
    t = torch.where(valid, s["top"].float() / tau, float("-inf"))
    e = torch.where(valid, (t - torch.where(live, t.amax(-1), 0.0)[:, None]).exp(), 0.0)
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
    zs = z / tau
    m = zs.amax(-1, keepdim=True)
    eq = (zs - m).exp()
    sq = eq.sum(-1, keepdim=True)
    logq = torch.gather(zs, 1, at) - m - sq.log()
    soft = torch.where(p > 0, p * (torch.where(p > 0, p, 1.0).log() - logq), 0.0).sum(-1)
    row = (1 - hard) * tau * tau * soft
    if hard > 0:
        word = targets.clamp(0, z.shape[1] - 1)[:, None]
        m1 = z.amax(-1, keepdim=True)
        e1 = (z - m1).exp()
        s1 = e1.sum(-1, keepdim=True)
        row = row + hard * (s1.log() + m1 - torch.gather(z, 1, word))[:, 0]
    scale = 1.0 / live.sum().clamp(min=1).float() if case["reduction"] == "mean" else torch.ones((), device=z.device)
    loss = torch.where(live, row, 0.0).sum() * scale
    if not case["train"]:
        return {"loss": loss}
    dz = (eq / sq).scatter_add_(1, at, -p).mul_((1 - hard) * tau)
    if hard > 0:
        dz = dz + hard * (e1 / s1).scatter_add_(1, word, torch.full_like(m1, -1.0))
    dz = torch.where(live[:, None], dz * scale, 0.0)
    return {"loss": loss, "dlogits": dz.to(s["logits"].dtype)}


def _plain_gated(s):
    case = s["case"]
    x, w = s["x"].detach().float(), s["w"].detach().float()
    gu = x @ w.t()
    g, u = gu.chunk(2, -1)
    if case["act"] == "silu":
        sig = 1.0 / (1.0 + (-g).exp())
        a, da = g * sig, sig * (1.0 + g * (1.0 - sig))
    elif case["act"] == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        a, da = g * cdf, cdf + g * (-0.5 * g * g).exp() * (1.0 / math.sqrt(2.0 * math.pi))
    else:
        c = math.sqrt(2.0 / math.pi)
        th = torch.tanh(c * (g + 0.044715 * g * g * g))
        a, da = 0.5 * g * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * g * (1.0 - th * th) * c * (1.0 + 3 * 0.044715 * g * g)
    y = (a * u).to(torch.bfloat16)
    if not case["train"]:
        return {"y": y}
    dy = s["dy"].float()
    dgu = torch.cat([dy * u * da, dy * a], -1)
    return {"y": y, "dx": (dgu @ w).to(torch.bfloat16), "dw": (dgu.t() @ x).to(torch.bfloat16)}


def _own(s):
    case = s["case"]
    if case["op"] == "layer_norm":
        from moodist_b200.ops.train import layer_norm

        y = layer_norm(s["x"], s["w"], s["b"], 1e-5)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if case["op"] == "rotary":
        from moodist_b200.ops.train import rotary

        q, k = rotary(s["q"], s["k"], s["cos"], s["sin"], s["positions"], interleaved=case["interleaved"])
        if not case["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if case["op"] == "distill":
        from moodist_b200.ops.train import distill_loss

        loss = distill_loss(s["logits"], s["ids"], s["top"], s["targets"], temperature=case["tau"], hard_weight=case["hard"],
                            reduction=case["reduction"])
        if not case["train"]:
            return {"loss": loss}
        (dz,) = torch.autograd.grad(loss, (s["logits"],))
        return {"loss": loss, "dlogits": dz}
    from moodist_b200.ops.gemm import gated_linear

    y = gated_linear(s["x"], s["w"], activation=case["act"])
    if not case["train"]:
        return {"y": y}
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        plain = {"layer_norm": _plain_layer_norm, "rotary": _plain_rotary, "distill": _plain_distill, "gated": _plain_gated}
        return plain[state["case"]["op"]](state)


def work(case):
    op, train = case["op"], case["train"]
    if op == "gated":
        t, d, f = case["rows"], case["dim"], case["ffn"]
        # x and w in, y out; training adds the output's gradient in and two gradients out
        fwd = 2 * (t * d + 2 * f * d + t * f)
        return {"bytes": fwd + (2 * (t * f + t * d + 2 * f * d) if train else 0), "flops": (3 if train else 1) * 4 * t * d * f}
    e = BYTES[case["dtype"]]
    if op == "layer_norm":
        n, d = case["rows"] * case["dim"], case["dim"]
        we = e if case["weights"] == "same" else 4
        return {"bytes": 2 * n * e + 2 * d * we + (2 * n * e + 2 * d * we if train else 0), "flops": n * (22 if train else 8)}
    if op == "rotary":
        tokens = case["batch"] * case["seq"]
        n = tokens * (case["heads"] + case["kv"]) * case["dim"]
        rows = min(tokens, case["length"]) if case["positions"] == "far" else min(case["seq"], case["length"])
        table = rows * case["rot"] * 4 + (0 if case["positions"] == "order" else tokens * 8)
        return {"bytes": (4 if train else 2) * n * e + table, "flops": (6 if train else 3) * n * case["rot"] // case["dim"]}
    n, top = case["rows"] * case["vocab"], case["rows"] * case["top"]
    return {"bytes": (2 if train else 1) * n * e + top * (8 + e), "flops": n * ((8 if train else 4) + (4 if case["hard"] > 0 else 0))}


def exact(case, seed):
    s = prepare(case, seed)
    op, train = case["op"], case["train"]
    if op == "layer_norm":
        x, w, b = (s[k].detach().double().requires_grad_(train) for k in ("x", "w", "b"))
        y = torch.nn.functional.layer_norm(x, (case["dim"],), w, b, 1e-5)
        if not train:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    if op == "rotary":
        # a pair is a complex number, the rotation a product with cos + i sin
        b, n, r = case["batch"], case["seq"], case["rot"]
        pos = s["positions"] if s["positions"] is not None else torch.arange(n, device="cuda").repeat(b, 1)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[pos.clamp(min=0)]
        turn[pos < 0] = 1.0

        def rotated(x, by):
            x = x.detach().double().clone()
            lo, hi = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
            v = torch.complex(x[..., lo].clone(), x[..., hi].clone()) * by[:, :, None]
            x[..., lo], x[..., hi] = v.real, v.imag
            return x

        out = {"q": rotated(s["q"], turn), "k": rotated(s["k"], turn)}
        if train:
            out.update(dq=rotated(s["dq"], turn.conj()), dk=rotated(s["dk"], turn.conj()))
        return out
    if op == "distill":
        tau, hard, v = case["tau"], case["hard"], case["vocab"]
        z = s["logits"].detach().double().requires_grad_(train)
        rows = torch.arange(case["rows"], device="cuda")[(s["ids"] >= 0).any(1)]
        if s["targets"] is not None:
            rows = rows[s["targets"][rows] >= 0]
        masked = s["ids"][rows] < 0
        logp = torch.log_softmax((s["top"][rows].double() / tau).masked_fill(masked, -math.inf), -1)
        logq = torch.log_softmax(z[rows] / tau, -1).gather(1, s["ids"][rows].masked_fill(masked, 0))
        loss = (1 - hard) * tau**2 * (logp.exp() * (logp - logq)).masked_fill(masked, 0.0).sum()
        if hard > 0:
            loss = loss + hard * torch.nn.functional.cross_entropy(z[rows], s["targets"][rows], reduction="sum")
        if case["reduction"] == "mean":
            loss = loss / max(1, rows.numel())
        if not train:
            return {"loss": loss.detach()}
        (dz,) = torch.autograd.grad(loss, (z,))
        return {"loss": loss.detach(), "dlogits": dz}
    x, w = (s[k].detach().double().requires_grad_(train) for k in ("x", "w"))
    g, u = x @ w[: case["ffn"]].t(), x @ w[case["ffn"] :].t()
    if case["act"] == "silu":
        y = torch.nn.functional.silu(g) * u
    else:
        y = torch.nn.functional.gelu(g, approximate="tanh" if case["act"] == "gelu_tanh" else "none") * u
    if not train:
        return {"y": y}
    dx, dw = torch.autograd.grad(y, (x, w), s["dy"].double())
    return {"y": y.detach(), "dx": dx, "dw": dw}
