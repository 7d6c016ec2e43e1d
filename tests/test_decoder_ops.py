"""Decoder operators on CPU tensors (layer norm, rotary positions, distillation loss, gated projection): the plain arithmetic
against 64-bit definitions, gradients against differences, and what the entry points refuse."""

import math

import pytest
import torch

import decoder_oracle as oracle
from moodist_b200.ops.gemm import gated_linear
from moodist_b200.ops.train import distill_loss, layer_norm, rotary, rotary_, rotary_tables

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 5, 7), (0, 16), (4, 33)])
def test_layer_norm(shape, dtype):
    torch.manual_seed(0)
    x = torch.randn(shape).to(dtype).requires_grad_()
    w, b = (torch.randn(shape[-1]).to(dtype).requires_grad_() for _ in range(2))
    y, dy = layer_norm(x, w, b, 1e-3), torch.randn(shape).to(dtype)
    assert y.dtype == dtype
    want = oracle.layer_norm(x, w, b, 1e-3, dy)
    oracle.assert_within(y, *want["y"], "y")
    for got, name in zip(torch.autograd.grad(y, (x, w, b), dy), ("dx", "dw", "db")):
        if dtype == torch.float32:  # torch's CPU backward pass of the cast rounds the 16-bit weight gradients elsewhere
            oracle.assert_within(got, *want[name], name)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary(dtype, interleaved):
    torch.manual_seed(1)
    cos, sin = rotary_tables(6, 9)
    q, k = torch.randn(2, 5, 3, 10).to(dtype), torch.randn(2, 5, 1, 10).to(dtype)
    pos = torch.tensor([[0, 8, -1, 9, 3], [4, 4, 4, -7, 1]])
    for p in (pos, pos[0].int(), None):
        for got, x in zip(rotary(q, k, cos, sin, p, interleaved), (q, k)):
            oracle.assert_within(got, *oracle.rotary(x, cos, sin, p, interleaved), "rotary")
    a, b = q.clone(), k.clone()
    rotary_(a, b, cos, sin, pos, interleaved)
    for got, want in zip((a, b), rotary(q, k, cos, sin, pos, interleaved)):
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    only, none = rotary(q[0], None, cos, sin, interleaved=interleaved)
    assert none is None
    oracle.assert_within(only, *oracle.rotary(q[0], cos, sin, None, interleaved), "3-d")


def test_rotary_tables_scalings():
    r, n, theta = 16, 40000, 10000.0
    inv = [theta ** (-2 * j / r) for j in range(r // 2)]
    cos, sin = rotary_tables(r, n, theta)
    # far positions keep their angle: exact to half a step of fp32
    for j, f in enumerate(inv):
        assert abs(float(cos[-1, j]) - math.cos((n - 1) * f)) <= 2.0**-24
        assert abs(float(sin[-1, j]) - math.sin((n - 1) * f)) <= 2.0**-24
    lin, _ = rotary_tables(r, n, theta, scaling="linear", factor=4.0)
    assert torch.equal(lin[4::4][:2000], cos[1:2001])
    c, s = rotary_tables(r, 2, theta, scaling="ntk", factor=4.0)
    angle = torch.atan2(s[1].double(), c[1].double())
    assert abs(float(angle[0]) - inv[0]) < 1e-6 and abs(float(angle[-1]) / (inv[-1] / 4.0) - 1) < 1e-5
    c, s = rotary_tables(r, 2, theta, scaling="by_parts", factor=8.0, original_length=4096, low=1.0, high=4.0)
    angle = torch.atan2(s[1].double(), c[1].double())
    for j, f in enumerate(inv):
        turns = 4096 * f / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / 3.0))
        assert abs(float(angle[j]) / (f * keep + f / 8.0 * (1 - keep)) - 1) < 1e-5
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(length=0), dict(scaling="other"), dict(factor=0.0), dict(theta=-1.0),
                dict(rotary_dim=2, scaling="ntk"), dict(scaling="by_parts"), dict(scaling="by_parts", original_length=8, low=4.0)):
        with pytest.raises(ValueError):
            rotary_tables(**{"rotary_dim": 8, "length": 4, **bad})


def distill_case(rows, V, K, dtype, device="cpu", seed=0):
    """Rows of every kind: full, padded, with a word twice, masked by -inf, empty, without target; NaN in masked places."""
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, V, generator=g) * 2).to(dtype)
    ids = torch.randint(0, V, (rows, K), generator=g)
    top = torch.randn(rows, K, generator=g).to(dtype)
    targets = torch.randint(0, V, (rows,), generator=g)
    if rows > 1:
        ids[1, :] = -1
        top[1, :] = float("nan")
        z[1, 0] = float("nan")  # a row left out may hold anything
    if rows > 2:
        targets[2] = -100
        z[2, -1] = float("inf")
    if rows > 3:
        ids[3, K // 2 :] = V + 5
        ids[3, 0] = 0
        top[3, K // 2 :] = float("nan")
    if rows > 4:
        ids[4, :] = int(ids[4, 0])
        targets[4] = int(ids[4, 0])
    if rows > 5:
        top[5, 1:] = -float("inf")
        z[5] = torch.where(torch.arange(V) % 3 == 0, z[5], -float("inf"))
        ids[5, 0] = 0
        targets[5] = 0
    if rows > 6:
        top[6, 1:] = torch.finfo(dtype).min
    if rows > 7:
        targets[7] = V
    return [t.to(device) for t in (z, ids, top, targets)]


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("tau,hard", [(1.0, 0.0), (2.0, 0.3), (0.5, 1.0)])
def test_distill_loss(tau, hard, reduction):
    z, ids, top, targets = distill_case(12, 37, 5, torch.float32)
    z.requires_grad_()
    loss = distill_loss(z, ids, top, targets, temperature=tau, hard_weight=hard, reduction=reduction, scale=1.5)
    want = oracle.distill(z, ids, top, targets, tau, hard, reduction, scale=1.5)
    oracle.assert_within(loss, *want["loss"], "loss")
    (dz,) = torch.autograd.grad(loss, z)
    oracle.assert_within(dz, *want["dz"], "dz")


def test_distill_loss_without_any_row():
    z, ids, top, _ = distill_case(3, 11, 2, torch.float32)
    z.requires_grad_()
    loss = distill_loss(z, torch.full_like(ids, -1), top)
    assert loss.item() == 0 and float(torch.autograd.grad(loss, z)[0].abs().max()) == 0


def test_distill_gradient_against_differences():
    z, ids, top, targets = distill_case(1, 19, 4, torch.float32)
    z.requires_grad_()

    def f(v):
        return oracle.distill(v, ids, top, targets, 2.0, 0.4, "mean")["loss"][0]

    (dz,) = torch.autograd.grad(distill_loss(z, ids, top, targets, temperature=2.0, hard_weight=0.4), z)
    step, base = 1e-4, z.detach().double()
    for j in range(19):
        d = torch.zeros_like(base)
        d[0, j] = step
        # a central difference is off by step^2 times the third derivative (at most 1), and 1e-12 of rounding over the step
        assert abs(float(dz[0, j]) - float(f(base + d) - f(base - d)) / (2 * step)) < 1e-6


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated_linear(act):
    torch.manual_seed(2)
    x, w = torch.randn(2, 3, 16).bfloat16(), (torch.randn(48, 16) * 0.3).bfloat16()
    h = gated_linear(x, w, act)
    want = oracle.gated(x, w, act)["h"]
    oracle.assert_within(h.reshape(-1, 24), *want, "h")


def test_refusals():
    refused = pytest.raises(RuntimeError, match="moodist")
    x = torch.randn(4, 8)
    for bad in (dict(weight=torch.ones(7)), dict(weight=torch.ones(8, 1)), dict(weight=torch.ones(8).half()), dict(eps=-1.0),
                dict(weight=torch.ones(8), bias=torch.ones(8).bfloat16()), dict(weight=torch.ones(8, dtype=torch.float64))):
        with refused:
            layer_norm(x, **bad)
    for bad in (x.double(), x.long(), torch.randn(4, 0), torch.tensor(1.0)):
        with refused:
            layer_norm(bad)

    cos, sin = rotary_tables(8, 6)
    q, k = torch.randn(2, 4, 3, 8), torch.randn(2, 4, 1, 8)
    for bad in (dict(q=q.double()), dict(q=q[0, 0]), dict(k=k[:, :3]), dict(k=k.half()), dict(k=k[..., :6]), dict(k=k[0]),
                dict(cos=cos[:, :3]), dict(cos=cos.half(), sin=sin.half()), dict(cos=cos[:0], sin=sin[:0]), dict(cos=cos.t(), sin=sin.t()),
                dict(cos=cos.clone().requires_grad_()), dict(q=q[..., :6], k=k[..., :6]), dict(positions=torch.zeros(2, 4)),
                dict(positions=torch.zeros(3, dtype=torch.long)), dict(positions=torch.zeros(4, 2, dtype=torch.long)),
                dict(q=torch.randn(1, 7, 1, 8), k=None)):
        args = {"q": q, "k": k, "cos": cos, "sin": sin, "positions": None, **bad}
        with refused:
            rotary(**args)
    for a, b in ((q.clone().requires_grad_(), k), (q[:, :, :1].expand(2, 4, 3, 8), k), (q.transpose(2, 3).contiguous().transpose(2, 3), k), (q, q)):
        with refused:
            rotary_(a, b, cos, sin)

    z, ids, top, t = torch.randn(3, 9), torch.zeros(3, 2, dtype=torch.long), torch.randn(3, 2), torch.zeros(3, dtype=torch.long)
    for bad in (dict(logits=z.double()), dict(teacher_ids=ids.float()), dict(teacher_ids=ids[:2]), dict(teacher_logits=top[:, :1]),
                dict(teacher_ids=ids[:, :0], teacher_logits=top[:, :0]), dict(teacher_logits=top.double()), dict(temperature=0.0),
                dict(temperature=float("nan")), dict(hard_weight=1.5), dict(hard_weight=0.5, targets=None), dict(targets=t.int()),
                dict(targets=t[:2]), dict(teacher_logits=top.clone().requires_grad_()), dict(teacher_ids=ids[0], teacher_logits=top[0])):
        args = {"logits": z, "teacher_ids": ids, "teacher_logits": top, "targets": t, **bad}
        with refused:
            distill_loss(**args)
    with pytest.raises(ValueError):
        distill_loss(z, ids, top, reduction="none")

    x, w = torch.randn(2, 8).bfloat16(), torch.randn(16, 8).bfloat16()
    for bad in (dict(activation="relu"), dict(x=x.float()), dict(w=w.float()), dict(w=w[:15]), dict(w=w[:8]), dict(w=w[0]),
                dict(x=x[:, :4]), dict(x=torch.randn(2, 6).bfloat16(), w=torch.randn(16, 6).bfloat16()), dict(x=torch.randn(2, 0).bfloat16(), w=w[:, :0])):
        with refused:
            gated_linear(**{"x": x, "w": w, **bad})


def test_sizes_beyond_the_kernels_counters_are_refused():
    wide = torch.zeros(1, 8).bfloat16()
    with pytest.raises(RuntimeError, match="moodist gated_linear"):
        gated_linear(wide, wide.expand(2**31, 8))
    cos, sin = rotary_tables(2, 1)
    for shape in ((1, 1, 2**20 + 1, 2), (1, 1, 1, 2**20 + 2)):
        with pytest.raises(RuntimeError, match="moodist rotary"):
            rotary(torch.zeros(1, 1, 1, 1).expand(shape), None, cos, sin)
    with pytest.raises(RuntimeError, match="moodist rotary"):
        rotary(torch.zeros(1, 1, 1, 2), torch.zeros(1, 1, 1, 2).expand(1, 1, 2**20 + 1, 2), cos, sin)
