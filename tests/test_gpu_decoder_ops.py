"""Decoder operators on the GPU: kernels against 64-bit definitions over types, sizes, strides, masks and streams, a decoder
block made of them, captured and replayed passes."""

import pytest
import torch

import decoder_oracle as oracle
from test_decoder_ops import distill_case

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _randn(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, device="cuda") * scale + shift).to(dtype)


# ---- layer norm ----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 7), (0, 16), (5, 256), (37, 1000), (130, 1537), (777, 4096), (64, 8192), (9, 16392), (3, 40001),
                                    (5000, 24), (1200, 512)])
def test_layer_norm(rows, D, dtype):
    from moodist_b200.ops.train import layer_norm

    torch.manual_seed(rows + D)
    x = _randn(rows, D, dtype=dtype, scale=2.0, shift=1.0).requires_grad_()
    dy = _randn(rows, D, dtype=dtype)
    for wt in {dtype, torch.float32}:
        w, b = (_randn(D, dtype=wt).requires_grad_() for _ in range(2))
        y = layer_norm(x, w, b, 1e-5)
        want = oracle.layer_norm(x, w, b, 1e-5, dy)
        oracle.assert_within(y, *want["y"], "y")
        for got, name in zip(torch.autograd.grad(y, (x, w, b), dy), ("dx", "dw", "db")):
            oracle.assert_within(got, *want[name], name)
        with torch.no_grad():
            assert torch.equal(layer_norm(x, w, b, 1e-5), y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_layouts(dtype):
    from moodist_b200.ops.train import layer_norm

    torch.manual_seed(7)
    base = _randn(6, 5, 80, dtype=dtype, shift=30.0)
    w = _randn(64, dtype=dtype)
    odd = _randn(6 * 64 + 1, dtype=dtype)[1:].view(6, 64)  # starts off a vector boundary
    for x in (base[..., :64], base[..., 3:67], base.transpose(0, 1)[..., 8:72], base[:1, :, :64].expand(6, 5, 64),
              _randn(64, 6, dtype=dtype).t(), odd):
        for weight, bias in ((None, None), (w, None), (None, w), (w[:1].expand(64), None)):
            leaves = [t for t in (x, weight, bias) if t is not None]
            x_ = x.detach().requires_grad_()
            w_, b_ = (None if t is None else t.detach().requires_grad_() for t in (weight, bias))
            y = layer_norm(x_, w_, b_, 1e-5)
            dy = _randn(*x.shape, dtype=dtype).transpose(0, -2 if x.dim() > 2 else 0)
            dy = dy if dy.shape == y.shape else torch.ones((), device="cuda", dtype=dtype).expand(y.shape)
            want = oracle.layer_norm(x, weight, bias, 1e-5, dy)
            oracle.assert_within(y, *want["y"], "y")
            names = [n for n, t in (("dx", x_), ("dw", w_), ("db", b_)) if t is not None]
            for got, name in zip(torch.autograd.grad(y, [t for t in (x_, w_, b_) if t is not None], dy), names):
                oracle.assert_within(got, *want[name], name)
            assert leaves


def test_layer_norm_partial_gradients_and_refusals():
    from moodist_b200.ops.train import layer_norm

    x, w, b = _randn(9, 40), _randn(40), _randn(40)
    dy = _randn(9, 40)
    want = oracle.layer_norm(x, w, b, 1e-5, dy)
    for i, name in enumerate(("dx", "dw", "db")):
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        y = layer_norm(*leaves)
        oracle.assert_within(torch.autograd.grad(y, leaves[i], dy)[0], *want[name], name)
    with pytest.raises(RuntimeError, match="moodist layer_norm.*once"):
        torch.autograd.grad(layer_norm(x.requires_grad_(), w), x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="device"):
        layer_norm(x, w.cpu())
    # the same inputs give the same bits
    big, bw = _randn(3000, 1000).requires_grad_(), _randn(1000).requires_grad_()
    one, two = (torch.autograd.grad(layer_norm(big, bw).square().sum(), (big, bw)) for _ in range(2))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer_norm_wide_weights_on_16_byte_boundaries(dtype):
    """fp32 weights that start 16 but not 32 bytes from a boundary, beside 16-bit rows that are read in vectors."""
    from moodist_b200.ops.train import layer_norm

    torch.manual_seed(8)
    for D in (64, 1024, 4096, 16384):
        x, dy = _randn(20, D, dtype=dtype), _randn(20, D, dtype=dtype)
        w, b = (_randn(D + 4)[4:].requires_grad_() for _ in range(2))
        x.requires_grad_()
        y = layer_norm(x, w, b)
        want = oracle.layer_norm(x, w, b, 1e-5, dy)
        oracle.assert_within(y, *want["y"], "y")
        for got, name in zip(torch.autograd.grad(y, (x, w, b), dy), ("dx", "dw", "db")):
            oracle.assert_within(got, *want[name], name)


def test_changes_between_forward_and_backward_are_noticed():
    """What the backward pass reads must not have been written since, views of it included."""
    from moodist_b200.ops.gemm import gated_linear
    from moodist_b200.ops.train import distill_loss, layer_norm, rotary, rotary_tables

    def changed(make, touch):
        out = make()
        with torch.no_grad():
            touch.add_(1)
        with pytest.raises(RuntimeError, match="inplace"):
            out.sum().backward()

    x3, w = _randn(2, 3, 16), _randn(16).requires_grad_()
    changed(lambda: layer_norm(x3, w), x3)
    changed(lambda: layer_norm(x3, w), w)
    x, wg = _randn(2, 3, 16, dtype=torch.bfloat16).requires_grad_(), _randn(32, 16, dtype=torch.bfloat16).requires_grad_()
    changed(lambda: gated_linear(x, wg), x)
    changed(lambda: gated_linear(x, wg), wg)
    cos, sin = rotary_tables(8, 4, device="cuda")
    changed(lambda: rotary(x3.view(2, 3, 2, 8).requires_grad_(), None, cos, sin)[0], cos)
    z = _randn(2, 3, 16, dtype=torch.float16).requires_grad_()
    ids, top = torch.zeros(2, 3, 2, device="cuda", dtype=torch.long), _randn(2, 3, 2)
    changed(lambda: distill_loss(z, ids, top), z)
    # bf16 logits are done with once the loss is there
    z = _randn(2, 3, 16, dtype=torch.bfloat16).requires_grad_()
    want = torch.autograd.grad(distill_loss(z, ids, top), z)[0]
    loss = distill_loss(z, ids, top)
    with torch.no_grad():
        z.zero_()
    assert torch.equal(torch.autograd.grad(loss, z)[0], want)


# ---- rotary positions ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,S,H,KV,D,R", [(1, 1, 1, 1, 2, 2), (2, 96, 8, 2, 128, 128), (3, 17, 5, 5, 80, 32), (64, 1, 32, 8, 128, 64),
                                          (1, 7, 3, 1, 36, 12), (2, 5, 2, 1, 7, 6), (0, 4, 2, 1, 8, 8), (1, 2050, 4, 2, 64, 64)])
def test_rotary(B, S, H, KV, D, R, dtype, interleaved):
    from moodist_b200.ops.train import rotary, rotary_, rotary_tables

    torch.manual_seed(S + D)
    length = max(S, 70)
    cos, sin = rotary_tables(R, length, device="cuda")
    qkv = _randn(B, S, H + 2 * KV, D, dtype=dtype)
    q, k = qkv[:, :, :H], qkv[:, :, H : H + KV]  # views of the fused projection
    pos = torch.randint(-2, length + 1, (B, S), device="cuda")
    for p in (pos, pos[0] if B else None, pos.int(), None):
        q_, k_ = q.detach().requires_grad_(), k.detach().requires_grad_()
        got = rotary(q_, k_, cos, sin, p, interleaved)
        for x, y in zip((q, k), got):
            oracle.assert_within(y, *oracle.rotary(x, cos, sin, p, interleaved), "rotary")
        dq, dk = _randn(*q.shape, dtype=dtype), _randn(B, KV, S, D, dtype=dtype).transpose(1, 2)
        grads = torch.autograd.grad(got, (q_, k_), (dq, dk))
        for g, x in zip(grads, (dq, dk)):
            oracle.assert_within(g, *oracle.rotary(x, cos, sin, p, interleaved, inverse=True), "gradient")
    # in place: the same bits, and nothing else of the fused rows changes
    want = rotary(q, k, cos, sin, pos, interleaved)
    rest = qkv[:, :, H + KV :].clone()
    rotary_(q, k, cos, sin, pos, interleaved)
    for y, x in zip(want, (q, k)):
        assert torch.equal(y.nan_to_num(5.0), x.nan_to_num(5.0))
    assert torch.equal(qkv[:, :, H + KV :], rest)


def test_rotary_single_uses_and_refusals():
    from moodist_b200.ops.train import rotary, rotary_, rotary_tables

    cos, sin = rotary_tables(8, 16, device="cuda")
    q, k = _randn(5, 3, 8).requires_grad_(), _randn(5, 1, 8).requires_grad_()
    a, b = rotary(q, k, cos, sin)
    dq, dk = torch.autograd.grad(a.sum(), (q, k), allow_unused=True)  # only one result used, its gradient expanded
    oracle.assert_within(dq, *oracle.rotary(torch.ones_like(q), cos, sin, None, False, inverse=True), "dq")
    assert dk is None or not dk.any()
    shared = _randn(5, 1, 8).requires_grad_()
    (g,) = torch.autograd.grad(rotary(shared.expand(5, 4, 8), None, cos, sin)[0].sum(), shared)
    value, bound = oracle.rotary(torch.ones(5, 1, 8, device="cuda"), cos, sin, None, False, inverse=True)
    oracle.assert_within(g, 4 * value, 8 * bound + 1e-6, "broadcast input")
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(rotary(q, k, cos, sin)[0].sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="gradient"):
        rotary_(q, None, cos, sin)
    with pytest.raises(RuntimeError, match="device"):
        rotary(q, None, cos.cpu(), sin.cpu())
    # infinities in padded tokens stay theirs
    x = torch.full((2, 1, 8), float("inf"), device="cuda")
    assert torch.equal(rotary(x, None, cos, sin, torch.tensor([-1, -5], device="cuda"))[0], x)
    # tables of an odd alignment
    c, s = torch.cat([cos.new_zeros(1), cos.reshape(-1)])[1:].view_as(cos), torch.cat([cos.new_zeros(1), sin.reshape(-1)])[1:].view_as(sin)
    assert torch.equal(rotary(q, None, c, s)[0], rotary(q, None, cos, sin)[0])


# ---- distillation loss --------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,K", [(1, 1, 1), (9, 37, 5), (12, 1000, 8), (10, 1003, 300), (8, 50257, 64), (9, 128256, 16), (0, 64, 4)])
def test_distill_loss(rows, V, K, dtype):
    from moodist_b200.ops.train import distill_loss

    z, ids, top, targets = distill_case(rows, V, K, dtype, "cuda", seed=V)
    for tau, hard, reduction, t in ((1.0, 0.0, "mean", None), (2.0, 0.3, "sum", targets), (0.7, 0.0, "mean", targets), (1.0, 1.0, "sum", targets)):
        if t is None:  # the rows whose logits may hold anything are left out through their target only
            z = z.nan_to_num(0.5, 0.5, -float("inf"))
        z.requires_grad_()
        loss = distill_loss(z, ids, top, t, temperature=tau, hard_weight=hard, reduction=reduction, scale=0.75)
        want = oracle.distill(z, ids, top, t, tau, hard, reduction, scale=0.75)
        oracle.assert_within(loss, *want["loss"], "loss")
        (dz,) = torch.autograd.grad(loss, z)
        oracle.assert_within(dz, *want["dz"], "dz")
        with torch.no_grad():
            assert torch.equal(distill_loss(z, ids, top, t, temperature=tau, hard_weight=hard, reduction=reduction, scale=0.75), loss)
        z = z.detach()


@pytest.mark.parametrize("rows,V,K,dtype", [(400, 9001, 3, torch.bfloat16), (310, 8200, 5, torch.float16), (40, 20000, 1100, torch.float32),
                                            (3000, 72, 9, torch.bfloat16), (150, 40000, 2, torch.float32)])
def test_distill_many_rows(rows, V, K, dtype):
    """More rows than CTAs, rows that do not count among them, entries beyond what is compared in shared memory."""
    from moodist_b200.ops.train import distill_loss

    z, ids, top, targets = distill_case(rows, V, K, dtype, "cuda", seed=rows)
    out = torch.rand(rows, device="cuda") < 0.3
    ids[out & (torch.arange(rows, device="cuda") % 2 == 0)] = V + 1
    targets[out & (torch.arange(rows, device="cuda") % 2 == 1)] = -100
    z.requires_grad_()
    for tau, hard, reduction in ((2.0, 0.5, "mean"), (1.0, 0.0, "sum")):
        loss = distill_loss(z, ids, top, targets, temperature=tau, hard_weight=hard, reduction=reduction)
        want = oracle.distill(z, ids, top, targets, tau, hard, reduction)
        oracle.assert_within(loss, *want["loss"], "loss")
        (dz,) = torch.autograd.grad(loss, z)
        oracle.assert_within(dz, *want["dz"], "dz")


@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_layouts_types_and_incoming_gradient(dtype):
    from moodist_b200.ops.train import distill_loss

    z, ids, top, targets = distill_case(10, 1000, 6, dtype, "cuda", seed=3)
    want = oracle.distill(z, ids, top, targets, 2.0, 0.25, "mean")
    wide = torch.zeros(10, 1024, device="cuda", dtype=dtype)
    odd = torch.zeros(10, 1001, device="cuda", dtype=dtype)
    wide[:, :1000], odd[:, 1:] = z, z
    for form in (z.view(2, 5, 1000), wide[:, :1000], odd[:, 1:], z.t().contiguous().t()):
        lead = form.shape[:-1]
        x = form.detach().requires_grad_()
        for i, p in ((ids, top), (ids.int(), top.float()), (ids.flip(1).contiguous().flip(1), top.bfloat16() if dtype == torch.bfloat16 else top)):
            loss = distill_loss(x, i.view(*lead, 6) if i.is_contiguous() else i.reshape(*lead, 6), p.reshape(*lead, 6), targets.view(lead),
                                temperature=2.0, hard_weight=0.25)
            oracle.assert_within(loss, *want["loss"], "loss")
            (dz,) = torch.autograd.grad(loss * 3.0, x)
            value, bound = want["dz"]
            # one more rounding where the gradient is scaled after it was written
            oracle.assert_within(dz.reshape(10, 1000), 3 * value, 6 * bound, "3 dz")


def test_distill_refusals_and_repeated_backward():
    from moodist_b200.ops.train import distill_loss

    z, ids, top, targets = distill_case(4, 64, 3, torch.float32, "cuda")
    z.requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(distill_loss(z, ids, top, targets), z, create_graph=True)
    with pytest.raises(RuntimeError, match="device"):
        distill_loss(z, ids.cpu(), top, targets)
    before = z.detach().clone()
    torch.autograd.grad(distill_loss(z, ids, top, targets), z)
    assert torch.equal(z.detach().nan_to_num(1.0), before.nan_to_num(1.0))  # the logits stay
    # one backward pass per forward pass, fp16 apart, whose gradient is not made beforehand
    for dtype in DTYPES:
        x = before.to(dtype).requires_grad_()
        loss = distill_loss(x, ids, top, targets)
        torch.autograd.grad(loss, x, retain_graph=True)
        if dtype == torch.float16:
            torch.autograd.grad(loss, x)
        else:
            with pytest.raises(RuntimeError, match="taken already"):
                torch.autograd.grad(loss, x)


# ---- gated projection ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("T,F,K", [(1, 8, 8), (0, 16, 16), (3, 200, 72), (17, 1000, 1016), (127, 136, 64), (128, 128, 512), (129, 264, 256), (301, 328, 200),
                                   (1000, 520, 264), (5, 264, 4096), (128, 1000, 1024), (100, 1184, 2056), (33, 10008, 256), (3, 19000, 136)])
def test_gated_linear(T, F, K, act):
    from moodist_b200.ops.gemm import gated_linear

    torch.manual_seed(T + F)
    x = _randn(T, K, dtype=torch.bfloat16).requires_grad_()
    w = _randn(2 * F, K, dtype=torch.bfloat16, scale=K**-0.5).requires_grad_()
    dh = _randn(T, F, dtype=torch.bfloat16)
    h = gated_linear(x, w, act)
    want = oracle.gated(x, w, act, dh)
    oracle.assert_within(h, *want["h"], "h")
    for got, name in zip(torch.autograd.grad(h, (x, w), dh), ("dx", "dw")):
        oracle.assert_within(got, *want[name], name)
        value = want[name][0]
        # four roundings to bf16 lie between the inputs and a gradient
        assert T == 0 or (got.double() - value).norm() <= 4 * 2.0**-8 * value.norm()
    with torch.no_grad():
        assert torch.equal(gated_linear(x, w, act), h)


def test_gated_linear_layouts_and_refusals():
    from moodist_b200.ops.gemm import gated_linear

    torch.manual_seed(5)
    base, wide = _randn(4, 9, 96, dtype=torch.bfloat16), _randn(48, 96, dtype=torch.bfloat16, scale=0.1)
    for x, w in ((base[..., :64], wide[:, :64]), (base[..., 4:68], wide[:, 3:67]), (base.transpose(0, 1)[..., 8:72], wide[:, :64]),
                 (base[:1, :, :64].expand(4, 9, 64), wide[:, 8:72]), (base[0, 0, :64], wide[:, :64]),
                 (_randn(64, 9, dtype=torch.bfloat16).t(), wide.t().contiguous().t()[:, :64])):
        x_, w_ = x.detach().requires_grad_(), w.detach().requires_grad_()
        h = gated_linear(x_, w_)
        assert h.shape == (*x.shape[:-1], 24)
        for dh in (_randn(*h.shape, dtype=torch.bfloat16), torch.ones((), device="cuda", dtype=torch.bfloat16).expand(h.shape)):
            want = oracle.gated(x, w, "silu", dh)
            oracle.assert_within(h.reshape(-1, 24), *want["h"], "h")
            dx, dw = torch.autograd.grad(h, (x_, w_), dh, retain_graph=True)
            oracle.assert_within(dx.reshape(-1, 64), *want["dx"], "dx")
            oracle.assert_within(dw, *want["dw"], "dw")
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(gated_linear(x_, w_).sum(), x_, create_graph=True)
    with pytest.raises(RuntimeError, match="device"):
        gated_linear(x_, w_.cpu())


# ---- more than 2^31 elements ----------------------------------------------------------------------------------------


def test_offsets_beyond_32_bits():
    """The last rows of tensors of more than 2^31 elements, against the same rows on their own."""
    from moodist_b200.ops.train import distill_loss, layer_norm, rotary, rotary_tables

    def big(*shape):
        return torch.empty(*shape, device="cuda", dtype=torch.bfloat16).normal_()

    x = big(140000, 16384)
    w = _randn(16384, dtype=torch.bfloat16)
    dy = x[-1:].expand(140000, 16384)
    x.requires_grad_()
    y = layer_norm(x, w)
    (dx,) = torch.autograd.grad(y, x, dy)
    last = x.detach()[-3:].clone().requires_grad_()
    y3 = layer_norm(last, w)
    assert torch.equal(y[-3:], y3) and torch.equal(dx[-3:], torch.autograd.grad(y3, last, dy[-3:])[0])
    del x, y, dx, dy

    q = big(2, 150000, 64, 128)
    cos, sin = rotary_tables(128, 150000, device="cuda")
    a, _ = rotary(q, None, cos, sin)
    at = torch.arange(149997, 150000, device="cuda")
    assert torch.equal(a[1:, -3:], rotary(q[1:, -3:], None, cos, sin, at)[0])
    del q, a

    z = big(17000, 128256).requires_grad_()
    ids, top = torch.randint(0, 128256, (17000, 4), device="cuda"), _randn(17000, 4)
    (dz,) = torch.autograd.grad(distill_loss(z, ids, top, reduction="sum"), z)
    last = z.detach()[-160:].clone().requires_grad_()
    (d3,) = torch.autograd.grad(distill_loss(last, ids[-160:], top[-160:], reduction="sum"), last)
    assert torch.equal(dz[-160:], d3)


# ---- together -----------------------------------------------------------------------------------------------------


class _Block:
    """A pre-norm decoder block and head of the operators, as a user strings them together."""

    def __init__(self, dim=256, heads=4, kv=2, ffn=512, vocab=1000, rot=32):
        from moodist_b200.ops.train import rotary_tables

        g = torch.Generator(device="cuda").manual_seed(11)

        def weight(*shape, scale):
            return (torch.randn(*shape, device="cuda", generator=g) * scale).bfloat16().requires_grad_()

        self.heads, self.kv, self.hd = heads, kv, dim // heads
        self.n1, self.b1, self.n2, self.b2 = (weight(dim, scale=0.1) for _ in range(4))
        self.wqkv, self.wo = weight((heads + 2 * kv) * self.hd, dim, scale=0.06), weight(dim, dim, scale=0.06)
        self.w13, self.w2, self.head = weight(2 * ffn, dim, scale=0.06), weight(dim, ffn, scale=0.04), weight(vocab, dim, scale=0.06)
        self.cos, self.sin = rotary_tables(rot, 512, scaling="by_parts", factor=4.0, original_length=128, device="cuda")

    def leaves(self):
        return [self.n1, self.b1, self.n2, self.b2, self.wqkv, self.wo, self.w13, self.w2, self.head]

    def loss(self, x, positions, ids, top, targets):
        from moodist_b200.ops.gemm import gated_linear, linear
        from moodist_b200.ops.train import distill_loss, layer_norm, rotary

        B, S, dim = x.shape
        qkv = linear(layer_norm(x, self.n1, self.b1), self.wqkv).view(B, S, -1, self.hd)
        q, k = rotary(qkv[:, :, : self.heads], qkv[:, :, self.heads : self.heads + self.kv], self.cos, self.sin, positions)
        v = qkv[:, :, self.heads + self.kv :]
        o = torch.nn.functional.scaled_dot_product_attention(*(t.transpose(1, 2) for t in (q, k, v)), is_causal=True, enable_gqa=True)
        x = x + linear(o.transpose(1, 2).reshape(B, S, dim), self.wo)
        x = x + linear(gated_linear(layer_norm(x, self.n2, self.b2), self.w13), self.w2)
        return distill_loss(linear(x, self.head), ids, top, targets, temperature=2.0, hard_weight=0.5)

    def reference(self, x, positions, ids, top, targets):
        """The same block in fp64 torch arithmetic; returns loss and gradients."""
        leaves = [t.detach().double().requires_grad_() for t in self.leaves()]
        n1, b1, n2, b2, wqkv, wo, w13, w2, head = leaves
        B, S, dim = x.shape
        x = x.double()
        F = torch.nn.functional
        qkv = (F.layer_norm(x, (dim,), n1, b1) @ wqkv.t()).view(B, S, -1, self.hd)
        half = self.cos.shape[1]
        c, s = (t.double()[positions.clamp(min=0)][:, :, None] for t in (self.cos, self.sin))

        def turn(t):
            a, b, rest = t[..., :half], t[..., half : 2 * half], t[..., 2 * half :]
            return torch.where((positions < 0)[..., None, None], t, torch.cat([a * c - b * s, b * c + a * s, rest], -1))

        q, k, v = turn(qkv[:, :, : self.heads]), turn(qkv[:, :, self.heads : self.heads + self.kv]), qkv[:, :, self.heads + self.kv :]
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        k, v = (t.repeat_interleave(self.heads // self.kv, 1) for t in (k, v))
        a = (q @ k.transpose(-1, -2) / self.hd**0.5).masked_fill(torch.ones(S, S, device="cuda").triu(1).bool(), -float("inf"))
        x = x + (a.softmax(-1) @ v).transpose(1, 2).reshape(B, S, dim) @ wo.t()
        g, u = (F.layer_norm(x, (dim,), n2, b2) @ w13.t()).chunk(2, -1)
        x = x + (F.silu(g) * u) @ w2.t()
        z = (x @ head.t()).reshape(B * S, -1)
        ids, top, t = ids.reshape(B * S, -1), top.reshape(B * S, -1).double(), targets.reshape(-1)
        live = (ids >= 0).any(-1) & (t >= 0)
        z, ids, top, t = z[live], ids[live], top[live], t[live]
        logp = torch.log_softmax((top / 2).masked_fill(ids < 0, -float("inf")), -1)
        logq = torch.log_softmax(z / 2, -1).gather(1, ids.clamp(min=0))
        kl = (logp.exp() * (logp - logq)).masked_fill(ids < 0, 0.0).sum(-1)
        loss = (0.5 * 4 * kl + 0.5 * F.cross_entropy(z, t, reduction="none")).mean()
        return loss, torch.autograd.grad(loss, leaves)


def _batch(seed, B=2, S=61, dim=256, vocab=1000, K=7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, S, dim, device="cuda", generator=g).bfloat16()
    length = torch.randint(1, S + 1, (B, 1), device="cuda", generator=g)
    order = torch.arange(S, device="cuda").expand(B, S)
    positions = torch.where(order < length, order, -1)
    ids = torch.randint(0, vocab, (B, S, K), device="cuda", generator=g)
    ids[order >= length] = -1
    ids[:, 0, 2:] = -1
    targets = torch.randint(0, vocab, (B, S), device="cuda", generator=g)
    targets[order >= length] = -100
    return x, positions, ids, torch.randn(B, S, K, device="cuda", generator=g), targets


def test_decoder_block_gradients():
    block = _Block()
    batch = _batch(0)
    loss = block.loss(*batch)
    grads = torch.autograd.grad(loss, block.leaves())
    ref, want = block.reference(*batch)
    # bf16 activations between some ten operators, each rounding by 2^-8 at most
    assert abs(loss.item() - ref.item()) <= 10 * 2.0**-8 * abs(ref.item())
    for got, value in zip(grads, want):
        assert (got.double() - value).norm() <= 16 * 2.0**-8 * value.norm()


def test_decoder_block_captured_and_replayed():
    """The whole pass, backward included, in a CUDA graph: replays over new inputs give the eager results, and two graphs
    replayed on two streams do not touch each other."""
    block = _Block()
    side = torch.cuda.Stream()

    def passed(held):
        # nothing of the autograd graph outlives the call
        loss = block.loss(*held)
        return torch.autograd.grad(loss, block.leaves()), loss.detach()

    def captured(seed):
        held = [t.clone() for t in _batch(seed)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                passed(held)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            grads, loss = passed(held)
        return graph, held, loss, grads

    graphs = [captured(seed) for seed in (1, 2)]
    streams = [torch.cuda.Stream() for _ in graphs]
    for seeds in ((3, 4), (5, 6)):
        for (graph, held, _, _), stream, seed in zip(graphs, streams, seeds):
            for into, new in zip(held, _batch(seed)):
                into.copy_(new)
        torch.cuda.synchronize()
        for _ in range(3):
            for (graph, _, _, _), stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, _, loss, grads), seed in zip(graphs, seeds):
            eager_grads, eager = passed(_batch(seed))
            assert torch.equal(loss, eager)
            for got, value in zip(grads, eager_grads):
                assert (got.double() - value.double()).norm() <= 2.0**-7 * value.double().norm()  # attention's library backward may reorder


def test_capture_beside_an_eager_graph_of_the_same_leaves():
    """A captured backward pass whose leaves an eager graph of the default stream still holds cannot be joined: it is refused
    by each operator, and runs once that graph is gone. One of another stream may live on."""
    from moodist_b200.ops.gemm import gated_linear
    from moodist_b200.ops.train import distill_loss, layer_norm, rotary, rotary_tables

    cos, sin = rotary_tables(32, 16, device="cuda")
    ids, top = torch.randint(0, 64, (16, 4), device="cuda"), _randn(16, 4)
    x = _randn(16, 64, dtype=torch.bfloat16).requires_grad_()
    w = _randn(64, 64, dtype=torch.bfloat16).requires_grad_()
    calls = (lambda: layer_norm(x), lambda: rotary(x.view(16, 2, 32), None, cos, sin)[0], lambda: distill_loss(x, ids, top),
             lambda: distill_loss(x.half(), ids, top), lambda: gated_linear(x, w))

    def captured(call):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = torch.autograd.grad(call().float().sum(), x)[0]
        return graph, out

    for call in (calls[0], calls[2], calls[4]):  # x is the operator's own leaf
        kept = call()
        want = torch.autograd.grad(call().float().sum(), x)[0]
        with pytest.raises(RuntimeError, match="default stream"):
            captured(call)
        del kept
        graph, out = captured(call)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    side = torch.cuda.Stream()
    for call in calls:
        want = torch.autograd.grad(call().float().sum(), x)[0]
        torch.cuda.synchronize()
        graph, out = captured(call)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        with torch.cuda.stream(side):
            kept = call()
        torch.cuda.synchronize()
        graph, out = captured(call)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del kept


def test_operators_on_a_side_stream():
    """Each operator runs on the stream that is current, in order with what was queued there before."""
    from moodist_b200.ops.gemm import gated_linear
    from moodist_b200.ops.train import distill_loss, layer_norm, rotary, rotary_tables

    cos, sin = rotary_tables(64, 64, device="cuda")
    x, w = _randn(64, 512, dtype=torch.bfloat16), _randn(1024, 512, dtype=torch.bfloat16, scale=0.05)
    ids, top = torch.randint(0, 512, (64, 4), device="cuda"), _randn(64, 4)

    def work(t):
        t = t.detach().requires_grad_()
        y = gated_linear(layer_norm(t), w)
        q, _ = rotary(y.view(64, 8, 64), None, cos, sin)
        loss = distill_loss(q.reshape(64, 512), ids, top)
        return loss, torch.autograd.grad(loss, t)[0]

    want = work(x * 2)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        late = torch.zeros_like(x)
        torch.cuda._sleep(20_000_000)  # 10 ms: work on another stream would read the zeros
        late.copy_(x * 2)
        got = work(late)
    stream.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.multigpu
def test_operators_on_another_device_than_the_current_one():
    from moodist_b200.ops.gemm import gated_linear
    from moodist_b200.ops.train import distill_loss, layer_norm, rotary, rotary_tables

    results = []
    for device in ("cuda:0", "cuda:1"):
        g = torch.Generator().manual_seed(9)
        x = torch.randn(300, 512, generator=g).bfloat16().to(device).requires_grad_()
        w = (torch.randn(1024, 512, generator=g) * 0.05).bfloat16().to(device).requires_grad_()
        ids, top = torch.randint(0, 512, (300, 4), generator=g).to(device), torch.randn(300, 4, generator=g).to(device)
        cos, sin = rotary_tables(64, 300)
        q, _ = rotary(gated_linear(layer_norm(x), w).view(300, 8, 64), None, cos.to(device), sin.to(device))
        loss = distill_loss(q.reshape(300, 512), ids, top)
        results.append([t.detach().cpu() for t in (loss, *torch.autograd.grad(loss, (x, w)))])
    for a, b in zip(*results):
        assert torch.equal(a, b)
