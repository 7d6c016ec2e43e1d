"""The decoder operators from their definitions in 64 bits, with elementwise bounds on what fp32 arithmetic and one rounding
may be off.  Each function returns {name: (value, bound)}; ``half_step`` is the largest relative error of one rounding."""

import torch

F32 = 2.0**-24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _rounded(value, dtype):
    # half a step of the value, or of the smallest subnormal
    return half_step(dtype) * value.abs() + torch.finfo(dtype).smallest_normal * half_step(dtype)


def assert_within(got, value, bound, what):
    assert got.shape == value.shape, (what, got.shape, value.shape)
    g = got.detach().double().cpu()
    v, b = value.cpu(), bound.cpu()
    same = (g == v) | (g.isnan() & v.isnan())
    bad = ~(same | ((g - v).abs() <= b))
    if bad.any():
        i = int(torch.nonzero(bad.reshape(-1))[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {i}: got {g.reshape(-1)[i]}, "
                             f"want {v.reshape(-1)[i]} within {b.reshape(-1)[i]}")


def layer_norm(x, w, b, eps, dy=None):
    """A sum of n fp32 terms in any order is off by at most n * 2^-24 of the sum of their magnitudes; 256 threads or a warp
    share a row, so n counts a thread's own terms and a tree of at most 16 levels."""
    dtype, D = x.dtype, x.shape[-1]
    wt = x.dtype if w is None else w.dtype
    x, dy = x.detach().double(), None if dy is None else dy.double()
    w64 = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    b64 = torch.zeros(D, dtype=torch.float64, device=x.device) if b is None else b.detach().double()
    n = D / 32 + 16
    c = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    h = c * r
    y = h * w64 + b64
    # the mean is off by n 2^-24 mean|x|; the centred row, and through it 1/sqrt(var), by as much over the deviation
    spread = 1 + x.abs().mean(-1, keepdim=True) * r
    mag = (h.abs() + spread) * w64.abs() + b64.abs()
    out = {"y": (y, _rounded(y, dtype) + (3 * n + 8) * F32 * mag * spread)}
    if dy is not None:
        g = dy * w64
        dx = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
        m2 = (g * h).abs().mean(-1, keepdim=True) + g.abs().mean(-1, keepdim=True) * spread
        mag = r * (g.abs() + g.abs().mean(-1, keepdim=True) + (h.abs() + spread) * m2) * spread
        out["dx"] = (dx, _rounded(dx, dtype) + (8 * n + 16) * F32 * mag)
        rows = dy.reshape(-1, D)
        h, spread = h.reshape(-1, D), spread.reshape(-1, 1)
        dw, db = (rows * h).sum(0), rows.sum(0)
        m = rows.shape[0]
        out["dw"] = (dw, _rounded(dw, wt) + (m + 3 * n + 8) * F32 * (rows.abs() * (h.abs() + spread) * spread).sum(0))
        out["db"] = (db, _rounded(db, wt) + (m + 8) * F32 * rows.abs().sum(0))
    return out


def rotary(x, cos, sin, positions, interleaved, inverse=False):
    """Two products and a sum, each rounded once in fp32."""
    half, length, seq = cos.shape[1], cos.shape[0], x.shape[-3]
    pos = torch.arange(seq, device=x.device) if positions is None else positions.long()
    at = pos.clamp(0, length - 1)
    c, s = cos.double()[at][..., None, :], sin.double()[at][..., None, :]
    if inverse:
        s = -s
    v = x.detach().double()
    a, b = (v[..., 0 : 2 * half : 2], v[..., 1 : 2 * half : 2]) if interleaved else (v[..., :half], v[..., half : 2 * half])
    ta, tb, ma, mb = a * c - b * s, b * c + a * s, (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()

    def join(p, q):
        return torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)

    value, bound = v.clone(), torch.zeros_like(v)
    turned, mag = join(ta, tb), join(ma, mb)
    still, beyond = (pos < 0)[..., None, None], (pos >= length)[..., None, None]
    value[..., : 2 * half] = torch.where(still, v[..., : 2 * half], torch.where(beyond, float("nan"), turned))
    bound[..., : 2 * half] = torch.where(still, 0.0, _rounded(turned, x.dtype) + 3 * F32 * mag)
    return value, bound


def distill(logits, ids, top, targets, tau, hard, reduction, ignore_index=-100, scale=1.0):
    """exp carries (2 + 1.2 |x|) steps of fp32 at x, sums of V terms over 512 threads V / 256 + 64 of them."""
    V, K = logits.shape[-1], ids.shape[-1]
    z, ids, top = logits.detach().double().reshape(-1, V), ids.reshape(-1, K).long(), top.detach().double().reshape(-1, K)
    R = z.shape[0]
    dz, tol, loss, loss_tol, count = torch.zeros_like(z), torch.zeros_like(z), 0.0, 0.0, 0
    for r in range(R):
        t = -1 if targets is None else int(targets.reshape(-1)[r])
        if targets is not None and (t == ignore_index or not 0 <= t < V):
            continue
        keep = (ids[r] >= 0) & (ids[r] < V) & (top[r] != -float("inf"))
        if not keep.any():
            continue
        count += 1
        at, p = ids[r][keep], torch.softmax(top[r][keep] / tau, 0)
        q, q1 = torch.softmax(z[r] / tau, 0), torch.softmax(z[r], 0)
        logq, logp = torch.log_softmax(z[r] / tau, 0)[at], torch.log_softmax(top[r][keep] / tau, 0)
        soft = torch.where(p > 0, p * (logp - logq), 0.0).sum()
        row = (1 - hard) * tau**2 * soft
        a, h = (1 - hard) * tau, hard
        grad, mag = a * q, a * q
        grad = grad.index_add(0, at, -a * p)
        mag = mag.index_add(0, at, a * p)
        if hard > 0:
            row = row - hard * torch.log_softmax(z[r], 0)[t]
            grad, mag = grad + h * q1, mag + h * q1
            grad[t] -= h
            mag[t] += h
        finite = z[r][z[r].isfinite()]
        reach = float(finite.max() - finite.min()) * max(1.0, 1 / tau) if finite.numel() else 0.0
        reach += float((top[r][keep].max() - top[r][keep][p > 0].min()) / tau) if (p > 0).any() else 0.0
        k = (V / 256 + 64 + K + 8 * reach + 40) * 2 * F32
        loss, loss_tol = loss + row, loss_tol + k * (1 + (1 - hard) * tau**2 + hard) + R * F32 * row.abs()
        dz[r], tol[r] = grad, k * mag
    f = scale / max(count, 1) if reduction == "mean" else scale
    dz, tol = (dz * f).reshape(logits.shape), (tol * f).reshape(logits.shape)
    loss = torch.as_tensor(loss * f, dtype=torch.float64)
    return {"loss": (loss, torch.as_tensor(loss_tol * abs(f), dtype=torch.float64) + 4 * F32 * loss.abs()),
            "dz": (dz, _rounded(dz, logits.dtype) + tol)}


def gated(x, w, act, dh=None):
    """Products of K terms in groups of 16 with fp32 accumulation: (K / 8 + 16) steps of 2^-23 of the sum of magnitudes.
    The backward pass rounds the two projections and their gradients to bf16 once each."""
    u16 = half_step(torch.bfloat16)
    x, w = x.detach().double(), w.detach().double()
    F, K = w.shape[0] // 2, w.shape[1]
    x = x.reshape(-1, K)
    acc = (K / 8 + 16) * 2 * F32
    g, u = x @ w[:F].t(), x @ w[F:].t()
    mg, mu = acc * (x.abs() @ w[:F].abs().t()), acc * (x.abs() @ w[F:].abs().t())
    g.requires_grad_(True)
    a = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g, approximate="tanh" if act == "gelu_tanh" else "none")
    (da,) = torch.autograd.grad(a.sum(), g)
    g, a = g.detach(), a.detach()
    h = a * u
    out = {"h": (h, _rounded(h, torch.bfloat16) + a.abs() * mu + u.abs() * (da.abs() + mg) * mg + 2.0**-19 * h.abs() + mu * mg)}
    if dh is not None:
        dh = dh.double().reshape(-1, F)
        dg, du = dh * u * da, dh * a
        # second derivatives of the three activations are at most 1.2
        eg = dh.abs() * (da.abs() * (u16 * u.abs() + mu) + 1.2 * u.abs() * (u16 * g.abs() + mg)) + 1.05 * u16 * dg.abs() + 1e-30
        eu = dh.abs() * (da.abs() + 0.1) * (u16 * g.abs() + mg) + 1.05 * u16 * du.abs() + 1e-30
        d, e = torch.cat([dg, du], -1), torch.cat([eg, eu], -1)
        dx, dw = d @ w, d.t() @ x
        T = x.shape[0]
        out["dx"] = (dx, 1.05 * u16 * dx.abs() + e @ w.abs() + (F / 4 + 16) * 2 * F32 * (d.abs() @ w.abs()) + 1e-30)
        out["dw"] = (dw, 1.05 * u16 * dw.abs() + e.t() @ x.abs() + (T / 8 + 16) * 2 * F32 * (d.abs().t() @ x.abs()) + 1e-30)
    return out
