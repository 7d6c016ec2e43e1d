"""Memory-bound pieces of the training step as single-pass sm_100a kernels, with autograd.

``rope_qkv_``     rotary embedding applied in place to the q and k heads of the fused QKV activations
``swiglu``        ``silu(gate) * up`` on the fused gate/up activations; the backward is one kernel too
``cross_entropy`` mean token cross-entropy over bf16 logits; the backward overwrites the logits with their
                  gradient, so no fp32 copy of the ``[tokens, vocab]`` matrix is ever made
``adamw_``        AdamW over a flat bf16 parameter shard with bf16 moments (gradient fp32 or bf16)
``rms_norm``      RMSNorm over the last dimension; the backward produces dx and dw in one pass over dy and x
``layer_norm``    layer normalisation over the last dimension with optional weight and bias, any width
``rotary``        rotary positions on q and k in one launch: either pair layout, part of the head, a position per token;
                  ``rotary_`` in place for serving, ``rotary_tables`` with the scalings for long contexts
``distill_loss``  distillation from a teacher's top logits, alone or with the hard targets' cross-entropy

On CUDA tensors these always run the kernels of ``csrc/kernels/`` (``train_ops.cu``, ``norm_ops.cu``, ``rotary.cu``,
``distill.cu``).  CPU tensors take plain PyTorch arithmetic so the sharded engine's host-side logic can be exercised on
``gloo`` ranks.
The reference library is a communication backend and has no counterpart of these ops.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from .._core import _C

_launches = 0


def train_op_launches() -> int:
    """Number of kernels launched by this module so far in this process."""
    return _launches + _C.decoder_op_launches()


def _count(n: int = 1) -> None:
    global _launches
    _launches += n


def _rope_reference(x2, cos, sin, seq, n_heads, head_dim, inverse):
    t = x2.shape[0]
    v = x2[:, : n_heads * head_dim].reshape(t, n_heads, head_dim).float()
    half = head_dim // 2
    pos = torch.arange(t, device=x2.device) % seq
    c = cos[pos][:, None, :]
    s = sin[pos][:, None, :] * (-1.0 if inverse else 1.0)
    a, b = v[..., :half], v[..., half:]
    out = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    x2[:, : n_heads * head_dim] = out.reshape(t, n_heads * head_dim).to(x2.dtype)


def _rope_apply(x2, cos, sin, seq, n_heads, head_dim, inverse):
    if x2.is_cuda:
        _count()
        _C.rope_(x2, cos, sin, seq, n_heads, head_dim, inverse)
    else:
        _rope_reference(x2, cos, sin, seq, n_heads, head_dim, inverse)


class _RopeQKV(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, cos, sin, seq, n_heads, head_dim):
        ctx.save_for_backward(cos, sin)
        ctx.args = (seq, n_heads, head_dim)
        x2 = qkv.view(-1, qkv.shape[-1])
        _rope_apply(x2, cos, sin, seq, n_heads, head_dim, False)
        ctx.mark_dirty(qkv)
        return qkv

    @staticmethod
    def backward(ctx, g):
        cos, sin = ctx.saved_tensors
        seq, n_heads, head_dim = ctx.args
        g = g.contiguous() if not g.is_contiguous() else g
        g2 = g.view(-1, g.shape[-1])
        # the incoming gradient is a fresh buffer (assembled from dq, dk, dv): rotate it in place
        _rope_apply(g2, cos, sin, seq, n_heads, head_dim, True)
        return g, None, None, None, None, None


def rope_qkv_(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, n_rot_heads: int, head_dim: int) -> torch.Tensor:
    """Rotate the first ``n_rot_heads`` heads (q then k) of ``qkv[B, S, (H + 2 KV) * head_dim]`` in place.

    Pairs are ``(j, j + head_dim/2)``; ``cos``/``sin`` are fp32 ``[>= S, head_dim/2]``.  ``qkv`` must be a
    tensor nobody else needs unrotated (the output of the QKV projection).
    """
    return _RopeQKV.apply(qkv, cos, sin, qkv.shape[-2], n_rot_heads, head_dim)


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu):
        ctx.save_for_backward(gu)
        gu2 = gu.reshape(-1, gu.shape[-1])
        if gu2.is_cuda:
            _count()
            out = _C.swiglu_fwd(gu2)
        else:
            g, u = gu2.float().chunk(2, dim=-1)
            out = (F.silu(g) * u).to(gu.dtype)
        return out.view(*gu.shape[:-1], gu.shape[-1] // 2)

    @staticmethod
    def backward(ctx, dout):
        (gu,) = ctx.saved_tensors
        gu2 = gu.reshape(-1, gu.shape[-1])
        d2 = dout.reshape(-1, dout.shape[-1])
        if gu2.is_cuda:
            if d2.stride(-1) != 1 or (d2.stride(0) * 2) % 16:
                d2 = d2.contiguous()
            _count()
            dgu = _C.swiglu_bwd(gu2, d2)
        else:
            g, u = gu2.float().chunk(2, dim=-1)
            sig = torch.sigmoid(g)
            sl = g * sig
            d = d2.float()
            dgu = torch.cat([d * u * (sig + sl * (1 - sig)), d * sl], dim=-1).to(gu.dtype)
        return dgu.view(gu.shape)


def swiglu(gu: torch.Tensor) -> torch.Tensor:
    """``silu(gu[..., :F]) * gu[..., F:]`` for the fused gate/up projection output."""
    return _SwiGLU.apply(gu)


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, ignore_index):
        l2 = logits.view(-1, logits.shape[-1])
        t = targets.reshape(-1).contiguous()
        # mean over the rows that are not ignored (kept on the device: no synchronisation)
        count = (t != ignore_index).sum().clamp(min=1).float()
        _count()
        rows, lse = _C.cross_entropy_fwd(l2, t, ignore_index)
        ctx.save_for_backward(l2, t, lse, count)
        ctx.ignore_index = ignore_index
        ctx.shape = logits.shape
        return rows.sum() / count

    @staticmethod
    def backward(ctx, g):
        l2, t, lse, count = ctx.saved_tensors
        gs = g.reshape(1).float() / count
        _count()
        _C.cross_entropy_bwd_(l2, t, lse, gs, 1.0, ctx.ignore_index)
        return l2.view(ctx.shape), None, None


def cross_entropy(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """Mean cross-entropy of bf16 ``logits[..., V]`` against int64 ``targets``.

    On CUDA the backward pass writes the gradient over ``logits`` (the output of the last projection,
    which nothing else reads); the returned loss is an fp32 scalar.
    """
    if not logits.is_cuda:
        return F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), targets.reshape(-1), ignore_index=ignore_index)
    if not logits.is_contiguous():
        logits = logits.contiguous()
    return _CrossEntropy.apply(logits, targets, ignore_index)


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, eps):
        x2 = x.reshape(-1, x.shape[-1])
        if x2.stride(-1) != 1 or (x2.stride(0) * 2) % 16:
            x2 = x2.contiguous()
        _count()
        y, rstd = _C.rmsnorm_fwd(x2, w, eps)
        ctx.save_for_backward(x2, w, rstd)
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2, w, rstd = ctx.saved_tensors
        d2 = dy.reshape(-1, dy.shape[-1])
        if d2.stride(-1) != 1 or (d2.stride(0) * 2) % 16:
            d2 = d2.contiguous()
        _count(2)
        dx, dw = _C.rmsnorm_bwd(x2, w, d2, rstd)
        return dx.view(dy.shape), dw, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """``x * rsqrt(mean(x^2, -1) + eps) * weight``; bf16 CUDA tensors whose last dimension is a multiple of 8
    (up to 8192) run the single-pass kernels, anything else ``torch.nn.functional.rms_norm``."""
    d = x.shape[-1]
    if (x.is_cuda and x.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16 and d % 8 == 0
            and d <= _C.rmsnorm_max_dim() and weight.is_contiguous()):
        return _RMSNorm.apply(x, weight, eps)
    return F.rms_norm(x, (d,), weight, eps)


def adamw_(p, g, m, v, lr: float, betas=(0.9, 0.95), eps: float = 1e-8, weight_decay: float = 0.1, step: int = 1,
           grad_scale: float = 1.0) -> None:
    """One AdamW update of the flat bf16 tensor ``p`` in place (decoupled decay, bias-corrected).

    ``g`` is the gradient (fp32 or bf16, multiplied by ``grad_scale`` first), ``m``/``v`` the bf16 moments.
    """
    b1, b2 = betas
    if p.is_cuda:
        _count()
        _C.adamw_(p, g, m, v, lr, b1, b2, eps, weight_decay, step, grad_scale)
        return
    gr = g.float() * grad_scale
    mf = m.float().mul_(b1).add_(gr, alpha=1 - b1)
    vf = v.float().mul_(b2).addcmul_(gr, gr, value=1 - b2)
    bc1 = 1 - b1**step
    bc2 = 1 - b2**step
    denom = vf.sqrt() / (bc2**0.5) + eps
    pf = p.float() * (1 - lr * weight_decay) - (lr / bc1) * mf / denom
    p.copy_(pf)
    m.copy_(mf)
    v.copy_(vf)


def adamw_master_(p, master, g, m, v, lr: float, betas=(0.9, 0.95), eps: float = 1e-8, weight_decay: float = 0.1,
                  step: int = 1) -> None:
    """AdamW on an fp32 master copy with fp32 moments; ``p`` (any float dtype, usually bf16) receives the rounded
    result.  The arithmetic mixed-precision FSDP keeps per shard: ``master``, ``m`` and ``v`` are fp32 tensors of
    ``p``'s shape, ``g`` the gradient in fp32 or bf16.  Plain PyTorch ops on whatever device the tensors live on
    (several passes over the shard; the single-pass kernel is ``adamw_``, which keeps bf16 state)."""
    b1, b2 = betas
    gr = g if g.dtype == torch.float32 else g.float()
    m.mul_(b1).add_(gr, alpha=1 - b1)
    v.mul_(b2).addcmul_(gr, gr, value=1 - b2)
    bc1 = 1 - b1**step
    bc2 = 1 - b2**step
    denom = v.sqrt().div_(bc2**0.5).add_(eps)
    master.mul_(1 - lr * weight_decay).addcdiv_(m, denom, value=-lr / bc1)
    p.copy_(master)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension; differentiable (once) in all three.

    ``x`` is bf16, fp16 or fp32 with any leading dimensions and any width; ``weight`` and ``bias`` are ``[width]``, both of
    ``x``'s type or both fp32, and may be left out.  Statistics and the sums of the weight's and bias's gradients are fp32
    with a fixed order of summation.
    """
    if x.is_cuda:
        return _C.layer_norm(x, weight, bias, eps)
    _C.layer_norm_check(x, weight, bias, eps)
    w = None if weight is None else weight.float()
    b = None if bias is None else bias.float()
    return F.layer_norm(x.float(), (x.shape[-1],), w, b, eps).to(x.dtype)


def rotary_tables(rotary_dim: int, length: int, theta: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                  original_length: int | None = None, low: float = 1.0, high: float = 4.0, device=None):
    """fp32 ``(cos, sin)`` tables ``[length, rotary_dim / 2]`` for :func:`rotary`, the angles computed in 64 bits.

    ``scaling`` stretches a model to contexts ``factor`` times longer than it was trained on: ``"linear"`` divides every
    angle by ``factor``; ``"ntk"`` raises the base to ``theta * factor ** (R / (R - 2))``, which divides the lowest
    frequency by ``factor`` and leaves the highest; ``"by_parts"`` leaves a frequency that turns ``high`` times or more
    within ``original_length`` positions, divides one that turns ``low`` times or less, and blends in between.
    """
    if rotary_dim < 2 or rotary_dim % 2 or length < 1:
        raise ValueError("moodist rotary_tables: an even rotary_dim and a length of at least 1 are required")
    if scaling not in (None, "linear", "ntk", "by_parts"):
        raise ValueError(f"moodist rotary_tables: unknown scaling {scaling!r}")
    if not theta > 0 or not factor > 0:
        raise ValueError("moodist rotary_tables: theta and factor must be positive")
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("moodist rotary_tables: ntk scaling needs a rotary_dim of at least 4")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    inv = theta ** (-torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float64) / rotary_dim)
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "by_parts":
        if original_length is None or original_length < 1 or not 0 <= low < high:
            raise ValueError("moodist rotary_tables: by_parts needs original_length and 0 <= low < high")
        turns = original_length * inv / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        inv = inv * (keep + (1 - keep) / factor)
    angle = torch.outer(torch.arange(length, device=device, dtype=torch.float64), inv)
    return angle.cos().float(), angle.sin().float()


def _turn_reference(x, cos, sin, positions, interleaved):
    length, half = cos.shape
    seq = x.shape[-3]
    pos = torch.arange(seq, device=x.device) if positions is None else positions.long()
    at = pos.clamp(0, length - 1)
    still, beyond = (pos < 0)[..., None, None], (pos >= length)[..., None, None]
    c, s = cos[at][..., None, :], sin[at][..., None, :]
    head = x[..., : 2 * half].float()
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :half], head[..., half:])
    ta, tb = a * c - b * s, b * c + a * s
    turned = torch.stack([ta, tb], -1).flatten(-2) if interleaved else torch.cat([ta, tb], -1)
    turned = torch.where(still, head, torch.where(beyond, float("nan"), turned))
    return torch.cat([turned.to(x.dtype), x[..., 2 * half :]], -1)


def rotary(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None = None,
           interleaved: bool = False):
    """``(q', k')``: rotary positions on ``q[B, S, H, D]`` and ``k[B, S, KV, D]`` (or without ``B``); ``k`` may be None.

    ``cos`` / ``sin`` are fp32 ``[positions, R / 2]`` (:func:`rotary_tables`): the first ``R <= D`` dimensions of a head turn,
    in pairs ``(j, j + R/2)`` or, ``interleaved``, ``(2j, 2j + 1)``, the others pass through.  ``positions`` (int64 or int32,
    ``[B, S]`` or ``[S]``; default ``0 .. S-1``) says where each token stands; a negative one marks padding, which passes
    through unchanged, and one that the tables do not have gives NaN.  bf16, fp16 or fp32, any strides (views of a fused
    projection's output go in as they are); the results are new contiguous tensors.  Differentiable (once) in q and k.
    """
    if q.is_cuda:
        return _C.rotary(q, k, cos, sin, positions, interleaved)
    _C.rotary_check(q, k, cos, sin, positions)
    return (_turn_reference(q, cos, sin, positions, interleaved),
            None if k is None else _turn_reference(k, cos, sin, positions, interleaved))


def rotary_(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None = None,
            interleaved: bool = False) -> None:
    """:func:`rotary` written over ``q`` and ``k``, for serving (no gradient passes through it).  Dimensions from ``R`` up and
    tokens at negative positions are not touched."""
    if q.is_cuda:
        _C.rotary_(q, k, cos, sin, positions, interleaved)
        return
    _C.rotary_check(q, k, cos, sin, positions)
    _C.rotary_in_place_check(q, k)
    for x in (q, k):
        if x is not None:
            x.copy_(_turn_reference(x, cos, sin, positions, interleaved))


def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, targets: torch.Tensor | None = None, *,
                 temperature: float = 1.0, hard_weight: float = 0.0, ignore_index: int = -100, reduction: str = "mean",
                 scale: float = 1.0) -> torch.Tensor:
    """Distillation loss of ``logits[..., V]`` against a teacher's top entries ``teacher_ids`` / ``teacher_logits[..., K]``.

    Per row ``(1 - hard_weight) * temperature^2 * KL(p || q) + hard_weight * cross_entropy(logits, targets)`` where ``p`` is
    the softmax of the teacher's entries over ``temperature`` (renormalised over the entries given) and ``q`` the softmax of
    ``logits / temperature`` over the vocabulary.  An entry whose id is outside ``[0, V)`` or whose logit is ``-inf`` is
    padding; a word named twice counts with both entries.  A row without any entry, or whose target is ``ignore_index`` (or
    outside ``[0, V)``), gives neither loss nor gradient.  The fp32 result is the sum over the other rows, or their mean
    (0 when there is none), times ``scale``.

    Logits are bf16, fp16 or fp32, ids int64 or int32, teacher logits bf16, fp16 or fp32, targets int64.  Differentiable
    (once) in ``logits``, which stay as they are: where :func:`cross_entropy` is wanted as well, take it in here through
    ``targets``, since its own backward pass overwrites the logits that this one reads.

    On CUDA the forward pass makes the gradient of bf16 and fp32 logits as well (when they require one), so that they are
    read once: call it under ``torch.no_grad()`` where only the loss is wanted.  The backward pass then hands that gradient
    out, once per forward pass, and only touches it if the loss was scaled afterwards (``scale`` costs nothing).
    """
    if reduction not in ("mean", "sum"):
        raise ValueError(f"moodist distill_loss: reduction must be 'mean' or 'sum', not {reduction!r}")
    if logits.is_cuda:
        return _C.distill_loss(logits, teacher_ids, teacher_logits, targets, temperature, hard_weight, ignore_index,
                               reduction == "mean", scale)
    _C.distill_check(logits, teacher_ids, teacher_logits, targets, temperature, hard_weight)
    V, K = logits.shape[-1], teacher_ids.shape[-1]
    ids, top = teacher_ids.reshape(-1, K).long(), teacher_logits.reshape(-1, K).float()
    valid = (ids >= 0) & (ids < V) & (top != float("-inf"))
    live = valid.any(-1)
    if targets is not None:
        t = targets.reshape(-1)
        live = live & (t != ignore_index) & (t >= 0) & (t < V)
    valid = valid & live[:, None]
    z = torch.where(live[:, None], logits.reshape(-1, V).float(), 0.0)
    at = torch.where(valid, ids, 0)
    top = torch.where(valid, top / temperature, float("-inf"))
    peak = torch.where(live, top.amax(-1), 0.0)[:, None]
    logp = top - peak - torch.where(live, (top - peak).exp().sum(-1), 1.0).log()[:, None]
    p = logp.exp()
    rows = z.new_zeros(z.shape[0])
    if hard_weight < 1:
        logq = torch.log_softmax(z / temperature, -1).gather(1, at)
        term = torch.where(p == 0, 0.0, p * (torch.where(p == 0, 0.0, logp) - torch.where(p == 0, 0.0, logq)))
        rows = rows + (1 - hard_weight) * temperature**2 * term.sum(-1)
    if hard_weight > 0:
        rows = rows + hard_weight * F.cross_entropy(z, torch.where(live, t, 0), reduction="none")
    factor = scale / live.sum().clamp(min=1) if reduction == "mean" else scale
    return torch.where(live, rows, 0.0).sum() * factor
