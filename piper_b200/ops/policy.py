"""Clipped policy loss with a KL term, on the log probabilities that ``token_logprobs`` gives.

``csrc/policy.cu`` has the formulas; one launch forward for up to 4,096 tokens, two above, one backward.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import native
from .packed import PackedSequences, _sequences
from .registry import custom_op, once_differentiable


class PolicyLoss(NamedTuple):
    """``loss`` is differentiable.  ``kl``: mean of e^u - 1 - u, u = ref_logprob - logprob, weighted as the loss is (0 without
    ``ref_logprob``).  ``clipped``: the share of clipped tokens among those that count.  All fp32, of no dimension."""

    loss: Tensor
    kl: Tensor
    clipped: Tensor


def _tokens_ref(logprob, old, adv, ref, low, high, kl_coef):
    """(loss, kl, gradient, clipped) of every token in fp64."""
    d = logprob.double() - old.double()
    a = adv.double()
    none = torch.zeros_like(d)
    clipped = torch.where(a > 0, d > math.log(high), (a < 0) & (d < (math.log(low) if low > 0 else -math.inf)))
    kept = torch.where(a == 0, none, -a * torch.exp(d))
    loss = torch.where(clipped, -a * torch.where(a > 0, high, low), kept)
    grad = torch.where(clipped, none, kept)
    kl = none
    if ref is not None:
        u = ref.double() - logprob.double()
        em1 = torch.expm1(u)
        kl = torch.where(u.abs() < 1e-3, u * u * (0.5 + u * (1 / 6 + u / 24)), torch.where(em1 == math.inf, em1, em1 - u))
        if kl_coef:
            loss, grad = loss + kl_coef * kl, grad - kl_coef * em1
    return loss, kl, grad, clipped


def _weights_ref(mask, table, T):
    """(which tokens count, their weights, weight tensor of the op) on the CPU."""
    on = torch.ones(T, dtype=torch.bool) if mask is None else mask.reshape(-1).clone()
    w = torch.zeros(T, dtype=torch.float64)
    if table is None:
        w[:] = 1.0 / max(1, int(on.sum()))
        weight = w[:1].clone() if T else torch.ones(1, dtype=torch.float64)
    else:
        parts = _sequences(table)
        inside = torch.zeros(T, dtype=torch.bool)
        weight = torch.zeros(table.shape[0], dtype=torch.float64)
        counts = [int(on[a:a + n].sum()) for a, n, _at in parts]
        weight[0] = 1.0 / max(1, sum(c > 0 for c in counts))
        for (a, n, at), c in zip(parts, counts):
            inside[a:a + n] = True
            if c:
                weight[1 + at // 128] = 1.0 / c
                w[a:a + n] = weight[0] / c
        on &= inside
    return on, torch.where(on, w, 0.0), weight


@custom_op("piper::clipped_policy_fwd")
def clipped_policy_fwd(logprob: Tensor, old: Tensor, adv: Tensor, ref: Optional[Tensor], mask: Optional[Tensor],
                       table: Optional[Tensor], low: float, high: float,
                       kl_coef: float) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(loss, kl, clipped, what the backward pass needs of the weights); low, high: borders of the ratio."""
    T = logprob.numel()
    if logprob.is_cuda:
        blocks = (T + 127) // 128 if table is None else table.shape[0] - 1
        loss, kl, clipped = (torch.empty((), dtype=torch.float32, device=logprob.device) for _ in range(3))
        weight = torch.empty(1 + (0 if table is None else blocks), dtype=torch.float32, device=logprob.device)
        scratch = torch.empty(32 * blocks, dtype=torch.uint8, device=logprob.device)
        native.lib().policy_fwd(_flat(logprob), _flat(old), _flat(adv), _flat(ref), _flat(mask), table, loss, kl, clipped, weight,
                                scratch, low, high, kl_coef)
        return loss, kl, clipped, weight
    on, w, weight = _weights_ref(mask, table, T)
    each, kl, _grad, clipped = _tokens_ref(*(t if t is None else t.reshape(-1) for t in (logprob, old, adv, ref)), low, high, kl_coef)

    def mean(x):
        return (torch.where(on, x, 0.0) * w).sum().float()

    share = (clipped & on).sum().double() / max(1, int(on.sum()))
    return mean(each), mean(kl), share.float(), weight.float()


def _flat(t: Optional[Tensor]) -> Optional[Tensor]:
    return None if t is None else t.reshape(-1).contiguous()


@clipped_policy_fwd.register_fake
def _(logprob, old, adv, ref, mask, table, low, high, kl_coef):
    scalars = (logprob.new_empty((), dtype=torch.float32) for _ in range(3))
    return (*scalars, logprob.new_empty((1 if table is None else table.shape[0],), dtype=torch.float32))


def _setup(ctx, inputs, output):
    logprob, old, adv, ref, mask, table, low, high, kl_coef = inputs
    _loss, kl, clipped, weight = output
    ctx.cfg = (low, high, kl_coef)
    ctx.mark_non_differentiable(kl, clipped, weight)
    ctx.save_for_backward(logprob, old, adv, ref, mask, table, weight)


def _backward(ctx, d_loss, _d_kl, _d_clipped, _d_weight):
    logprob, old, adv, ref, mask, table, weight = ctx.saved_tensors
    none = (None,) * 8
    if d_loss is None:
        return torch.zeros_like(logprob), *none
    if logprob.is_cuda:
        d = torch.empty(logprob.numel(), dtype=torch.float32, device=logprob.device)
        native.lib().policy_bwd(_flat(logprob), _flat(old), _flat(adv), _flat(ref), _flat(mask), table, weight,
                                d_loss.to(torch.float32).contiguous(), d, *ctx.cfg)
        return once_differentiable("clipped_policy_loss", d.view(logprob.shape), logprob), *none
    with torch.no_grad():
        on, w, _ = _weights_ref(mask, table, logprob.numel())
        parts = _tokens_ref(*(t if t is None else t.reshape(-1) for t in (logprob, old, adv, ref)), *ctx.cfg)
        d = (torch.where(on, parts[2], 0.0) * w * d_loss.double()).float().view(logprob.shape)
    return once_differentiable("clipped_policy_loss", d, logprob), *none


clipped_policy_fwd.register_autograd(_backward, setup_context=_setup)
clipped_policy_fwd = clipped_policy_fwd.overload


def clipped_policy_loss(logprob: Tensor, old_logprob: Tensor, advantages: Tensor, *, ref_logprob: Optional[Tensor] = None,
                        mask: Optional[Tensor] = None, sequences: Optional[PackedSequences] = None,
                        clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0) -> PolicyLoss:
    """Mean over the tokens that count of max(-A r, -A clip(r, 1 - clip[0], 1 + clip[1])) + ``kl_coef`` x (e^u - 1 - u), where
    r = e^(logprob - old_logprob) and u = ref_logprob - logprob.

    All fp32 of one shape; ``mask`` (bool) says which tokens count, and nothing that stands at others reaches a result.  With
    ``sequences`` the mean is taken within every sequence first, then over those that have tokens that count; tokens behind the
    last sequence do not count.  Without any the loss is 0.  Only ``logprob`` gets a gradient (the rest are constants), which
    has no derivative of its own.  A token without advantage adds its KL term alone, whatever its ratio.
    """
    low, high = clip
    if not (0 <= low <= 1 and 0 <= high < math.inf):
        raise ValueError(f"clipped_policy_loss: clip must be 0 to 1 below and 0 or more above, got {tuple(clip)}")
    if not math.isfinite(kl_coef):
        raise ValueError(f"clipped_policy_loss: kl_coef must be finite, got {kl_coef}")
    if kl_coef and ref_logprob is None:
        raise ValueError("clipped_policy_loss: a KL term needs ref_logprob")
    if sequences is not None and logprob.numel() != sequences.tokens:
        raise ValueError(f"clipped_policy_loss: {logprob.numel()} tokens, the packed batch has {sequences.tokens}")
    table = None if sequences is None else sequences.table
    if not logprob.is_cuda:                          # on a GPU the op makes these checks by itself
        for name, t, dtype in (("logprob", logprob, torch.float32), ("old_logprob", old_logprob, torch.float32),
                               ("advantages", advantages, torch.float32), ("ref_logprob", ref_logprob, torch.float32),
                               ("mask", mask, torch.bool)):
            if t is None:
                continue
            if t.dtype != dtype:
                raise TypeError(f"clipped_policy_loss: {name} must be {dtype}, got {t.dtype}")
            if t.shape != logprob.shape or t.device != logprob.device:
                raise ValueError(f"clipped_policy_loss: {name} is {tuple(t.shape)} on {t.device}, logprob "
                                 f"{tuple(logprob.shape)} on {logprob.device}")
        if table is not None and table.device != logprob.device:
            raise ValueError(f"clipped_policy_loss: sequences are on {table.device}, logprob on {logprob.device}")
    return PolicyLoss(*clipped_policy_fwd(logprob, old_logprob, advantages, ref_logprob, mask, table, 1.0 - low, 1.0 + high,
                                          float(kl_coef))[:3])
