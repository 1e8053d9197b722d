"""Log probabilities of given tokens with the entropy and the most probable alternatives of their rows of logits.

What a policy update, a distillation loss and a scoring request need of the logits, next to ``cross_entropy``, which
gives a loss and nothing else.  One pass over the logits in the forward pass (``csrc/logprobs.cu``), one read and one
write of them in the backward pass; no probabilities are kept.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch import Tensor

from . import native
from .registry import custom_op, once_differentiable

MAX_TOP = 32
MAX_VOCAB = 1 << 30


class TokenLogprobs(NamedTuple):
    """Log probabilities in fp32, shaped like the tokens; the alternatives have a last dimension of ``top``."""

    logprob: Tensor
    entropy: Tensor
    top_logprob: Tensor
    top_id: Tensor


def _counted(tokens: Tensor, V: int, ignore_index: int) -> Tensor:
    return (tokens != ignore_index) & (tokens >= 0) & (tokens < V)


def _stats_ref(logits: Tensor, temperature: float) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(log p, p, entropy, largest logit, log of the sum) of [T, V] logits in fp32 or more."""
    x = logits.double() if logits.dtype == torch.float64 else logits.float()
    lowest = torch.finfo(x.dtype).min
    top = torch.where(x == x, x, torch.full_like(x, -math.inf)).amax(1, keepdim=True).clamp(min=lowest)
    z = (x - top) / temperature
    total = torch.exp(z).sum(1, keepdim=True)
    logp = torch.where(total == 0, torch.full_like(z, -math.inf), z - torch.log(total))
    p = torch.exp(logp)
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(1)
    return logp, p, entropy, top.squeeze(1), torch.log(total).squeeze(1)


@custom_op("piper::token_logprobs_fwd")
def token_logprobs_fwd(logits: Tensor, tokens: Tensor, top: int, temperature: float,
                       ignore_index: int) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """logits [T, V], tokens [T] -> (logprob [T], entropy [T], top_logprob [T, top], top_id [T, top], stats [T, 2])."""
    T, V = logits.shape
    if logits.is_cuda:
        if logits.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"the sm_100a kernels take bfloat16 or float32 logits, got {logits.dtype}")
        lg = logits if logits.stride(1) == 1 else logits.contiguous()
        logprob, entropy, stats = (torch.empty(s, dtype=torch.float32, device=lg.device) for s in ((T,), (T,), (T, 2)))
        top_logprob = torch.empty((T, top), dtype=torch.float32, device=lg.device)
        top_id = torch.empty((T, top), dtype=torch.int64, device=lg.device)
        native.lib().logprobs_fwd(lg, tokens.contiguous(), logprob, entropy, top_logprob, top_id, stats, temperature,
                                  ignore_index)
        return logprob, entropy, top_logprob, top_id, stats
    logp, _p, entropy, largest, log_s = _stats_ref(logits, temperature)
    at = tokens.clamp(0, V - 1).unsqueeze(1)
    logprob = torch.where(_counted(tokens, V, ignore_index), logp.gather(1, at).squeeze(1), torch.zeros((), dtype=logp.dtype))
    ranked = torch.where(logits == logits, logits, torch.full_like(logits, -math.inf))
    top_id = torch.sort(ranked, dim=1, descending=True, stable=True).indices[:, :top].contiguous()
    stats = torch.stack((largest, log_s / math.log(2.0)), 1)
    return logprob.float(), entropy.float(), logp.gather(1, top_id).float(), top_id, stats.float()


@token_logprobs_fwd.register_fake
def _(logits, tokens, top, temperature, ignore_index):
    T = logits.shape[0]
    f32 = torch.float32
    return (logits.new_empty((T,), dtype=f32), logits.new_empty((T,), dtype=f32), logits.new_empty((T, top), dtype=f32),
            logits.new_empty((T, top), dtype=torch.int64), logits.new_empty((T, 2), dtype=f32))


def _setup(ctx, inputs, output):
    logits, tokens, _top, temperature, ignore_index = inputs
    _logprob, entropy, _top_logprob, top_id, stats = output
    ctx.cfg = (temperature, ignore_index)
    ctx.mark_non_differentiable(top_id, stats)
    ctx.save_for_backward(logits, tokens, entropy, top_id, stats)


def _backward(ctx, d_logprob, d_entropy, d_top, _d_id, _d_stats):
    logits, tokens, entropy, top_id, stats = ctx.saved_tensors
    temperature, ignore_index = ctx.cfg
    T, V = logits.shape

    def dense(g):
        return None if g is None else g.to(torch.float32).contiguous()

    if d_logprob is None and d_entropy is None and d_top is None:
        return torch.zeros_like(logits), None, None, None, None
    if logits.is_cuda:
        lg = logits if logits.stride(1) == 1 else logits.contiguous()
        d = torch.empty((T, V), dtype=logits.dtype, device=logits.device)
        native.lib().logprobs_bwd(lg, tokens.contiguous(), stats, entropy, top_id, dense(d_logprob), dense(d_entropy), dense(d_top),
                                  d, temperature, ignore_index)
        return once_differentiable("token_logprobs on a GPU", d, logits), None, None, None, None
    logp, p, h, _largest, log_s = _stats_ref(logits, temperature)
    up = torch.zeros_like(p)                         # gradient with respect to log p
    if d_logprob is not None:
        on = _counted(tokens, V, ignore_index)
        up.scatter_add_(1, tokens.clamp(0, V - 1).unsqueeze(1), torch.where(on, d_logprob, 0).to(p.dtype).unsqueeze(1))
    if d_top is not None:
        up.scatter_add_(1, top_id, d_top.to(p.dtype))
    d = up - p * up.sum(1, keepdim=True)
    if d_entropy is not None:
        d = d - d_entropy.to(p.dtype).unsqueeze(1) * torch.where(p == 0, torch.zeros_like(p), p * (logp + h.unsqueeze(1)))
    # nothing asks for a row (padding, whatever its logits are), or nothing is left in it
    live = torch.zeros(T, dtype=torch.bool)
    if d_logprob is not None:
        live |= (d_logprob != 0) & on
    if d_entropy is not None:
        live |= d_entropy != 0
    if d_top is not None:
        live |= (d_top != 0).any(1)
    d = torch.where((live & ~torch.isinf(log_s)).unsqueeze(1), d / temperature, torch.zeros_like(d))
    return d.to(logits.dtype), None, None, None, None


token_logprobs_fwd.register_autograd(_backward, setup_context=_setup)
token_logprobs_fwd = token_logprobs_fwd.overload


def token_logprobs(logits: Tensor, tokens: Tensor, *, top: int = 0, temperature: float = 1.0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Of every row of ``logits`` [..., V] at ``temperature``: the log probability of its token, the entropy, and the ``top``
    most probable ids with their log probabilities, equal logits by rising id.

    Logits are bf16 or fp32; everything is computed and returned in fp32.  ``logprob``, ``entropy`` and ``top_logprob`` are
    differentiable with respect to the logits (the ids are taken as given).  A token that is ``ignore_index`` or no id
    of the vocabulary has log probability 0 and no gradient through it.  Masked ids (-inf) have probability 0; a row that
    has nothing else has entropy 0, log probabilities of -inf and no gradient.  A row with a NaN or +inf is NaN; its ids
    are some of the vocabulary's.  A row whose outputs get no gradient but zeros gives none, whatever its logits are.  Gradients
    of the gradient exist on the CPU only; on a GPU they raise.
    """
    if logits.is_cuda and logits.dim() == 2:         # the op makes the checks below by itself
        return TokenLogprobs(*token_logprobs_fwd(logits, tokens, top, temperature, ignore_index)[:4])
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"token_logprobs: logits have no vocabulary: {tuple(logits.shape)}")
    if logits.shape[-1] > MAX_VOCAB:
        raise ValueError(f"token_logprobs: at most {MAX_VOCAB} ids, got {logits.shape[-1]}")
    if not logits.is_floating_point():
        raise TypeError(f"token_logprobs: logits must be floating point, got {logits.dtype}")
    if tokens.dtype != torch.int64 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"token_logprobs: tokens must be int64 {tuple(logits.shape[:-1])}, got {tokens.dtype} "
                         f"{tuple(tokens.shape)}")
    if tokens.device != logits.device:
        raise ValueError(f"token_logprobs: tokens are on {tokens.device}, logits on {logits.device}")
    V = logits.shape[-1]
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"token_logprobs: top must be 0 to {min(MAX_TOP, V)}, got {top}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"token_logprobs: temperature must be 1e-6 to 1e6, got {temperature}")
    lg = logits if logits.dim() == 2 else logits.reshape(-1, V)
    lead = tokens.shape
    logprob, entropy, top_logprob, top_id, _ = token_logprobs_fwd(lg, tokens.reshape(-1), top, float(temperature), ignore_index)
    if len(lead) != 1:
        logprob, entropy = logprob.view(lead), entropy.view(lead)
        top_logprob, top_id = top_logprob.view(*lead, top), top_id.view(*lead, top)
    return TokenLogprobs(logprob, entropy, top_logprob, top_id)
