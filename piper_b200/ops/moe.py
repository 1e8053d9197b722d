"""Mixture-of-experts ops: router, dispatch into padded expert segments, grouped linear, combine.

Row layout.  ``moe_dispatch`` copies each token once per selected expert into a row buffer in which the
entries of expert ``e`` occupy rows ``[g_start[e], g_start[e] + counts[e])``; every segment is padded with
zero rows to a multiple of 128 (``g_len``), so a segment is a whole number of tensor-core M tiles and the
weight-gradient GEMM can contract over padded segments.  The grouped linear op takes such a buffer plus a
*group table* ``(g_start, g_len)`` with ``G = sources * experts`` groups, group ``g`` using expert
``g % experts``; ``sources`` is 1 without expert parallelism and the expert-parallel degree after a token
exchange, when rows arrive grouped by (source rank, local expert).

The reference's expert compute pads every expert to ``T*k`` rows and runs ``bmm``
(``examples/models/qwen3_bmm_experts_patch.py:24-37``, an ``E``-fold waste); its un-permute and weighted
combine are separate index-put / ``bmm`` calls (``examples/models/qwen3.py:265-283``).  Here dispatch,
combine and their gradients are one kernel each and the expert GEMMs are ragged.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import core, native
from .registry import custom_op, host_op, once_differentiable
from .core import _is_native, _require_bf16, grad_sinks, wgrad_store

PAD = 128

# Set by the executor around a segment run when the expert-parallel exchanges are lowered to peer-memory kernels
# (``parallel/ep_fused.py``): ``_EP_RUNTIME.dispatch`` replaces the local permutation of ``moe_dispatch`` by a
# gather straight into the expert owners' receive regions, and ``_EP_TABLE`` is the group table of the receive
# region that the expert segment reads in place.
_EP_RUNTIME = None
_EP_TABLE = None


def set_ep_context(runtime, table) -> None:
    global _EP_RUNTIME, _EP_TABLE
    _EP_RUNTIME, _EP_TABLE = runtime, table
    native.set_flag(native.EXPERT_RUNTIME, runtime is not None or table is not None)


def row_capacity(tokens: int, k: int, experts: int) -> int:
    """Rows a dispatch buffer needs in the worst case (every segment padded by up to PAD-1 rows)."""
    return (tokens * k + experts * (PAD - 1) + PAD - 1) // PAD * PAD


# ------------------------------------------------------------------ router
@custom_op("piper::moe_route")
def moe_route(logits: Tensor, k: int, renorm: bool) -> tuple[Tensor, Tensor, Tensor]:
    """softmax over experts, top-k, optional renormalisation -> (weights fp32 [T,k], idx int32 [T,k], counts int32 [E])."""
    T, E = logits.shape
    if _is_native(logits):
        _require_bf16(logits)
        w = torch.empty((T, k), dtype=torch.float32, device=logits.device)
        idx = torch.empty((T, k), dtype=torch.int32, device=logits.device)
        counts = torch.zeros(E, dtype=torch.int32, device=logits.device)
        native.lib().moe_route(logits.contiguous(), w, idx, counts, k, renorm)
        return w, idx, counts
    p = torch.softmax(logits.float(), dim=-1)
    w, idx = torch.topk(p, k, dim=-1)
    if renorm:
        w = w / w.sum(-1, keepdim=True)
    counts = torch.bincount(idx.reshape(-1), minlength=E).to(torch.int32)
    return w.contiguous(), idx.to(torch.int32).contiguous(), counts


@moe_route.register_fake
def _(logits, k, renorm):
    T, E = logits.shape
    return (logits.new_empty((T, k), dtype=torch.float32), logits.new_empty((T, k), dtype=torch.int32),
            logits.new_empty((E,), dtype=torch.int32))


def _route_setup(ctx, inputs, output):
    logits, k, renorm = inputs
    w, idx, _counts = output
    ctx.renorm = renorm
    ctx.save_for_backward(logits, idx, w)


def _route_backward(ctx, dw, _didx, _dcounts):
    logits, idx, w = ctx.saved_tensors
    if dw is None:
        dw = torch.zeros_like(w)
    if _is_native(logits):
        d = torch.empty_like(logits, memory_format=torch.contiguous_format)
        native.lib().moe_route_bwd(logits.contiguous(), idx, w, dw.contiguous().float(), d, ctx.renorm)
        return d, None, None
    p = torch.softmax(logits.float(), dim=-1)
    dp = torch.zeros_like(p)
    g = dw.float()
    if ctx.renorm:
        S = torch.gather(p, 1, idx.long()).sum(-1, keepdim=True)
        g = (g - (g * w).sum(-1, keepdim=True)) / S
    dp.scatter_(1, idx.long(), g)
    d = p * (dp - (dp * p).sum(-1, keepdim=True))
    return d.to(logits.dtype), None, None


moe_route.register_autograd(_route_backward, setup_context=_route_setup)


# ------------------------------------------------------------ balance loss
MAX_BALANCE_EXPERTS = 256


class BalanceLoss(NamedTuple):
    """``loss`` fp32 of no dimension, differentiable; ``counts`` int32 [E]: choices of every expert by the tokens that count;
    ``prob`` fp32 [E]: its mean probability over them."""

    loss: Tensor
    counts: Tensor
    prob: Tensor


def _probabilities(logits: Tensor) -> Tensor:
    """Softmax in fp64; rows without a finite logit become 0."""
    x = logits.double()
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - torch.where(top == -float("inf"), torch.zeros_like(top), top))
    total = e.sum(1, keepdim=True)
    return torch.where(total == 0, e, e / total)


@custom_op("piper::moe_balance_fwd")
def moe_balance_fwd(logits: Tensor, idx: Tensor, mask: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(loss, counts, prob, what the gradient of a probability is, up to that of the loss)."""
    T, E = logits.shape
    if _is_native(logits):
        def empty(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device=logits.device)

        loss, counts, prob, factor = empty(), empty(E, dtype=torch.int32), empty(E), empty(E)
        scratch = empty(native.lib().balance_ctas(T, E) * 2 * (E + 1))
        native.lib().balance_fwd(logits.contiguous(), idx.contiguous(), None if mask is None else mask.contiguous(), loss, counts,
                                 prob, factor, scratch, native.status_tensor(logits.device))
        return loss, counts, prob, factor
    on = torch.ones(T, dtype=torch.bool) if mask is None else mask
    n = max(1, int(on.sum()))
    chosen = idx[on].reshape(-1).long()
    if bool(((chosen < 0) | (chosen >= E)).any()):
        raise ValueError(f"moe_balance_loss: idx holds what is no expert of {E}")
    counts = torch.bincount(chosen, minlength=E)
    prob = _probabilities(logits[on]).sum(0) / n
    share = counts.double() * (E / (n * idx.shape[1]))
    return (share * prob).sum().float(), counts.to(torch.int32), prob.float(), (share / n).float()


@moe_balance_fwd.register_fake
def _(logits, idx, mask):
    E = logits.shape[1]
    return (logits.new_empty((), dtype=torch.float32), logits.new_empty((E,), dtype=torch.int32),
            logits.new_empty((E,), dtype=torch.float32), logits.new_empty((E,), dtype=torch.float32))


def _balance_setup(ctx, inputs, output):
    logits, idx, mask = inputs
    _loss, counts, prob, factor = output
    ctx.mark_non_differentiable(counts, prob, factor)
    ctx.save_for_backward(logits, idx, mask, factor)


def _balance_backward(ctx, d_loss, _d_counts, _d_prob, _d_factor):
    logits, idx, mask, factor = ctx.saved_tensors
    if d_loss is None:
        return torch.zeros_like(logits), None, None
    if _is_native(logits):
        d = torch.empty_like(logits, memory_format=torch.contiguous_format)
        native.lib().balance_bwd(logits.contiguous(), idx.contiguous(), None if mask is None else mask.contiguous(), factor,
                                 d_loss.to(torch.float32).contiguous(), d)
    else:
        with torch.no_grad():
            p, c = _probabilities(logits), factor.double() * d_loss.double()
            d = p * (c - (p * c).sum(1, keepdim=True))
            if mask is not None:
                d = torch.where(mask.unsqueeze(1), d, 0.0)
            d = d.to(logits.dtype)
    return once_differentiable("moe_balance_loss", d, logits), None, None


moe_balance_fwd.register_autograd(_balance_backward, setup_context=_balance_setup)
moe_balance_fwd = moe_balance_fwd.overload


def moe_balance_loss(logits: Tensor, idx: Tensor, *, mask: Optional[Tensor] = None) -> BalanceLoss:
    """E sum_e f_e P_e of a router: f_e the share of the choices ``idx`` (int32 [T, k], as ``moe_route`` gives) that went to expert
    e, P_e its mean probability under ``logits`` [T, E], both over the tokens that count (``mask``, bool [T]).  1 where all
    experts get the same, 0 without a token that counts.

    Logits are bf16 or fp32, at most 256 experts; the choices have no gradient, and nothing at tokens that do not count reaches a
    result.  A row of -inf alone has no probabilities and no gradient.  The gradient has no derivative of its own.  On
    a GPU a choice that is no expert is left out, and the next status check raises.
    """
    if not logits.is_cuda:                           # on a GPU the op makes these checks by itself
        if not logits.is_floating_point():
            raise TypeError(f"moe_balance_loss: logits must be floating point, got {logits.dtype}")
        if logits.dim() != 2 or not 1 <= logits.shape[1] <= MAX_BALANCE_EXPERTS:
            raise ValueError(f"moe_balance_loss: logits must be [T, E] with 1 to {MAX_BALANCE_EXPERTS} experts, got {tuple(logits.shape)}")
        T, E = logits.shape
        if idx.dtype != torch.int32 or idx.dim() != 2 or idx.shape[0] != T or not 1 <= idx.shape[1] <= E:
            raise ValueError(f"moe_balance_loss: idx must be int32 [{T}, 1 to {E}], got {idx.dtype} {tuple(idx.shape)}")
        if idx.device != logits.device:
            raise ValueError(f"moe_balance_loss: idx is on {idx.device}, logits on {logits.device}")
        if mask is not None and (mask.dtype != torch.bool or mask.shape != (T,) or mask.device != logits.device):
            raise ValueError(f"moe_balance_loss: mask must be bool [{T}] on {logits.device}, got {mask.dtype} {tuple(mask.shape)} on "
                             f"{mask.device}")
    return BalanceLoss(*moe_balance_fwd(logits, idx, mask)[:3])


@custom_op("piper::moe_attach_loss")
def moe_attach_loss(weights: Tensor, loss: Tensor, coef: float) -> Tensor:
    """The routing weights as they are; in a backward pass that reaches them ``loss`` gets the gradient ``coef``, as if coef x loss had
    been added to what the pass began with, whatever factor that had.  So a stage's auxiliary loss need not travel to the last stage."""
    return weights.clone()


@moe_attach_loss.register_fake
def _(weights, loss, coef):
    return torch.empty_like(weights)


def _attach_setup(ctx, inputs, output):
    _weights, loss, coef = inputs
    ctx.coef, ctx.like = coef, (loss.shape, loss.dtype, loss.device)


def _attach_backward(ctx, d_weights):
    shape, dtype, device = ctx.like
    return d_weights, torch.full(shape, ctx.coef, dtype=dtype, device=device), None


moe_attach_loss.register_autograd(_attach_backward, setup_context=_attach_setup)
moe_attach_loss = moe_attach_loss.overload


# -------------------------------------------------------------- group table
@custom_op("piper::moe_group_table")
def moe_group_table(counts: Tensor, expert_weights: Tensor) -> tuple[Tensor, Tensor]:
    """counts [G] int32 (source-major) -> (g_start, g_len): padded segments laid out back to back.

    The number of local experts is read from ``expert_weights.shape[0]`` when the op runs, not baked in as a
    traced constant, so the same graph serves any expert-parallel degree.
    """
    experts = expert_weights.shape[0]
    if _is_native(counts):
        if _EP_TABLE is not None and _EP_TABLE[0].numel() == counts.numel():
            return _EP_TABLE[0].clone(), _EP_TABLE[1].clone()
        g_start = torch.empty_like(counts)
        g_len = torch.empty_like(counts)
        total = torch.empty(1, dtype=torch.int32, device=counts.device)
        native.lib().moe_group_table(counts.contiguous(), experts, None, g_start, g_len, total)
        return g_start, g_len
    g_len = (counts + (PAD - 1)) // PAD * PAD
    g_start = torch.cumsum(g_len, 0) - g_len
    return g_start.to(torch.int32), g_len.to(torch.int32)


host_op("moe_group_table_host", moe_group_table._body)


@moe_group_table.register_fake
def _(counts, expert_weights):
    return torch.empty_like(counts), torch.empty_like(counts)


# ---------------------------------------------------------------- dispatch
@custom_op("piper::moe_dispatch")
def moe_dispatch(x: Tensor, idx: Tensor, counts: Tensor) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """x [T, D] -> (rows [cap, D], pos int32 [T*k], g_start int32 [E], g_len int32 [E], ep_counts int32 [E]).

    ``ep_counts`` is a copy of ``counts`` meant for the expert region alone: an expert-parallel token exchange
    replaces it by the counts received from the peers, while ``counts`` keeps describing the local layout.
    """
    T, D = x.shape
    k = idx.shape[1]
    E = counts.shape[0]
    cap = row_capacity(T, k, E)
    if _is_native(x):
        _require_bf16(x)
        if _EP_RUNTIME is not None and _EP_RUNTIME.active is not None:
            return _EP_RUNTIME.dispatch(x, idx, counts)
        g_start = torch.empty_like(counts)
        g_len = torch.empty_like(counts)
        cursor = torch.empty_like(counts)
        copy = torch.empty_like(counts)
        native.lib().moe_dispatch_table(counts, g_start, g_len, cursor, copy)
        rows = torch.empty((cap, D), dtype=x.dtype, device=x.device)
        pos = torch.empty(T * k, dtype=torch.int32, device=x.device)
        native.lib().moe_permute(x.contiguous(), idx, g_start, g_len, counts, cursor, pos, rows)
        return rows, pos, g_start, g_len, copy
    g_len = (counts + (PAD - 1)) // PAD * PAD
    g_start = (torch.cumsum(g_len, 0) - g_len).to(torch.int32)
    flat_e = idx.reshape(-1).long()
    order = torch.argsort(flat_e, stable=True)
    rank_in_e = torch.empty_like(order)
    sorted_e = flat_e[order]
    first = torch.searchsorted(sorted_e, sorted_e)
    rank_in_e[order] = torch.arange(order.numel()) - first
    pos = (g_start.long()[flat_e] + rank_in_e).to(torch.int32)
    rows = torch.zeros((cap, D), dtype=x.dtype)
    rows[pos.long()] = x.repeat_interleave(k, dim=0)
    return rows, pos, g_start, g_len.to(torch.int32), counts.clone()


host_op("moe_dispatch_host", moe_dispatch._body)


@moe_dispatch.register_fake
def _(x, idx, counts):
    T, D = x.shape
    k, E = idx.shape[1], counts.shape[0]
    return (x.new_empty((row_capacity(T, k, E), D)), x.new_empty((T * k,), dtype=torch.int32),
            torch.empty_like(counts), torch.empty_like(counts), torch.empty_like(counts))


def _dispatch_setup(ctx, inputs, output):
    x, idx, _counts = inputs
    ctx.k = idx.shape[1]
    ctx.xshape, ctx.xdtype = x.shape, x.dtype
    ctx.save_for_backward(output[1])


def _dispatch_backward(ctx, drows, _dpos, _dgs, _dgl, _dec):
    (pos,) = ctx.saved_tensors
    T, D = ctx.xshape
    if drows is None:
        return torch.zeros((T, D), dtype=ctx.xdtype, device=pos.device), None, None
    if _is_native(drows):
        dx = torch.empty((T, D), dtype=drows.dtype, device=drows.device)
        native.lib().moe_permute_bwd(drows.contiguous(), pos, dx, ctx.k)
        return dx, None, None
    dx = drows[pos.long()].float().reshape(T, ctx.k, D).sum(1)
    return dx.to(drows.dtype), None, None


moe_dispatch.register_autograd(_dispatch_backward, setup_context=_dispatch_setup)


# ----------------------------------------------------------- grouped linear
def _grouped(mode: int, x, dy, w, out, g_start, g_len, experts: int, N: int, K: int, accumulate: bool = False):
    native.lib().grouped_gemm(mode, x, dy, w, out, g_start, g_len, experts, N, K, accumulate,
                              native.status_tensor(out.device))
    return out


def _grouped_ref_segments(g_start: Tensor, g_len: Tensor):
    gs, gl = g_start.tolist(), g_len.tolist()
    return [(g, s, s + n) for g, (s, n) in enumerate(zip(gs, gl)) if n > 0]


@custom_op("piper::grouped_linear")
def grouped_linear(rows: Tensor, w: Tensor, g_start: Tensor, g_len: Tensor) -> Tensor:
    """out[r] = rows[r] @ w[expert(group of r)]^T for w [experts, N, K]; rows outside every group are undefined."""
    E, N, K = w.shape
    if _is_native(rows):
        _require_bf16(rows, w)
        out = torch.empty((rows.shape[0], N), dtype=rows.dtype, device=rows.device)
        return _grouped(0, rows.contiguous(), None, w, out, g_start, g_len, E, N, K)
    out = torch.zeros((rows.shape[0], N), dtype=rows.dtype)
    for g, a, b in _grouped_ref_segments(g_start, g_len):
        out[a:b] = rows[a:b] @ w[g % E].t()
    return out


@grouped_linear.register_fake
def _(rows, w, g_start, g_len):
    return rows.new_empty((rows.shape[0], w.shape[1]))


def _grouped_wgrad(rows: Tensor, dy: Tensor, w: Tensor, g_start: Tensor, g_len: Tensor) -> Optional[Tensor]:
    E, N, K = w.shape
    sink = grad_sinks.get(w)
    if _is_native(rows):
        if sink is not None:
            _grouped(2, rows, dy, None, sink, g_start, g_len, E, N, K, accumulate=True)
            return None
        # every tile of dW is written once (zeros for an expert without rows), rounded from the fp32 accumulator
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device)
        return _grouped(2, rows, dy, None, dw, g_start, g_len, E, N, K, accumulate=False)
    dw = torch.zeros(w.shape, dtype=torch.float32)
    for g, a, b in _grouped_ref_segments(g_start, g_len):
        dw[g % E] += dy[a:b].float().t() @ rows[a:b].float()
    if sink is not None:
        sink.add_(dw)
        return None
    return dw.to(w.dtype)


def _glinear_setup(ctx, inputs, output):
    rows, w, g_start, g_len = inputs
    ctx.save_for_backward(rows, w, g_start, g_len)


def _glinear_backward(ctx, dy):
    rows, w, g_start, g_len = ctx.saved_tensors
    E, N, K = w.shape
    dyc = dy.contiguous()
    if (core._GEMM_FORK and ctx.needs_input_grad[0] and ctx.needs_input_grad[1] and wgrad_store.active is None
            and _is_native(rows) and grad_sinks.get(w) is not None):
        # same fork as in the dense linear backward: the weight-gradient GEMM runs on a side stream
        cur = torch.cuda.current_stream(rows.device)
        side = core._side_stream(cur)
        side.wait_stream(cur)
        with torch.cuda.stream(side):
            _grouped_wgrad(rows, dyc, w, g_start, g_len)
        drows = torch.empty_like(rows, memory_format=torch.contiguous_format)
        _grouped(1, None, dyc, w, drows, g_start, g_len, E, N, K)
        if core._GEMM_FORK == 2 and core.deferred_join.depth > 0:
            for t in (rows, dyc, g_start, g_len):
                t.record_stream(side)
            core.deferred_join.pending[(cur.device.index, cur.cuda_stream)] = (cur, side)
        else:
            cur.wait_stream(side)
        return drows, None, None, None
    drows = None
    if ctx.needs_input_grad[0]:
        if _is_native(rows):
            drows = torch.empty_like(rows, memory_format=torch.contiguous_format)
            _grouped(1, None, dyc, w, drows, g_start, g_len, E, N, K)
        else:
            drows = torch.zeros_like(rows)
            for g, a, b in _grouped_ref_segments(g_start, g_len):
                drows[a:b] = dyc[a:b] @ w[g % E]
    dw = None
    if ctx.needs_input_grad[1]:
        if wgrad_store.active is not None:
            rd, dd = rows.detach(), dyc.detach()
            wgrad_store.active.append((lambda: _grouped_wgrad(rd, dd, w, g_start, g_len), w))
        else:
            dw = _grouped_wgrad(rows, dyc, w, g_start, g_len)
    return drows, dw, None, None


grouped_linear.register_autograd(_glinear_backward, setup_context=_glinear_setup)


def _glinear_backward_host(dy: Tensor, rows: Tensor, w: Tensor, g_start: Tensor, g_len: Tensor, need_rows: bool,
                           need_w: bool) -> tuple[Tensor, Tensor]:
    drows, dw, _, _ = _glinear_backward(core.HostContext((rows, w, g_start, g_len), (need_rows, need_w)), dy)
    none = torch.empty(0)
    return none if drows is None else drows, none if dw is None else dw


host_op("grouped_linear_backward_host", _glinear_backward_host)


# ----------------------------------------------------------------- combine
@custom_op("piper::moe_combine")
def moe_combine(rows: Tensor, pos: Tensor, weights: Tensor, g_start: Tensor, g_len: Tensor, counts: Tensor) -> Tensor:
    """out[t] = sum_j weights[t, j] * rows[pos[t*k + j]]."""
    T, k = weights.shape
    D = rows.shape[1]
    if _is_native(rows):
        _require_bf16(rows)
        out = torch.empty((T, D), dtype=rows.dtype, device=rows.device)
        native.lib().moe_combine(rows.contiguous(), pos, weights.contiguous(), out)
        return out
    picked = rows[pos.long()].float().reshape(T, k, D)
    return (picked * weights.float().unsqueeze(-1)).sum(1).to(rows.dtype)


@moe_combine.register_fake
def _(rows, pos, weights, g_start, g_len, counts):
    return rows.new_empty((weights.shape[0], rows.shape[1]))


def _combine_setup(ctx, inputs, output):
    rows, pos, weights, g_start, g_len, counts = inputs
    ctx.save_for_backward(rows, pos, weights, g_start, g_len, counts)


def _combine_backward(ctx, dout):
    rows, pos, weights, g_start, g_len, counts = ctx.saved_tensors
    T, k = weights.shape
    D = rows.shape[1]
    if _is_native(rows):
        drows = torch.empty_like(rows, memory_format=torch.contiguous_format)
        dweights = torch.empty_like(weights, memory_format=torch.contiguous_format)
        native.lib().moe_combine_bwd(rows.contiguous(), dout.contiguous(), pos, weights.contiguous(), drows, dweights,
                                     g_start, g_len, counts)
        return drows, None, dweights, None, None, None
    drows = torch.zeros_like(rows)
    g = dout.float().unsqueeze(1) * weights.float().unsqueeze(-1)
    drows[pos.long()] = g.reshape(T * k, D).to(rows.dtype)
    dweights = (rows[pos.long()].float().reshape(T, k, D) * dout.float().unsqueeze(1)).sum(-1)
    return drows, None, dweights.to(weights.dtype), None, None, None


moe_combine.register_autograd(_combine_backward, setup_context=_combine_setup)

# The registered overloads are what programs call and tracers record.
moe_route = moe_route.overload
moe_group_table = moe_group_table.overload
moe_dispatch = moe_dispatch.overload
grouped_linear = grouped_linear.overload
moe_combine = moe_combine.overload
