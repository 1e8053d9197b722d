"""Packed batches: sequences of any lengths, one behind the other in a batch of tokens, and causal attention within each of them.

What fine-tuning on conversations and replies wants in place of ``attention``, whose sequences all have one length, a multiple of
128.  ``pack_sequences`` lays out a batch once; every layer, forward and backward, and ``clipped_policy_loss`` take the result.
Kernels: ``csrc/pack.cu``, ``csrc/attention_sm100.cu``.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import native
from .core import _is_native, _require_bf16
from .registry import custom_op, once_differentiable

BLOCK = 128                      # rows of a query or key block
MAX_TOKENS = 1 << 21
# Short neighbours share blocks where that saves a fifth of some 5,800 cycles a pair of a query and a key block and 7,500 a block, and where
# the query blocks of all heads are more than two for each of 148 SMs.  Time of both passes with groups, of that without, by that
# share of cycles, on 340 to 16,000 tokens in up to 871 sequences: 1.0-1.06 at 0.9 and above, 0.90-1.03 at 0.77 to 0.9, 0.24-0.76 below; with
# 112 blocks of all heads 1.16 at 0.29.
GROUP_GAIN = 1.25
GROUP_BLOCKS = 296


class PackedSequences(NamedTuple):
    """Where the sequences of a packed batch lie.  ``longest`` (blocks of the longest sequence), ``work`` and ``tile_work`` (pairs of a
    query and a key block) only choose launch shapes: where the offsets are on a GPU, they are those of equal sequences."""

    offsets: Tensor              # int32 [n + 1]: sequence i has rows offsets[i] to offsets[i + 1]
    table: Tensor                # int32 [blocks + 1, 4]: blocks of the sequences, see _table_ref
    tiles: Optional[Tensor]      # the same with groups of short sequences, if there are enough of them, and
    own: Optional[Tensor]        # uint8 [128 * blocks, 2]: see _groups_ref
    tokens: int                  # rows of the batch, those behind the last sequence included
    longest: int
    work: int
    tile_work: int

    def inside(self) -> Tensor:
        """bool [tokens]: whether a token belongs to a sequence."""
        # by the table, where all is behind the last sequence if offsets on a GPU do not rise from 0 to at most `tokens`
        return torch.arange(self.tokens, device=self.offsets.device) < self.table[0, 1]

    def positions(self) -> Tensor:
        """int64 [tokens]: a token's place in its sequence, 0 behind the last one."""
        at = torch.arange(self.tokens, device=self.offsets.device)
        of = torch.searchsorted(self.offsets, at, right=True) - 1
        return torch.where(self.inside(), at - self.offsets[of.clamp(min=0)], 0)


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _table_ref(offsets: list, tokens: int, blocks: int, marks: Optional[list] = None) -> Tensor:
    """Row 0: blocks in use, end of the last sequence, tokens, sequences that have rows.  Then, for every block of 128 rows, those with
    most blocks of their sequence in front of them first: first row of the sequence, its rows, place of the block in it, and 128 times the
    number of blocks of the sequences before, the sequence's mark added."""
    rows, before = [], 0
    for s, (a, b) in enumerate(zip(offsets, offsets[1:])):
        rows += [(a, b - a, i, before * BLOCK + (marks[s] if marks else 0)) for i in range(_blocks(b - a))]
        before += _blocks(b - a)
    rows.sort(key=lambda r: (-r[2], -_blocks(r[1]), r[0]))
    table = torch.zeros(blocks + 1, 4, dtype=torch.int32)
    table[0] = torch.tensor([len(rows), offsets[-1], tokens, sum(r[2] == 0 for r in rows)])
    if rows:
        table[1:len(rows) + 1] = torch.tensor(rows, dtype=torch.int32)
    return table


def _groups(offsets: list) -> list:
    """Neighbouring sequences that fit one block together, as lists of their indices, greedily within each of 32 parts."""
    n = len(offsets) - 1
    chunk, out = max(64, -(-n // 32)), []
    for c in range(0, n, chunk):
        group = []
        for s in range(c, min(n, c + chunk)):
            if offsets[s + 1] == offsets[s]:
                continue
            if group and offsets[s + 1] - offsets[group[0]] <= BLOCK:
                group.append(s)
            else:
                out.append(group := [s])
    return out


def _groups_ref(offsets: list, tokens: int, blocks: int) -> tuple[Tensor, Tensor]:
    """The table in which neighbouring sequences that fit one block together count as one, marked by 1; and for row i of such a group,
    at the place that its lse begins at plus i, the first and the last row of its own sequence in the group."""
    groups = _groups(offsets)
    ends = [offsets[g[0]] for g in groups] + [offsets[-1]]
    own, before = torch.zeros(blocks * BLOCK, 2, dtype=torch.uint8), 0
    for g, (a, b) in zip(groups, zip(ends, ends[1:])):
        for s in g if len(g) > 1 else []:
            first, last = offsets[s] - a, offsets[s + 1] - 1 - a
            own[before * BLOCK + first:before * BLOCK + last + 1] = torch.tensor([first, last], dtype=torch.uint8)
        before += _blocks(b - a)
    return _table_ref(ends, tokens, blocks, [int(len(g) > 1) for g in groups]), own


def _check_offsets(offsets: list, tokens: int) -> None:
    if offsets[0] != 0 or any(b < a for a, b in zip(offsets, offsets[1:])) or offsets[-1] > tokens:
        raise ValueError(f"pack_sequences: offsets must rise from 0 to at most {tokens}")


@custom_op("piper::pack_table")
def pack_table(offsets: Tensor, tokens: int, blocks: int, grouped: bool) -> tuple[Tensor, Tensor]:
    """(table, rows of groups)"""
    if _is_native(offsets):
        def empty(*shape, dtype=torch.int32):
            return torch.empty(shape, dtype=dtype, device=offsets.device)

        table, own = empty(blocks + 1, 4), empty(blocks * BLOCK if grouped else 0, 2, dtype=torch.uint8)
        native.lib().pack_table(offsets, tokens, table, own, empty(2 * (offsets.numel() - 1) if grouped else 0),
                                native.status_tensor(offsets.device))
        return table, own
    values = offsets.tolist()
    _check_offsets(values, tokens)
    if grouped:
        return _groups_ref(values, tokens, blocks)
    return _table_ref(values, tokens, blocks), torch.empty(0, 2, dtype=torch.uint8)


@pack_table.register_fake
def _(offsets, tokens, blocks, grouped):
    return (offsets.new_empty((blocks + 1, 4), dtype=torch.int32),
            offsets.new_empty((blocks * BLOCK if grouped else 0, 2), dtype=torch.uint8))


pack_table = pack_table.overload


def pack_sequences(offsets: Tensor, tokens: int, device: Optional[torch.device] = None) -> PackedSequences:
    """Lays out a batch of ``tokens`` rows in which sequence i has rows ``offsets[i]`` to ``offsets[i + 1]`` (int32 or int64 [n + 1],
    rising from 0; sequences may be empty).  Rows behind the last sequence belong to none.

    Offsets in host memory are checked here and give exact launch shapes; ``device`` is where the batch is.  Offsets
    on a GPU stay there, nothing waits for them: if they do not rise from 0 to at most ``tokens``, the batch counts as empty and the
    next status check raises.
    """
    if offsets.dim() != 1 or offsets.numel() < 1 or offsets.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"pack_sequences: offsets must be int32 or int64 [n + 1], got {offsets.dtype} {tuple(offsets.shape)}")
    if not 0 <= tokens <= MAX_TOKENS:
        raise ValueError(f"pack_sequences: 0 to {MAX_TOKENS} tokens, got {tokens}")
    n = offsets.numel() - 1
    if offsets.device.type == "cpu":
        values = offsets.tolist()
        _check_offsets(values, tokens)
        ends = [values[g[0]] for g in _groups(values)] + [values[-1]]
        counts, fewer = ([_blocks(b - a) for a, b in zip(v, v[1:])] for v in (values, ends))
        blocks, tiles, longest = sum(counts), sum(fewer), max(counts, default=0)
        work, tile_work = (sum(c * (c + 1) // 2 for c in v) for v in (counts, fewer))
        grouped = GROUP_GAIN * (tile_work * 5800 + tiles * 7500) < work * 5800 + blocks * 7500
        # a copy of what was checked; nothing waits for its way to the device
        offsets = torch.tensor(values, dtype=torch.int32).to("cpu" if device is None else device, non_blocking=True)
    else:
        if device is not None and torch.empty(0, device=device).device != offsets.device:
            raise ValueError(f"pack_sequences: offsets are on {offsets.device}, not on {device}")
        blocks = (tokens + (BLOCK - 1) * min(n, tokens)) // BLOCK
        grouped = tokens < n * BLOCK // 2
        # two neighbouring groups have more than 128 rows together, but at long sequences and the ends of the 32 parts
        tiles = min(blocks, 3 * tokens // BLOCK + 33)
        longest = _blocks(-(-tokens // max(n, 1)))
        work, tile_work = (min(max(n, 1), b) * longest * (longest + 1) // 2 for b in (blocks, tiles))
        # a copy: the caller may fill the same buffer for the next batch; what does not fit becomes an offset that is refused
        offsets = offsets.clamp(-1, (1 << 31) - 1).to(torch.int32).contiguous()
    pair = pack_table(offsets, tokens, tiles, True) if grouped else (None, None)
    return PackedSequences(offsets, pack_table(offsets, tokens, blocks, False)[0], *pair, tokens, longest, work, tile_work)


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------


def _sequences(table: Tensor, own: Optional[Tensor] = None) -> list:
    """(first row, rows, place of lse) of the sequences in a table on the CPU."""
    rows = table.tolist()
    out = []
    for a, n, i, at in rows[1:rows[0][0] + 1]:
        if i > 0:
            continue
        if at % 2 == 0:
            out.append((a, n, at))
            continue
        first = 0
        while first < n:
            last = int(own[at - 1 + first, 1])
            out.append((a + first, last + 1 - first, at - 1 + first))
            first = last + 1
    return out


def _attention_ref(q: Tensor, k: Tensor, v: Tensor, scale: float) -> tuple[Tensor, Tensor]:
    """[H, n, hd] in fp32 -> (out, lse)."""
    s = (q @ k.transpose(-1, -2)) * scale
    n = q.shape[1]
    s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), float("-inf"))
    return torch.softmax(s, -1) @ v, torch.logsumexp(s, -1)


def _heads(x: Tensor, Hq: int, Hkv: int, hd: int) -> tuple[Tensor, Tensor, Tensor]:
    """Rows of qkv as [H, n, hd] each, keys and values repeated over their group."""
    x = x.float().view(x.shape[0], Hq + 2 * Hkv, hd).transpose(0, 1)
    return x[:Hq], x[Hq:Hq + Hkv].repeat_interleave(Hq // Hkv, 0), x[Hq + Hkv:].repeat_interleave(Hq // Hkv, 0)


@custom_op("piper::packed_attention_fwd")
def packed_attention_fwd(qkv: Tensor, tiles: Tensor, own: Optional[Tensor], longest: int, work: int, Hq: int, Hkv: int, hd: int,
                         scale: float, keep: bool) -> tuple[Tensor, Tensor, Tensor]:
    """qkv [T, (Hq + 2 Hkv) * hd] -> (out [T, Hq * hd], lse [Hq, 128 * blocks], by the blocks of the tiles, and, if ``keep``, what
    rounding has taken from out, int8 [128 * blocks, Hq * hd] in the kernels' own order, which only they use).  The formula keeps it."""
    T, padded = qkv.shape[0], (tiles.shape[0] - 1) * BLOCK
    if _is_native(qkv):
        _require_bf16(qkv)
        out = torch.empty((T, Hq * hd), dtype=qkv.dtype, device=qkv.device)
        lse = torch.empty((Hq, padded), dtype=torch.float32, device=qkv.device)
        rest = torch.empty((padded if keep else 0, Hq * hd), dtype=torch.int8, device=qkv.device)
        native.lib().attn_packed_fwd(_aligned(qkv), tiles, own, out, lse, rest, longest, work, Hq, Hkv, hd, scale,
                                     native.status_tensor(qkv.device))
        return out, lse, rest
    out, lse = torch.zeros(T, Hq * hd, dtype=qkv.dtype), torch.zeros(Hq, padded)
    for a, n, at in _sequences(tiles, own):
        o, lse[:, at:at + n] = _attention_ref(*_heads(qkv[a:a + n], Hq, Hkv, hd), scale)
        out[a:a + n] = o.transpose(0, 1).reshape(n, Hq * hd).to(qkv.dtype)
    return out, lse, torch.zeros((padded if keep else 0, Hq * hd), dtype=torch.int8)


def _aligned(t: Tensor) -> Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


@packed_attention_fwd.register_fake
def _(qkv, tiles, own, longest, work, Hq, Hkv, hd, scale, keep):
    return (qkv.new_empty((qkv.shape[0], Hq * hd)),
            qkv.new_empty((Hq, (tiles.shape[0] - 1) * BLOCK), dtype=torch.float32),
            qkv.new_empty(((tiles.shape[0] - 1) * BLOCK if keep else 0, Hq * hd), dtype=torch.int8))


def _forward(ctx, qkv, tiles, own, longest, work, Hq, Hkv, hd, scale, _keep):
    out, lse, rest = packed_attention_fwd(qkv, tiles, own, longest, work, Hq, Hkv, hd, scale, True)
    ctx.set_materialize_grads(False)
    ctx.cfg = (longest, work, Hq, Hkv, hd, scale)
    ctx.mark_non_differentiable(lse, rest)
    ctx.save_for_backward(qkv, tiles, own, out, lse, rest)
    return out, lse, rest


def _backward(ctx, dout, _dlse, _drest):
    longest, work, Hq, Hkv, hd, scale = ctx.cfg
    qkv, tiles, own, out, lse, rest = ctx.saved_tensors
    none = (None,) * 9
    if dout is None:
        return torch.zeros_like(qkv), *none
    if _is_native(qkv):
        qc = _aligned(qkv)
        dqkv = torch.empty_like(qc)
        floats = native.lib().attn_packed_bwd_floats(tiles.shape[0] - 1, longest, work, Hq, Hkv, hd)
        scratch = torch.empty(floats, dtype=torch.float32, device=qkv.device)
        native.lib().attn_packed_bwd(qc, tiles, own, _aligned(out), _aligned(rest), _aligned(dout), _aligned(lse), scratch, dqkv, longest,
                                     work, Hq, Hkv, hd, scale, native.status_tensor(qkv.device))
        return once_differentiable("packed_attention", dqkv, qkv), *none
    dqkv = torch.zeros_like(qkv, memory_format=torch.contiguous_format)
    for a, n, _at in _sequences(tiles, own):
        with torch.enable_grad():
            rows = qkv[a:a + n].detach().float().requires_grad_(True)
            o, _ = _attention_ref(*_heads(rows, Hq, Hkv, hd), scale)
            (g,) = torch.autograd.grad(o, rows, dout[a:a + n].float().view(n, Hq, hd).transpose(0, 1))
        dqkv[a:a + n] = g.to(qkv.dtype)
    return once_differentiable("packed_attention", dqkv, qkv), *none


packed_attention_fwd.register_autograd(_backward, forward=_forward)
packed_attention_fwd = packed_attention_fwd.overload


def packed_attention(qkv: Tensor, sequences: PackedSequences, Hq: int, Hkv: int, hd: int, scale: float) -> Tensor:
    """Causal grouped-query attention within every sequence of a packed batch: ``qkv`` [tokens, (Hq + 2 Hkv) * hd] -> [tokens, Hq *
    hd].  Rows behind the last sequence give zeros and get a gradient of zero, whatever stands in them.

    bf16 and heads of 64 or 128 on a GPU; ``scale`` above 0.  What stands in one sequence, infinities and NaN included, does not reach
    another.  The gradient has no derivative of its own; for it ``qkv``, the output, and a byte an output and a number a row and head are
    kept, these two for whole blocks: by the batch's own number of them where the offsets were in host memory, by the most that
    ``tokens`` rows in as many sequences can have where they were on a GPU.
    """
    if qkv.dim() != 2 or qkv.shape[0] != sequences.tokens:
        raise ValueError(f"packed_attention: qkv is {tuple(qkv.shape)}, the batch has {sequences.tokens} tokens")
    tiles, own, work = sequences.table, None, sequences.work
    if sequences.own is not None and Hq * (tiles.shape[0] - 1) > GROUP_BLOCKS:
        tiles, own, work = sequences.tiles, sequences.own, sequences.tile_work
    if qkv.is_cuda:                              # the op makes the checks below by itself
        return packed_attention_fwd(qkv, tiles, own, sequences.longest, work, Hq, Hkv, hd, scale, False)[0]
    if Hq < 1 or Hkv < 1 or Hq % Hkv or qkv.shape[1] != (Hq + 2 * Hkv) * hd:
        raise ValueError(f"packed_attention: qkv must be [T, (Hq + 2 Hkv) * hd] with whole groups of heads, got "
                         f"{tuple(qkv.shape)} for {Hq} / {Hkv} heads of {hd}")
    if not 0 < scale < math.inf:
        raise ValueError(f"packed_attention: scale must be above 0, got {scale}")
    if tiles.device != qkv.device:
        raise ValueError(f"packed_attention: sequences are on {tiles.device}, qkv on {qkv.device}")
    return packed_attention_fwd(qkv, tiles, own, sequences.longest, work, Hq, Hkv, hd, scale, False)[0]
