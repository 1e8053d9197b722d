"""AdamW over many tensors at once, with moments in 32 or in 8 bits (``csrc/adamw.cu``).

The executor steps flat buckets (``runtime/storage.py``, which uses this state where ``state_bits`` is 8); a program with
tensors of its own steps them all in one launch::

    state = ops.AdamWState(params, bits=8)
    ...
    ops.adamw_step(params, [p.grad for p in params], state, lr=3e-4, betas=(0.9, 0.95), weight_decay=0.1)

8-bit moments take 2.03 bytes an element in place of 8.  A block of 256 elements keeps its largest magnitude as an fp32 scale;
an element is an 8-bit number relative to it with three bits of mantissa (the first moment 16 binades and a sign, the
second 32 binades), rounded up or down at random in proportion to the distance.  The random bits depend on the step, the
tensor's place in the list (counted from the state's ``first``) and the element alone: a step from the same state gives the same bits.

The kernel's square root and quotient are approximate, each within two units of the last place: an update differs by up to 2^-20 of itself
from the same formula with rounded operations, which is what the executor's 32-bit buckets use (``adam_flat``).
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch
from torch import Tensor

from . import native

BLOCK = 256
_PIECE = BLOCK << 14               # elements of a state that are encoded or decoded at a time
_M_BASE, _V_BASE = 889, 761        # fp32 bits >> 20 of code 0; those of 1.0 are 1016, codes 127 and 255


def _mix32(h: Tensor) -> Tensor:
    """The mixer of ``csrc/adamw.h`` (C. Wellons, 2018)."""
    for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B)):
        h = ((h ^ (h >> shift)) * factor) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _random16(step: int, ordinal: int, n: int, device) -> tuple[Tensor, Tensor]:
    seed = int(_mix32(torch.tensor((step * 0x9E3779B1 + ordinal * 0x85EBCA77) & 0xFFFFFFFF)))
    h = _mix32((torch.arange(n, device=device) + seed) & 0xFFFFFFFF)
    return h & 0xFFFF, h >> 16


def _decode(codes: Tensor, scale: Tensor, signed: bool) -> Tensor:
    c = codes.to(torch.int32)
    low = c & 127 if signed else c
    x = torch.where(low > 0, (low + (_M_BASE if signed else _V_BASE)) << 20, torch.zeros_like(low)).view(torch.float32)
    x = (x.view(-1, BLOCK) * scale.unsqueeze(1)).view(-1)
    return torch.where(c >= 128, -x, x) if signed else x


def _encode(x: Tensor, r: Tensor, signed: bool) -> tuple[Tensor, Tensor]:
    """Codes and scales of whole blocks of fp32 values; r: 16 random bits for each."""
    a = x.abs().view(-1, BLOCK)
    scale = torch.where(torch.isfinite(a).all(1), a.amax(1), torch.full((), math.nan, device=x.device))
    y = (a / torch.where(scale > 0, scale, torch.ones_like(scale)).unsqueeze(1)).view(-1)
    base = _M_BASE if signed else _V_BASE
    least = float(torch.tensor((base + 1) << 20, dtype=torch.int32).view(torch.float32))
    codes = ((y.view(torch.int32) + (r << 4).to(torch.int32)) >> 20) - base
    small = (r.to(torch.float32) * (least / 65536) < y) if signed else x > 0      # y may be below all numbers
    codes = torch.where(y < least, small.to(torch.int32), codes)
    if signed:
        codes = codes + 128 * (x < 0)
    return (codes & 255).to(torch.uint8), scale


def _check_apart(params: Sequence[Tensor], what: str) -> None:
    at = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in params if p.numel())
    if any(a[1] > b[0] for a, b in zip(at, at[1:])):
        raise ValueError(f"{what}: two parameters share memory, or one is listed twice")


class AdamWState:
    """Moments, master copies and step counts of a list of parameters (bf16 or fp32, contiguous, on one device, no two of which
    share memory).

    Everything is flat: parameter ``i`` owns the elements ``[offsets[i], offsets[i] + numel)`` of ``m`` and ``v`` (fp32, or
    uint8 codes with the scales ``m_scale`` and ``v_scale`` of their blocks of 256) and, where a parameter is bf16, of the
    fp32 ``master``, from which its update starts.  Tensors begin at whole blocks; what is between them stays zero.  With 8 bits, a
    moment that is infinite or NaN makes its block NaN.  ``first`` is the place of the first parameter among those of other states of
    the same model, which would otherwise round with the same random bits.
    """

    def __init__(self, params: Sequence[Tensor], *, bits: int = 32, first: int = 0) -> None:
        params = list(params)
        if bits not in (8, 32):
            raise ValueError(f"AdamWState: bits must be 8 or 32, got {bits}")
        if not params:
            raise ValueError("AdamWState: no parameters")
        if not 0 <= first < 1 << 32:
            raise ValueError(f"AdamWState: first must be 0 to 2^32 - 1, got {first}")
        self.bits, self.first, self.device = bits, first, params[0].device
        self.shapes = [tuple(p.shape) for p in params]
        self.dtypes = [p.dtype for p in params]
        self.offsets, at = [], 0
        for p in params:
            if p.dtype not in (torch.bfloat16, torch.float32):
                raise TypeError(f"AdamWState: parameters are bfloat16 or float32, got {p.dtype}")
            if p.device != self.device:
                raise ValueError(f"AdamWState: parameters on {self.device} and {p.device}")
            if not p.is_contiguous():
                raise ValueError("AdamWState: parameters must be contiguous")
            self.offsets.append(at)
            at += (p.numel() + BLOCK - 1) // BLOCK * BLOCK
        _check_apart(params, "AdamWState")
        self.numel = at
        # what the library reads and counts on: offsets, twice the elements and one for bf16, steps
        self._table = torch.tensor([self.offsets, [2 * p.numel() + (p.dtype == torch.bfloat16) for p in params],
                                    [0] * len(params)], dtype=torch.int64)
        moment = dict(dtype=torch.uint8 if bits == 8 else torch.float32, device=self.device)
        self.m, self.v = torch.zeros(at, **moment), torch.zeros(at, **moment)
        self.m_scale = self.v_scale = self.master = None
        if bits == 8:
            self.m_scale, self.v_scale = (torch.zeros(at // BLOCK, dtype=torch.float32, device=self.device) for _ in range(2))
        if torch.bfloat16 in self.dtypes:
            self.master = torch.zeros(at, dtype=torch.float32, device=self.device)
            self.read_masters(params)

    def read_masters(self, params: Sequence[Tensor]) -> None:
        """Master copies from the parameters as they are now (after somebody else wrote them)."""
        with torch.no_grad():
            for o, p in zip(self.offsets, params):
                if p.dtype == torch.bfloat16:
                    self.master[o:o + p.numel()].copy_(p.detach().reshape(-1))

    @property
    def steps(self) -> list:
        """The number of steps taken so far, of each parameter."""
        return self._table[2].tolist()

    def set_step(self, step: int) -> None:
        """The number of steps taken so far, of all parameters."""
        if step < 0:
            raise ValueError(f"AdamWState: steps are counted from 0, got {step}")
        self._table[2] = int(step)

    def moments(self) -> tuple[Tensor, Tensor]:
        """Both moments in fp32, flat as ``m`` and ``v`` are (those themselves if they have 32 bits)."""
        if self.bits == 32:
            return self.m, self.v
        if not self.m.is_cuda:
            return _decode(self.m, self.m_scale, True), _decode(self.v, self.v_scale, False)
        out = [torch.empty(self.numel, dtype=torch.float32, device=self.device) for _ in range(2)]
        native.lib().moments_decode(self.m, self.m_scale, self.v, self.v_scale, out[0], out[1])
        return out[0], out[1]

    def set_moments(self, m: Tensor, v: Tensor) -> None:
        """The reverse of ``moments()``; 8-bit codes are the nearest ones, so what came out of it goes back unchanged.  What is
        missing at the end counts as zeros."""
        if m.dim() != 1 or m.shape != v.shape or m.numel() > self.numel:
            raise ValueError(f"AdamWState: moments are two tensors of at most {self.numel} elements, got {tuple(m.shape)} and {tuple(v.shape)}")
        with torch.no_grad():
            if self.bits == 32:
                for x, own in ((m, self.m), (v, self.v)):
                    own[:x.numel()] = x
                    own[x.numel():] = 0
                return
            # in pieces: encoding takes some fifty bytes an element, many times what the state holds
            half = torch.full((min(self.numel, _PIECE),), 1 << 15, dtype=torch.int64, device=self.device)
            for x, codes, scale, signed in ((m, self.m, self.m_scale, True), (v, self.v, self.v_scale, False)):
                for a in range(0, self.numel, _PIECE):
                    z = min(a + _PIECE, self.numel)
                    part = torch.zeros(z - a, dtype=torch.float32, device=self.device)
                    part[:max(min(x.numel(), z) - a, 0)] = x[a:z]
                    codes[a:z], scale[a // BLOCK:z // BLOCK] = _encode(part, half[:z - a], signed)

    def state_dict(self) -> dict:
        return {"bits": self.bits, "shapes": list(self.shapes), "dtypes": list(self.dtypes), "steps": list(self.steps),
                "m": self.m, "v": self.v, "m_scale": self.m_scale, "v_scale": self.v_scale, "master": self.master}

    def load_state_dict(self, state: dict) -> None:
        """Takes over a state of the same parameters, of either width.  Nothing is written if it is of others."""
        if [tuple(s) for s in state["shapes"]] != self.shapes:
            raise ValueError("AdamWState: the state is of other parameters")
        # which of its parameters have a master copy; a state that does not say had better be of one type
        dtypes = state.get("dtypes")
        if (state["master"] is None) != (self.master is None) or (
                list(dtypes) != self.dtypes if dtypes is not None else len(set(self.dtypes)) > 1):
            raise ValueError("AdamWState: the state is of parameters of another type")
        if len(state["steps"]) != len(self.shapes) or any(
                state[n].numel() != self.numel for n in ("m", "v", "master") if state[n] is not None):
            raise ValueError("AdamWState: the state is of another layout")
        with torch.no_grad():
            if state["bits"] == self.bits:
                for name in ("m", "v", "m_scale", "v_scale"):
                    if getattr(self, name) is not None:
                        getattr(self, name).copy_(state[name])
            else:
                if state["bits"] == 32:
                    self.set_moments(state["m"], state["v"])
                for name, signed in (("m", True), ("v", False)) if state["bits"] == 8 else ():
                    for a in range(0, self.numel, _PIECE):
                        z = min(a + _PIECE, self.numel)
                        getattr(self, name)[a:z] = _decode(state[name][a:z].to(self.device),
                                                           state[name + "_scale"][a // BLOCK:z // BLOCK].to(self.device), signed)
            if self.master is not None:
                self.master.copy_(state["master"])
        self._table[2] = torch.tensor([int(s) for s in state["steps"]], dtype=torch.int64)


def adamw_step(params: Sequence[Tensor], grads: Sequence[Optional[Tensor]], state: AdamWState, *, lr: float = 1e-3,
               betas: tuple = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, grad_scale: float = 1.0) -> None:
    """One step of AdamW (decoupled weight decay) for all ``params`` with a gradient, in place.

    ``grads`` are bf16 or fp32, shaped like their parameters, and are multiplied by ``grad_scale`` (the mean over
    microbatches, a clipping factor); a parameter whose gradient is None is left as it is and its step count with it.  The
    step counts live on the host, so a step cannot be captured into a CUDA graph, which would repeat one bias correction.
    """
    params, grads = list(params), list(grads)
    b1, b2 = betas
    if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and 0 <= b1 < 1 and 0 <= b2 < 1):
        raise ValueError(f"adamw_step: lr={lr}, betas={betas}, eps={eps}, weight_decay={weight_decay}")
    if state.device.type == "cuda":
        if params and params[0].device != state.device:
            raise ValueError(f"adamw_step: the state is on {state.device}, a parameter on {params[0].device}")
        # the library checks every tensor, and that its stream is not captured, before it launches anything
        native.lib().adamw.default(params, grads, state.m, state.v, state.m_scale, state.v_scale, state.master, state._table,
                                   state.first, lr, b1, b2, eps, weight_decay, grad_scale)
    else:
        if len(params) != len(state.shapes) or len(grads) != len(params):
            raise ValueError(f"adamw_step: {len(params)} parameters, {len(grads)} gradients, a state of {len(state.shapes)}")
        for p, g, size, dtype in zip(params, grads, state._table[1].tolist(), state.dtypes):
            if p.dtype != dtype or 2 * p.numel() + (p.dtype == torch.bfloat16) != size or p.device != state.device:
                raise ValueError(f"adamw_step: the state is of a {dtype} parameter of {size // 2} elements on {state.device}, got "
                                 f"{p.dtype} {tuple(p.shape)} on {p.device}")
            if not p.is_contiguous():
                raise ValueError("adamw_step: parameters must be contiguous")
            if g is not None and (g.shape != p.shape or g.device != p.device):
                raise ValueError(f"adamw_step: a gradient is {tuple(g.shape)} on {g.device}, its parameter {tuple(p.shape)}")
            if g is not None and g.dtype not in (torch.float32, torch.bfloat16):
                raise ValueError(f"adamw_step: gradients are bfloat16 or float32, got {g.dtype}")
        _check_apart(params, "adamw_step")
        with torch.no_grad():
            for i, (p, g, done) in enumerate(zip(params, grads, state.steps)):
                if g is not None and p.numel():
                    _step_ref(state, i, p, g, done + 1, lr, b1, b2, eps, weight_decay, grad_scale)
        torch.autograd.graph.increment_version([p for p, g in zip(params, grads) if g is not None and not p.is_inference()])
        state._table[2] += torch.tensor([g is not None for g in grads], dtype=torch.int64)


def _step_ref(state: AdamWState, i: int, p: Tensor, grad: Tensor, step: int, lr: float, b1: float, b2: float, eps: float,
              wd: float, grad_scale: float) -> None:
    n, o = p.numel(), state.offsets[i]
    whole = (n + BLOCK - 1) // BLOCK * BLOCK
    part, blocks = slice(o, o + whole), slice(o // BLOCK, (o + whole) // BLOCK)
    g = torch.zeros(whole, dtype=torch.float32, device=p.device)
    g[:n] = grad.reshape(-1)
    g *= grad_scale
    if state.bits == 8:
        m, v = _decode(state.m[part], state.m_scale[blocks], True), _decode(state.v[part], state.v_scale[blocks], False)
    else:
        m, v = state.m[part], state.v[part]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * (1 - b2) * g
    m[n:] = 0
    v[n:] = 0
    w = state.master[o:o + n] if p.dtype == torch.bfloat16 else p.detach().view(-1)
    update = m[:n] / (torch.sqrt(v[:n]) * (1 / math.sqrt(1 - b2 ** step)) + eps)
    w.copy_(w * (1 - lr * wd) - update * (lr / (1 - b1 ** step)))
    if p.dtype == torch.bfloat16:
        p.detach().view(-1).copy_(w)
    if state.bits == 8:
        rm, rv = _random16(step, state.first + i, whole, p.device)
        state.m[part], state.m_scale[blocks] = _encode(m, rm, True)
        state.v[part], state.v_scale[blocks] = _encode(v, rv, False)
    else:
        state.m[part], state.v[part] = m, v
