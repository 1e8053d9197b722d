"""Matrix products in 8-bit floating point with a scale for every 128 elements of the contraction.

Operands are rounded to e4m3.  Activations and output gradients have a scale for every 128 neighbouring elements along the
contraction (``1 x 128``), weights one for every ``128 x 128``, so that a weight and its transpose have the same codes.
A scale is the smallest power of two that brings the group's largest magnitude to 448, the largest e4m3 number; scaling
is then exact, and an operand is rounded once.  Sums are kept in fp32 (``csrc/fp8_gemm_sm100.cu``).

``fp8_linear`` is ``linear`` with all three products of a training step in 8 bits: the gradient of the input contracts
over the weights' rows, the gradient of the weights over the tokens, for which input and output gradient are rounded in
groups of 128 tokens.  Between the passes it keeps the input as that 8-bit operand, half the bytes of the bf16 input, and of the
weight nothing but the weight, which is rounded again: every microbatch in flight would have a copy of its own, and a sharded
parameter would stay gathered.  A group with a NaN or an infinity is NaN.
"""
from __future__ import annotations

from typing import Optional, Union

import torch
from torch import Tensor

from . import native
from .core import grad_sinks, wgrad_store
from .registry import custom_op, host_op, once_differentiable

GROUP = 128
_NAN_SCALE = 255


def _sizes(rows: int, cols: int) -> tuple[int, int, int]:
    """Bytes of a row of codes, words of scales for a group of four, groups of four."""
    return (cols + 15) // 16 * 16, (rows + GROUP - 1) // GROUP * GROUP, (cols + 4 * GROUP - 1) // (4 * GROUP)


def _bytes(rows: int, cols: int) -> int:
    ld, pad, groups = _sizes(rows, cols)
    return rows * ld + 4 * groups * pad


class Fp8Matrix:
    """A matrix ``[rows, cols]`` in e4m3, ready as an operand of a product along ``cols``.

    ``data`` is one piece of memory, uint8: the ``codes`` ``[rows, cols rounded up to 16]`` and, behind them, the ``scales``, the
    exponents of the powers of two, with a bias of 127 (255: NaN), of four neighbouring groups of a row in one int32,
    ``[ceil(cols / 512), rows rounded up to 128]``.
    """

    def __init__(self, data: Tensor, rows: int, cols: int) -> None:
        self.data, self.rows, self.cols = data, rows, cols

    @property
    def codes(self) -> Tensor:
        ld = _sizes(self.rows, self.cols)[0]
        return self.data[:self.rows * ld].view(self.rows, ld)

    @property
    def scales(self) -> Tensor:
        ld, pad, groups = _sizes(self.rows, self.cols)
        return self.data[self.rows * ld:].view(torch.int32).view(groups, pad)

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.cols

    @property
    def device(self) -> torch.device:
        return self.data.device

    def dequantize(self) -> Tensor:
        """The values that the codes stand for, in fp32."""
        if self.data.is_cuda:
            out = torch.empty(self.rows, self.cols, dtype=torch.float32, device=self.device)
            native.lib().fp8_dequantize(self.data, out)
            return out
        return _values_ref(self.data, self.rows, self.cols)

    def __repr__(self) -> str:
        return f"Fp8Matrix({self.rows}, {self.cols}, device={self.device})"


# ------------------------------------------------------------------ plain form (CPU)
def _quantize_ref(x: Tensor, square: bool) -> Tensor:
    """x [rows, cols] as an operand along its columns."""
    rows, cols = x.shape
    if x.numel() == 0:
        return torch.zeros(_bytes(rows, cols), dtype=torch.uint8)
    R, C = (rows + GROUP - 1) // GROUP, (cols + GROUP - 1) // GROUP
    pad = torch.zeros(R * GROUP, C * GROUP, dtype=torch.float32)
    pad[:rows, :cols] = x
    h = GROUP if square else 1
    tiles = pad.view(R * GROUP // h, h, C, GROUP)
    most = tiles.abs().amax((1, 3), keepdim=True)
    most = torch.where(torch.isfinite(tiles).all(3, keepdim=True).all(1, keepdim=True), most, torch.full_like(most, float("inf")))
    bits = most.view(torch.int32)
    byte = torch.where(torch.isinf(most), torch.full_like(bits, _NAN_SCALE),
                       ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=0))
    inverse = torch.where(byte == _NAN_SCALE, torch.zeros_like(byte), (254 - byte) << 23).view(torch.float32)
    codes = torch.zeros(rows, _sizes(rows, cols)[0], dtype=torch.uint8)
    codes[:, :cols] = (tiles * inverse).view(pad.shape)[:rows, :cols].contiguous().to(torch.float8_e4m3fn).view(torch.uint8)
    words = torch.zeros((C + 3) // 4 * 4, R * GROUP, dtype=torch.uint8)
    words[:C] = byte.view(R * GROUP // h, 1, C).expand(-1, h, C).reshape(R * GROUP, C).t().to(torch.uint8)
    return torch.cat((codes.view(-1), words.view(-1, 4, R * GROUP).transpose(1, 2).reshape(-1)))


def _values_ref(data: Tensor, rows: int, cols: int) -> Tensor:
    ld, pad, groups = _sizes(rows, cols)
    codes = data[:rows * ld].view(rows, ld)
    byte = data[rows * ld:].view(groups, pad, 4).transpose(1, 2).reshape(groups * 4, pad)
    byte = byte[:(cols + GROUP - 1) // GROUP, :rows].t().to(torch.int32)
    scale = torch.where(byte > 0, byte << 23, torch.full_like(byte, 1 << 22)).view(torch.float32)
    scale = torch.where(byte == _NAN_SCALE, torch.full_like(scale, float("nan")), scale)
    values = codes[:, :cols].contiguous().view(torch.float8_e4m3fn).to(torch.float32)
    return values * scale.repeat_interleave(GROUP, 1)[:, :cols]


# ------------------------------------------------------------------ rounding
def _quantize(x: Tensor, square: bool, plain: bool, turned: bool) -> tuple[Tensor, Tensor]:
    """x as an operand along its columns, and x^T along the rows of x; what is not wanted is empty."""
    rows, cols = x.shape
    if not x.is_cuda:
        none = torch.empty(0, dtype=torch.uint8)
        return _quantize_ref(x, square) if plain else none, _quantize_ref(x.t(), square) if turned else none
    if x.stride(1) != 1 or x.stride(0) % 8 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    p = torch.empty(_bytes(rows, cols) if plain else 0, dtype=torch.uint8, device=x.device)
    t = torch.empty(_bytes(cols, rows) if turned else 0, dtype=torch.uint8, device=x.device)
    native.lib().fp8_quantize(x, square, p if plain else None, t if turned else None, None, None, None)
    return p, t


def _product(a: Tensor, b: Tensor, M: int, N: int, K: int, out: Tensor) -> Tensor:
    """a [M, K] b [N, K]^T into ``out``; on a GPU into bf16, or added to fp32."""
    if out.is_cuda:
        if M and N:
            native.lib().fp8_gemm(a, b, out, K, native.status_tensor(out.device))
        return out
    return out.copy_(_values_ref(a, M, K) @ _values_ref(b, N, K).t())


def _check_matrix(x: Tensor, what: str) -> None:
    if x.dim() != 2 or x.shape[0] == 0 or x.shape[1] == 0 or x.shape[1] % 16:
        raise ValueError(f"{what}: expected [rows, cols] with a multiple of 16 columns, got {tuple(x.shape)}")
    _check_type(x, what)


def _check_type(x: Tensor, what: str) -> None:
    if x.dtype != torch.bfloat16 and (x.is_cuda or x.dtype != torch.float32):
        raise TypeError(f"{what}: the sm_100a kernels take bfloat16 tensors, got {x.dtype}")


def fp8_quantize(x: Tensor, *, square: bool = False, transpose: bool = False) -> Fp8Matrix:
    """``x`` [rows, cols] (or, with ``transpose``, its transpose) in e4m3, with a scale for every 128 elements along the columns
    of the result, or with ``square`` for every 128 x 128, as weights have it.  No gradient passes."""
    _check_matrix(x, "fp8_quantize")
    with torch.no_grad():
        plain, turned = _quantize(x.detach(), square, not transpose, transpose)
    return Fp8Matrix(turned, x.shape[1], x.shape[0]) if transpose else Fp8Matrix(plain, *x.shape)


def fp8_matmul(a: Fp8Matrix, b: Fp8Matrix) -> Tensor:
    """a [M, K] b [N, K]^T in bf16 (fp32 on the CPU); N must be a multiple of 8."""
    if a.cols != b.cols:
        raise ValueError(f"fp8_matmul: contraction mismatch: {a.shape} and {b.shape}")
    if a.device != b.device:
        raise ValueError(f"fp8_matmul: operands on {a.device} and {b.device}")
    if b.rows % 8:
        raise ValueError(f"fp8_matmul: the product must have a multiple of 8 columns, got {b.rows}")
    out = torch.empty(a.rows, b.rows, dtype=torch.bfloat16 if a.data.is_cuda else torch.float32, device=a.device)
    return _product(a.data, b.data, a.rows, b.rows, a.cols, out)


# ------------------------------------------------------------------ linear layer
@custom_op("piper::fp8_linear_keep")
def fp8_linear_keep(x: Tensor, w: Tensor) -> tuple[Tensor, Tensor]:
    """y [T, N] = x [T, K] w [N, K]^T, and x^T [K, T] as the operand that the gradient of w wants."""
    (T, K), N = x.shape, w.shape[0]
    xp, xt = _quantize(x, False, True, True)
    return _product(xp, _quantize(w, True, True, False)[0], T, N, K, torch.empty(T, N, dtype=x.dtype, device=x.device)), xt


@fp8_linear_keep.register_fake
def _(x, w):
    T, (N, K) = x.shape[0], w.shape
    return x.new_empty((T, N)), x.new_empty((_bytes(K, T),), dtype=torch.uint8)


@custom_op("piper::fp8_linear")
def fp8_linear_op(x: Tensor, w: Tensor) -> Tensor:
    """y [T, N] = x [T, K] w [N, K]^T.  Whether the backward pass needs x is decided where it is known, when the op runs, and
    not by the caller, whose program may be traced without gradients."""
    (T, K), N = x.shape, w.shape[0]
    xp, wp = _quantize(x, False, True, False)[0], _quantize(w, True, True, False)[0]
    return _product(xp, wp, T, N, K, torch.empty(T, N, dtype=x.dtype, device=x.device))


@fp8_linear_op.register_fake
def _(x, w):
    return x.new_empty((x.shape[0], w.shape[0]))


def _linear_forward(ctx, x, w):
    y, xt = fp8_linear_keep(x, w) if w.requires_grad else (fp8_linear_op(x, w), None)
    ctx.rows = x.shape[0]
    ctx.save_for_backward(w, xt)
    # only to be found by gradients of the gradients, which raise: its values are not read, and the caller may write over them.  On a
    # GPU it would keep what xt is there to save.
    ctx.x = None if x.is_cuda else x
    return y


def _fp8_wgrad(dyt: Tensor, xt: Tensor, w: Tensor, T: int):
    """dW [N, K] = dY^T X, into the weight's fp32 bucket if it has one (returns None then)."""
    N, K = w.shape
    sink = grad_sinks.get(w)
    if T == 0:
        return None if sink is not None else torch.zeros_like(w)
    if sink is None:
        return _product(dyt, xt, N, K, T, torch.empty_like(w, memory_format=torch.contiguous_format))
    if w.is_cuda:
        _product(dyt, xt, N, K, T, sink)
    else:
        sink.add_(_values_ref(dyt, N, T) @ _values_ref(xt, K, T).t())
    return None


def _linear_backward(dy: Tensor, w: Tensor, xt: Optional[Tensor], T: int, need_x: bool, need_w: bool):
    N, K = w.shape
    dyp, dyt = _quantize(dy, False, need_x, need_w)
    dx = dw = None
    if need_x:
        wt = _quantize(w, True, False, True)[1]
        dx = _product(dyp, wt, T, K, N, torch.empty((T, K), dtype=dy.dtype, device=dy.device))
    if need_w:
        if wgrad_store.active is not None:
            wgrad_store.active.append((lambda: _fp8_wgrad(dyt, xt, w, T), w))
        else:
            dw = _fp8_wgrad(dyt, xt, w, T)
    return dx, dw


def _linear_formula(ctx, dy):
    w, xt = ctx.saved_tensors
    grads = _linear_backward(dy, w, xt, ctx.rows, *ctx.needs_input_grad[:2])
    return tuple(once_differentiable("fp8_linear", g, dy, w, *([] if ctx.x is None else [ctx.x])) for g in grads)


fp8_linear_op.register_autograd(_linear_formula, forward=_linear_forward)


def _linear_backward_host(dy: Tensor, w: Tensor, xt: Tensor, T: int, need_x: bool, need_w: bool) -> tuple[Tensor, Tensor]:
    dx, dw = _linear_backward(dy, w, xt, T, need_x, need_w)
    none = torch.empty(0)
    return none if dx is None else dx, none if dw is None else dw


host_op("fp8_linear_backward_host", _linear_backward_host)


@custom_op("piper::fp8_linear_kept")
def fp8_linear_kept(x: Tensor, w: Tensor, N: int) -> Tensor:
    """y [T, N] = x [T, K] w^T of a weight [N, K] that was rounded before."""
    T, K = x.shape
    return _product(_quantize(x, False, True, False)[0], w, T, N, K, torch.empty(T, N, dtype=x.dtype, device=x.device))


@fp8_linear_kept.register_fake
def _(x, w, N):
    return x.new_empty((x.shape[0], N))


fp8_linear_keep = fp8_linear_keep.overload
fp8_linear_op = fp8_linear_op.overload
fp8_linear_kept = fp8_linear_kept.overload


def fp8_linear(x: Tensor, w: Union[Tensor, Fp8Matrix]) -> Tensor:
    """y[..., N] = x[..., K] @ w[N, K]^T with both operands rounded to e4m3; so are those of its gradients' products.

    ``w`` may be a weight that was rounded before (``fp8_quantize(w, square=True)``), for calls without gradients.  K and N are
    multiples of 16; there may be any number of rows.  Gradients of the gradients raise.
    """
    kept = isinstance(w, Fp8Matrix)
    if x.is_cuda and x.dim() == 2 and not kept:
        return fp8_linear_op(x, w)                   # makes the checks below by itself
    N, K = w.shape
    _check_type(x, "fp8_linear")
    if x.dim() < 1 or x.shape[-1] != K or K == 0 or N == 0 or K % 16 or N % 16:
        raise ValueError(f"fp8_linear: x {tuple(x.shape)} and w {(N, K)}: features must agree and be multiples of 16")
    if x.device != w.device:
        raise ValueError(f"fp8_linear: x is on {x.device}, w on {w.device}")
    lead = x.shape[:-1]
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    if kept:
        if torch.is_grad_enabled() and x.requires_grad:
            raise ValueError("fp8_linear: a weight that was rounded before has no backward pass; give the bf16 weight")
        y = fp8_linear_kept(x2, w.data, N)
    else:
        if w.dtype != x.dtype:
            raise TypeError(f"fp8_linear: x is {x.dtype}, w {w.dtype}")
        y = fp8_linear_op(x2, w)
    return y if x.dim() == 2 else y.view(*lead, N)
