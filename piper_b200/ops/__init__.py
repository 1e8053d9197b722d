"""Compute ops of the framework: ``torch.ops.piper.*`` custom ops backed by sm_100a kernels."""
from . import moe, native
from .core import (
    add_rmsnorm,
    attention,
    cross_entropy,
    embedding,
    grad_sinks,
    linear,
    qk_rope,
    residual_add,
    rmsnorm,
    rope_tables,
    swiglu,
    wgrad_store,
)
from .fp8 import Fp8Matrix, fp8_linear, fp8_matmul, fp8_quantize
from .logprobs import TokenLogprobs, token_logprobs
from .optim import AdamWState, adamw_step
from .packed import PackedSequences, pack_sequences, packed_attention
from .policy import PolicyLoss, clipped_policy_loss

__all__ = [
    "moe", "native", "linear", "rmsnorm", "add_rmsnorm", "qk_rope", "residual_add", "rope_tables", "attention", "swiglu",
    "embedding", "cross_entropy", "token_logprobs", "TokenLogprobs", "AdamWState",
    "adamw_step", "Fp8Matrix", "fp8_linear", "fp8_matmul", "fp8_quantize", "grad_sinks", "wgrad_store",
    "PackedSequences", "pack_sequences", "packed_attention", "PolicyLoss", "clipped_policy_loss",
]
