"""Model building blocks on top of ``torch.ops.piper.*``."""
from .layers import (Attention, CrossEntropyLoss, Embedding, FeedForward, Linear, RMSNorm, clipped_policy_loss,
                     cross_entropy_loss, packed_rope, policy_gradient_loss)

__all__ = ["Linear", "RMSNorm", "Embedding", "Attention", "FeedForward", "CrossEntropyLoss", "cross_entropy_loss",
           "policy_gradient_loss", "clipped_policy_loss", "packed_rope"]
