"""CyFA operators on the MI355X HIP path: the reference's entry points
(cyclic_flow_attention/ops/__init__.py:4-7), and the operators around a
causal language model's blocks."""

from .chunk import chunk_cyfa
from .distill import distill_loss
from .fused_recurrent import fused_recurrent_cyfa
from .residual import residual_norm
from .sampling import SampledTokens, adjust_logits, sample_tokens
from .vocab import TokenLogprobs, embed_tokens, token_logprobs, token_loss

__all__ = ["SampledTokens", "TokenLogprobs", "adjust_logits", "chunk_cyfa", "distill_loss", "embed_tokens",
           "fused_recurrent_cyfa", "residual_norm", "sample_tokens", "token_logprobs", "token_loss"]
