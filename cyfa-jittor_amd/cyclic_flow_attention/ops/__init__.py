"""CyFA operators on the MI355X HIP path: the reference's entry points
(cyclic_flow_attention/ops/__init__.py:4-7), and the operators around a
causal language model's blocks."""

from .chunk import chunk_cyfa
from .fused_recurrent import fused_recurrent_cyfa
from .residual import residual_norm
from .vocab import TokenLogprobs, embed_tokens, token_logprobs, token_loss

__all__ = ["TokenLogprobs", "chunk_cyfa", "embed_tokens", "fused_recurrent_cyfa", "residual_norm", "token_logprobs", "token_loss"]
