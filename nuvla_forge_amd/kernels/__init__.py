"""MI355X (gfx950) fused kernels for VLA-style driving models.

Drop-in for ``nuvla_forge.kernels`` (reference ``nuvla_forge/kernels/__init__.py:8-18``):
the same three ops and the same ``HAS_TRITON`` flag, backed by hand-written HIP
kernels in ``libnf_hip.so`` instead of Triton; plus ``fused_gate_up_swiglu``,
the SwiGLU fused into its gate/up projection GEMM, and the operators around a
language model's vocabulary table and between its layers: ``embedding_lookup``,
``chunked_token_logprobs`` and ``fused_dropout``; and a transformer block's
attention: ``fused_rotary`` for the positions of its queries and keys,
``fused_attention``.
"""

from .adaln_rmsnorm import fused_adaln_residual_rmsnorm
from .attention import fused_attention
from .chunked_ce import chunked_cross_entropy
from .dropout import fused_dropout
from .embedding import embedding_lookup
from .rotary import fused_rotary
from .swiglu import fused_gate_up_swiglu, fused_swiglu
from .token_logprobs import TokenLogprobs, chunked_token_logprobs
from .utils import HAS_HIP, HAS_TRITON

__all__ = [
    "HAS_HIP",
    "HAS_TRITON",
    "TokenLogprobs",
    "chunked_cross_entropy",
    "chunked_token_logprobs",
    "embedding_lookup",
    "fused_adaln_residual_rmsnorm",
    "fused_attention",
    "fused_dropout",
    "fused_gate_up_swiglu",
    "fused_rotary",
    "fused_swiglu",
]
