"""
nanospeaker_amd: nanoSpeaker's dropless MoE hot path (routing, dispatch, grouped SwiGLU
experts, combine, backward) as hand-written HIP kernels for MI355X (gfx950), behind a
C ABI (include/nsmoe.h) and the reference's Python interface (MoEBlock, TopKRouter,
moe_kernel ops); and the operators of generation (rotary positions, attention over a shared
prefix and caches, eviction, penalties on logits).
"""

from .cache import cache_evict, shared_prefix_attention
from .glu import GLUFeedForward, glu_hidden_dim, make_glu
from .logits import penalize_logits
from .moe import AUTO_CAPACITY, MoEBlock
from .rope import rotary_embed, rotary_frequencies
from .router import TopKRouter
from .utils import ACTIVATIONS, resolve_activation

__all__ = [
    "ACTIVATIONS", "AUTO_CAPACITY", "GLUFeedForward", "MoEBlock", "TopKRouter", "cache_evict",
    "glu_hidden_dim", "make_glu", "penalize_logits", "resolve_activation", "rotary_embed",
    "rotary_frequencies", "shared_prefix_attention",
]
