"""MI355X (gfx950) native Morphottention: fused morpho-attention on HIP kernels.

Drop-in for the reference package ``morphottention``
(``packages/morphottention/torch-ext/morphottention/__init__.py:1-3``).
"""

from .autograd import MorphoAttention, MorphoAttentionFunction, morpho_attention
from .cache import (CacheStep, MorphoCache, MorphoLoop, SharedPrefix, morpho_cache_append, morpho_cache_attention,
                    morpho_cache_compact, morpho_cache_copy_pages, morpho_cache_plan, pack_cache_weights)
from .soft_morph import SoftMorphAttention, SoftMorphAttentionFunction, soft_morph_attention
from .verify import morpho_verify_drafts

__all__ = ["MorphoAttention", "MorphoAttentionFunction", "morpho_attention", "SoftMorphAttention",
           "SoftMorphAttentionFunction", "soft_morph_attention", "CacheStep", "MorphoCache", "MorphoLoop", "SharedPrefix",
           "morpho_cache_append", "morpho_cache_attention", "morpho_cache_compact", "morpho_cache_copy_pages",
           "morpho_cache_plan", "morpho_verify_drafts", "pack_cache_weights"]
