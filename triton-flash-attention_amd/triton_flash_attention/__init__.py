"""MI355X-native FlashAttention-2 with the public API of triton_flash_attention.

The reference package's import surface (triton_flash_attention/__init__.py:3-15), and the
operators that a decoder runs around the attention call: the norm and rotation of queries and
keys (:mod:`.rotary`) and the paged key/value cache of a serving program (:mod:`.paged`).
"""

from .attention import (
    DispatchDecision,
    TritonAttention,
    explain_dispatch,
    scaled_dot_product_attention,
)
from .paged import PagedPlan as PagedPlan
from .paged import paged_attention as paged_attention
from .paged import paged_cache_plan as paged_cache_plan
from .paged import paged_cache_store as paged_cache_store
from .rotary import qk_norm_rope as qk_norm_rope

__version__ = "0.2.0+gfx950"

# `import *` brings the reference's names alone; the others are imported by name.
__all__ = [
    "DispatchDecision",
    "TritonAttention",
    "explain_dispatch",
    "scaled_dot_product_attention",
]
