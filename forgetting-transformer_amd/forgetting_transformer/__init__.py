"""Forgetting Attention for AMD MI355X (gfx950).

Same import path and call signature as the reference package
(``src/forgetting_transformer/__init__.py:1-3``)::

    from forgetting_transformer import forgetting_attention
"""
from .ops.forgetting_attention import (forgetting_attention, forgetting_attention_from_logits,
                                         forgetting_attention_norm_gate, qk_norm_threshold)
from .ops.norm_gate import group_norm, group_norm_gated, rms_norm
from .ops.packed import forgetting_attention_packed
from .ops.paged import PageSlots, page_release, page_slots, paged_append, paged_forgetting_attention
from .ops.paged8 import paged_append_8bit, paged_forgetting_attention_8bit, paged_gather
from .ops.rotary import qk_norm_rotary, rotary, rotary_frequencies
from .ops.token_shift import token_shift
from .fgate_cache import FgateDynamicCache
from .paged_cache import PagedFgateCache

__version__ = "0.1.0"
__all__ = ["forgetting_attention", "forgetting_attention_from_logits", "forgetting_attention_norm_gate", "forgetting_attention_packed", "qk_norm_threshold", "group_norm",
           "group_norm_gated", "rms_norm", "token_shift", "FgateDynamicCache", "rotary", "qk_norm_rotary", "rotary_frequencies", "PageSlots", "page_slots", "page_release",
           "paged_append", "paged_forgetting_attention", "paged_append_8bit", "paged_gather", "paged_forgetting_attention_8bit", "PagedFgateCache"]
