from .forgetting_attention import (forgetting_attention, forgetting_attention_from_logits,
                                         forgetting_attention_norm_gate, qk_norm_threshold)
from .norm_gate import group_norm, group_norm_gated, rms_norm
from .packed import forgetting_attention_packed
from .paged import PageSlots, page_release, page_slots, paged_append, paged_forgetting_attention
from .paged8 import paged_append_8bit, paged_forgetting_attention_8bit, paged_gather
from .rotary import qk_norm_rotary, rotary, rotary_frequencies
from .token_shift import token_shift

__all__ = ["forgetting_attention", "forgetting_attention_from_logits", "forgetting_attention_norm_gate", "forgetting_attention_packed", "qk_norm_threshold", "group_norm",
           "group_norm_gated", "rms_norm", "token_shift", "rotary", "qk_norm_rotary", "rotary_frequencies", "PageSlots", "page_slots", "page_release", "paged_append",
           "paged_forgetting_attention", "paged_append_8bit", "paged_gather", "paged_forgetting_attention_8bit"]
