"""Key / value / forget-gate cache of a model's layers for requests that come and go, in pages.

The counterpart of ``FgateDynamicCache`` for serving: its rows have one length, here every request has its own.  All layers share one block table
and one stack of free pages, since a token has the same slot in each; every layer has pages of its own.  A step is::

    step = cache.schedule(new_tokens, max_tokens)             # slots, positions and requests of the step's tokens
    for layer in ...:
        q, k = qk_norm_rotary(q, k, ..., positions=step.positions[None])       # (1, tokens, H, D)
        cache.update(k[0], v, log_fgate, layer)
        out = cache.attend(q[0], layer)

A step that holds prompts is scheduled with ``prompts=True`` and ends in ``cache.attend_prompts(q[0], layer)``, which goes through the prompts as packed sequences.  With ``cache_dtype`` the pages hold keys and
values in 8 bits, quantised as they are written (``paged8.py``), and the query heads may share key heads.

``cache.release(done)`` gives a request's pages back.  Nothing waits for the device, and the state stays in the same tensors, so a step can be captured.
It keeps no states of a token shift (``FgateDynamicCache`` does), and ``token_shift`` takes whole batches, not a step of several requests' tokens: layers
with the shift are not served from pages.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from .ops.packed import forgetting_attention_packed
from .ops.paged import MAX_REQUESTS, PageSlots, _check_page_size, page_release, page_slots, paged_append, paged_forgetting_attention
from .ops.paged8 import CODE_DTYPES, paged_append_8bit, paged_forgetting_attention_8bit, paged_gather, scale_block

__all__ = ["PagedFgateCache"]


class PagedFgateCache:
    """Pages of ``num_layers`` layers for up to ``max_requests`` requests of up to ``max_length`` tokens (rounded up to whole pages), ``num_pages`` pages of
    ``page_size`` tokens in all.  ``dtype`` is that of the model's keys and values, and of the pages unless ``cache_dtype`` is ``torch.float8_e4m3fn`` or ``torch.int8``; then
    ``num_kv_heads`` may be a divisor of ``num_heads``."""

    def __init__(self, num_layers: int, num_heads: int, head_dim: int, *, num_pages: int, max_requests: int, max_length: int, page_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device=None, cache_dtype: Optional[torch.dtype] = None, num_kv_heads: Optional[int] = None) -> None:
        _check_page_size(page_size)
        assert num_layers > 0 and num_heads > 0 and num_pages > 0 and max_length > 0, "layers, heads, pages and max_length must be positive"
        assert 0 < max_requests <= MAX_REQUESTS, f"between 1 and {MAX_REQUESTS} requests"
        assert head_dim in {16, 32, 64, 128}, "head dim must be one of 16, 32, 64, 128"
        assert dtype in (torch.bfloat16, torch.float16), "keys and values must be bfloat16 or float16"
        assert cache_dtype is None or cache_dtype == dtype or cache_dtype in CODE_DTYPES, "cache_dtype must be float8_e4m3fn, int8, or the dtype"
        cache_dtype = dtype if cache_dtype is None else cache_dtype
        num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        assert num_kv_heads > 0 and num_heads % num_kv_heads == 0, "num_heads must be a multiple of num_kv_heads"
        assert num_kv_heads == num_heads or cache_dtype in CODE_DTYPES, "16-bit pages hold a key head for every query head"
        device = torch.device("cuda" if device is None else device)
        self.page_size, self.dtype = page_size, dtype
        width = (max_length + page_size - 1) // page_size
        shape, kv_shape = (num_pages, num_heads, page_size), (num_pages, num_kv_heads, page_size)

        def per_layer(*s, fill=torch.zeros, dtype=cache_dtype) -> List[torch.Tensor]:
            return [fill(s, dtype=dtype, device=device) for _ in range(num_layers)]

        self.key_pages, self.value_pages = per_layer(*kv_shape, head_dim), per_layer(*kv_shape, head_dim)
        self.key_scales: Optional[List[torch.Tensor]] = None
        self.value_scales: Optional[List[torch.Tensor]] = None
        if cache_dtype in CODE_DTYPES:
            blocks = (num_pages, num_kv_heads, page_size // scale_block(page_size))
            self.key_scales, self.value_scales = (per_layer(*blocks, fill=torch.ones, dtype=torch.float32) for _ in range(2))
        self.log_fgate_pages: List[torch.Tensor] = [torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(num_layers)]
        self.block_table = torch.full((max_requests, width), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(max_requests, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)   # page 0 on top
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=device)
        self.step: Optional[PageSlots] = None
        self._ends = None          # of the step's tokens and of the keys they see, request by request

    def __len__(self) -> int:
        return len(self.key_pages)

    def schedule(self, new_tokens: torch.Tensor, max_tokens: int, prompts: bool = False) -> PageSlots:
        """Room for ``new_tokens[b]`` tokens of every request (``(max_requests,)`` int32), the step that ``update`` and ``attend`` work on; with ``prompts`` for
        ``attend_prompts`` as well."""
        self.step = page_slots(self.lengths, new_tokens, self.block_table, self.free_pages, self.free_count, page_size=self.page_size,
                               max_tokens=max_tokens, in_place=True)
        self._ends = None
        if prompts:
            # requests that were refused, or bring nothing, need no keys: without any their tokens give zeros
            keys = torch.where(self.step.granted & (new_tokens > 0), self.lengths, 0)
            self._ends = [torch.nn.functional.pad(n.cumsum(0).clamp(max=2**31 - 1).int(), (1, 0)) for n in (new_tokens.clamp(min=0), keys)]
        return self.step

    def release(self, done: torch.Tensor) -> None:
        """Give back the pages of the requests with ``done[b]`` (``(max_requests,)`` bool); their places are free for new requests."""
        page_release(self.lengths, done, self.block_table, self.free_pages, self.free_count, page_size=self.page_size, in_place=True)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, log_fgate_states: torch.Tensor, layer_idx: int) -> None:
        """Keys and values ``(tokens, heads, head_dim)`` and log gates ``(tokens, heads)`` of the step's tokens into the pages of a layer."""
        assert self.step is not None, "schedule a step first"
        k_pages, v_pages, g_pages = self.key_pages[layer_idx], self.value_pages[layer_idx], self.log_fgate_pages[layer_idx]
        if self.key_scales is None:
            paged_append(key_states, value_states, log_fgate_states, k_pages, v_pages, g_pages, self.step.slots)
        else:
            paged_append_8bit(key_states, value_states, log_fgate_states, k_pages, v_pages, self.key_scales[layer_idx], self.value_scales[layer_idx], g_pages, self.step.slots)

    def attend(self, q: torch.Tensor, layer_idx: int, sm_scale: Optional[float] = None) -> torch.Tensor:
        """Attention of the step's tokens ``(tokens, heads, head_dim)`` over their requests, each up to itself; tokens without a slot give zeros.

        Every token reads all keys in front of it, which is what a step of one token per request needs; the prompts of a step are cheaper through ``attend_prompts``.
        """
        assert self.step is not None, "schedule a step first"
        k_pages, v_pages, g_pages = self.key_pages[layer_idx], self.value_pages[layer_idx], self.log_fgate_pages[layer_idx]
        if self.key_scales is None:
            return paged_forgetting_attention(q, k_pages, v_pages, g_pages, self.block_table, self.step.keys, requests=self.step.requests, sm_scale=sm_scale)
        return paged_forgetting_attention_8bit(q, k_pages, v_pages, self.key_scales[layer_idx], self.value_scales[layer_idx], g_pages, self.block_table, self.step.keys,
                                               requests=self.step.requests, sm_scale=sm_scale)

    def attend_prompts(self, q: torch.Tensor, layer_idx: int, sm_scale: Optional[float] = None, max_keys: Optional[int] = None) -> torch.Tensor:
        """What ``attend`` gives, for steps whose requests bring many tokens: the keys of the requests that bring any are read back from the pages, and every request's tokens go
        through ``forgetting_attention_packed`` over them.

        ``max_keys`` promises that those requests hold no more tokens together: one whose tokens end behind them gives zeros, and so do those that follow.  Without it there is room for all
        that the step's requests can hold, ``max_length`` each or the whole pool if that is less: 16-bit keys and values, and sums of the gates, for so many tokens in every layer.
        """
        assert self._ends is not None, "schedule a step with prompts first"
        assert max_keys is None or max_keys > 0, "max_keys must be positive"
        pages = self.key_pages[layer_idx]
        if max_keys is None:
            (requests, width), (num_pages, _, page_size, _) = self.block_table.shape, pages.shape
            max_keys = min(num_pages, min(requests, self.step.slots.shape[0]) * width) * page_size
        scales = {} if self.key_scales is None else dict(k_scales=self.key_scales[layer_idx], v_scales=self.value_scales[layer_idx], dtype=self.dtype)
        k, v, log_fgate = paged_gather(pages, self.value_pages[layer_idx], self.log_fgate_pages[layer_idx], self.block_table, self._ends[1],
                                       max_tokens=max_keys, **scales)
        return forgetting_attention_packed(q, k, v, log_fgate, *self._ends, sm_scale=sm_scale)
