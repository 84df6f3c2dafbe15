"""Key / value / forget-gate cache of a model's layers for requests that come and go, in pages.

The counterpart of ``FgateDynamicCache`` for serving: its rows have one length, here every request has its own.  All layers share one block table
and one stack of free pages, since a token has the same slot in each; every layer has pages of its own.  A step is::

    step = cache.schedule(new_tokens, max_tokens)             # slots, positions and requests of the step's tokens
    for layer in ...:
        q, k = qk_norm_rotary(q, k, ..., positions=step.positions[None])       # (1, tokens, H, D)
        cache.update(k[0], v, log_fgate, layer)
        out = cache.attend(q[0], layer)

and ``cache.release(done)`` gives a request's pages back.  Nothing waits for the device, and the state stays in the same tensors, so a step can be captured.
It keeps no states of a token shift (``FgateDynamicCache`` does), and ``token_shift`` takes whole batches, not a step of several requests' tokens: layers
with the shift are not served from pages.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from .ops.paged import MAX_REQUESTS, PageSlots, _check_page_size, page_release, page_slots, paged_append, paged_forgetting_attention

__all__ = ["PagedFgateCache"]


class PagedFgateCache:
    """Pages of ``num_layers`` layers for up to ``max_requests`` requests of up to ``max_length`` tokens (rounded up to whole pages), ``num_pages`` pages of
    ``page_size`` tokens in all."""

    def __init__(self, num_layers: int, num_heads: int, head_dim: int, *, num_pages: int, max_requests: int, max_length: int, page_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device=None) -> None:
        _check_page_size(page_size)
        assert num_layers > 0 and num_heads > 0 and num_pages > 0 and max_length > 0, "layers, heads, pages and max_length must be positive"
        assert 0 < max_requests <= MAX_REQUESTS, f"between 1 and {MAX_REQUESTS} requests"
        assert head_dim in {16, 32, 64, 128}, "head dim must be one of 16, 32, 64, 128"
        assert dtype in (torch.bfloat16, torch.float16), "keys and values must be bfloat16 or float16"
        device = torch.device("cuda" if device is None else device)
        self.page_size = page_size
        width = (max_length + page_size - 1) // page_size
        shape = (num_pages, num_heads, page_size)
        self.key_pages: List[torch.Tensor] = [torch.zeros(*shape, head_dim, dtype=dtype, device=device) for _ in range(num_layers)]
        self.value_pages: List[torch.Tensor] = [torch.zeros(*shape, head_dim, dtype=dtype, device=device) for _ in range(num_layers)]
        self.log_fgate_pages: List[torch.Tensor] = [torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(num_layers)]
        self.block_table = torch.full((max_requests, width), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(max_requests, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)   # page 0 on top
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=device)
        self.step: Optional[PageSlots] = None

    def __len__(self) -> int:
        return len(self.key_pages)

    def schedule(self, new_tokens: torch.Tensor, max_tokens: int) -> PageSlots:
        """Room for ``new_tokens[b]`` tokens of every request (``(max_requests,)`` int32), the step that ``update`` and ``attend`` work on."""
        self.step = page_slots(self.lengths, new_tokens, self.block_table, self.free_pages, self.free_count, page_size=self.page_size,
                               max_tokens=max_tokens, in_place=True)
        return self.step

    def release(self, done: torch.Tensor) -> None:
        """Give back the pages of the requests with ``done[b]`` (``(max_requests,)`` bool); their places are free for new requests."""
        page_release(self.lengths, done, self.block_table, self.free_pages, self.free_count, page_size=self.page_size, in_place=True)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, log_fgate_states: torch.Tensor, layer_idx: int) -> None:
        """Keys and values ``(tokens, heads, head_dim)`` and log gates ``(tokens, heads)`` of the step's tokens into the pages of a layer."""
        assert self.step is not None, "schedule a step first"
        paged_append(key_states, value_states, log_fgate_states, self.key_pages[layer_idx], self.value_pages[layer_idx], self.log_fgate_pages[layer_idx],
                     self.step.slots)

    def attend(self, q: torch.Tensor, layer_idx: int, sm_scale: Optional[float] = None) -> torch.Tensor:
        """Attention of the step's tokens ``(tokens, heads, head_dim)`` over their requests, each up to itself; tokens without a slot give zeros.

        Every token reads all keys in front of it, which is what a step of one token per request needs; the prompts of a step are cheaper through
        ``forgetting_attention`` on the prompt itself.
        """
        assert self.step is not None, "schedule a step first"
        return paged_forgetting_attention(q, self.key_pages[layer_idx], self.value_pages[layer_idx], self.log_fgate_pages[layer_idx], self.block_table,
                                          self.step.keys, requests=self.step.requests, sm_scale=sm_scale)
