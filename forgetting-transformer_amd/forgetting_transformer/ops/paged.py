"""Serving from a pool of pages on AMD MI355X: slots of new tokens, the append into them, and attention of one new token per request.

The dense cache of the reference (``model/forgetting_transformer/fgate_cache.py:5-203``) holds a batch whose rows all have the same length.  Requests that come and go
with lengths of their own share a pool instead: ``P`` pages of ``S`` tokens (a power of two, 8 to 4096), keys and values ``(P, H, S, D)``, log forget gates
``(P, H, S)``.  Row ``b`` of ``block_table`` ``(B, W)`` names the pages of request ``b`` in order; token ``i`` of it is in slot ``page * S + i % S``.  ``free_pages[:free_count]``
is the stack of the pages nobody has.  Lengths, tables and counts are int32 tensors on the device, and no call waits for it: a step can be captured into a
graph.  The device work is done by the gfx950 kernels behind ``fox_page_slots``, ``fox_page_release``, ``fox_paged_append`` and ``fox_paged_decode``; there is no fallback
path, and none of them has a gradient.
"""
from __future__ import annotations

import operator
from typing import NamedTuple, Optional, Tuple

import torch

from . import _native
from .forgetting_attention import _DTYPES
from .rotary import aligned

__all__ = ["PageSlots", "page_slots", "page_release", "paged_append", "paged_forgetting_attention"]

MAX_REQUESTS = 4096


class PageSlots(NamedTuple):
    """What ``page_slots`` gives: four values for every new token, and the state behind them."""
    slots: torch.Tensor        # (max_tokens,) int64: place in the pool, -1 for none
    positions: torch.Tensor    # (max_tokens,) int64: place in its request
    requests: torch.Tensor     # (max_tokens,) int32: the request, -1 for none
    keys: torch.Tensor         # (max_tokens,) int32: tokens of the request up to this one, 0 without a request
    lengths: torch.Tensor      # (B,) int32: tokens of each request, the new ones included
    free_count: torch.Tensor   # (1,) int32
    granted: torch.Tensor      # (B,) bool


def _check_page_size(page_size: int) -> None:
    page_size = operator.index(page_size)
    assert 8 <= page_size <= 4096 and page_size & (page_size - 1) == 0, f"page_size must be a power of two from 8 to 4096, got {page_size}"


def _ints(t: torch.Tensor, dim: int, name: str, device=None) -> None:
    assert t.dtype == torch.int32 and t.dim() == dim, f"{name} must be an int32 tensor of {dim} dimension{'s' if dim > 1 else ''}"
    assert device is None or t.device == device, f"{name} must be on the device of the others"


def _check_state(lengths, block_table, free_pages, free_count, page_size):
    _check_page_size(page_size)
    _ints(lengths, 1, "lengths")
    if not lengths.is_cuda:
        raise RuntimeError("the pages need tensors on an AMD GPU (there is no CPU path)")
    for t, dim, name in ((block_table, 2, "block_table"), (free_pages, 1, "free_pages"), (free_count, 1, "free_count")):
        _ints(t, dim, name, lengths.device)
    B, W = block_table.shape
    assert lengths.shape == (B,) and W > 0, "block_table must have a row of at least one page for every length"
    assert 0 < B <= MAX_REQUESTS, f"between 1 and {MAX_REQUESTS} requests"
    assert W * page_size <= 1 << 30, "a request's pages must hold at most 2**30 tokens"
    assert free_pages.numel() > 0 and free_count.numel() == 1, "free_pages must have a place for every page, free_count one element"
    for t, name in ((lengths, "lengths"), (free_pages, "free_pages"), (free_count, "free_count")):
        assert t.is_contiguous(), f"{name} must be contiguous"
    assert block_table.stride(1) == 1 and (B == 1 or block_table.stride(0) >= W), "the rows of block_table must be contiguous and apart"


def _refused(what: str):
    raise RuntimeError(f"{what} does not take these tensors: they may not overlap, require grad, be inference tensors to write outside inference mode or "
                       "tensor subclasses, and function transforms, traces and dispatch modes are not supported")


def page_slots(lengths: torch.Tensor, new_tokens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor, *,
               page_size: int, max_tokens: int, in_place: bool = False) -> PageSlots:
    """Pages and slots for the ``new_tokens[b]`` tokens that each request adds to the ``lengths[b]`` it has cached.

    The tokens of a step lie one request after the other in ``max_tokens`` places.  New pages come from the top of the stack, in request order, and their numbers go
    into ``block_table`` (in place).  A request gets all its tokens or none (``granted``): none if they end behind ``max_tokens``, if it would need more than W pages or if the
    stack does not hold its pages and those of the requests in front of it; then its length stays and its tokens have no slot.  A request without new tokens ends where the one in
    front of it ends, so it counts as refused behind ``max_tokens`` too, though nothing of it changes: who preempts by this asks for ``granted | (new_tokens == 0)``.  Places that hold no token, and tokens without a slot,
    have slot and request -1 and see no keys.  ``in_place`` writes the new state into ``lengths`` and ``free_count`` (what a captured step needs), else both are new tensors and the call can be repeated.
    """
    ext = _native.load()
    out = ext.page_slots(lengths, new_tokens, block_table, free_pages, free_count, page_size, max_tokens, in_place)
    if out is None:
        _check_state(lengths, block_table, free_pages, free_count, page_size)
        _ints(new_tokens, 1, "new_tokens", lengths.device)
        assert new_tokens.shape == lengths.shape, "new_tokens must have an element for every length"
        assert 0 <= operator.index(max_tokens) < 1 << 31, "max_tokens must not be negative"
        with torch.cuda.device(lengths.device):
            out = ext.page_slots(lengths, new_tokens.contiguous(), block_table, free_pages, free_count, page_size, max_tokens, in_place)
        if out is None:
            _refused("page_slots")
    return PageSlots._make(out)


def page_release(lengths: torch.Tensor, done: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor, *,
                 page_size: int, in_place: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """The pages of the requests with ``done[b]`` (bool) back onto the stack (``free_pages``, in place), their lengths to 0.

    Returns ``(lengths, free_count)``, the tensors given with ``in_place``, else new ones.
    """
    ext = _native.load()
    out = ext.page_release(lengths, done, block_table, free_pages, free_count, page_size, in_place)
    if out is None:
        _check_state(lengths, block_table, free_pages, free_count, page_size)
        assert done.dtype == torch.bool and done.shape == lengths.shape and done.device == lengths.device, "done must be a bool for every length"
        with torch.cuda.device(lengths.device):
            out = ext.page_release(lengths, done.contiguous(), block_table, free_pages, free_count, page_size, in_place)
        if out is None:
            _refused("page_release")
    return out


def _check_pages(k_pages, v_pages, log_fgate_pages):
    assert k_pages.dim() == 4 and k_pages.shape == v_pages.shape, "k_pages and v_pages must be (P, H, S, D)"
    assert log_fgate_pages.shape == k_pages.shape[:3], "log_fgate_pages must be (P, H, S) like the keys"
    assert k_pages.dtype in _DTYPES and v_pages.dtype == k_pages.dtype, "k_pages and v_pages must both be bfloat16 or both float16"
    assert log_fgate_pages.dtype == torch.float32, "log_fgate_pages must be float32"
    assert k_pages.shape[-1] in {16, 32, 64, 128}, "head dim must be one of 16, 32, 64, 128"
    _check_page_size(k_pages.shape[2])
    if not k_pages.is_cuda:
        raise RuntimeError("the pages need tensors on an AMD GPU (there is no CPU path)")
    assert k_pages.device == v_pages.device == log_fgate_pages.device, "the pages must be on one device"
    assert k_pages.numel() > 0, "there must be a page"
    for t in (k_pages, v_pages):
        assert aligned(t) is t, "pages must be 16-byte aligned with unit stride on the head dim and the others multiples of 8"


def _check_tokens(t, k_pages, name):
    P, H, S, D = k_pages.shape
    assert t.dim() == 3 and t.shape[1:] == (H, D), f"{name} must be (tokens, H, D) with the heads of the pages"
    assert t.dtype == k_pages.dtype and t.device == k_pages.device, f"{name} must have the type and device of the pages"
    return aligned(t)


def paged_append(k: torch.Tensor, v: torch.Tensor, log_fgate: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 log_fgate_pages: torch.Tensor, slots: torch.Tensor) -> None:
    """Keys and values ``(T, H, D)`` and log gates ``(T, H)`` of new tokens into their slots of the pages, in place.

    slots: ``(T,)`` int64, each slot at most once; tokens with a slot outside the pool (-1) are left out.
    """
    ext = _native.load()
    if ext.paged_append(k, v, log_fgate, k_pages, v_pages, log_fgate_pages, slots):
        return
    _check_pages(k_pages, v_pages, log_fgate_pages)
    k, v = _check_tokens(k, k_pages, "k"), _check_tokens(v, k_pages, "v")
    assert k.shape == v.shape, "k and v must have the same shape"
    assert k.numel() // 8 < 1 << 31, "too many tokens for one call"
    assert log_fgate.dtype == torch.float32 and log_fgate.shape == k.shape[:2] and log_fgate.device == k.device, "log_fgate must be float32 (tokens, H)"
    assert slots.dtype == torch.int64 and slots.shape == k.shape[:1] and slots.device == k.device, "slots must be int64, one for every token"
    with torch.cuda.device(k.device):
        done = ext.paged_append(k, v, log_fgate, k_pages, v_pages, log_fgate_pages, slots.contiguous())
    if not done:
        _refused("paged_append")


def paged_forgetting_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, log_fgate_pages: torch.Tensor, block_table: torch.Tensor,
                               lengths: torch.Tensor, *, requests: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None,
                               max_length: Optional[int] = None) -> torch.Tensor:
    """``forgetting_attention`` of one token per row, ``q`` ``(B, H, D)``, against the first ``lengths[b]`` tokens of its request in the pages.

    The token itself is the last of them (append first).  Row ``b`` belongs to request ``requests[b]`` (int32), or, without ``requests``, to request ``b`` of as many.  A row
    without keys, or whose request is not in the table (-1), gives zeros.  Keys on pages outside the pool are left out and their gates count as 0.  ``sm_scale`` defaults
    to ``1 / sqrt(D)``.  ``max_length`` promises that no length is larger (larger ones are cut) and saves scratch and launches where the table is much wider.
    """
    ext = _native.load()
    out = ext.paged_attention(q, k_pages, v_pages, log_fgate_pages, block_table, lengths, requests, sm_scale, max_length)
    if out is not None:
        return out
    _check_pages(k_pages, v_pages, log_fgate_pages)
    q = _check_tokens(q, k_pages, "q")
    B = q.shape[0]
    _ints(block_table, 2, "block_table", q.device)
    _ints(lengths, 1, "lengths", q.device)
    assert lengths.shape == (B,), "lengths must have an element for every row of q"
    if requests is None:
        assert block_table.shape[0] == B, "block_table must have a row for every row of q where requests is not given"
    else:
        _ints(requests, 1, "requests", q.device)
        assert requests.shape == (B,), "requests must have an element for every row of q"
        requests = requests.contiguous()
    assert block_table.shape[0] > 0 and 0 < block_table.shape[1] * k_pages.shape[2] <= 1 << 30, "block_table must hold between 1 and 2**30 tokens a request"
    assert B * k_pages.shape[1] <= 1 << 23, "at most 2**23 rows and heads"
    assert max_length is None or max_length > 0, "max_length must be positive"
    block_table = block_table if block_table.stride(1) == 1 else block_table.contiguous()
    with torch.cuda.device(q.device):
        out = ext.paged_attention(q, k_pages, v_pages, log_fgate_pages, block_table, lengths.contiguous(), requests, sm_scale, max_length)
    return out if out is not None else _refused("paged_forgetting_attention")
