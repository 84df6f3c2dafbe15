"""Pages whose keys and values are held in 8 bits, on AMD MI355X: the append that quantises, the gather that reads back, and attention of one new token per request.

The pool is that of ``paged.py`` with half the bytes: ``k_pages`` and ``v_pages`` ``(P, Hk, S, D)`` are codes, ``torch.float8_e4m3fn`` or ``torch.int8``, and ``k_scales`` and
``v_scales`` ``(P, Hk, S // G)`` hold a float32 scale for every block of ``G = min(S, 16)`` tokens and key head: an element stands for ``code * scale``.  Log gates stay in 32 bits and belong to the
``H`` query heads, ``(P, H, S)``; ``H`` is a multiple of ``Hk`` and query head ``h`` reads key head ``h // (H // Hk)``.  Block tables, lengths and slots are those of ``page_slots``; no call waits
for the device.  The reference keeps 16 bits and has no pages (``model/forgetting_transformer/fgate_cache.py:5-203``).  The device work is done by the gfx950 kernels behind
``fox_paged8_append``, ``fox_paged_gather`` and ``fox_paged8_decode``; there is no fallback path, and none of them has a gradient.
"""
from __future__ import annotations

import operator
from typing import Optional, Tuple

import torch

from . import _native
from .forgetting_attention import _DTYPES
from .paged import MAX_REQUESTS, _check_page_size, _ints, _refused
from .rotary import aligned

__all__ = ["paged_append_8bit", "paged_gather", "paged_forgetting_attention_8bit"]

CODE_DTYPES = (torch.float8_e4m3fn, torch.int8)


def scale_block(page_size: int) -> int:
    """Tokens that share a scale."""
    return min(page_size, 16)


def _check_pages(k_pages, v_pages, log_fgate_pages, k_scales, v_scales, plain: bool = False):
    assert k_pages.dim() == 4 and k_pages.shape == v_pages.shape, "k_pages and v_pages must be (P, key heads, S, D)"
    assert v_pages.dtype == k_pages.dtype, "k_pages and v_pages must be of one type"
    P, Hk, S, D = k_pages.shape
    sixteen = plain and k_pages.dtype in _DTYPES
    assert sixteen or k_pages.dtype in CODE_DTYPES, "k_pages and v_pages must be float8_e4m3fn or int8" + (", or bfloat16 or float16" if plain else "")
    assert D in {16, 32, 64, 128}, "head dim must be one of 16, 32, 64, 128"
    _check_page_size(S)
    assert log_fgate_pages.dtype == torch.float32, "log_fgate_pages must be float32"
    assert log_fgate_pages.dim() == 3 and log_fgate_pages.shape[0] == P and log_fgate_pages.shape[2] == S, "log_fgate_pages must be (P, H, S) like the keys"
    H = log_fgate_pages.shape[1]
    assert H > 0 and Hk > 0 and H % Hk == 0, f"the query heads must be a multiple of the key heads, got {H} and {Hk}"
    if sixteen:
        assert k_scales is None and v_scales is None, "16-bit pages have no scales"
    else:
        for t, name in ((k_scales, "k_scales"), (v_scales, "v_scales")):
            assert t is not None and t.dtype == torch.float32 and t.shape == (P, Hk, S // scale_block(S)), f"{name} must be float32 (P, key heads, S // min(S, 16))"
    if not k_pages.is_cuda:
        raise RuntimeError("the pages need tensors on an AMD GPU (there is no CPU path)")
    for t in (v_pages, log_fgate_pages, k_scales, v_scales):
        assert t is None or t.device == k_pages.device, "the pages and their scales must be on one device"
    assert k_pages.numel() > 0, "there must be a page"
    step = 8 if sixteen else 16
    for t in (k_pages, v_pages):
        assert t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % step == 0 for s in t.stride()[:-1]), \
            f"pages must be 16-byte aligned with unit stride on the head dim and the others multiples of {step}"


def _check_tokens(t, heads, k_pages, name):
    assert t.dim() == 3 and t.shape[1:] == (heads, k_pages.shape[3]), f"{name} must be (tokens, {heads}, {k_pages.shape[3]}), with the heads of the pages"
    assert t.dtype in _DTYPES and t.device == k_pages.device, f"{name} must be bfloat16 or float16, on the device of the pages"
    return aligned(t)


def _check_table(block_table, k_pages, rows, requests, what):
    _ints(block_table, 2, "block_table", k_pages.device)
    if requests is None:
        assert block_table.shape[0] == rows, f"block_table must have a row for every {what} where requests is not given"
    else:
        _ints(requests, 1, "requests", k_pages.device)
        assert requests.shape == (rows,), f"requests must have an element for every {what}"
    assert block_table.shape[0] > 0 and 0 < block_table.shape[1] * k_pages.shape[2] <= 1 << 30, "block_table must hold between 1 and 2**30 tokens a request"
    return block_table if block_table.stride(1) == 1 else block_table.contiguous(), None if requests is None else requests.contiguous()


def paged_append_8bit(k: torch.Tensor, v: torch.Tensor, log_fgate: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scales: torch.Tensor,
                      v_scales: torch.Tensor, log_fgate_pages: torch.Tensor, slots: torch.Tensor) -> None:
    """Keys and values ``(T, Hk, D)`` and log gates ``(T, H)`` of new tokens into their slots of the pages, in place, quantised.

    slots: ``(T,)`` int64, each at most once; tokens with a slot outside the pool (-1) are left out.  Slots within one block must be those of consecutive tokens and follow each
    other, which is how ``page_slots`` hands them out.  A block whose first slot is among them starts anew: its scale becomes the smallest power of two by which the largest finite
    magnitude of the new rows fits the codes (448 in e4m3, 127 in int8; at least ``2**-126``).  Another block keeps the rows in front of the new ones and takes the larger of
    that scale and its own; where it grows, the rows in front are rounded again to it.  Every code is the nearest to ``x / scale``, ties to the even one; infinities become
    the largest code, NaN stays NaN in e4m3 and becomes 0 in int8.
    """
    ext = _native.load()
    if ext.paged8_append(k, v, log_fgate, k_pages, v_pages, k_scales, v_scales, log_fgate_pages, slots):
        return
    _check_pages(k_pages, v_pages, log_fgate_pages, k_scales, v_scales)
    Hk, H = k_pages.shape[1], log_fgate_pages.shape[1]
    k, v = _check_tokens(k, Hk, k_pages, "k"), _check_tokens(v, Hk, k_pages, "v")
    assert k.shape == v.shape and k.dtype == v.dtype, "k and v must have the same shape and type"
    assert k.shape[0] * Hk <= 1 << 28, "too many tokens for one call"
    assert log_fgate.dtype == torch.float32 and log_fgate.shape == (k.shape[0], H) and log_fgate.device == k.device, "log_fgate must be float32 (tokens, query heads)"
    assert slots.dtype == torch.int64 and slots.shape == k.shape[:1] and slots.device == k.device, "slots must be int64, one for every token"
    with torch.cuda.device(k.device):
        done = ext.paged8_append(k, v, log_fgate, k_pages, v_pages, k_scales, v_scales, log_fgate_pages, slots.contiguous())
    if not done:
        _refused("paged_append_8bit")


def paged_gather(k_pages: torch.Tensor, v_pages: torch.Tensor, log_fgate_pages: torch.Tensor, block_table: torch.Tensor, cu_seqlens: torch.Tensor, *, max_tokens: int,
                 requests: Optional[torch.Tensor] = None, k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None,
                 dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The cached tokens of B requests out of their pages, one request after the other: ``k, v`` ``(max_tokens, Hk, D)`` and ``log_fgate`` ``(max_tokens, H)``.

    Places ``cu_seqlens[b]`` to ``cu_seqlens[b + 1] - 1`` (int32 ``(B + 1,)`` on the device) get the first tokens of the request in row ``b`` of the table, or in row ``requests[b]``: what
    ``forgetting_attention_packed`` takes as the keys of prompts that continue what is cached.  Places behind the last request, and tokens on pages or of requests that the table does
    not name, are zeros.  Of 8-bit pages, with their scales, the values ``code * scale`` in ``dtype`` (bfloat16 where it is not given); 16-bit pages without scales are read as they are.
    """
    ext = _native.load()
    known = dtype is None or dtype == k_pages.dtype or (dtype in _DTYPES and k_pages.dtype not in _DTYPES)
    out = ext.paged_gather(k_pages, v_pages, log_fgate_pages, block_table, cu_seqlens, requests, max_tokens, k_scales, v_scales, dtype == torch.float16) if known else None
    if out is not None:
        return out
    _check_pages(k_pages, v_pages, log_fgate_pages, k_scales, v_scales, plain=True)
    assert known, "dtype must be bfloat16 or float16, and that of the pages where they hold 16 bits"
    _ints(cu_seqlens, 1, "cu_seqlens", k_pages.device)
    B = cu_seqlens.shape[0] - 1
    assert 0 < B <= MAX_REQUESTS, f"cu_seqlens must be the ends of between 1 and {MAX_REQUESTS} requests, with a 0 in front"
    assert 0 <= operator.index(max_tokens) <= 1 << 30, "max_tokens must be between 0 and 2**30"
    block_table, requests = _check_table(block_table, k_pages, B, requests, "request of cu_seqlens")
    with torch.cuda.device(k_pages.device):
        out = ext.paged_gather(k_pages, v_pages, log_fgate_pages, block_table, cu_seqlens.contiguous(), requests, max_tokens, k_scales, v_scales, dtype == torch.float16)
    return out if out is not None else _refused("paged_gather")


def paged_forgetting_attention_8bit(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor,
                                    log_fgate_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, *, requests: Optional[torch.Tensor] = None,
                                    sm_scale: Optional[float] = None, max_length: Optional[int] = None) -> torch.Tensor:
    """``paged_forgetting_attention`` over 8-bit pages: one token per row, ``q`` ``(B, H, D)``, against the first ``lengths[b]`` tokens of its request.

    The token itself is the last of them (append first).  Row ``b`` belongs to request ``requests[b]`` (int32), or, without ``requests``, to request ``b`` of as many.  A row without
    keys, or whose request is not in the table (-1), gives zeros.  Keys on pages outside the pool are left out and their gates count as 0.  ``sm_scale`` defaults to
    ``1 / sqrt(D)``.  ``max_length`` promises that no length is larger (larger ones are cut) and saves scratch and launches where the table is much wider.
    """
    ext = _native.load()
    out = ext.paged8_attention(q, k_pages, v_pages, k_scales, v_scales, log_fgate_pages, block_table, lengths, requests, sm_scale, max_length)
    if out is not None:
        return out
    _check_pages(k_pages, v_pages, log_fgate_pages, k_scales, v_scales)
    H = log_fgate_pages.shape[1]
    q = _check_tokens(q, H, k_pages, "q")
    B = q.shape[0]
    _ints(lengths, 1, "lengths", q.device)
    assert lengths.shape == (B,), "lengths must have an element for every row of q"
    block_table, requests = _check_table(block_table, k_pages, B, requests, "row of q")
    assert B * H <= 1 << 23, "at most 2**23 rows and heads"
    assert max_length is None or max_length > 0, "max_length must be positive"
    with torch.cuda.device(q.device):
        out = ext.paged8_attention(q, k_pages, v_pages, k_scales, v_scales, log_fgate_pages, block_table, lengths.contiguous(), requests, sm_scale, max_length)
    return out if out is not None else _refused("paged_forgetting_attention_8bit")
