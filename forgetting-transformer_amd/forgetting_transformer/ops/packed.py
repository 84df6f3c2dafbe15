"""Forgetting Attention over sequences packed one after the other, on AMD MI355X.

The reference's operator (``ops/forgetting_attention.py:403-455``) takes a batch whose rows have one length, padded on the left.  Here sequences of lengths of their
own lie one after the other in ``(tokens, heads, head_dim)`` tensors: the documents of a training step, or the prompts of a step as ``page_slots`` lays them out.
Query heads may share key heads, every query head keeps its own forget gates.  The device work is done by the gfx950 kernels behind ``fox_packed_fwd`` and
``fox_packed_bwd``; there is no fallback path.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from .forgetting_attention import _DTYPES
from .rotary import aligned

__all__ = ["forgetting_attention_packed"]

MAX_SEQUENCES = 65535


def _check_packed(q, k, v, log_fgate, cu_seqlens, cu_seqlens_k):
    assert q.dim() == 3, "q must be (tokens, heads, head_dim)"
    assert k.dim() == 3 and k.shape == v.shape, "k and v must both be (tokens, key heads, head_dim)"
    assert q.dtype in _DTYPES and k.dtype == q.dtype and v.dtype == q.dtype, "q, k and v must all be bfloat16 or all float16"
    assert q.shape[2] in {16, 32, 64, 128} and k.shape[2] == q.shape[2], "head dim must be one of 16, 32, 64, 128, the same for q, k and v"
    H, Hk = q.shape[1], k.shape[1]
    assert H > 0 and Hk > 0 and H % Hk == 0, f"the heads of q must be a multiple of the key heads, got {H} and {Hk}"
    assert log_fgate.dtype == torch.float32 and log_fgate.shape == (k.shape[0], H), "log_fgate must be float32 (tokens of k, heads of q)"
    for t, name in ((cu_seqlens, "cu_seqlens"), (cu_seqlens_k, "cu_seqlens_k")):
        if t is not None:
            assert t.dtype == torch.int32 and t.dim() == 1 and t.shape[0] >= 2, f"{name} must be int32, the ends of the sequences with a 0 in front"
    assert cu_seqlens.shape[0] - 1 <= MAX_SEQUENCES, f"at most {MAX_SEQUENCES} sequences"
    if cu_seqlens_k is None:
        assert k.shape[0] == q.shape[0], "without cu_seqlens_k, q and k must have the same tokens"
    else:
        assert cu_seqlens_k.shape == cu_seqlens.shape, "cu_seqlens and cu_seqlens_k must be of the same sequences"
    assert max(q.shape[0], k.shape[0]) <= 1 << 30, "at most 2**30 tokens"
    if not q.is_cuda:
        raise RuntimeError("forgetting_attention_packed needs tensors on an AMD GPU (there is no CPU path)")
    for t in (k, v, log_fgate, cu_seqlens, cu_seqlens_k):
        assert t is None or t.device == q.device, "all tensors must be on one device"


def _rows(t: torch.Tensor) -> torch.Tensor:
    """As the kernels read it: ``aligned``, and tokens behind each other with less than 2**23 elements from one to the next."""
    return aligned(t) if 0 < t.stride(0) < 1 << 23 else t.clone(memory_format=torch.contiguous_format)


def forgetting_attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_fgate: torch.Tensor, cu_seqlens: torch.Tensor,
                                cu_seqlens_k: Optional[torch.Tensor] = None, *, sm_scale: Optional[float] = None) -> torch.Tensor:
    """``forgetting_attention`` of every one of B packed sequences with itself, causal.

    q: ``(T, H, D)``; k, v: ``(N, Hk, D)``, with ``H`` a multiple of ``Hk`` (query head ``h`` reads key head ``h // (H // Hk)``); log_fgate: ``(N, H)`` float32.
    cu_seqlens: ``(B + 1,)`` int32 on the device, 0 and the ends of the sequences' queries, not decreasing; cu_seqlens_k: the same of their keys, which
    are those of the queries where it is not given.  Of a sequence with m queries and n keys, query i sees the keys ``j <= i + n - m``: the keys of a prompt's earlier pieces
    lie in front of those of the piece.  A query that sees no key gives zeros, and so do places that belong to no sequence (as a step with room for more tokens
    has them behind its last one); no gradient reaches them or comes from them.  A sequence whose queries (keys) end behind the last of the tensor has none, and neither have those
    that follow.  ``sm_scale`` defaults to ``1 / sqrt(D)``.

    Gradients for q, k, v and log_fgate.  Nothing waits for the device.  There is no ``adaptive_threshold`` here: where strong gates prune most of a long batch, the dense operator on padded rows
    may be the faster one.
    """
    ext = _native.load()
    out = ext.packed_attention(q, k, v, log_fgate, cu_seqlens, cu_seqlens_k, sm_scale)
    if out is not None:
        return out
    _check_packed(q, k, v, log_fgate, cu_seqlens, cu_seqlens_k)
    with torch.cuda.device(q.device):
        out = ext.packed_attention(_rows(q), _rows(k), _rows(v), log_fgate, cu_seqlens.contiguous(), None if cu_seqlens_k is None else cu_seqlens_k.contiguous(), sm_scale)
    if out is None:
        raise RuntimeError("forgetting_attention_packed does not take these tensors: tensor subclasses, function transforms, traces and dispatch modes are not supported")
    return out
