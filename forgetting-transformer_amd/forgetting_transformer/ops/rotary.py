"""Position rotation of queries and keys on AMD MI355X, alone and in the pass of their per-head RMS norms.

The FoX layer can rotate queries and keys (``rotary.py`` of the reference's ``model/forgetting_transformer``, off by default) behind its
QK-norm (``modeling_forgetting_transformer.py:258-265, 314-325``).  ``rotary`` is the rotation alone, ``qk_norm_rotary`` norms and rotates queries and keys
in one pass over both.  Angles are formed on the device from positions and frequencies, in 64 bits; there is no table whose length would bound
the positions.  The device work is done by the gfx950 kernels behind ``fox_rotary_fwd`` / ``fox_rotary_bwd``; there is no fallback path.
"""
from __future__ import annotations

import math
import operator
from typing import Optional, Tuple, Union

import torch

from . import _native
from .forgetting_attention import _DTYPES

__all__ = ["rotary", "qk_norm_rotary", "rotary_frequencies"]

Positions = Union[None, int, torch.Tensor]


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, slow: float = 1.0, fast: float = 32.0, device=None) -> torch.Tensor:
    """The ``rotary_dim / 2`` frequencies ``base ** (-2 i / rotary_dim)``, radians per position, as float64.

    For contexts ``factor`` times as long as those trained on:

    * ``scaling="linear"``: every frequency divided by ``factor`` (positions squeezed into the old range);
    * ``scaling="base"``: the base raised so that the lowest frequency is divided by ``factor`` and the highest stays;
    * ``scaling="parts"``: frequencies that turn more than ``fast`` times over ``original_length`` positions stay, those that turn less
      than ``slow`` times are divided by ``factor``, those between are blended linearly in the number of turns.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not base > 0 or not factor > 0:
        raise ValueError("base and factor must be positive")
    if scaling == "base":
        base = base * factor ** (rotary_dim / (rotary_dim - 2)) if rotary_dim > 2 else base
    freq = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "parts":
        if original_length is None or not fast > slow:
            raise ValueError('scaling="parts" needs original_length, and fast above slow')
        keep = [min(1.0, max(0.0, (original_length * f / (2.0 * math.pi) - slow) / (fast - slow))) for f in freq]
        freq = [f * (k + (1.0 - k) / factor) for f, k in zip(freq, keep)]
    elif scaling not in (None, "base"):
        raise ValueError(f"Unsupported scaling: {scaling}")
    return torch.tensor(freq, dtype=torch.float64, device=device)


def aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the kernels read it, in 16-byte vectors: unit inner stride, an aligned base, the other strides multiples of 8; a copy where it is not."""
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in t.stride()[:-1])
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _check_size(elements: int) -> None:
    assert elements <= 1 << 34, "at most 2**34 elements in one call"


def _check_heads(t: torch.Tensor, name: str) -> torch.Tensor:
    assert t.dim() == 4, f"{name} must be (B, T, H, D), or (B, H, T, D) with head_first"
    assert t.dtype in _DTYPES, f"{name} must be bfloat16 or float16"
    assert t.shape[-1] in {16, 32, 64, 128}, "head dim must be one of 16, 32, 64, 128"
    if not t.is_cuda:
        raise RuntimeError("the rotation needs tensors on an AMD GPU (there is no CPU path)")
    return aligned(t)


def _check_angles(x, inv_freq, positions, interleaved, head_first):
    """Frequencies and positions as the kernels take them."""
    B, T = x.shape[0], x.shape[2 if head_first else 1]
    assert B * T <= 1 << 30 and x.shape[1 if head_first else 2] <= 65535, "at most 2**30 tokens of 65535 heads"
    assert inv_freq.dim() == 1 and inv_freq.is_floating_point(), "inv_freq must be a floating (rotary_dim / 2,) tensor"
    assert not inv_freq.requires_grad, "the frequencies have no gradient"
    R, step = 2 * inv_freq.shape[0], 2 if interleaved else 16
    assert 0 < R <= x.shape[-1] and R % step == 0, f"rotary_dim (twice the frequencies) must be a multiple of {step} up to the head dim, got {R}"
    if isinstance(positions, torch.Tensor):
        assert not positions.is_floating_point() and not positions.is_complex() and positions.dtype != torch.bool, "positions must be integers"
        assert positions.dim() in (1, 2) and positions.shape[-1] in ((T,) if positions.dim() == 1 else (T, 1)), "positions must be (T,), (B, T) or (B, 1)"
        assert positions.dim() == 1 or positions.shape[0] in (B, 1), "positions must be (T,), (B, T) or (B, 1)"
        positions = positions.to(device=x.device, dtype=torch.int64)
    elif positions is not None:
        positions = operator.index(positions)
    return inv_freq.to(device=x.device, dtype=torch.float64).contiguous(), positions


def _refused(what: str):
    raise RuntimeError(f"{what} does not take these tensors (function transforms, traces, dispatch modes and tensor subclasses are not supported)")


def rotary(x: torch.Tensor, inv_freq: torch.Tensor, *, positions: Positions = None, interleaved: bool = False,
           head_first: bool = False) -> torch.Tensor:
    """``x`` with the first ``2 * len(inv_freq)`` elements of every head rotated by ``positions * inv_freq``.

    x: ``(B, T, H, D)`` bfloat16/float16 (``(B, H, T, D)`` with ``head_first``), D one of 16, 32, 64, 128.  The pairs are ``(i, i + R/2)``,
    R a multiple of 16, or ``(2i, 2i+1)`` with ``interleaved``, R even.  positions: the first position as a number p (p, p + 1, ...), None (0, 1, ...),
    or integers ``(T,)``, ``(B, T)`` or ``(B, 1)`` that are the positions themselves, not offsets: ``(B, 1)`` is one position for all tokens of a row, and tokens that follow
    each other from a start of their own per row are ``start[:, None] + torch.arange(T)``.  At most 2**30 tokens and 2**34 elements.  Differentiable with
    respect to ``x``, any number of times.
    """
    y = _native.load().rotary(x, inv_freq, positions, interleaved, head_first)   # None: not a call for the native path as it is
    if y is not None:
        return y
    _check_size(x.numel())
    x = _check_heads(x, "x")
    inv_freq, positions = _check_angles(x, inv_freq, positions, interleaved, head_first)
    with torch.cuda.device(x.device):
        y = _native.load().rotary(x, inv_freq, positions, interleaved, head_first)
    return y if y is not None else _refused("rotary")


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, inv_freq: torch.Tensor, *,
                   positions: Positions = None, interleaved: bool = False, eps: float = 1e-5,
                   head_first: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``rotary(rms_norm(q) * q_weight)`` and the same for ``k``, per head, in one pass and rounded once.

    q, k: ``(B, T, H, D)`` (``(B, H, T, D)`` with ``head_first``), alike but for the number of heads; weights: ``(H * D,)`` each
    (``GroupNorm(num_groups=heads)`` of the layer), or ``(D,)`` each, shared by the heads (``RMSNorm(head_dim)``).  The other arguments are those of
    ``rotary``.  Differentiable with respect to q, k and both weights, once.
    """
    out = _native.load().qk_norm_rotary(q, k, q_weight, k_weight, inv_freq, positions, interleaved, eps, head_first)
    if out is not None:
        return out
    _check_size(q.numel() + k.numel())
    q, k = _check_heads(q, "q"), _check_heads(k, "k")
    heads = 1 if head_first else 2
    assert q.dtype == k.dtype and q.device == k.device, "q and k must have the same type and device"
    assert q.shape[:heads] + q.shape[heads + 1:] == k.shape[:heads] + k.shape[heads + 1:], "q and k may differ in their heads only"
    D, Hq, Hk = q.shape[-1], q.shape[heads], k.shape[heads]
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        assert w.dim() == 1 and w.is_floating_point() and w.device == q.device, f"{name} must be a floating vector on the device of q"
    assert (q_weight.shape[0], k_weight.shape[0]) in ((Hq * D, Hk * D), (D, D)), "the weights must have (heads * head dim) or, both, (head dim) elements"
    inv_freq, positions = _check_angles(q, inv_freq, positions, interleaved, head_first)
    with torch.cuda.device(q.device):
        out = _native.load().qk_norm_rotary(q, k, q_weight, k_weight, inv_freq, positions, interleaved, float(eps), head_first)
    return out if out is not None else _refused("qk_norm_rotary")
