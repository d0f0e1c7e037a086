"""Operators for sequences of different lengths, packed one behind another without padding: rotary positions, and
attention with grouped heads, causal or both ways, for training and for single new tokens against a cache.

The reference has neither; they are what a trunk over sequences beside the Evoformer needs.  Both run on CUDA
tensors (bfloat16, float16, float32) in kernels of this package, with sums in a fixed order: the same bits in every
run.  They can be captured in a CUDA graph, and can be differentiated once, in reverse mode.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib

_LAYOUTS = {"half": 0, "interleaved": 1}


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, slow: float = 1.0, fast: float = 4.0,
                       device=None) -> torch.Tensor:
    """Frequencies ``base ** (-2 i / dim)`` of ``dim / 2`` pairs, radians a position, float64.  ``scaling`` fits a model to
    contexts ``factor`` times as long as it was trained on:

    * ``"linear"``: all frequencies divided by ``factor``.
    * ``"base"``: the base grows so that the slowest pair is divided by ``factor`` and the fastest stays as it is.
    * ``"bands"``: pairs that make fewer than ``slow`` turns in ``original_length`` positions are divided by ``factor``, those
      that make more than ``fast`` stay, with a line between the two over the number of turns."""
    dim = int(dim)
    if dim < 2 or dim % 2:
        raise ValueError("dim must be even and at least 2")
    if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor > 0):
        raise ValueError("base and factor must be positive")
    if scaling not in (None, "linear", "base", "bands"):
        raise ValueError("scaling must be None, 'linear', 'base' or 'bands'")
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    f = base ** (torch.arange(0, dim, 2, dtype=torch.float64) / -dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "bands":
        if original_length is None or original_length < 1 or not 0 <= slow < fast:
            raise ValueError("'bands' needs original_length and 0 <= slow < fast")
        keep = ((original_length * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
    return f.to(device)


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor, *,
                     layout: str = "half", amplitude: float = 1.0):
    """q and k (``[..., N, H, D]`` and ``[..., N, H_k, D]``, up to two axes before N) with the first ``2 n`` values of every
    head turned by ``position * frequency``: ``(a cos - b sin, a sin + b cos) * amplitude``.  Returns both (q alone where k is
    None), dense; what lies behind the ``2 n`` values is copied.

    ``positions``: int64 or int32, ``[N]`` or the axes before the heads.  ``frequencies``: ``[n]``, float64 or float32, as of
    ``rotary_frequencies``; angles are formed in 64 bits, so far positions are as exact as near ones.  ``layout``: pairs are
    values ``(i, i + n)`` (``"half"``) or ``(2 i, 2 i + 1)`` (``"interleaved"``).  q and k may be strided (slices of one
    projection).  Gradients: q and k."""
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be one of {', '.join(map(repr, _LAYOUTS))}")
    return _lib.host().rotary_embedding(q, k, positions, frequencies, _LAYOUTS[layout], amplitude)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor,
                     key_offsets: Optional[torch.Tensor] = None, *, causal: bool = True,
                     scale: Optional[float] = None) -> torch.Tensor:
    """``softmax(scale q k^T) v`` within each of B sequences whose rows lie one behind another: q ``[T, H, D]``, k and v
    ``[T_k, H_k, D]``, H a multiple of H_k (query head h reads key head ``h // (H // H_k)``), D up to 256.  ``scale`` is
    ``D ** -0.5`` by default.

    ``offsets`` (``[B + 1]``, int32 or int64, ascending): sequence b has the queries ``offsets[b]`` to ``offsets[b + 1]``.
    ``key_offsets``: the same for the keys where they differ; or ``[B, 2]``, begin and end of each sequence's keys, which may
    then lie anywhere, as in the slots of a cache (``cache.view(-1, H_k, D)``), in any order and shared.  Both are read on
    the device, so that a call never waits for it; no row outside the tensors is touched whatever they hold.

    With ``causal``, query i of n sees the keys up to ``i + n_k - n``: the last query sees all, a single one is a new token
    against the keys so far.  A query that sees no key gets zeros (and gives no gradient), as do rows outside every sequence.
    Values there, and in key rows outside the sequence, may be anything; within a sequence q, k and v have to be finite (where a
    score is NaN or plus infinity, the queries that see it get what is not finite either).

    16-bit types: P enters its products rounded to the type, as in the package's other attention (in two pieces of it for a few
    queries without a gradient); statistics and sums are fp32.  Gradients: q, k, v (k and v not with ``[B, 2]`` ranges)."""
    return _lib.host().packed_attention(q, k, v, offsets, key_offsets, causal, scale)
