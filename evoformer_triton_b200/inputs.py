"""The operators that make the attention's inputs: layer norm, a learned relative position bias, and the
projection of the pair representation to a pair bias.

The reference's op begins at Q, K, V and a finished pair bias; these are the steps of a block before it.  All
three run on CUDA tensors (bfloat16, float16, float32) in kernels of this package, forward and backward, with
sums in fp32 taken in a fixed order: the same bits in every run.  They can be captured in a CUDA graph,
and can be differentiated once, in reverse mode.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _lib

_SCHEMES = {"clip": 0, "log": 1, "log_causal": 2}
MAX_BUCKETS = 1024
MAX_LOG_BUCKETS = 256  # (causal ones have 127 borders, which are handed over with every launch)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, in the type of ``x``.

    ``weight`` and ``bias`` (``[C]``, either may be left out) may be of another type than ``x``, as fp32 weights
    beside 16-bit activations.  ``x`` may be strided (transposed rows, a slice of a wider tensor): rows are read
    where they lie as long as their C values are contiguous.  The result and the gradient of ``x`` are dense."""
    return _lib.host().layer_norm(x, weight, bias, eps)


@functools.lru_cache(maxsize=None)
def _log_buckets(n: int, max_distance: int, causal: bool):
    """``(exact, edges)`` of logarithmic buckets: distances below ``exact`` have a bucket each, and ``edges[k - 1]`` is
    the smallest distance of bucket ``exact + k``: the smallest whole d with
    ``exact + floor(log(d / exact) / log(max_distance / exact) * m) >= exact + k``, m the number of wide buckets, which
    is ``d ** m * exact ** k >= max_distance ** k * exact ** m`` in whole numbers (a logarithm in floating point
    puts some distances that lie on a border, 16 for n = 32 up to 128, on one side or the other)."""
    side = n if causal else n // 2  # buckets of one direction
    exact = side // 2
    m = side - exact
    edges = []
    for k in range(1, m):
        reached = lambda d: d ** m * exact ** k >= max_distance ** k * exact ** m  # noqa: B023, E731
        d = int(exact * (max_distance / exact) ** (k / m))  # (floating point says where to look)
        while not reached(d):
            d += 1
        while d > exact and reached(d - 1):
            d -= 1
        edges.append(max(d, exact))
    return exact, edges


def relative_position_bias(table: torch.Tensor, positions: torch.Tensor, key_positions: Optional[torch.Tensor] = None, *,
                           max_distance: int, buckets: str = "clip", pair_bias: Optional[torch.Tensor] = None,
                           dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """A pair bias ``[B, 1, H, N, N_keys]`` looked up in ``table`` (``[n, H]``) by the distance of two residues.

    ``positions`` are the residue numbers (int64 or int32) ``[N]``, or ``[B, N]`` where they differ over the batch;
    ``key_positions`` those of the keys where they are not the same, for an attention that has them (the one of this
    package has the queries' residues as keys).  With ``[N]`` the
    result has B = 1: ``expand`` it, the attention reads it in place.  ``buckets``:

    * ``"clip"``: ``clamp(position - key_position, -max_distance, max_distance) + max_distance``; n = 2 max_distance + 1.
    * ``"log"`` (n a multiple of 4): each direction has n / 2 buckets, keys that follow the query the upper ones;
      distances below n / 4 have one each, longer ones share them logarithmically up to ``max_distance``, beyond
      which all have the last.
    * ``"log_causal"`` (n even): the same with n buckets for keys before the query; those that follow it have bucket 0.

    ``pair_bias`` (``[B, 1, H, N, N_keys]``) is a bias to which this one is added, in fp32, before the one rounding to
    ``dtype`` (by default that of ``pair_bias``, else of ``table``).  Rows of the result begin on 16-byte boundaries, so
    the attention takes it as it is for any N.  Gradients: ``table`` and ``pair_bias``."""
    if buckets not in _SCHEMES:
        raise ValueError(f"buckets must be one of {', '.join(map(repr, _SCHEMES))}")
    n, max_distance = (table.shape[0] if table.dim() == 2 else 0), int(max_distance)
    exact, edges = max_distance, []
    if buckets == "clip":
        if max_distance < 0 or n != 2 * max_distance + 1 or n > MAX_BUCKETS:
            raise ValueError(f"clipped buckets need a table of 2 * max_distance + 1 rows, at most {MAX_BUCKETS}")
    else:
        causal = buckets == "log_causal"
        per = 2 if causal else 4
        if n < per or n % per or n > MAX_LOG_BUCKETS:
            raise ValueError(f"{buckets!r} buckets need a table of a multiple of {per} rows, at most {MAX_LOG_BUCKETS}")
        if not n // per < max_distance < 1 << 20:
            raise ValueError(f"max_distance must be above {n // per}, the number of distances with a bucket of their own, and below 2 ** 20")
        exact, edges = _log_buckets(n, max_distance, causal)
    return _lib.host().relative_position_bias(table, positions, key_positions, pair_bias, dtype, _SCHEMES[buckets], exact, edges)


def pair_bias_projection(pair: torch.Tensor, weight: torch.Tensor, norm_weight: Optional[torch.Tensor] = None,
                         norm_bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """The pair bias ``[B, 1, H, N_res, N_res]`` of a pair representation ``[B, N_res, N_res, C]``:
    ``linear(layer_norm(pair, norm_weight, norm_bias, eps), weight)`` with the heads first, in the type of ``pair``, in one
    pass over ``pair``; the normalised representation is not written.

    ``weight`` is ``[H, C]`` as a linear layer holds it; all weights may be of another type than ``pair``.  ``pair`` may be
    strided with its C values contiguous (``pair.transpose(1, 2)`` around ending nodes).  C up to 512, H up to 64.
    Where ``pair`` has 16 bits, ``weight * norm_weight`` enters the products with 16 bits (bfloat16; 22 in the forward of
    float16), fp32 weights too: a result is off by up to 2 ** -16 of the sum of its terms' magnitudes beside its rounding.
    The gradients of the weights are fp32 sums of fp32 factors.
    Rows of the result begin on 16-byte boundaries, so the attention takes it as it is for any N_res."""
    return _lib.host().pair_bias_projection(pair, weight, norm_weight, norm_bias, eps)
