"""Products with weights of 4 bits that have a scale for each group of a
channel's values: what serves the experts (or any linear layer) at a quarter of
the bytes of 16-bit weights.

``pack_int4`` lays out weights that are quantised already, ``quantize_int4``
makes them from floats; ``int4_matmul`` multiplies rows with them, and
``int4_grouped_matmul`` with those of each row's expert, in the order of
``experts.sort_experts``. No gradients: these serve. The reference has no 4-bit
path.

Everything runs on torch's current stream with no host synchronisation, and
can be captured into a graph. There is no CPU path.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .layer import _mi_layer


class Int4Weights(NamedTuple):
    """Weights [N, K] or [E, N, K] as the products read them.

    ``packed`` uint8 [(E,) N / 16, K / 128, 1024] (both rounded up): tiles of 16
    channels x 128 values in the order of a wave's registers. ``scale``
    [(E,) K / group_size, N] (N rounded up to 16), float32 or of the products'
    type. ``Int4Weights(w.packed[e], w.scale[e], *w[2:])`` is one expert's.
    """
    packed: torch.Tensor
    scale: torch.Tensor
    N: int
    K: int
    group_size: int


def pack_int4(q: torch.Tensor, scale: torch.Tensor, group_size: int = 128) -> Int4Weights:
    """Weights ``q[n, k] * scale[n, k // group_size]`` laid out for the products:
    ``q`` int8 [N, K] or [E, N, K] with values -8 .. 7 (others are cut to
    that), ``scale`` [.., N, ceil(K / group_size)] in float32, or in the type of
    the rows that it will multiply. ``group_size`` is a power of two from 32."""
    return Int4Weights(*_mi_layer.pack_int4(q, scale, group_size), q.shape[-2], q.shape[-1], group_size)


def quantize_int4(w: torch.Tensor, group_size: int = 128) -> Int4Weights:
    """4-bit weights of ``w`` [N, K] or [E, N, K] (bfloat16, float16 or float32):
    for each group of ``group_size`` values of a channel ``scale = max(amax,
    1e-10) / 7`` in float32 and ``q = w / scale`` rounded to nearest even. A
    group that holds a NaN or an infinity gets a scale that is not finite."""
    return Int4Weights(*_mi_layer.quantize_int4(w, group_size), w.shape[-2], w.shape[-1], group_size)


def int4_matmul(x: torch.Tensor, w: Int4Weights, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[m, n] = sum_g scale[n, g] (sum_{k in g} x[m, k] q[n, k]) + bias[n]``
    for ``x`` [M, K] in bfloat16 or float16 and dense weights [N, K]. Weights
    are not rounded to x's type: sums of a group are of x times whole numbers,
    and the scale is applied to them, in fp32. ``bias`` [N] in any of the three
    float types. ``out`` [M, N] in ``out_dtype`` (x's if None; that of ``out``
    if one is passed), rounded once.

    Rows may lie at any distance; those that do not start at multiples of 16
    bytes, or whose K is no multiple of 8, are copied first."""
    return _mi_layer.int4_matmul("int4_matmul", x, *w, bias, None, None, out_dtype, out)


def int4_grouped_matmul(x: torch.Tensor, w: Int4Weights, expert_offsets: torch.Tensor,
                        row_ids: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """``int4_matmul`` of each row with the weights of its expert: ``w`` of [E, N,
    K]; rows ``expert_offsets[e] .. expert_offsets[e+1] - 1`` are expert e's
    (``ExpertPlan.expert_offsets``).

    Row m of the product is row m of ``x``, or with ``row_ids`` (int32 [R]) row
    ``row_ids[m]``: ``plan.token_of_row`` multiplies tokens without laying them
    out first. Result [R, N]. Rows that no expert has are zeros, or stay as
    they were in ``out`` (a shard that has few of the rows writes only those).
    An id that is no row of ``x`` gives a row of NaN."""
    return _mi_layer.int4_matmul("int4_grouped_matmul", x, *w, None, expert_offsets, row_ids, out_dtype, out)
