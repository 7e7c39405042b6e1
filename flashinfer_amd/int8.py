"""Products of 8-bit integers with a scale for each token and output channel.

The counterpart of the FP8 path of ``kernel.run`` for weights in int8:
``quantize_int8`` and ``swiglu_quantize_int8`` make int8 rows with a scale
each, ``int8_matmul`` multiplies them with a layer's weights, and
``int8_grouped_matmul`` with the weights of each row's expert, in the order of
``experts.sort_experts``. Sums are exact in int32. No gradients: these serve.
The reference has no integer path.

Everything runs on torch's current stream with no host synchronisation, and
can be captured into a graph. There is no CPU path.
"""
from __future__ import annotations

import torch

from .experts import _mi_experts


def quantize_int8(x: torch.Tensor, num_rows: torch.Tensor | None = None, q: torch.Tensor | None = None,
                  scale: torch.Tensor | None = None):
    """``(q, scale)`` of ``x`` [M, K] (bfloat16, float16 or float32): int8 [M, K]
    and fp32 [M] with ``scale[m] = max(amax, 1e-10) / 127`` and ``q = x / scale``
    rounded to nearest even. A row that holds a NaN or an infinity gets a scale
    that is not finite, so that what is made of it is NaN.

    ``num_rows`` (int32, one element, on the device) limits the work to the
    first rows, e.g. ``plan.expert_offsets[-1:]``; the others are zeros, or stay
    as they were in ``q`` and ``scale`` passed in."""
    return _mi_experts.quantize(x, False, num_rows, q, scale)


def swiglu_quantize_int8(x: torch.Tensor, num_rows: torch.Tensor | None = None,
                         q: torch.Tensor | None = None, scale: torch.Tensor | None = None):
    """``quantize_int8`` of ``silu(x[:, I:]) * x[:, :I]`` for ``x`` [M, 2I], in fp32
    without rounding in between: what stands between the two products of an
    expert (the halves as in solution/triton/kernel.py:297-330)."""
    return _mi_experts.quantize(x, True, num_rows, q, scale)


def int8_matmul(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[m, n] = (sum_k a[m, k] b[n, k]) a_scale[m] b_scale[n] + bias[n]`` for
    int8 ``a`` [M, K] and ``b`` [N, K] (weights as a linear layer holds them),
    fp32 ``a_scale`` [M] and ``b_scale`` [N]. K is 1 to 131071. ``bias`` [N] in
    any of the three float types. ``out`` [M, N] in ``out_dtype`` (bfloat16,
    float16 or float32; that of ``out`` if one is passed), rounded once.

    Rows may lie at any distance; K, strides and addresses that are multiples
    of 16 take the fast kernels, and large products of another K are copied to
    such rows first."""
    return _mi_experts.int8_matmul(a, a_scale, b, b_scale, bias, out_dtype, out)


def int8_grouped_matmul(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                        expert_offsets: torch.Tensor, row_ids: torch.Tensor | None = None,
                        out_dtype: torch.dtype = torch.bfloat16,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """``int8_matmul`` of each row with the weights of its expert: ``b`` int8
    [E, N, K], ``b_scale`` fp32 [E, N]; rows ``expert_offsets[e] ..
    expert_offsets[e+1] - 1`` are expert e's (``ExpertPlan.expert_offsets``).

    Row m of the product is row m of ``a``, or with ``row_ids`` (int32 [R]) row
    ``row_ids[m]``: ``plan.token_of_row`` multiplies tokens without laying them
    out first. Result [R, N]. Rows that no expert has are zeros, or stay as
    they were in ``out`` (a shard that has few of the rows writes only those).
    An id that is no row of ``a`` gives a row of NaN."""
    return _mi_experts.int8_grouped_matmul(a, a_scale, b, b_scale, expert_offsets, row_ids, out_dtype, out)
