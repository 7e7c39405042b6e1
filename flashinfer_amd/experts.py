"""Tokens to the order of their experts and back, with gradients.

``kernel.run`` is the whole layer for FP8 weights. These operators are its
token side alone, for experts of a caller's own: ``sort_experts`` places every
(token, expert) slot of a routing at a row, ``permute`` lays the tokens' rows
out in that order, and ``unpermute`` brings the experts' rows back to their
tokens, weighted and summed. ``permute`` and ``unpermute`` are differentiable
(once, in reverse mode; tensors with a forward-mode tangent are refused); the
reference has neither (its sort and combine serve its one entry point,
solution/triton/kernel.py:460-505, :337-368).

Everything runs on torch's current stream with no host synchronisation, and
can be captured into a graph. There is no CPU path.
"""
from __future__ import annotations

from typing import NamedTuple

import torch


class _Extension:
    """flashinfer_amd/_mi_experts, loaded at the first call: the package has to
    import before it is built. Loud if it is missing, as there is no other
    implementation."""

    def __getattr__(self, name):
        try:
            from . import _mi_experts as ext
        except ImportError as e:
            raise RuntimeError("flashinfer_amd/_mi_experts is missing or does not load: build it with "
                               f"`python -m flashinfer_amd.build` ({e})") from e
        for n in ("sort_experts", "permute", "unpermute", "quantize", "int8_matmul", "int8_grouped_matmul"):
            self.__dict__[n] = getattr(ext, n)
        return getattr(ext, name)


_mi_experts = _Extension()


class ExpertPlan(NamedTuple):
    """Where the T * k slots of a routing lie once sorted by local expert.

    ``expert_offsets`` int32 [E+1]: first row of each expert; the last entry is
    S, the number of local rows. ``token_of_row`` int32 [T*k] and
    ``row_of_slot`` int32 [T, k]: the two directions. Rows from S on belong to
    the slots of other shards' experts.
    """
    expert_offsets: torch.Tensor
    token_of_row: torch.Tensor
    row_of_slot: torch.Tensor


def sort_experts(topk_ids: torch.Tensor, num_experts: int, expert_offset: int = 0) -> ExpertPlan:
    """Sorts the slots of ``topk_ids`` (int32 [T, k] of global expert ids, e.g.
    those of ``kernel.route``) by the experts ``expert_offset ..
    expert_offset + num_experts - 1`` of this shard. The order is stable: rows
    of one expert are ascending in token, then in slot. Ids outside the shard
    (negative ones too) go behind the last expert. A token may name an expert
    twice. k up to 64, up to 1024 experts."""
    return ExpertPlan(*_mi_experts.sort_experts(topk_ids, num_experts, expert_offset))


def permute(hidden: torch.Tensor, plan: ExpertPlan, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows [T*k, H] in the plan's order: row ``p`` is ``hidden[token_of_row[p]]``
    for the S local rows. The rows behind them are zeros; in a buffer passed as
    ``out`` they stay as they were (a shard that has few of the slots writes
    only those).

    Any real dtype of 1 to 8 bytes; bfloat16, float16 and float32 are
    differentiable (without ``out``). The gradient of a token is the sum of the
    gradients of its local rows, in fp32 in slot order, rounded once."""
    return _mi_experts.permute(hidden, plan[0], plan[2], out)


def unpermute(rows: torch.Tensor, plan: ExpertPlan, weights: torch.Tensor | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Tokens [T, H] from their experts' rows [T*k, H] (bfloat16, float16 or
    float32): the sum over a token's local slots of ``weights[t, j]`` (fp32
    [T, k]; ones if None) times row ``row_of_slot[t, j]``, in fp32 in slot
    order, rounded once. Zeros for a token without a local slot. Rows behind
    the local ones are not read.

    Differentiable in ``rows`` and ``weights`` (without ``out``): rows get
    ``weights[t, j]`` times their token's gradient (zeros behind the local
    ones), weights the fp32 dot product of their row and their token's
    gradient (0 for slots of other shards)."""
    return _mi_experts.unpermute(rows, plan[0], plan[2], weights, out)
