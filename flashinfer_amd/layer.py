"""Inside a mixture-of-experts layer of a caller's own: the balance loss of its
router and the gate between its experts' products, both with gradients.

``experts.sort_experts``, ``permute`` and ``unpermute`` bring tokens to their
experts and back; ``balance_loss`` keeps a router that is being trained from
preferring a few of them, and ``swiglu`` is what stands between the experts'
two products, with dropout. The reference serves a trained layer and has
neither by itself (its gate is part of solution/triton/kernel.py:297-330).

Everything runs on torch's current stream with no host synchronisation, and
can be captured into a graph. Gradients are once, in reverse mode; tensors
with a forward-mode tangent are refused. There is no CPU path.
"""
from __future__ import annotations

import operator

import torch

from .experts import _Extension

_mi_layer = _Extension("_mi_layer", ("balance_loss", "swiglu", "pack_int4", "quantize_int4", "int4_matmul"))

_SCORES = {"softmax": 0, "sigmoid": 1}


def balance_loss(logits: torch.Tensor, topk_ids: torch.Tensor, seq_offsets: torch.Tensor | None = None,
                 mask: torch.Tensor | None = None, score: str = "softmax"):
    """``(loss, counts)`` of a router: how unevenly it loads its experts.

    ``logits`` [T, E] (bfloat16, float16 or float32; up to 1024 experts) and
    the experts chosen from them, ``topk_ids`` (int32 [T, k], k up to 64; ids
    outside 0 .. E - 1 count nowhere). ``P[t]`` is the softmax of ``logits[t]``,
    or with ``score="sigmoid"`` its sigmoids divided by their sum (a row that is
    -inf throughout has zeros). Of a sequence's n tokens and the c[e] slots of
    theirs that name expert e,

        sum_e (E c[e] / (k n)) (sum_t P[t, e] / n)

    is 1 for an even load, and ``loss`` (fp32, a scalar) its mean over the
    sequences that have a token. Sequence s has the tokens ``seq_offsets[s] ..
    seq_offsets[s + 1] - 1`` (int32 [S + 1], non-decreasing; tokens outside
    belong to none), without them the batch is one. ``mask`` (bool [T]) leaves
    tokens out: whatever they hold, NaN too, changes nothing. ``counts`` are
    c as int32 [S, E], or [E] without ``seq_offsets``.

    Differentiable in ``logits`` through ``P``; a token left out gets zeros.
    Sums are fp32 in a fixed order, so the same call gives the same bits."""
    if score not in _SCORES:
        raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    return _mi_layer.balance_loss(logits, topk_ids, seq_offsets, mask, _SCORES[score])


def swiglu(x: torch.Tensor, dropout: float = 0.0, seed: int | torch.Tensor | None = None,
           num_rows: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(x[:, I:]) * x[:, :I]`` for ``x`` [M, 2I] (bfloat16, float16 or
    float32; the halves as ``swiglu_quantize_int8`` takes them), in fp32 and
    rounded once.

    ``dropout`` sets elements to zero (whatever they were) with this
    probability, to the nearest 1 / 65536 below 1, and divides the others by
    what it leaves. Which ones depends on ``seed`` and the element's place alone
    (Philox4x32-10, 16 bits each), so no mask is stored and the backward pass
    makes it again: an int in -2^63 .. 2^64 - 1, or int64 with one element on
    the device, which a captured graph can read anew at each replay. Each layer and step wants a
    seed of its own.

    ``num_rows`` (int32, one element, on the device) limits the work to the
    first rows, e.g. ``plan.expert_offsets[-1:]``; the others are zeros, or stay
    as they were in ``out``. Differentiable in ``x`` (without ``out``); rows past
    ``num_rows`` get zeros."""
    threshold = 0
    if dropout:
        threshold = round(dropout * 65536) if 0.0 <= dropout < 1.0 else 65536
        if threshold >= 65536:
            raise ValueError(f"dropout must be 0 to 1 - 2^-16, got {dropout}")
        if seed is None:
            raise ValueError("dropout needs a seed")
    number, tensor = 0, None
    if isinstance(seed, torch.Tensor):
        tensor = seed
    elif threshold:
        number = operator.index(seed)
        if not -(1 << 63) <= number < 1 << 64:
            raise ValueError(f"seed must have 64 bits, got {number}")
        number -= (number >> 63) << 64 if number > 0 else 0
    return _mi_layer.swiglu(x, threshold, number, tensor, num_rows, out)
