"""Distillation from a teacher's most probable tokens on MI355X: host side.

The reference trains on labels alone (``ForCausalLMLoss``, transformers
loss/loss_utils.py:32-71).  A teacher says more of each position: its most
probable tokens and their log-probabilities, as ``fused_linear_token_stats``
(``siq_vl_amd.log_probs``) gives them.  ``fused_linear_distillation`` is the loss
of a student against them, on the same packed batch and with the kernels of the
fused cross-entropy: no logits, ignored rows compacted away, and both gradients
made in the forward, which the backward scales by the upstream gradient.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .cross_entropy import IGNORE_INDEX, _raise_bad, default_chunk_tokens
from .log_probs import _validated

_DIVERGENCES = ("forward", "reverse")


class TeacherError(ValueError):
    """A token of a teacher outside [0, vocab) that is not -1, or named twice for
    one position."""


class DistillationLoss(NamedTuple):
    """``loss = (1 - ce_weight) * divergence + ce_weight * cross_entropy``, fp32
    scalars; only ``loss`` has a gradient."""

    loss: torch.Tensor
    divergence: torch.Tensor
    cross_entropy: torch.Tensor | None


def _judge(vocab: int, ignore_index: int):
    def judge(vals):
        if vals[1] > 0:
            _raise_bad(int(vals[1]), vocab, ignore_index)
        if vals[2] > 0:
            raise TeacherError(f"fused_linear_distillation: {int(vals[2])} of the teacher's tokens lie outside "
                               f"[0, {vocab}) and are not -1, or are named twice for one position")

    return judge


def fused_linear_distillation(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor | None,
                              top_ids: torch.Tensor, top_log_probs: torch.Tensor, ignore_index: int = IGNORE_INDEX,
                              temperature: float = 1.0, ce_weight: float = 0.0, divergence: str = "forward",
                              tail: bool = True, num_items_in_batch=None, chunk_tokens: int | None = None,
                              validate="lazy") -> DistillationLoss:
    """The divergence of ``softmax(hidden @ weight.T / temperature)`` from a teacher's
    distribution, without logits, and the labels' cross-entropy beside it.

    ``top_ids`` (int64 or int32) and ``top_log_probs``: the teacher's tokens, up to 128
    a position, and their log-probabilities at ``temperature`` (shape
    ``[..., top_k]`` over ``hidden[..., 0]``'s).  An id of -1 or a log-probability of
    ``-inf`` names no token.  With t, s the teacher's and the student's probabilities
    of the named tokens, r = max(1 - sum t, 0) and q what both give to all others:

    * ``"forward"``: ``sum t (ln t - ln s)``, and with ``tail`` ``+ r (ln r - ln q)``, so
      that tokens which the teacher does not name are held to what it left them;
    * ``"reverse"``: ``sum s (ln s - ln t) + q (ln q - ln r)`` with r at least 2^-24; it
      needs ``tail``.

    ``loss = (1 - ce_weight) * divergence + ce_weight * cross_entropy``, each the mean
    over the rows whose label counts (``labels`` and ``ignore_index`` as for
    ``fused_linear_cross_entropy``), or the sum over ``num_items_in_batch``; NaN if no
    row counts.  ``ce_weight`` goes with ``temperature`` 1 alone; no factor of
    temperature squared is applied.  Without labels every row counts, ``ce_weight`` is
    0 and ``cross_entropy`` None.

    Labels outside ``[0, vocab)`` raise ``LabelError``, a teacher's bad tokens
    ``TeacherError``: lazily by default (``validate``), at a later call or at
    ``cross_entropy.check_pending_labels()``.  Without gradients only the losses are
    computed; a frozen ``weight`` gives the dH-only call.
    """
    if divergence not in _DIVERGENCES:
        raise ValueError(f"divergence must be one of {_DIVERGENCES}, got {divergence!r}")
    shape = hidden.shape[:-1]
    if top_ids.shape[:-1] != shape or top_log_probs.shape != top_ids.shape:
        raise ValueError(f"top_ids and top_log_probs must be {tuple(shape)} with the teacher's tokens behind it, got "
                         f"{tuple(top_ids.shape)} and {tuple(top_log_probs.shape)}")
    vocab = weight.shape[0]
    given = labels is not None
    if not given:
        if ce_weight != 0:
            raise ValueError("ce_weight needs labels")
        if top_ids.shape[-1] == 0:
            raise ValueError("top_ids names no token")
        first = top_ids[..., 0]
        labels = torch.where((first >= 0) & (first < vocab), first, 0).to(torch.int64)
        ignore_index = IGNORE_INDEX
    if labels.shape != shape:
        raise ValueError(f"labels must be {tuple(shape)}, got {tuple(labels.shape)}")
    h = hidden if hidden.dtype == torch.bfloat16 else hidden.to(torch.bfloat16)
    w = weight if weight.dtype == torch.bfloat16 else weight.to(torch.bfloat16)
    teacher = top_log_probs
    if teacher.dtype != torch.float32 and teacher.dtype.is_floating_point:
        teacher = teacher.to(torch.float32)
    if chunk_tokens is None:
        chunk_tokens = default_chunk_tokens(vocab)
    ignore_index = int(ignore_index)
    divisor = None if num_items_in_batch is None else _lib.scalar_on(hidden.device, num_items_in_batch)
    loss, div, ce = _validated(
        3, h, validate, _judge(vocab, ignore_index),
        lambda host: _lib.native().distillation(h, w, labels, top_ids, teacher, ignore_index, float(temperature),
                                                float(ce_weight), divergence == "reverse", bool(tail), int(chunk_tokens),
                                                divisor, host))
    return DistillationLoss(loss, div, ce if given else None)


__all__ = ["DistillationLoss", "TeacherError", "fused_linear_distillation"]
