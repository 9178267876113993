"""Losses of preference and policy training on MI355X: host side.

The reference ends at supervised fine-tuning (scripts/train.py:685-745).  What
follows it trains on pairs of answers, or on sampled answers with advantages,
over the same packed batches (``cu_seqlens``) and labels:

* ``preference_loss`` -- paired log ratios against a frozen reference model
  (sigmoid, ipo or hinge);
* ``policy_loss`` -- the clipped policy loss with an optional second clip and KL
  term, averaged over tokens or sequence by sequence.

Both take fp32 per-token log-probabilities (``fused_linear_log_probs`` gives
them without logits) with a mask of the tokens that count; masked tokens count
nowhere, whatever their values, and have gradient zero.  The forward leaves the
gradients but for the upstream factor, which the backward applies.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

_LOSS_TYPES = {"sigmoid": 0, "ipo": 1, "hinge": 2}  # SIQ_PREF_*
_ORDERS = {"interleaved": 0, "halves": 1}  # SIQ_ORDER_*
_AGGREGATIONS = {"token": 0, "sequence": 1}  # SIQ_AGG_*
_KL_TYPES = {"k1": 0, "k2": 1, "k3": 2}  # SIQ_KL_*


class PreferenceLoss(NamedTuple):
    """``loss`` (differentiable), and ``beta`` times the scores of both sides of each pair."""

    loss: torch.Tensor
    chosen_rewards: torch.Tensor
    rejected_rewards: torch.Tensor


class PolicyLoss(NamedTuple):
    """``loss`` (differentiable), and over the counted tokens the mean KL estimate and the share that was cut."""

    loss: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor


def _choice(name: str, value: str, of: dict) -> int:
    if value not in of:
        raise ValueError(f"{name} must be one of {sorted(of)}, got {value!r}")
    return of[value]


def _divisor(items, device: torch.device) -> torch.Tensor | None:
    if items is None:
        return None
    if torch.is_tensor(items) and items.numel() != 1:
        raise ValueError(f"num_items_in_batch must be one number, got {tuple(items.shape)}")
    return _lib.scalar_on(device, items)


def preference_loss(policy_logps: torch.Tensor, reference_logps: torch.Tensor | None, cu_seqlens: torch.Tensor,
                    mask: torch.Tensor | None = None, beta: float = 0.1, loss_type: str = "sigmoid",
                    label_smoothing: float = 0.0, length_normalized: bool = False, order: str = "interleaved",
                    num_items_in_batch=None) -> PreferenceLoss:
    """The loss of paired sequences from their per-token log-probabilities.

    ``policy_logps`` / ``reference_logps``: fp32, one per token of the packed
    batch, any one shape (``reference_logps`` None: no reference model);
    ``cu_seqlens`` int32 ``[2 * pairs + 1]``; ``mask`` (bool or uint8): the
    answers' tokens.  Pair ``i`` is sequences ``2 i`` (chosen) and ``2 i + 1``
    (rejected), or with ``order="halves"`` ``i`` and ``pairs + i``.  A sequence's
    score is the sum of its counted tokens' policy - reference
    (``length_normalized``: their mean), ``x`` the difference of a pair's scores:

    * ``"sigmoid"``: ``-logsigmoid(beta x)``, with ``label_smoothing`` e
      ``-(1 - e) logsigmoid(beta x) - e logsigmoid(-beta x)``;
    * ``"ipo"``: ``(x - 1 / (2 beta))^2``;
    * ``"hinge"``: ``max(0, 1 - beta x)``.

    The loss is the mean over the pairs, or their sum over
    ``num_items_in_batch``.  A sequence of which nothing counts has score 0.
    """
    kind, order = _choice("loss_type", loss_type, _LOSS_TYPES), _choice("order", order, _ORDERS)
    return PreferenceLoss(*_lib.native().preference_loss(
        policy_logps, reference_logps, cu_seqlens, mask, kind, order, float(beta), float(label_smoothing),
        bool(length_normalized), _divisor(num_items_in_batch, policy_logps.device)))


def policy_loss(logps: torch.Tensor, old_logps: torch.Tensor, advantages: torch.Tensor,
                cu_seqlens: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                reference_logps: torch.Tensor | None = None, clip_low: float = 0.2, clip_high: float | None = None,
                dual_clip: float | None = None, kl_coef: float = 0.0, kl_type: str = "k3",
                aggregation: str = "token", num_items_in_batch=None) -> PolicyLoss:
    """The clipped policy loss of sampled tokens.

    ``logps`` / ``old_logps`` (the sampling policy's) / ``reference_logps``: fp32,
    one per token of the packed batch, any one shape; ``advantages`` fp32, of
    that shape (one a token) or ``[sequences]`` (where both fit: one a token);
    ``cu_seqlens`` int32 ``[sequences + 1]`` (None: one sequence); ``mask`` (bool
    or uint8): the answers' tokens.  With ``r = exp(logps - old_logps)`` a token's
    loss is

        ``-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef kl``

    (``clip_high`` None: ``clip_low``; ``dual_clip`` c > 1: for ``A < 0`` the
    objective is not below ``c A``), with ``x = reference_logps - logps`` and
    ``kl`` = ``-x`` (``"k1"``), ``x^2 / 2`` (``"k2"``) or ``e^x - 1 - x`` (``"k3"``);
    at ``kl_coef`` 0 the estimate is reported alone.
    ``aggregation="token"`` averages over the counted tokens, ``"sequence"`` each
    sequence's counted tokens and then the sequences; ``num_items_in_batch``
    replaces the number of counted tokens, or of sequences, divided by.  A batch
    that counts nothing has loss 0 and gradient 0, divided by 0 too.
    """
    agg, kind = _choice("aggregation", aggregation, _AGGREGATIONS), _choice("kl_type", kl_type, _KL_TYPES)
    high = clip_low if clip_high is None else clip_high
    if dual_clip is not None and not dual_clip > 1:
        raise ValueError(f"dual_clip must be above 1, got {dual_clip}")
    return PolicyLoss(*_lib.native().policy_loss(
        logps, old_logps, advantages, cu_seqlens, mask, reference_logps, agg, kind, float(clip_low), float(high),
        float(dual_clip or 0.0), float(kl_coef), _divisor(num_items_in_batch, logps.device)))


__all__ = ["PolicyLoss", "PreferenceLoss", "policy_loss", "preference_loss"]
