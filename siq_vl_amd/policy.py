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


def _logps(name: str, t: torch.Tensor, like: torch.Tensor | None = None, frozen: bool = False) -> torch.Tensor:
    if t.dtype != torch.float32:
        raise ValueError(f"{name} must be float32, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must live on the GPU, got {t.device}")
    if like is not None and (t.shape != like.shape or t.device != like.device):
        raise ValueError(f"{name} must be {tuple(like.shape)} on {like.device}, got {tuple(t.shape)} on {t.device}")
    if frozen and t.requires_grad:
        raise ValueError(f"gradients with respect to {name} are not supported (detach it)")
    return t.contiguous()


def _mask(mask: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor | None:
    if mask is None:
        return None
    if mask.dtype not in (torch.bool, torch.uint8):
        raise ValueError(f"mask must be bool or uint8, got {mask.dtype}")
    if mask.shape != like.shape or mask.device != like.device:
        raise ValueError(f"mask must be {tuple(like.shape)} on {like.device}, got {tuple(mask.shape)} on {mask.device}")
    return mask.contiguous()


def _offsets(cu: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    if cu.dtype != torch.int32 or cu.dim() != 1 or cu.numel() < 2 or cu.device != like.device:
        raise ValueError(f"cu_seqlens must be int32 [sequences + 1] on {like.device}, got {tuple(cu.shape)} {cu.dtype} on "
                         f"{cu.device}")
    return cu.contiguous()


def _divisor(items, device: torch.device) -> torch.Tensor | None:
    if items is None:
        return None
    if torch.is_tensor(items):
        if items.numel() != 1:
            raise ValueError(f"num_items_in_batch must be one number, got {tuple(items.shape)}")
        return items.detach().to(device=device, dtype=torch.float32).reshape(())
    return torch.tensor(float(items), dtype=torch.float32, device=device)


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, policy, reference, cu, mask, loss_type, order, beta, smoothing, normalized, divisor):
        dev, tokens, pairs = policy.device, policy.numel(), (cu.numel() - 1) // 2
        loss, chosen, rejected = policy.new_empty(()), policy.new_empty(pairs), policy.new_empty(pairs)
        coef = policy.new_empty(2 * pairs)
        L = _lib.lib()
        ws = torch.empty(L.siq_pref_workspace_bytes(pairs, tokens), dtype=torch.uint8, device=dev)
        with _lib.on_device(dev):
            rc = L.siq_pref_fwd(policy.data_ptr(), _ptr(reference), _ptr(mask), cu.data_ptr(), pairs, tokens, loss_type,
                                order, beta, smoothing, normalized, _ptr(divisor), loss.data_ptr(), chosen.data_ptr(),
                                rejected.data_ptr(), coef.data_ptr(), ws.data_ptr(), ws.numel(), _lib.stream(dev))
        _lib.check(rc, "siq_pref_fwd")
        ctx.save_for_backward(coef, cu, *(() if mask is None else (mask,)))
        ctx.shape, ctx.pairs = policy.shape, pairs
        ctx.mark_non_differentiable(chosen, rejected)
        ctx.set_materialize_grads(False)
        return loss, chosen, rejected

    @staticmethod
    def backward(ctx, grad_loss, *_):
        _lib.first_order("preference_loss")
        if grad_loss is None:
            return (None,) * 10
        coef, cu, *mask = ctx.saved_tensors
        grad = grad_loss.to(torch.float32)
        dev = coef.device
        dpolicy = torch.empty(ctx.shape, dtype=torch.float32, device=dev)
        with _lib.on_device(dev):
            rc = _lib.lib().siq_pref_bwd(grad.data_ptr(), coef.data_ptr(), mask[0].data_ptr() if mask else None,
                                         cu.data_ptr(), ctx.pairs, dpolicy.numel(), dpolicy.data_ptr(),
                                         _lib.stream(dev))
        _lib.check(rc, "siq_pref_bwd")
        return dpolicy, *(None,) * 9


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
    policy = _logps("policy_logps", policy_logps)
    reference = None if reference_logps is None else _logps("reference_logps", reference_logps, policy, frozen=True)
    mask, cu = _mask(mask, policy), _offsets(cu_seqlens, policy)
    if cu.numel() % 2 == 0:
        raise ValueError(f"preference pairs need an even number of sequences, got {cu.numel() - 1}")
    return PreferenceLoss(*_Preference.apply(policy, reference, cu, mask, kind, order, float(beta),
                                             float(label_smoothing), int(length_normalized),
                                             _divisor(num_items_in_batch, policy.device)))


class _Policy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, old, advantages, cu, mask, reference, per_token, aggregation, kl_type, low, high, dual,
                kl_coef, divisor):
        dev, tokens = logps.device, logps.numel()
        seqs = 1 if cu is None else cu.numel() - 1
        loss, kl, cut = logps.new_empty(()), logps.new_empty(()), logps.new_empty(())
        dtoken, weight = logps.new_empty(tokens), logps.new_empty(seqs if aggregation else 1)
        L = _lib.lib()
        ws = torch.empty(L.siq_policy_workspace_bytes(seqs, tokens), dtype=torch.uint8, device=dev)
        with _lib.on_device(dev):
            rc = L.siq_policy_fwd(logps.data_ptr(), old.data_ptr(), advantages.data_ptr(), _ptr(mask), _ptr(reference),
                                  _ptr(cu), seqs, tokens, per_token, aggregation, kl_type, low, high, dual, kl_coef,
                                  _ptr(divisor), loss.data_ptr(), kl.data_ptr(), cut.data_ptr(), dtoken.data_ptr(),
                                  weight.data_ptr(), ws.data_ptr(), ws.numel(), _lib.stream(dev))
        _lib.check(rc, "siq_policy_fwd")
        ctx.save_for_backward(dtoken, weight, *(() if cu is None else (cu,)))
        ctx.shape, ctx.seqs, ctx.aggregation = logps.shape, seqs, aggregation
        ctx.mark_non_differentiable(kl, cut)
        ctx.set_materialize_grads(False)
        return loss, kl, cut

    @staticmethod
    def backward(ctx, grad_loss, *_):
        _lib.first_order("policy_loss")
        if grad_loss is None:
            return (None,) * 14
        dtoken, weight, *cu = ctx.saved_tensors
        grad = grad_loss.to(torch.float32)
        dev = dtoken.device
        dlogps = torch.empty(ctx.shape, dtype=torch.float32, device=dev)
        with _lib.on_device(dev):
            rc = _lib.lib().siq_policy_bwd(grad.data_ptr(), dtoken.data_ptr(), weight.data_ptr(),
                                           cu[0].data_ptr() if cu else None, ctx.seqs, dtoken.numel(), ctx.aggregation,
                                           dlogps.data_ptr(), _lib.stream(dev))
        _lib.check(rc, "siq_policy_bwd")
        return dlogps, *(None,) * 13


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
    ``kl`` = ``-x`` (``"k1"``), ``x^2 / 2`` (``"k2"``) or ``e^x - 1 - x`` (``"k3"``).
    ``aggregation="token"`` averages over the counted tokens, ``"sequence"`` each
    sequence's counted tokens and then the sequences; ``num_items_in_batch``
    replaces the number of counted tokens, or of sequences, divided by.  A batch
    that counts nothing has loss 0 and gradient 0.
    """
    agg, kind = _choice("aggregation", aggregation, _AGGREGATIONS), _choice("kl_type", kl_type, _KL_TYPES)
    lp = _logps("logps", logps)
    old = _logps("old_logps", old_logps, lp, frozen=True)
    ref = None if reference_logps is None else _logps("reference_logps", reference_logps, lp, frozen=True)
    mask = _mask(mask, lp)
    cu = None if cu_seqlens is None else _offsets(cu_seqlens, lp)
    per_token = advantages.shape == lp.shape
    adv = _logps("advantages", advantages, lp if per_token else None, frozen=True)
    seqs = 1 if cu is None else cu.numel() - 1
    if not per_token and (adv.shape != (seqs,) or adv.device != lp.device):
        raise ValueError(f"advantages must be {tuple(lp.shape)} (one a token) or [{seqs}] (one a sequence) on {lp.device}, "
                         f"got {tuple(adv.shape)} on {adv.device}")
    high = clip_low if clip_high is None else clip_high
    if dual_clip is not None and not dual_clip > 1:
        raise ValueError(f"dual_clip must be above 1, got {dual_clip}")
    return PolicyLoss(*_Policy.apply(lp, old, adv, cu, mask, ref, int(per_token), agg, kind, float(clip_low), float(high),
                                     float(dual_clip or 0.0), float(kl_coef), _divisor(num_items_in_batch, lp.device)))


__all__ = ["PolicyLoss", "PreferenceLoss", "policy_loss", "preference_loss"]
