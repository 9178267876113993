"""Log-probabilities of the labels from hidden states, without logits, on MI355X: host side.

The reference's loss is the mean of them (``lm_head``, transformers
models/qwen2/modeling_qwen2.py:465, and ``ForCausalLMLoss``,
loss/loss_utils.py:32-71); the losses of preference and policy training
(``siq_vl_amd.policy``) weight each token's.  ``fused_linear_log_probs`` gives
them with the kernels of the fused cross-entropy: ignored rows are compacted
away, the logits exist only as one chunk's softmax numerators, and the gradient,
which is known per token only in the backward, is applied there as one factor a
row.

The backward starts from the numerators where the forward could keep them
(``keep_bytes``), and forms the logits again, chunk by chunk, otherwise: a
quarter of the work in full training, a third with a frozen ``lm_head``.
"""

from __future__ import annotations

import torch

from . import _lib
from .cross_entropy import _LABEL_CHECKS, IGNORE_INDEX, _judge, _track_bad, default_chunk_tokens

# What the forward may keep for its backward: rows x vocab bf16.  The head's
# backward is a step's first, so this is held beside all other activations, but
# not for long; 8 GiB are 28,000 rows at vocab 151,936 and 3% of the card.
DEFAULT_KEEP_BYTES = 8 << 30


def flp_fwd(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, ignore_index: int = IGNORE_INDEX,
            temperature: float = 1.0, keep: bool = False):
    """Raw forward: ``(logp fp32 [n], count, bad_labels, saved | None)``."""
    logp, counts, saved = _lib.native().flp_fwd(hidden, weight, labels, int(ignore_index), float(temperature), bool(keep))
    return logp, counts[0], counts[1], saved


def flp_bwd(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, dlogp: torch.Tensor,
            ignore_index: int = IGNORE_INDEX, temperature: float = 1.0, saved: torch.Tensor | None = None,
            need_dhidden: bool = True, need_dweight: bool = True, chunk_tokens: int | None = None):
    """Raw backward: ``(dhidden | None, dweight | None)``; ``saved`` is the
    forward's on the same inputs, or None (the logits are formed again)."""
    if hidden.dim() == weight.dim() == 2 and chunk_tokens is None:
        chunk_tokens = default_chunk_tokens(weight.shape[0])
    return _lib.native().flp_bwd(hidden, weight, labels, dlogp, int(ignore_index), float(temperature), saved,
                                 bool(need_dhidden), bool(need_dweight), int(chunk_tokens or 0))


def fused_linear_log_probs(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                           ignore_index: int = IGNORE_INDEX, temperature: float = 1.0, chunk_tokens: int | None = None,
                           keep_bytes: int = DEFAULT_KEEP_BYTES, validate="lazy") -> torch.Tensor:
    """``log_softmax(hidden @ weight.T / temperature)`` at ``labels``, without logits.

    ``labels`` are the already-shifted targets (same shape as ``hidden[..., 0]``);
    the result has their shape, fp32, with 0 where a label is ``ignore_index``
    (such rows take no part and have gradient 0).  Labels outside ``[0, vocab)``
    raise ``LabelError`` as ``fused_linear_cross_entropy``'s do (``validate``).
    ``temperature``: what sampled answers were drawn with.

    ``keep_bytes`` bounds what the forward may keep for the backward (2 * rows *
    vocab bytes, ignored rows counted: how many there are is known on the device
    alone); a batch above it keeps nothing, and the backward forms the logits
    again, ``chunk_tokens`` rows at a time (None: 2 GiB of them).
    Without gradients nothing is kept.  A frozen ``weight`` gives the dH-only
    backward.
    """
    if labels.shape != hidden.shape[:-1]:
        raise ValueError(f"labels must be {tuple(hidden.shape[:-1])}, got {tuple(labels.shape)}")
    h = hidden if hidden.dtype == torch.bfloat16 else hidden.to(torch.bfloat16)
    w = weight if weight.dtype == torch.bfloat16 else weight.to(torch.bfloat16)
    if chunk_tokens is None:
        chunk_tokens = default_chunk_tokens(w.shape[0])
    ignore_index = int(ignore_index)
    host = _LABEL_CHECKS.landing(2) if h.is_cuda and validate not in (None, False, "sync") else None
    try:
        logp, counts = _lib.native().linear_log_probs(h, w, labels, ignore_index, float(temperature), int(chunk_tokens),
                                                      int(keep_bytes), host)
    except BaseException:  # (a checkpoint's recomputation ends in one, behind the launch)
        if host is not None:
            _LABEL_CHECKS.hold(h.device, host)
        raise
    if host is not None:
        _LABEL_CHECKS.landed_on(h.device, host, _judge(w.shape[0], ignore_index))
    else:
        _track_bad(counts[1], w.shape[0], ignore_index, validate)
    return logp


__all__ = ["DEFAULT_KEEP_BYTES", "flp_bwd", "flp_fwd", "fused_linear_log_probs"]
