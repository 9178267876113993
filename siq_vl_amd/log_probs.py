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
from .cross_entropy import IGNORE_INDEX, _check_operands, _track_bad, default_chunk_tokens

# What the forward may keep for its backward: rows x vocab bf16.  The head's
# backward is a step's first, so this is held beside all other activations, but
# not for long; 8 GiB are 28,000 rows at vocab 151,936 and 3% of the card.
DEFAULT_KEEP_BYTES = 8 << 30


def flp_fwd(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, ignore_index: int = IGNORE_INDEX,
            temperature: float = 1.0, keep: bool = False):
    """Raw forward: ``(logp fp32 [n], count, bad_labels, saved | None)``."""
    logp, counts, saved = _forward(hidden, weight, labels, ignore_index, temperature, keep, labels.shape)
    return logp, counts[0], counts[1], saved


def _forward(hidden, weight, labels, ignore_index, temperature, keep, shape):
    """``(logp of that shape, [count, bad_labels] int64, saved | None)``."""
    _check_operands(hidden, weight, labels)
    for name, t in (("weight", weight), ("labels", labels)):
        if t.device != hidden.device:
            raise ValueError(f"{name} must live on {hidden.device}, got {t.device}")
    (n, hdim), vocab, dev = hidden.shape, weight.shape[0], hidden.device
    hidden, weight, labels = hidden.contiguous(), weight.contiguous(), labels.contiguous()
    L = _lib.lib()
    logp = torch.empty(shape, dtype=torch.float32, device=dev)
    counts = torch.empty(2, dtype=torch.int64, device=dev)
    saved = torch.empty(L.siq_flp_saved_bytes(n, vocab), dtype=torch.uint8, device=dev) if keep else None
    ws = torch.empty(L.siq_flp_fwd_workspace_bytes(n, hdim, vocab, int(keep)), dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        rc = L.siq_flp_fwd(hidden.data_ptr(), weight.data_ptr(), labels.data_ptr(), n, hdim, vocab, int(ignore_index),
                           float(temperature), logp.data_ptr(), counts.data_ptr(), counts.data_ptr() + 8,
                           saved.data_ptr() if keep else None, saved.numel() if keep else 0, ws.data_ptr(), ws.numel(),
                           _lib.stream(dev))
    _lib.check(rc, "siq_flp_fwd")
    return logp, counts, saved


def flp_bwd(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, dlogp: torch.Tensor,
            ignore_index: int = IGNORE_INDEX, temperature: float = 1.0, saved: torch.Tensor | None = None,
            need_dhidden: bool = True, need_dweight: bool = True, chunk_tokens: int | None = None):
    """Raw backward: ``(dhidden | None, dweight | None)``; ``saved`` is the
    forward's on the same inputs, or None (the logits are formed again)."""
    _check_operands(hidden, weight, labels)
    (n, hdim), vocab, dev = hidden.shape, weight.shape[0], hidden.device
    if dlogp.shape != (n,) or dlogp.dtype != torch.float32:
        raise ValueError(f"dlogp must be float32 [{n}], got {dlogp.dtype} {tuple(dlogp.shape)}")
    for name, t in (("weight", weight), ("labels", labels), ("dlogp", dlogp)):
        if t.device != dev:
            raise ValueError(f"{name} must live on {dev}, got {t.device}")
    hidden, weight, labels, dlogp = (t.contiguous() for t in (hidden, weight, labels, dlogp))
    chunk = default_chunk_tokens(vocab) if chunk_tokens is None else int(chunk_tokens)
    if chunk <= 0:
        raise ValueError("chunk_tokens must be positive")
    L = _lib.lib()
    dh = torch.empty_like(hidden) if need_dhidden else None
    dw = torch.empty_like(weight) if need_dweight else None
    have = saved is not None
    ws = torch.empty(L.siq_flp_bwd_workspace_bytes(n, hdim, vocab, chunk, int(need_dweight), int(have)),
                     dtype=torch.uint8, device=dev)
    with _lib.on_device(dev):
        rc = L.siq_flp_bwd(hidden.data_ptr(), weight.data_ptr(), labels.data_ptr(), dlogp.data_ptr(), n, hdim, vocab,
                           int(ignore_index), float(temperature), saved.data_ptr() if have else None,
                           saved.numel() if have else 0, dh.data_ptr() if need_dhidden else None,
                           dw.data_ptr() if need_dweight else None, chunk, ws.data_ptr(), ws.numel(), _lib.stream(dev))
    _lib.check(rc, "siq_flp_bwd")
    return dh, dw


def _rows(hidden: torch.Tensor) -> torch.Tensor:
    return hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])


class _FusedLinearLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, temperature, chunk_tokens, keep_bytes, validate):
        h2, y = _rows(hidden), labels if labels.dim() == 1 else labels.reshape(-1)
        keep = _lib.lib().siq_flp_saved_bytes(h2.shape[0], weight.shape[0]) <= keep_bytes
        logp, counts, saved = _forward(h2, weight, y, ignore_index, temperature, keep, labels.shape)
        _track_bad(counts[1], weight.shape[0], ignore_index, validate)
        ctx.save_for_backward(hidden, weight, labels, *((saved,) if keep else ()))
        ctx.ignore_index, ctx.temperature, ctx.chunk_tokens = ignore_index, temperature, chunk_tokens
        return logp

    @staticmethod
    def backward(ctx, dlogp):
        _lib.first_order("fused_linear_log_probs")
        hidden, weight, labels, *saved = ctx.saved_tensors
        dh, dw = flp_bwd(_rows(hidden), weight, labels.reshape(-1), dlogp.reshape(-1),
                         ctx.ignore_index, ctx.temperature, saved[0] if saved else None, ctx.needs_input_grad[0],
                         ctx.needs_input_grad[1], ctx.chunk_tokens)
        return None if dh is None else dh.view(hidden.shape), dw, *(None,) * 6


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
    vocab bytes); a batch above it keeps nothing, and the backward forms the
    logits again, ``chunk_tokens`` rows at a time (None: 2 GiB of them).
    Without gradients nothing is kept.  A frozen ``weight`` gives the dH-only
    backward.
    """
    if labels.shape != hidden.shape[:-1]:
        raise ValueError(f"labels must be {tuple(hidden.shape[:-1])}, got {tuple(labels.shape)}")
    h = hidden if hidden.dtype == torch.bfloat16 else hidden.to(torch.bfloat16)
    w = weight if weight.dtype == torch.bfloat16 else weight.to(torch.bfloat16)
    if not torch.is_grad_enabled() or not (h.requires_grad or w.requires_grad):
        logp, counts, _ = _forward(_rows(h), w, labels.reshape(-1), int(ignore_index), temperature, False, labels.shape)
        _track_bad(counts[1], w.shape[0], int(ignore_index), validate)
        return logp
    return _FusedLinearLogProbs.apply(h, w, labels, int(ignore_index), float(temperature), chunk_tokens, int(keep_bytes),
                                      validate)


__all__ = ["DEFAULT_KEEP_BYTES", "flp_bwd", "flp_fwd", "fused_linear_log_probs"]
