"""Activations kept in 8 bits for the backward pass, on MI355X: host side.

The reference trains with ``gradient_checkpointing=True``
(scripts/train.py:714): every decoder layer keeps its bf16 input and is run
again in the backward.  Here that input is kept in 8 bits, and the widest
activations of a layer that is not run again, the two inputs of its gated MLP
activation, are too:

* ``pack8`` / ``unpack8`` -- raw operators: 32 neighbours share one
  power-of-two step, codes are ``"int8"`` (steps of the group's largest
  magnitude / 64 .. 127) or ``"e4m3"`` (4 significant bits, for groups whose
  values span many orders); 1.03 bytes an element;
* ``checkpoint8(function, x, *args)`` -- runs ``function(x, *args)`` as
  ``torch.utils.checkpoint`` does, with ``x`` kept packed: the backward unpacks
  it and runs ``function`` again, so gradients are those at the unpacked ``x``;
* ``swiglu8(gate, up)`` -- ``silu(gate) * up`` as an autograd op that packs both
  inputs in the pass that reads them; its backward works on the unpacked values;
* ``swiglu8_linear(gate, up, weight)`` -- the down projection after it too,
  whose weight gradient takes the activation recomputed by that backward
  instead of a saved one;
* ``enable_8bit_checkpoints(model)`` / ``enable_8bit_mlp(model)`` -- install them
  on a transformers model (gradient checkpointing of every layer, or every
  Qwen2 MLP).

Forward results are the unpacked ones' exactly (nothing is rounded on the way
out); only what the backward reads is in 8 bits.
"""

from __future__ import annotations

import functools
import types
from typing import NamedTuple

import torch

from . import _lib

GROUP = 32
_FORMATS = {"int8": 0, "e4m3": 1}  # SIQ_FORMAT_*
_DTYPES = {torch.bfloat16: 0, torch.float32: 1}  # SIQ_DTYPE_*


class Packed8(NamedTuple):
    """An activation in 8 bits: ``codes`` uint8 [numel], ``scales`` uint8 [ceil(numel / 32)]."""

    codes: torch.Tensor
    scales: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype
    format: str

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def _format(fmt: str) -> int:
    if fmt not in _FORMATS:
        raise ValueError(f"format must be one of {sorted(_FORMATS)}, got {fmt!r}")
    return _FORMATS[fmt]


def _check(t: torch.Tensor, name: str) -> None:
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be bfloat16 or float32, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must live on the GPU, got {t.device}")


def pack8(x: torch.Tensor, format: str = "int8") -> Packed8:
    """``x`` (bf16 or fp32, any shape) in 8 bits, in memory order."""
    codes, scales = _lib.native().pack8(x, _format(format))
    return Packed8(codes, scales, x.shape, x.dtype, format)


def unpack8(packed: Packed8, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The values that ``packed`` stands for (``dtype``: bf16 or fp32, the packed tensor's by default)."""
    fmt = _format(packed.format)
    dtype = packed.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        raise ValueError(f"dtype must be bfloat16 or float32, got {dtype}")
    return _lib.native().unpack8(packed.codes, packed.scales, packed.shape, dtype == torch.float32, fmt)


# --------------------------------------------------------------------------- gated MLP activation
def swiglu8_fwd(gate: torch.Tensor, up: torch.Tensor, format: str = "int8", keep: bool = True):
    """Raw forward on ``[..., cols]``: ``(h, stores)`` with ``stores`` the packed
    gate and up (codes, scales, codes, scales), or None without ``keep``."""
    h, stores = _lib.native().swiglu8_fwd(gate, up, _format(format), keep)
    return h, stores if keep else None


def swiglu8_bwd(dh: torch.Tensor, stores, format: str = "int8", need_h: bool = False, fused: bool = False):
    """Raw backward: ``(dgate, dup, h | None)`` like ``dh``; with ``fused`` both
    gradients side by side in one tensor, ``(dgate_dup [..., 2 * cols], None, h | None)``."""
    return _lib.native().swiglu8_bwd(dh, stores, _format(format), need_h, fused)


def swiglu8(gate: torch.Tensor, up: torch.Tensor | None = None, format: str = "int8") -> torch.Tensor:
    """``silu(gate) * up`` that keeps gate and up in 8 bits for its backward.
    With ``up`` None, ``gate`` holds both side by side in its last dimension."""
    return _lib.native().swiglu8(gate, up, _format(format))


class _Swiglu8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, weight, fmt):
        h, stores = swiglu8_fwd(gate, up, fmt)
        ctx.save_for_backward(weight, *stores)
        ctx.fmt = fmt
        return torch.nn.functional.linear(h, weight)

    @staticmethod
    def backward(ctx, dy):
        _lib.first_order("swiglu8_linear")
        weight, *stores = ctx.saved_tensors
        need_in, need_w = any(ctx.needs_input_grad[:2]), ctx.needs_input_grad[2]
        dgate, dup, h = swiglu8_bwd(dy @ weight, stores, ctx.fmt, need_h=need_w)
        dw = dy.reshape(-1, dy.shape[-1]).T @ h.reshape(-1, h.shape[-1]) if need_w else None
        return (dgate, dup, dw, None) if need_in else (None, None, dw, None)


def swiglu8_linear(gate: torch.Tensor, up: torch.Tensor, weight: torch.Tensor, format: str = "int8") -> torch.Tensor:
    """``linear(silu(gate) * up, weight)`` that keeps gate and up in 8 bits and
    no activation in between: the weight's gradient takes the one recomputed
    from them."""
    if weight.dim() != 2 or weight.shape[1] != gate.shape[-1]:
        raise ValueError(f"weight must be [out, {gate.shape[-1]}], got {tuple(weight.shape)}")
    weight = weight.to(gate.dtype)
    _lib.native().no_tangent("swiglu8_linear", [gate, up, weight])
    with torch.autocast(gate.device.type, enabled=False):
        if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad or weight.requires_grad):
            return _Swiglu8Linear.apply(gate, up, weight, format)
        return torch.nn.functional.linear(swiglu8_fwd(gate, up, format, keep=False)[0], weight)


def _only_forward(mod: torch.nn.Module) -> bool:
    """Whether a call of ``mod`` is its class's forward and nothing else (no
    hooks, no forward of its own), so that what computes the same may take its place."""
    every = torch.nn.modules.module
    return not (mod._forward_pre_hooks or mod._forward_hooks or mod._backward_pre_hooks or mod._backward_hooks
                or every._global_forward_pre_hooks or every._global_forward_hooks
                or every._global_backward_pre_hooks or every._global_backward_hooks or "forward" in vars(mod))


def checkpointed_qwen2_mlp_forward(self, x: torch.Tensor) -> torch.Tensor:
    """``Qwen2MLP.forward`` (``down_proj(act_fn(gate_proj(x)) * up_proj(x))``) on
    ``swiglu8``.  Projections that are not bf16 or fp32 on the GPU, and an
    activation with hooks or a forward of its own, take the stock forward; a
    down projection that is more than a Linear's product is called as it is."""
    gate, up = self.gate_proj(x), self.up_proj(x)
    if not (gate.is_cuda and gate.dtype in _DTYPES and gate.dtype == up.dtype and _only_forward(self.act_fn)):
        return self.down_proj(self.act_fn(gate) * up)
    down = self.down_proj
    if type(down) is torch.nn.Linear and _only_forward(down) and down.bias is None and down.weight.requires_grad:
        return swiglu8_linear(gate, up, down.weight, self.siq_mlp_format)
    return down(swiglu8(gate, up, self.siq_mlp_format))


def enable_8bit_mlp(model: torch.nn.Module, format: str = "int8") -> int:
    """Installs ``checkpointed_qwen2_mlp_forward`` on every Qwen2 MLP of
    ``model`` whose activation is SiLU; returns the number of MLPs patched."""
    _format(format)
    from transformers.models.qwen2.modeling_qwen2 import Qwen2MLP

    n = 0
    for mod in model.modules():
        if isinstance(mod, Qwen2MLP) and mod.config.hidden_act in ("silu", "swish"):
            mod.siq_mlp_format = format
            mod.forward = types.MethodType(checkpointed_qwen2_mlp_forward, mod)
            n += 1
    return n


# --------------------------------------------------------------------------- checkpoints of whole functions
class _Unpacked(torch.autograd.Function):
    """The unpacked input as no leaf (``source`` requires grad), so that the function may change it in place where it
    may change the forward's.  Gradients flow through the forward's input, not through this one."""

    @staticmethod
    def forward(ctx, source, packed, strides):
        return _unpacked(packed, strides)

    @staticmethod
    def backward(ctx, grad):
        return None, None, None


def _unpacked(packed: Packed8, strides) -> torch.Tensor:
    """``unpack8(packed)`` with its dimensions in the order of ``strides`` in memory (None: as they are)."""
    x = unpack8(packed)
    return x if strides is None else torch.empty_strided(x.shape, strides, dtype=x.dtype, device=x.device).copy_(x)


def checkpoint8(function, x: torch.Tensor, *args, format: str = "int8", **kwargs):
    """``function(x, *args)``, run again in the backward as
    ``torch.utils.checkpoint.checkpoint(..., use_reentrant=False)`` does
    (``kwargs`` go there), with ``x`` kept in 8 bits instead of as it is.  The
    forward runs on ``x`` itself; what the backward recomputes, and so the
    gradients, are those at the unpacked ``x``, with the forward's random numbers.
    ``function`` may change ``x`` in place, and view it as its strides allow."""
    _format(format)
    _check(x, "x")
    if not torch.is_grad_enabled():
        return function(x, *args)
    packed, first, trained = pack8(x, format), [x], x.requires_grad
    # (a transposed input is recomputed as one: the function may view it as its strides allow)
    strides = None if x.is_contiguous() else torch.empty_like(x, device="meta").stride()
    # torch keeps the random state of the GPUs that its arguments' tensors are on: an empty one stands for x there
    there = x.new_empty(0)
    del x

    def run(there, *rest):
        # the forward takes x from the list, so that nothing here keeps it
        if first:
            value = first.pop()
        elif trained:
            value = _Unpacked.apply(there.detach().requires_grad_(), packed, strides)
        else:
            value = _unpacked(packed, strides)
        return function(value, *rest)

    return torch.utils.checkpoint.checkpoint(run, there, *args, use_reentrant=False, **kwargs)


def _layer_checkpoint(format: str, function, *args):
    if args and torch.is_tensor(args[0]) and args[0].is_cuda and args[0].dtype in _DTYPES:
        return checkpoint8(function, *args, format=format)
    return torch.utils.checkpoint.checkpoint(function, *args, use_reentrant=False)


def enable_8bit_checkpoints(model: torch.nn.Module, format: str = "int8") -> int:
    """Gradient checkpointing of every layer of a transformers model
    (``gradient_checkpointing_enable``) with the layers' inputs kept in 8 bits;
    returns the number of modules it holds for.  A ``Trainer`` with
    ``gradient_checkpointing=True`` enables the stock one at its start: leave that
    argument False and call this before."""
    _format(format)
    if not hasattr(model, "gradient_checkpointing_enable"):
        raise TypeError("expected a transformers model (gradient_checkpointing_enable)")
    model.gradient_checkpointing_enable(gradient_checkpointing_kwargs={"use_reentrant": False})
    func = functools.partial(_layer_checkpoint, format)
    n = 0
    for mod in model.modules():
        if getattr(mod, "gradient_checkpointing", False) and hasattr(mod, "_gradient_checkpointing_func"):
            mod._gradient_checkpointing_func = func
            n += 1
    return n


__all__ = [
    "Packed8",
    "checkpoint8",
    "checkpointed_qwen2_mlp_forward",
    "enable_8bit_checkpoints",
    "enable_8bit_mlp",
    "pack8",
    "swiglu8",
    "swiglu8_bwd",
    "swiglu8_fwd",
    "swiglu8_linear",
    "unpack8",
]
