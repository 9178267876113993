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


def _flat(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _align(n: int) -> int:
    return (n + 255) & ~255


def _stores(numel: int, count: int, device: torch.device) -> list[torch.Tensor]:
    """``count`` pairs of code and scale bytes for ``numel`` elements each, in one allocation."""
    groups = (numel + GROUP - 1) // GROUP
    step = _align(numel) + _align(groups)
    buf = torch.empty(step * count, dtype=torch.uint8, device=device)
    out = []
    for i in range(count):
        at = i * step
        out += [buf[at:at + numel], buf[at + _align(numel):at + _align(numel) + groups]]
    return out


def pack8(x: torch.Tensor, format: str = "int8") -> Packed8:
    """``x`` (bf16 or fp32, any shape) in 8 bits, in memory order."""
    fmt = _format(format)
    _check(x, "x")
    x = _flat(x.detach())
    codes, scales = _stores(x.numel(), 1, x.device)
    with _lib.on_device(x.device):
        rc = _lib.lib().siq_pack8(x.data_ptr(), x.numel(), _DTYPES[x.dtype], fmt, codes.data_ptr(), scales.data_ptr(),
                                  _lib.stream(x.device))
    _lib.check(rc, "siq_pack8")
    return Packed8(codes, scales, x.shape, x.dtype, format)


def unpack8(packed: Packed8, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The values that ``packed`` stands for (``dtype``: bf16 or fp32, the packed tensor's by default)."""
    fmt = _format(packed.format)
    dtype = packed.dtype if dtype is None else dtype
    numel = packed.shape.numel()
    if dtype not in _DTYPES:
        raise ValueError(f"dtype must be bfloat16 or float32, got {dtype}")
    for name, t, n in (("codes", packed.codes, numel), ("scales", packed.scales, (numel + GROUP - 1) // GROUP)):
        if t.dtype != torch.uint8 or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"{name} must be {n} contiguous uint8, got {tuple(t.shape)} {t.dtype}")
        if t.device.type != "cuda" or t.device != packed.codes.device:
            raise ValueError(f"codes and scales must live on one GPU, got {packed.codes.device} and {t.device}")
    x = torch.empty(packed.shape, dtype=dtype, device=packed.codes.device)
    with _lib.on_device(x.device):
        rc = _lib.lib().siq_unpack8(packed.codes.data_ptr(), packed.scales.data_ptr(), numel, _DTYPES[dtype], fmt,
                                    x.data_ptr(), _lib.stream(x.device))
    _lib.check(rc, "siq_unpack8")
    return x


# --------------------------------------------------------------------------- gated MLP activation
def _rows(t: torch.Tensor) -> torch.Tensor:
    """A [rows, cols] view of ``t`` that the kernels read in place, or a contiguous copy."""
    t = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    step = 4 if t.dtype == torch.float32 else 8
    if t.is_contiguous() or (t.stride(1) == 1 and t.stride(0) >= t.shape[1] and t.stride(0) % step == 0
                             and t.shape[1] % 8 == 0):
        return t.clone() if t.data_ptr() % 16 else t
    return t.contiguous()


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 and not t.is_contiguous() else t.shape[1]


def swiglu8_fwd(gate: torch.Tensor, up: torch.Tensor, format: str = "int8", keep: bool = True):
    """Raw forward on ``[..., cols]``: ``(h, stores)`` with ``stores`` the packed
    gate and up (codes, scales, codes, scales), or None without ``keep``."""
    fmt = _format(format)
    for name, t in (("gate", gate), ("up", up)):
        _check(t, name)
        if t.dim() == 0:
            raise ValueError(f"{name} must have at least one dimension")
    if gate.shape != up.shape or gate.dtype != up.dtype or gate.device != up.device:
        raise ValueError(f"gate and up must be alike, got {tuple(gate.shape)} {gate.dtype} on {gate.device} and "
                         f"{tuple(up.shape)} {up.dtype} on {up.device}")
    h = torch.empty(gate.shape, dtype=gate.dtype, device=gate.device)
    stores = _stores(h.numel(), 2, h.device) if keep else None
    if h.numel() == 0:
        return h, stores
    g, u = _rows(gate), _rows(up)
    ptrs = [s.data_ptr() for s in stores] if keep else [None] * 4
    with _lib.on_device(h.device):
        rc = _lib.lib().siq_swiglu8_fwd(g.data_ptr(), u.data_ptr(), g.shape[0], g.shape[1], _ld(g), _ld(u),
                                        _DTYPES[h.dtype], fmt, h.data_ptr(), *ptrs, _lib.stream(h.device))
    _lib.check(rc, "siq_swiglu8_fwd")
    return h, stores


def swiglu8_bwd(dh: torch.Tensor, stores, format: str = "int8", need_h: bool = False, fused: bool = False):
    """Raw backward: ``(dgate, dup, h | None)`` like ``dh``; with ``fused`` both
    gradients side by side in one tensor, ``(dgate_dup [..., 2 * cols], None, h | None)``."""
    fmt = _format(format)
    _check(dh, "dh")
    if dh.dim() == 0:
        raise ValueError("dh must have at least one dimension")
    numel, cols = dh.numel(), dh.shape[-1]
    groups = (numel + GROUP - 1) // GROUP
    for s, n in zip(stores, (numel, groups, numel, groups), strict=True):
        if s.dtype != torch.uint8 or s.numel() != n or not s.is_contiguous() or s.device != dh.device:
            raise ValueError(f"the packed gate and up do not belong to a gradient of shape {tuple(dh.shape)}")
    rows = numel // cols if cols else 0
    both = torch.empty(*dh.shape[:-1], 2 * cols, dtype=dh.dtype, device=dh.device) if fused else None
    # the halves are written in place where their rows start at 16-byte boundaries
    halves = fused and cols % 8 == 0
    if halves:
        dgate, dup, ld = both[..., :cols], both[..., cols:], 2 * cols
    else:
        dgate = torch.empty(dh.shape, dtype=dh.dtype, device=dh.device)
        dup, ld = torch.empty_like(dgate), cols
    h = torch.empty(dh.shape, dtype=dh.dtype, device=dh.device) if need_h else None
    if numel:
        dh = _flat(dh)
        with _lib.on_device(dh.device):
            rc = _lib.lib().siq_swiglu8_bwd(dh.data_ptr(), *(s.data_ptr() for s in stores), rows, cols, ld, ld,
                                            _DTYPES[dh.dtype], fmt, dgate.data_ptr(), dup.data_ptr(),
                                            None if h is None else h.data_ptr(), _lib.stream(dh.device))
        _lib.check(rc, "siq_swiglu8_bwd")
        if fused and not halves:
            both[..., :cols], both[..., cols:] = dgate, dup
    return (both, None, h) if fused else (dgate, dup, h)


class _Swiglu8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, fmt):
        h, stores = swiglu8_fwd(gate, up, fmt)
        ctx.save_for_backward(*stores)
        ctx.fmt = fmt
        return h

    @staticmethod
    def backward(ctx, dh):
        _lib.first_order("swiglu8")
        dgate, dup, _ = swiglu8_bwd(dh, ctx.saved_tensors, ctx.fmt)
        return dgate, dup, None


class _Swiglu8Fused(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate_up, fmt):
        cols = gate_up.shape[-1] // 2
        h, stores = swiglu8_fwd(gate_up[..., :cols], gate_up[..., cols:], fmt)
        ctx.save_for_backward(*stores)
        ctx.fmt = fmt
        return h

    @staticmethod
    def backward(ctx, dh):
        _lib.first_order("swiglu8")
        return swiglu8_bwd(dh, ctx.saved_tensors, ctx.fmt, fused=True)[0], None


def swiglu8(gate: torch.Tensor, up: torch.Tensor | None = None, format: str = "int8") -> torch.Tensor:
    """``silu(gate) * up`` that keeps gate and up in 8 bits for its backward.
    With ``up`` None, ``gate`` holds both side by side in its last dimension."""
    _format(format)
    if up is None:
        if gate.dim() == 0 or gate.shape[-1] % 2:
            raise ValueError(f"gate and up side by side need an even last dimension, got {tuple(gate.shape)}")
        if torch.is_grad_enabled() and gate.requires_grad:
            return _Swiglu8Fused.apply(gate, format)
        cols = gate.shape[-1] // 2
        return swiglu8_fwd(gate[..., :cols], gate[..., cols:], format, keep=False)[0]
    if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad):
        return _Swiglu8.apply(gate, up, format)
    return swiglu8_fwd(gate, up, format, keep=False)[0]


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
    with torch.autocast(gate.device.type, enabled=False):
        if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad or weight.requires_grad):
            return _Swiglu8Linear.apply(gate, up, weight, format)
        return torch.nn.functional.linear(swiglu8_fwd(gate, up, format, keep=False)[0], weight)


def checkpointed_qwen2_mlp_forward(self, x: torch.Tensor) -> torch.Tensor:
    """``Qwen2MLP.forward`` (``down_proj(act_fn(gate_proj(x)) * up_proj(x))``) on
    ``swiglu8``.  Projections that are not bf16 or fp32 on the GPU take the
    stock forward."""
    gate, up = self.gate_proj(x), self.up_proj(x)
    if not (gate.is_cuda and gate.dtype in _DTYPES and gate.dtype == up.dtype):
        return self.down_proj(self.act_fn(gate) * up)
    down = self.down_proj
    if type(down) is torch.nn.Linear and down.bias is None and down.weight.requires_grad:
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
def checkpoint8(function, x: torch.Tensor, *args, format: str = "int8", **kwargs):
    """``function(x, *args)``, run again in the backward as
    ``torch.utils.checkpoint.checkpoint(..., use_reentrant=False)`` does
    (``kwargs`` go there), with ``x`` kept in 8 bits instead of as it is.  The
    forward runs on ``x`` itself; what the backward recomputes, and so the
    gradients, are those at the unpacked ``x``."""
    _format(format)
    _check(x, "x")
    if not torch.is_grad_enabled():
        return function(x, *args)
    packed, first, trained = pack8(x, format), [x], x.requires_grad
    del x

    def run(*rest):
        # the forward takes x from the list, so that nothing here keeps it
        value = first.pop() if first else unpack8(packed).requires_grad_(trained)
        return function(value, *rest)

    return torch.utils.checkpoint.checkpoint(run, *args, use_reentrant=False, **kwargs)


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
