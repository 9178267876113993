"""8-bit storage of activations on the CPU: the oracle against its definition, and every refusal."""

import numpy as np
import pytest
import torch

from oracle import pack8 as op
from siq_vl_amd import _lib
from siq_vl_amd import checkpoint8 as K

FAKE = 1 << 20
OK, INVALID, UNSUPPORTED, ALIGN = (_lib.SIQ_OK, _lib.SIQ_ERR_INVALID_ARGUMENT, _lib.SIQ_ERR_UNSUPPORTED,
                                   _lib.SIQ_ERR_ALIGNMENT)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("scale", [1.0, 1e-30, 3e30])
def test_oracle_rounds_by_half_a_step(fmt, scale):
    x = scale * np.random.default_rng(0).standard_normal(32 * 40 + 7)
    codes, scales = op.encode(x, fmt)
    y = op.decode(codes, scales, fmt)
    step = 2.0 ** (np.repeat(scales.astype(int), 32)[:x.size] - (133 if fmt == "int8" else 135))
    if fmt == "int8":
        assert (np.abs(x - y) <= step / 2).all()
        assert np.abs(codes.view(np.int8).astype(int)).max() >= 64  # the range is used
    else:  # half a unit of the last of 4 significant bits, and of the smallest number
        assert (np.abs(x - y) <= np.maximum(np.abs(x) * 2.0 ** -4, step * 2.0 ** -10)).all()
    # packing what was unpacked changes nothing
    assert np.array_equal(op.rounded(y, fmt), y)


def test_oracle_e4m3_is_torchs():
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(op.E4M3, table, equal_nan=True)
    x = np.random.default_rng(1).uniform(-448, 448, 4096)
    x[:32] = 448.0  # the first group's step is 1
    t = torch.tensor(x[:32 * 128], dtype=torch.float32)
    groups = t.view(-1, 32)
    for i in (0, 5, 127):
        c, s = op.encode(groups[i].double().numpy(), "e4m3")
        step = 2.0 ** (int(s[0]) - 135)
        want = (groups[i] / step).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        assert np.array_equal(c, want)


def test_oracle_swiglu_gradients_are_differences():
    rng = np.random.default_rng(2)
    g, u, dh = rng.standard_normal((3, 50)) * 3
    dg, du = op.swiglu_bwd(dh, g, u)
    eps = 1e-6
    # central differences: truncation ~ eps^2, rounding ~ 1e-16 / eps
    assert np.allclose(dg, dh * (op.swiglu(g + eps, u) - op.swiglu(g - eps, u)) / (2 * eps), atol=1e-8)
    assert np.allclose(du, dh * (op.swiglu(g, u + eps) - op.swiglu(g, u - eps)) / (2 * eps), atol=1e-8)


def test_pack_validation(lib):
    def pack(x=FAKE, n=64, dtype=0, fmt=0, codes=FAKE, scales=FAKE):
        return lib.siq_pack8(x, n, dtype, fmt, codes, scales, None), lib.siq_unpack8(codes, scales, n, dtype, fmt, x, None)

    assert pack(n=0, x=None, codes=None, scales=None) == (OK, OK)
    assert pack(n=-1) == (INVALID, INVALID)
    assert pack(n=2 ** 35 + 1) == (INVALID, INVALID)
    assert pack(dtype=2) == (INVALID, INVALID)
    assert pack(fmt=2) == (INVALID, INVALID)
    assert pack(x=None) == (INVALID, INVALID)
    assert pack(scales=None) == (INVALID, INVALID)
    assert pack(x=FAKE + 8) == (ALIGN, ALIGN)
    assert pack(codes=FAKE + 1) == (ALIGN, ALIGN)


def test_swiglu_validation(lib):
    def fwd(rows=4, cols=64, gs=64, us=64, dtype=0, fmt=0, gate=FAKE, h=FAKE, keep=(FAKE,) * 4):
        return lib.siq_swiglu8_fwd(gate, FAKE, rows, cols, gs, us, dtype, fmt, h, *keep, None)

    def bwd(rows=4, cols=64, gs=64, us=64, dtype=0, fmt=0, dh=FAKE, dgate=FAKE, h=None, keep=(FAKE,) * 4):
        return lib.siq_swiglu8_bwd(dh, *keep, rows, cols, gs, us, dtype, fmt, dgate, FAKE, h, None)

    for f in (fwd, bwd):
        assert f(rows=0) == OK and f(cols=0, gs=0, us=0) == OK
        assert f(rows=-1) == INVALID and f(cols=-1) == INVALID
        assert f(rows=2 ** 33, cols=64) == INVALID
        assert f(dtype=3) == INVALID and f(fmt=-1) == INVALID
        assert f(gs=63) == ALIGN          # rows would overlap
        assert f(gs=68) == ALIGN          # not a multiple of 8 bf16
        assert f(gs=66, dtype=1) == ALIGN
        assert f(cols=60, gs=64, us=64) == UNSUPPORTED
    assert fwd(gate=None) == INVALID and fwd(h=None) == INVALID and fwd(gate=FAKE + 2) == ALIGN
    assert fwd(keep=(FAKE, FAKE, None, FAKE)) == INVALID
    assert fwd(keep=(None, None, None, FAKE)) == INVALID
    assert bwd(dh=None) == INVALID and bwd(dgate=None) == INVALID and bwd(h=FAKE + 4) == ALIGN
    assert bwd(keep=(None, FAKE, FAKE, FAKE)) == INVALID


def test_python_refusals():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="GPU"):
        K.pack8(x)
    with pytest.raises(ValueError, match="float16"):
        K.pack8(x.half())
    with pytest.raises(ValueError, match="format"):
        K.pack8(x, "int4")
    with pytest.raises(ValueError, match="format"):
        K.swiglu8(x, x, "fp8")
    with pytest.raises(ValueError, match="GPU"):
        K.swiglu8(x, x)
    with pytest.raises(ValueError, match="even last dimension"):
        K.swiglu8(torch.zeros(3, 5))
    with pytest.raises(ValueError, match=r"weight must be \[out, 64\]"):
        K.swiglu8_linear(x, x, torch.zeros(8, 32))
    with pytest.raises(ValueError, match="GPU"):
        K.checkpoint8(lambda t: t, x)
    codes, scales = torch.zeros(64, dtype=torch.uint8), torch.zeros(2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="codes must be 65"):
        K.unpack8(K.Packed8(codes, scales, torch.Size([65]), torch.float32, "int8"))
    with pytest.raises(ValueError, match="GPU"):
        K.unpack8(K.Packed8(codes, scales, torch.Size([64]), torch.float32, "int8"))
    with pytest.raises(ValueError, match="dtype"):
        K.unpack8(K.Packed8(codes, scales, torch.Size([64]), torch.float16, "int8"))
    with pytest.raises(TypeError, match="transformers"):
        K.enable_8bit_checkpoints(torch.nn.Linear(2, 2))
    assert K.enable_8bit_mlp(torch.nn.Linear(2, 2)) == 0
    with pytest.raises(ValueError, match="format"):
        K.enable_8bit_mlp(torch.nn.Linear(2, 2), "int4")


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_seen_where_they_are(grad):
    fw, native = torch.autograd.forward_ad, _lib.native()
    x, y = torch.ones(2, 3), torch.ones(3)
    with torch.set_grad_enabled(grad):
        native.no_tangent("an operator", [x, y])
        with fw.dual_level():
            native.no_tangent("an operator", [x, y])
            d = fw.make_dual(y, y)
            for args in ([x, d], [d], [d * 2, x]):
                with pytest.raises(NotImplementedError, match="an operator has no forward-mode derivative"):
                    native.no_tangent("an operator", args)
            native.no_tangent("an operator", [fw.unpack_dual(d).primal, x])
        native.no_tangent("an operator", [y])


def test_modules_that_are_more_than_their_forward():
    def plain():
        return torch.nn.Linear(2, 2)

    assert K._only_forward(plain())
    for register in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook",
                     "register_full_backward_pre_hook"):
        mod = plain()
        handle = getattr(mod, register)(lambda *a: None)
        assert not K._only_forward(mod)
        handle.remove()
        assert K._only_forward(mod)
    for register in ("register_module_forward_hook", "register_module_forward_pre_hook",
                     "register_module_full_backward_hook", "register_module_full_backward_pre_hook"):
        handle = getattr(torch.nn.modules.module, register)(lambda *a: None)
        try:
            assert not K._only_forward(plain())
        finally:
            handle.remove()
    mod = plain()
    mod.forward = lambda x: x
    assert not K._only_forward(mod)
