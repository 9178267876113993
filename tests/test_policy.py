"""Preference and policy losses on the CPU: the oracle against differences, and every refusal."""

import warnings

import numpy as np
import pytest
import torch

from oracle import policy as op
from siq_vl_amd import _lib
from siq_vl_amd import policy as P

FAKE = 1 << 20
OK, INVALID, UNSUPPORTED, WS, ALIGN = (_lib.SIQ_OK, _lib.SIQ_ERR_INVALID_ARGUMENT, _lib.SIQ_ERR_UNSUPPORTED,
                                       _lib.SIQ_ERR_WORKSPACE, _lib.SIQ_ERR_ALIGNMENT)


def differences(f, x, eps=1e-6):
    out = np.empty_like(x)
    for i in range(x.size):
        a, b = x.copy(), x.copy()
        a[i] += eps
        b[i] -= eps
        out[i] = (f(a) - f(b)) / (2 * eps)
    return out


@pytest.mark.parametrize("kw", [dict(), dict(smoothing=0.2), dict(loss_type="ipo", normalized=True),
                                dict(loss_type="hinge", order="halves"), dict(items=7.0, normalized=True)])
def test_oracle_preference_gradient_is_a_difference(kw):
    rng = np.random.default_rng(0)
    cu = [0, 5, 9, 9, 20]
    pi, ref, mask = -rng.random(20), -rng.random(20), rng.random(20) < 0.7
    grad = op.preference(pi, ref, cu, mask, **kw)[3]
    num = differences(lambda v: op.preference(v, ref, cu, mask, **kw)[0], pi)
    assert np.allclose(grad, num, atol=1e-8)


@pytest.mark.parametrize("kw", [dict(), dict(kl_coef=0.3), dict(kl_coef=0.3, kl_type="k1", aggregation="sequence"),
                                dict(kl_coef=0.1, kl_type="k2", dual=1.5, items=3.0), dict(high=0.4, low=0.1)])
@pytest.mark.parametrize("per_token", [True, False])
def test_oracle_policy_gradient_is_a_difference(kw, per_token):
    rng = np.random.default_rng(1)
    cu = [0, 5, 9, 9, 20]
    old = -rng.random(20)
    lp, ref, mask = old + 0.5 * rng.standard_normal(20), old + 0.3 * rng.standard_normal(20), rng.random(20) < 0.7
    adv = rng.standard_normal(20 if per_token else 4)
    args = dict(cu=cu, mask=mask, reference=ref, **kw)
    loss, kl, cut, grad = op.policy(lp, old, adv, **args)
    assert 0 <= cut <= 1 and (kw.get("kl_type") == "k1" or kl >= 0)
    assert np.allclose(grad, differences(lambda v: op.policy(v, old, adv, **args)[0], lp), atol=1e-8)


def _pref(lib, **kw):
    a = dict(policy=FAKE, ref=FAKE, mask=FAKE, cu=FAKE, pairs=3, tokens=100, kind=0, order=0, beta=0.1, smooth=0.0, norm=0,
             div=None, loss=FAKE, c=FAKE, r=FAKE, coef=FAKE, ws=FAKE, bytes=lib.siq_pref_workspace_bytes(3, 100))
    a.update(kw)
    return lib.siq_pref_fwd(*(a[k] for k in ("policy", "ref", "mask", "cu", "pairs", "tokens", "kind", "order", "beta",
                                             "smooth", "norm", "div", "loss", "c", "r", "coef", "ws", "bytes")), None)


@pytest.mark.parametrize("kw,code", [
    (dict(pairs=0), INVALID), (dict(pairs=2 ** 23 + 1), INVALID), (dict(tokens=-1), INVALID), (dict(tokens=2 ** 31), INVALID),
    (dict(kind=3), INVALID), (dict(order=2), INVALID), (dict(beta=0.0), INVALID), (dict(beta=float("nan")), INVALID),
    (dict(beta=float("inf")), INVALID), (dict(smooth=0.6), INVALID), (dict(smooth=-0.1), INVALID),
    (dict(smooth=0.1, kind=1), UNSUPPORTED), (dict(cu=None), INVALID), (dict(loss=None), INVALID), (dict(c=None), INVALID),
    (dict(coef=None), INVALID), (dict(policy=None), INVALID), (dict(ws=None), WS), (dict(bytes=16), WS),
    (dict(ws=FAKE + 8), WS),
])
def test_preference_validation(lib, kw, code):
    assert _pref(lib, **kw) == code


def _policy(lib, **kw):
    a = dict(lp=FAKE, old=FAKE, adv=FAKE, mask=FAKE, ref=FAKE, cu=FAKE, seqs=3, tokens=100, per=0, agg=0, kl=2, low=0.2,
             high=0.2, dual=0.0, coef=0.1, div=None, loss=FAKE, mean=FAKE, frac=FAKE, dtoken=FAKE, weight=FAKE, ws=FAKE,
             bytes=lib.siq_policy_workspace_bytes(3, 100))
    a.update(kw)
    return lib.siq_policy_fwd(*(a[k] for k in ("lp", "old", "adv", "mask", "ref", "cu", "seqs", "tokens", "per", "agg", "kl",
                                               "low", "high", "dual", "coef", "div", "loss", "mean", "frac", "dtoken", "weight", "ws",
                                               "bytes")), None)


@pytest.mark.parametrize("kw,code", [
    (dict(seqs=0), INVALID), (dict(seqs=2 ** 24 + 1), INVALID), (dict(tokens=-1), INVALID), (dict(agg=2), INVALID),
    (dict(kl=3), INVALID), (dict(kl=-1), INVALID), (dict(low=1.5), INVALID), (dict(low=-0.1), INVALID),
    (dict(high=-0.1), INVALID), (dict(high=float("nan")), INVALID), (dict(dual=1.0), INVALID), (dict(dual=0.5), INVALID),
    (dict(coef=float("nan")), INVALID), (dict(ref=None), INVALID), (dict(cu=None), INVALID), (dict(loss=None), INVALID), (dict(mean=None), INVALID), (dict(frac=None), INVALID),
    (dict(weight=None), INVALID), (dict(lp=None), INVALID), (dict(adv=None), INVALID), (dict(dtoken=None), INVALID),
    (dict(dtoken=FAKE + 4), ALIGN), (dict(bytes=0), WS),
])
def test_policy_validation(lib, kw, code):
    assert _policy(lib, **kw) == code


def test_backward_validation(lib):
    f, g = lib.siq_pref_bwd, lib.siq_policy_bwd
    assert f(None, None, None, None, 3, 0, None, None) == OK and g(None, None, None, None, 1, 0, 0, None, None) == OK
    assert f(None, FAKE, None, FAKE, 3, 10, FAKE, None) == INVALID
    assert f(FAKE, FAKE, None, FAKE, 0, 10, FAKE, None) == INVALID
    assert f(FAKE, FAKE, None, None, 3, 10, FAKE, None) == INVALID
    assert g(FAKE, FAKE, FAKE, None, 2, 10, 0, FAKE, None) == INVALID
    assert g(FAKE, FAKE, FAKE, FAKE, 2, 10, 5, FAKE, None) == INVALID
    assert g(FAKE, FAKE, FAKE, FAKE, 2, 10, 1, FAKE + 4, None) == ALIGN
    assert lib.siq_pref_workspace_bytes(0, 10) == 0 and lib.siq_policy_workspace_bytes(1, -1) == 0
    assert lib.siq_pref_workspace_bytes(2 ** 23, 2 ** 31 - 1) > 0


def test_python_refusals():
    lp, cu = torch.zeros(10), torch.tensor([0, 5, 10], dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        P.preference_loss(lp, lp, cu)
    with pytest.raises(ValueError, match="float32"):
        P.preference_loss(lp.double(), lp, cu)
    with pytest.raises(ValueError, match="loss_type"):
        P.preference_loss(lp, lp, cu, loss_type="other")
    with pytest.raises(ValueError, match="order"):
        P.preference_loss(lp, lp, cu, order="random")
    with pytest.raises(ValueError, match="aggregation"):
        P.policy_loss(lp, lp, lp, aggregation="mean")
    with pytest.raises(ValueError, match="kl_type"):
        P.policy_loss(lp, lp, lp, kl_type="k4")
    with pytest.raises(ValueError, match="GPU"):
        P.policy_loss(lp, lp, lp)


def test_missing_extension_fails_loudly(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_NATIVE", None)
    monkeypatch.setattr(_lib._build, "NATIVE_PATH", tmp_path / "absent.so")
    with pytest.raises(RuntimeError, match="build"):
        _lib.native()


def test_the_extension_calls_entries_of_the_library():
    native = _lib.native()
    assert set(native.entries()) <= set(_lib.EXPORTED)
    with pytest.raises(IndexError):  # refused at the first entry without an address: what is bound stays
        native.bind({})


def test_errors_come_from_the_extension_as_python_errors():
    x = torch.zeros(3, 4)
    with pytest.raises(ValueError, match="policy_logps must be float32, got torch.float16"):
        P.preference_loss(x.half(), None, x)
    with pytest.raises(TypeError):
        P.policy_loss(x, None, x)


@pytest.mark.parametrize("value", [7, 7.0, 0, torch.tensor(7), torch.tensor([7.0]), torch.tensor(7.0, requires_grad=True),
                                   2 ** 24 + 1, torch.tensor(2 ** 24 + 1)])
def test_numbers_become_fp32_scalars(value):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        t = _lib.scalar_on(torch.device("cpu"), value)
    assert t.shape == () and t.dtype == torch.float32 and not t.requires_grad
    assert t.item() == np.float32(value.item() if torch.is_tensor(value) else value)
