"""Token statistics on the CPU: the oracle against differences, workspace sizes and every refusal."""

import numpy as np
import pytest
import torch

from oracle import token_stats as ots
from siq_vl_amd import _lib
from siq_vl_amd import log_probs as LP

FAKE = 1 << 20
OK, INVALID, UNSUPPORTED, WS, ALIGN = (_lib.SIQ_OK, _lib.SIQ_ERR_INVALID_ARGUMENT, _lib.SIQ_ERR_UNSUPPORTED,
                                       _lib.SIQ_ERR_WORKSPACE, _lib.SIQ_ERR_ALIGNMENT)


@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_oracle_against_torch_and_differences(temperature):
    rng = np.random.default_rng(0)
    h, w = rng.standard_normal((6, 5)), rng.standard_normal((9, 5))
    w[7] = w[2]  # equal logits
    y = np.array([3, -100, 0, 8, 3, 2])
    g, e = rng.standard_normal(6), rng.standard_normal(6)
    out = ots.linear_token_stats(h, w, y, 9, g, e, temperature)
    at = y >= 0
    lp = torch.log_softmax(torch.tensor(h) @ torch.tensor(w).T / temperature, 1)
    assert np.allclose(out["logp"][at], lp[torch.tensor(at), torch.tensor(y[at])], atol=1e-12)
    assert np.allclose(out["entropy"][at], torch.distributions.Categorical(logits=lp).entropy()[torch.tensor(at)], atol=1e-12)
    assert (out["logp"][1] == 0) and (out["entropy"][1] == 0) and (out["top_ids"][1] == -1).all()
    got = np.take_along_axis(lp.numpy()[at], out["top_ids"][at], 1)
    assert np.allclose(got, out["top_logp"][at], atol=1e-12) and (np.diff(got) <= 1e-12).all()
    place = np.argsort(out["top_ids"][at], 1)
    assert (place[:, 2] + 1 == place[:, 7]).all()  # the lower id first

    def f(h, w):
        o = ots.linear_token_stats(h, w, y, temperature=temperature)
        return float(o["logp"] @ g + o["entropy"] @ e)

    for name, x in (("dh", h), ("dw", w)):
        num = np.empty_like(x)
        for i in np.ndindex(x.shape):
            old = x[i]
            x[i] = old + 1e-6
            up = f(h, w)
            x[i] = old - 1e-6
            num[i] = (up - f(h, w)) / 2e-6
            x[i] = old
        assert np.allclose(out[name], num, atol=1e-8)
    assert (out["dh"][1] == 0).all()


def _fwd(lib, **kw):
    a = dict(h=FAKE, w=FAKE, y=FAKE, n=300, hdim=256, vocab=1000, ign=-100, t=1.0, k=5, lp=FAKE, ent=FAKE, state=FAKE, tl=FAKE,
             ti=FAKE, count=FAKE, bad=FAKE, saved=None, sb=0, ws=FAKE)
    a.update(kw)
    a.setdefault("wb", lib.siq_stats_fwd_workspace_bytes(300, 256, 1000, 5, int(a["saved"] is not None)))
    return lib.siq_stats_fwd(*(a[k] for k in ("h", "w", "y", "n", "hdim", "vocab", "ign", "t", "k", "lp", "ent", "state", "tl",
                                              "ti", "count", "bad", "saved", "sb", "ws", "wb")), None)


def _bwd(lib, **kw):
    a = dict(h=FAKE, w=FAKE, y=FAKE, state=FAKE, g=FAKE, e=FAKE, n=300, hdim=256, vocab=1000, ign=-100, t=1.0,
             saved=None, sb=0, dh=FAKE + (1 << 24), dw=FAKE, chunk=128, ws=FAKE)
    a.update(kw)
    a.setdefault("wb", lib.siq_stats_bwd_workspace_bytes(300, 256, 1000, 128, int(a["dw"] is not None),
                                                         int(a["saved"] is not None)))
    return lib.siq_stats_bwd(*(a[k] for k in ("h", "w", "y", "state", "g", "e", "n", "hdim", "vocab", "ign", "t",
                                              "saved", "sb", "dh", "dw", "chunk", "ws", "wb")), None)


@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), INVALID), (dict(n=2 ** 31), INVALID), (dict(hdim=0), INVALID), (dict(hdim=100), UNSUPPORTED),
    (dict(vocab=1001), UNSUPPORTED), (dict(vocab=2 ** 23), INVALID), (dict(h=None), INVALID), (dict(h=FAKE + 8), ALIGN),
    (dict(w=None), INVALID), (dict(w=FAKE + 2), ALIGN), (dict(y=None), INVALID), (dict(t=0.0), INVALID),
    (dict(t=float("nan")), INVALID), (dict(t=1e-45), INVALID), (dict(saved=FAKE, sb=100), WS), (dict(saved=FAKE + 8, sb=1 << 30), WS), (dict(ws=None), WS),
    (dict(wb=64), WS),
])
def test_validation_of_both_directions(lib, kw, code):
    assert _fwd(lib, **kw) == code
    assert _bwd(lib, **kw) == code


def test_validation_of_one_direction(lib):
    for kw in (dict(k=-1), dict(k=129), dict(k=9, vocab=8), dict(tl=None), dict(ti=None), dict(count=None), dict(bad=None),
               dict(lp=None), dict(ent=None)):
        assert _fwd(lib, wb=1 << 40, **kw) == INVALID
    assert _fwd(lib, k=129) == INVALID and "top_k must be in [0, 128]" in lib.siq_last_error().decode()
    assert _bwd(lib, chunk=0, wb=1 << 40) == INVALID and _bwd(lib, state=None) == INVALID
    assert _bwd(lib, dh=FAKE + 8) == ALIGN and _bwd(lib, dw=FAKE + 8) == ALIGN
    assert _bwd(lib, dh=FAKE) == INVALID and _bwd(lib, dh=FAKE + 1024) == INVALID  # over hidden
    assert _bwd(lib, dh=None, dw=None) == OK  # nothing to do


def test_workspace_sizes(lib):
    n, h, v = 16384, 1536, 151936
    saved = lib.siq_stats_saved_bytes(n, v)
    assert 2 * n * v < saved < 2.2 * n * v
    # scores alone hold sums of parts of rows, alternatives at most 2 GiB of logits besides
    none, some = (lib.siq_stats_fwd_workspace_bytes(n, h, v, k, 0) for k in (0, 20))
    assert none < 512 << 20 and some < (2 << 30) + (512 << 20)
    chunk = 6912
    assert lib.siq_stats_bwd_workspace_bytes(n, h, v, chunk, 0, 0) > 2 * chunk * v
    assert lib.siq_stats_bwd_workspace_bytes(n, h, v, chunk, 1, 1) < 5 << 30
    for f in (lambda *a: lib.siq_stats_fwd_workspace_bytes(*a, 5, 0), lambda *a: lib.siq_stats_bwd_workspace_bytes(*a, 64, 1, 0)):
        assert f(-1, 64, 8) == 0 and f(0, 64, 8) > 0 and f(5, 0, 8) == 0
    assert lib.siq_stats_fwd_workspace_bytes(5, 64, 8, 129, 0) == 0 and lib.siq_stats_saved_bytes(-1, 8) == 0


def test_python_refusals():
    h, w, y = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16), torch.zeros(4).long()
    with pytest.raises(ValueError, match="GPU"):
        LP.fused_linear_token_stats(h, w, y)
    with pytest.raises(ValueError, match="GPU"):
        LP.fused_linear_token_stats(h, w)
    with pytest.raises(ValueError, match=r"labels must be \(4,\)"):
        LP.fused_linear_token_stats(h, w, y[:3])
    with pytest.raises(ValueError, match="hdim"):
        LP.fused_linear_token_stats(h, w[:, :32], y)
    with pytest.raises(ValueError, match="chunk_tokens"):
        LP.fused_linear_token_stats(h, w, y, chunk_tokens=0)
