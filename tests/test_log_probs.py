"""Log-probabilities of labels on the CPU: the oracle against differences, workspace sizes and every refusal."""

import numpy as np
import pytest
import torch

from oracle import log_probs as olp
from siq_vl_amd import _lib
from siq_vl_amd import log_probs as LP

FAKE = 1 << 20
OK, INVALID, UNSUPPORTED, WS, ALIGN = (_lib.SIQ_OK, _lib.SIQ_ERR_INVALID_ARGUMENT, _lib.SIQ_ERR_UNSUPPORTED,
                                       _lib.SIQ_ERR_WORKSPACE, _lib.SIQ_ERR_ALIGNMENT)


@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_oracle_gradients_are_differences(temperature):
    rng = np.random.default_rng(0)
    h, w, g = rng.standard_normal((5, 6)), rng.standard_normal((7, 6)), rng.standard_normal(5)
    y = np.array([3, -100, 0, 6, 3])

    def f(h, w):
        return float(olp.linear_log_probs(h, w, y, temperature=temperature)["logp"] @ g)

    out = olp.linear_log_probs(h, w, y, g, temperature)
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
    assert (out["dh"][1] == 0).all() and out["logp"][1] == 0 and out["count"] == 4
    z = torch.tensor(h) @ torch.tensor(w).T / temperature
    want = torch.log_softmax(z, 1)[torch.arange(5), torch.tensor(y).clamp(min=0)].numpy()
    assert np.allclose(out["logp"], np.where(y >= 0, want, 0), atol=1e-12)


def _fwd(lib, **kw):
    a = dict(h=FAKE, w=FAKE, y=FAKE, n=300, hdim=256, vocab=1000, ign=-100, t=1.0, lp=FAKE, count=FAKE, bad=FAKE,
             saved=None, sb=0, ws=FAKE)
    a.update(kw)
    a.setdefault("wb", lib.siq_flp_fwd_workspace_bytes(300, 256, 1000, int(a["saved"] is not None)))
    return lib.siq_flp_fwd(*(a[k] for k in ("h", "w", "y", "n", "hdim", "vocab", "ign", "t", "lp", "count", "bad", "saved",
                                            "sb", "ws", "wb")), None)


def _bwd(lib, **kw):
    a = dict(h=FAKE, w=FAKE, y=FAKE, g=FAKE, n=300, hdim=256, vocab=1000, ign=-100, t=1.0, saved=None, sb=0,
             dh=FAKE + (1 << 24), dw=FAKE, chunk=128, ws=FAKE)
    a.update(kw)
    a.setdefault("wb", lib.siq_flp_bwd_workspace_bytes(300, 256, 1000, 128, int(a["dw"] is not None),
                                                       int(a["saved"] is not None)))
    return lib.siq_flp_bwd(*(a[k] for k in ("h", "w", "y", "g", "n", "hdim", "vocab", "ign", "t", "saved", "sb", "dh", "dw",
                                            "chunk", "ws", "wb")), None)


@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), INVALID), (dict(n=2 ** 31), INVALID), (dict(hdim=0), INVALID), (dict(hdim=100), UNSUPPORTED),
    (dict(vocab=1001), UNSUPPORTED), (dict(vocab=2 ** 23), INVALID), (dict(h=None), INVALID), (dict(h=FAKE + 8), ALIGN),
    (dict(w=None), INVALID), (dict(w=FAKE + 2), ALIGN), (dict(y=None), INVALID), (dict(t=0.0), INVALID),
    (dict(t=-1.0), INVALID), (dict(t=float("inf")), INVALID), (dict(t=float("nan")), INVALID), (dict(t=1e-45), INVALID),
    (dict(saved=FAKE, sb=100), WS), (dict(saved=FAKE + 8, sb=1 << 30), WS), (dict(ws=None), WS), (dict(wb=64), WS),
])
def test_validation_of_both_directions(lib, kw, code):
    assert _fwd(lib, **kw) == code
    assert _bwd(lib, **kw) == code


def test_validation_of_one_direction(lib):
    assert _fwd(lib, lp=None) == INVALID and _fwd(lib, count=None) == INVALID and _fwd(lib, bad=None) == INVALID
    assert _bwd(lib, g=None) == INVALID and _bwd(lib, chunk=0, wb=1 << 40) == INVALID
    assert _bwd(lib, dh=FAKE + 8) == ALIGN and _bwd(lib, dw=FAKE + 8) == ALIGN
    assert _bwd(lib, dh=FAKE) == INVALID and _bwd(lib, dh=FAKE + 1024) == INVALID  # over hidden
    assert _bwd(lib, dh=None, dw=None) == OK  # nothing to do


def test_workspace_sizes(lib):
    n, h, v = 16384, 1536, 151936
    saved = lib.siq_flp_saved_bytes(n, v)
    assert 2 * n * v < saved < 2 * n * v + (1 << 20)
    # a forward that keeps nothing, or its numerators elsewhere, needs no logits-sized buffer
    assert lib.siq_flp_fwd_workspace_bytes(n, h, v, 0) < 300 << 20
    assert lib.siq_flp_fwd_workspace_bytes(n, h, v, 1) < 300 << 20
    # the backward holds one chunk of them, or none
    chunk = 6912
    assert lib.siq_flp_bwd_workspace_bytes(n, h, v, chunk, 0, 0) > 2 * chunk * v
    assert lib.siq_flp_bwd_workspace_bytes(n, h, v, chunk, 1, 1) < 2 << 30
    for f in (lambda *a: lib.siq_flp_fwd_workspace_bytes(*a, 0), lambda *a: lib.siq_flp_bwd_workspace_bytes(*a, 64, 1, 0)):
        assert f(-1, 64, 8) == 0 and f(0, 64, 8) > 0 and f(5, 0, 8) == 0


def test_python_refusals():
    h, w, y = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16), torch.zeros(4).long()
    with pytest.raises(ValueError, match="GPU"):
        LP.fused_linear_log_probs(h, w, y)
    with pytest.raises(ValueError, match=r"labels must be \(4,\)"):
        LP.fused_linear_log_probs(h, w, y[:3])
    with pytest.raises(ValueError, match="hdim"):
        LP.fused_linear_log_probs(h, w[:, :32], y)
    with pytest.raises(ValueError, match="bfloat16"):
        LP.flp_bwd(h.float(), w, y, torch.zeros(4))


def test_log_probs_of_a_model_need_labels_and_the_gpu():
    transformers = pytest.importorskip("transformers")
    from siq_vl_amd.text_model import enable_fused_cross_entropy

    cfg = transformers.Qwen2Config(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=1,
                                   num_attention_heads=2, num_key_value_heads=1, use_cache=False)
    model = transformers.Qwen2ForCausalLM(cfg)
    enable_fused_cross_entropy(model)
    ids = torch.randint(0, 64, (1, 5))
    with pytest.raises(ValueError, match="return_log_probs needs labels"):
        model(input_ids=ids, return_log_probs=True)
    with pytest.raises(ValueError, match="GPU"):
        model(input_ids=ids, labels=ids, return_log_probs=True)
    assert model(input_ids=ids).logits.shape == (1, 5, 64)
