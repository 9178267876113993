"""Distillation on the CPU: the oracle against torch and differences, workspace sizes and every refusal."""

import numpy as np
import pytest
import torch

from oracle import distillation as od
from siq_vl_amd import _lib
from siq_vl_amd import distillation as D

FAKE = 1 << 20
OK, INVALID, UNSUPPORTED, WS, ALIGN = (_lib.SIQ_OK, _lib.SIQ_ERR_INVALID_ARGUMENT, _lib.SIQ_ERR_UNSUPPORTED,
                                       _lib.SIQ_ERR_WORKSPACE, _lib.SIQ_ERR_ALIGNMENT)


def problem(seed=0, n=5, hdim=4, vocab=9, k=3, mass=0.9):
    rng = np.random.default_rng(seed)
    h, w = rng.standard_normal((n, hdim)), rng.standard_normal((vocab, hdim))
    ids = np.stack([rng.permutation(vocab)[:k] for _ in range(n)])
    t = rng.random((n, k))
    lt = np.log(mass * t / t.sum(1, keepdims=True))
    y = rng.integers(0, vocab, n)
    y[0] = ids[0, 1]
    return h, w, y, ids, lt


@pytest.mark.parametrize("kw", [
    dict(), dict(tail=False), dict(ce_weight=0.3), dict(ce_weight=0.3, tail=False), dict(ce_weight=1.0), dict(temperature=1.7),
    dict(divergence="reverse"), dict(divergence="reverse", ce_weight=0.2), dict(divisor=11.0),
])
def test_oracle_gradients_are_differences(kw):
    h, w, y, ids, lt = problem()
    y[2] = -100
    ids[1, 2], lt[3, 0] = -1, -np.inf
    out = od.linear_distillation(h, w, y, ids, lt, **kw)

    def f():
        return od.linear_distillation(h, w, y, ids, lt, **kw)["loss"]

    for name, x in (("dh", h), ("dw", w)):
        num = np.empty_like(x)
        for i in np.ndindex(x.shape):
            old = x[i]
            x[i] = old + 1e-6
            up = f()
            x[i] = old - 1e-6
            num[i] = (up - f()) / 2e-6
            x[i] = old
        assert np.allclose(out[name], num, atol=1e-8)
    assert (out["dh"][2] == 0).all() and out["count"] == 4


def test_oracle_against_torch():
    h, w, y, ids, lt = problem(3)
    lp = torch.log_softmax(torch.tensor(h) @ torch.tensor(w).T, 1)
    ls, t = lp.gather(1, torch.tensor(ids)), torch.tensor(lt).exp()
    # the tokens and their tail as one distribution of k + 1
    both = [torch.cat([x, 1 - x.sum(1, keepdim=True)], 1) for x in (t, ls.exp())]
    kl = torch.nn.functional.kl_div
    assert np.isclose(od.linear_distillation(h, w, y, ids, lt)["divergence"],
                      kl(both[1].log(), both[0], reduction="batchmean"), atol=1e-12)
    assert np.isclose(od.linear_distillation(h, w, y, ids, lt, divergence="reverse")["divergence"],
                      kl(both[0].log(), both[1], reduction="batchmean"), atol=1e-12)
    assert np.isclose(od.linear_distillation(h, w, y, ids, lt)["cross_entropy"],
                      torch.nn.functional.nll_loss(lp, torch.tensor(y)), atol=1e-12)
    # a teacher that names every token, and the student itself as the teacher
    every = np.tile(np.arange(9), (5, 1))
    out = od.linear_distillation(h, w, y, every, lp.numpy())
    assert abs(out["loss"]) < 1e-12 and np.abs(out["dh"]).max() < 1e-12


def test_oracle_names_tokens_once():
    ids, lts, bad = od.named([3, -1, 3, 9, 5, -2, 5], [-1.0, -1.0, -2.0, -1.0, -np.inf, -1.0, -3.0], 9)
    assert ids.tolist() == [3, 5] and lts.tolist() == [-1.0, -3.0] and bad == 3


def _call(lib, **kw):
    a = dict(h=FAKE, w=FAKE, y=FAKE, ids=FAKE, ib=8, t=FAKE, n=300, hdim=256, vocab=1000, k=5, ign=-100, temp=1.0, ce=0.0, div=0,
             tail=1, divisor=None, loss=FAKE, md=FAKE, mc=FAKE, counts=FAKE, dh=FAKE + (1 << 24), dw=FAKE, chunk=128, ws=FAKE)
    a.update(kw)
    grads = a["dh"] is not None or a["dw"] is not None
    a.setdefault("wb", lib.siq_distill_workspace_bytes(300, 256, 1000, 5, 128, int(grads), int(a["dw"] is not None)))
    return lib.siq_distill(*(a[k] for k in ("h", "w", "y", "ids", "ib", "t", "n", "hdim", "vocab", "k", "ign", "temp", "ce", "div",
                                            "tail", "divisor", "loss", "md", "mc", "counts", "dh", "dw", "chunk", "ws", "wb")),
                           None)


@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), INVALID), (dict(n=2 ** 31), INVALID), (dict(hdim=0), INVALID), (dict(hdim=100), UNSUPPORTED),
    (dict(vocab=1001), UNSUPPORTED), (dict(vocab=2 ** 23), INVALID), (dict(h=None), INVALID), (dict(h=FAKE + 8), ALIGN),
    (dict(w=None), INVALID), (dict(w=FAKE + 2), ALIGN), (dict(y=None), INVALID), (dict(ids=None), INVALID),
    (dict(t=None), INVALID), (dict(ib=2), INVALID), (dict(k=0), INVALID), (dict(k=129), INVALID), (dict(k=9, vocab=8), INVALID),
    (dict(temp=0.0), INVALID), (dict(temp=float("inf")), INVALID), (dict(ce=-0.1), INVALID), (dict(ce=1.1), INVALID),
    (dict(ce=float("nan")), INVALID), (dict(ce=0.1, temp=2.0), UNSUPPORTED), (dict(div=2), INVALID),
    (dict(div=1, tail=0), UNSUPPORTED), (dict(loss=None), INVALID), (dict(md=None), INVALID), (dict(mc=None), INVALID),
    (dict(counts=None), INVALID), (dict(chunk=0, wb=1 << 40), INVALID), (dict(dh=FAKE + 8), ALIGN), (dict(dw=FAKE + 8), ALIGN),
    (dict(dh=FAKE), INVALID), (dict(dh=FAKE + 1024), INVALID), (dict(ws=None), WS), (dict(wb=64), WS),
])
def test_validation(lib, kw, code):
    assert _call(lib, **kw) == code


def test_workspace_sizes(lib):
    n, h, v, chunk = 16384, 1536, 151936, 6912
    f = lib.siq_distill_workspace_bytes
    loss, dh, dw = (f(n, h, v, 64, chunk, *x) for x in ((0, 0), (1, 0), (1, 1)))
    assert loss < 1 << 30 < 2 * chunk * v < dh < dw < 7 << 30
    assert f(-1, 64, 8, 1, 64, 1, 1) == 0 and f(5, 0, 8, 1, 64, 1, 1) == 0 and f(5, 64, 8, 0, 64, 1, 1) == 0
    assert f(5, 64, 8, 129, 64, 1, 1) == 0 and f(5, 64, 8, 1, 0, 1, 1) == 0 and f(0, 64, 8, 1, 64, 1, 1) > 0


def test_scaling_two_tensors(lib):
    f = lib.siq_scale2_bf16
    assert f(None, None, 0, None, None, 0, None, None) == OK
    assert f(FAKE, FAKE, -1, FAKE, FAKE, 8, FAKE, None) == INVALID and f(FAKE, FAKE, 8, FAKE, FAKE, -1, FAKE, None) == INVALID
    assert f(None, FAKE, 8, FAKE, FAKE, 8, FAKE, None) == INVALID and f(FAKE, FAKE, 8, FAKE, FAKE, 8, None, None) == INVALID
    assert f(FAKE, FAKE, 8, FAKE + 8, FAKE, 8, FAKE, None) == ALIGN and f(FAKE, FAKE + 2, 8, FAKE, FAKE, 8, FAKE, None) == ALIGN


def test_python_refusals():
    h, w, y = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16), torch.zeros(4).long()
    ids, lt = torch.zeros(4, 2).long(), torch.zeros(4, 2)

    def f(*a, **kw):
        args = dict(zip(("hidden", "weight", "labels", "top_ids", "top_log_probs"), (h, w, y, ids, lt)))
        args.update(kw)
        return D.fused_linear_distillation(**args)

    for kw, text in ((dict(), "GPU"), (dict(labels=None), "GPU"), (dict(labels=y[:3]), r"labels must be \(4,\)"),
                     (dict(top_ids=ids[:3]), "top_ids and top_log_probs"), (dict(top_log_probs=lt[:, :1]), "top_log_probs must be"),
                     (dict(divergence="both"), "divergence must be one of"), (dict(labels=None, ce_weight=0.5), "needs labels"),
                     (dict(labels=None, top_ids=ids[:, :0], top_log_probs=lt[:, :0]), "names no token"),
                     (dict(weight=w[:, :32]), "hdim"), (dict(chunk_tokens=0), "chunk_tokens"),
                     (dict(top_log_probs=lt.clone().requires_grad_()), "detach")):
        with pytest.raises(ValueError, match=text):
            f(**kw)


def test_a_model_with_a_teacher_needs_labels_and_the_gpu():
    transformers = pytest.importorskip("transformers")
    from siq_vl_amd.text_model import enable_fused_cross_entropy

    cfg = transformers.Qwen2Config(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=1,
                                   num_attention_heads=2, num_key_value_heads=1, use_cache=False)
    model = transformers.Qwen2ForCausalLM(cfg)
    enable_fused_cross_entropy(model)
    ids = torch.randint(0, 64, (1, 5))
    teacher = (torch.zeros(1, 5, 2).long(), torch.zeros(1, 5, 2))
    with pytest.raises(ValueError, match="teacher needs labels"):
        model(input_ids=ids, teacher=teacher)
    with pytest.raises(ValueError, match="not both"):
        model(input_ids=ids, labels=ids, teacher=teacher, return_log_probs=True)
    with pytest.raises(ValueError, match="GPU"):
        model(input_ids=ids, labels=ids, teacher=teacher)
    with pytest.raises(ValueError, match="GPU"):
        model(input_ids=ids, labels=ids, return_log_probs=True, top_k=4)
    with pytest.raises(ValueError, match="top_k goes with return_log_probs"):
        model(input_ids=ids, labels=ids, top_k=4)


def test_distillation_options_need_a_teacher():
    transformers = pytest.importorskip("transformers")
    from siq_vl_amd.text_model import enable_fused_cross_entropy

    cfg = transformers.Qwen2Config(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=1,
                                   num_attention_heads=2, num_key_value_heads=1, use_cache=False)
    model = transformers.Qwen2ForCausalLM(cfg)
    enable_fused_cross_entropy(model)
    ids = torch.randint(0, 64, (1, 5))
    with pytest.raises(ValueError, match="go with a teacher"):
        model(input_ids=ids, labels=ids, distillation={"ce_weight": 0.5})
