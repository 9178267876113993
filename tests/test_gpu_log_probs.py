"""Log-probabilities of labels on the GPU against the oracle in 64 bits, kept and recomputed, alone and with the losses
that read them."""

import numpy as np
import pytest
import torch

from oracle import log_probs as olp
from oracle import policy as op
from siq_vl_amd import cross_entropy as C
from siq_vl_amd import log_probs as LP
from siq_vl_amd import policy as P

pytestmark = pytest.mark.gpu
DEV = "cuda"


def np64(t):
    return t.detach().double().cpu().numpy()


def make(n, hdim, vocab, seed=0, ignored=0.3, wscale=0.05, lean=0.0):
    g = torch.Generator().manual_seed(seed)
    w = (wscale * torch.randn(vocab, hdim, generator=g)).to(torch.bfloat16)
    y = torch.randint(0, vocab, (n,), generator=g)
    h = torch.randn(n, hdim, generator=g) + lean * torch.rand(n, 1, generator=g) * w[y].float() / (wscale ** 2 * hdim)
    y[torch.rand(n, generator=g) < ignored] = -100
    up = torch.randn(n, generator=g) * torch.rand(n, generator=g)
    up[torch.rand(n, generator=g) < 0.2] = 0.0
    return h.to(torch.bfloat16), w, y, up


def check(h, w, y, up, temperature=1.0, keep=True, chunk=None, need_dw=True, rounds=1.0):
    hd, wd, yd = h.to(DEV), w.to(DEV), y.to(DEV)
    logp, count, bad, saved = LP.flp_fwd(hd, wd, yd, temperature=temperature, keep=keep)
    assert (saved is not None) == keep
    dh, dw = LP.flp_bwd(hd, wd, yd, up.to(DEV), temperature=temperature, saved=saved, need_dweight=need_dw,
                        chunk_tokens=chunk)
    torch.cuda.synchronize()
    ref = olp.linear_log_probs(np64(h), np64(w), y.numpy(), np64(up), temperature)
    assert int(count) == ref["count"] and int(bad) == ref["bad"]
    assert (np.abs(np64(logp) - ref["logp"]) <= ref["logp_off"]).all()
    out = (y == -100) | (y < 0) | (y >= w.shape[0])
    assert bool((logp.cpu()[out] == 0).all()) and bool((dh.cpu()[out] == 0).all())
    assert (np.abs(np64(dh) - ref["dh"]) <= rounds * ref["dh_off"]).all()
    if need_dw:
        assert (np.abs(np64(dw) - ref["dw"]) <= rounds * ref["dw_off"]).all()
    else:
        assert dw is None
    return logp, dh, dw


@pytest.mark.parametrize("keep,chunk", [(True, None), (False, None), (False, 128), (False, 64), (False, 100)])
@pytest.mark.parametrize("n,hdim,vocab", [(50, 896, 520), (100, 1152, 1000), (64, 64, 2000), (65, 192, 1000), (128, 320, 4104), (129, 320, 4104), (1, 64, 8), (3, 64, 1000), (255, 320, 264), (257, 128, 2000), (300, 896, 1000)])
def test_against_the_oracle(n, hdim, vocab, keep, chunk):
    print(f"logp n={n} h={hdim} V={vocab} keep={keep} chunk={chunk}", flush=True)
    h, w, y, up = make(n, hdim, vocab, seed=n, ignored=0.3 if n > 1 else 0.0)
    check(h, w, y, up, 1.0, keep, chunk)
    check(h, w, y, up, 0.7, keep, chunk)
    check(h, w, y, up, 1.9, keep, chunk, need_dw=False)


@pytest.mark.parametrize("keep", [True, False])
def test_likely_labels_keep_their_digits(keep):
    h, w, y, up = make(400, 256, 1000, seed=5, lean=40.0)
    logp, _, _ = check(h, w, y, up, 1.0, keep)
    assert float(logp[y.to(DEV) >= 0].max()) > -1e-3


@pytest.mark.parametrize("n", [50, 100, 300])
@pytest.mark.parametrize("keep", [True, False])
def test_labels_far_below_the_largest_logit(n, keep):
    """Logits a hundred apart: whole tiles are formed again relative to their own maximum, and rounded twice."""
    h, w, y, up = make(n, 128, 1000, seed=6, wscale=2.0)
    logp, _, _ = check(h, w, y, up, 1.0, keep, rounds=2.0)
    assert float(logp.min()) < -60
    check(h, w, y, up, 0.25, keep, rounds=2.0)


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("n", [40, 700])
def test_one_label_for_all_rows_and_labels_at_the_ends(n, keep):
    h, w, y, up = make(n, 128, 264, seed=7)
    y[y >= 0] = 17
    check(h, w, y, up, 1.0, keep)
    y[::2], y[1::2] = 0, 263
    check(h, w, y, up, 1.0, keep)


@pytest.mark.parametrize("keep", [True, False])
def test_nothing_counts_no_rows_and_bad_labels(keep):
    h, w, y, up = make(300, 128, 1000, seed=8)
    y[:] = -100
    _, dh, dw = check(h, w, y, up, 1.0, keep)
    assert bool((dw == 0).all())
    logp, count, bad, saved = LP.flp_fwd(h[:0].to(DEV), w.to(DEV), y[:0].to(DEV), keep=keep)
    dh, dw = LP.flp_bwd(h[:0].to(DEV), w.to(DEV), y[:0].to(DEV), up[:0].to(DEV), saved=saved)
    assert logp.shape == (0,) and int(count) == 0 and dh.shape == (0, 128) and bool((dw == 0).all())
    y[:] = 5
    y[3], y[200] = 1000, -7
    check(h, w, y, up, 1.0, keep)
    with pytest.raises(C.LabelError):
        LP.fused_linear_log_probs(h.to(DEV), w.to(DEV), y.to(DEV), validate="sync")
    # upstream gradients of rows that do not count are not read
    up[3] = up[200] = float("nan")
    dh, dw = LP.flp_bwd(h.to(DEV), w.to(DEV), y.to(DEV), up.to(DEV))
    assert not bool(dh.isnan().any()) and not bool(dw.isnan().any())


def test_mean_is_the_cross_entropy():
    h, w, y, _ = make(600, 320, 2000, seed=9)
    hd, wd, yd = h.to(DEV), w.to(DEV), y.to(DEV)
    loss, count, _, dh, dw = C.flce_fwd_bwd(hd, wd, yd, chunk_tokens=1024)
    logp, _, _, saved = LP.flp_fwd(hd, wd, yd, keep=True)
    assert abs(float(loss) + float(logp.double().sum()) / int(count)) <= 1e-6 * float(loss)
    up = torch.full((600,), -1.0, device=DEV) / count.float()
    ref = olp.linear_log_probs(np64(h), np64(w), y.numpy(), np64(up))
    for s in (saved, None):
        dh2, dw2 = LP.flp_bwd(hd, wd, yd, up, saved=s, chunk_tokens=1024)
        # each side is at most dh_off / dw_off from the exact gradient
        assert (np.abs(np64(dh) - np64(dh2)) <= 2 * ref["dh_off"]).all()
        assert (np.abs(np64(dw) - np64(dw2)) <= 2 * ref["dw_off"]).all()


@pytest.mark.parametrize("keep", [True, False])
def test_near_certain_labels_are_exact_relative_to_their_distance_from_certainty(keep):
    """Log-probabilities of -1e-9 and their gradients: sums that held the label's own term would lose them."""
    g = torch.Generator().manual_seed(3)
    w = (0.05 * torch.randn(1000, 256, generator=g)).to(torch.bfloat16)
    y = torch.randint(0, 1000, (40,), generator=g)
    # logits of 12 .. 32 above the others'
    h = (torch.linspace(12, 32, 40)[:, None] * w[y].float() / (0.05 ** 2 * 256)).to(torch.bfloat16)
    up = torch.ones(40)
    logp, _, _, saved = LP.flp_fwd(h.to(DEV), w.to(DEV), y.to(DEV), keep=keep)
    ref = olp.linear_log_probs(np64(h), np64(w), y.numpy(), np64(up))
    z = np64(h) @ np64(w).T
    off = 2 * 36 * 2.0 ** -24 * (np.abs(np64(h)) @ np.abs(np64(w)).T).max(1) + 64 * 2.0 ** -24
    exact = -np.log1p(np.array([np.exp(np.delete(r, k) - r[k]).sum() for r, k in zip(z, y.numpy())]))
    assert exact.max() > -1e-8 and (np.abs(np64(logp) - exact) <= off * np.abs(exact)).all()
    dh, _ = LP.flp_bwd(h.to(DEV), w.to(DEV), y.to(DEV), up.to(DEV), saved=saved, need_dweight=False)
    # every term of a row's gradient is as small as 1 - p: errors are relative to it
    size = -np.expm1(exact)[:, None] * (np.abs(np64(w)).max(0)[None] + np.abs(np64(w))[y.numpy()])
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    p[np.arange(40), y.numpy()] = np.expm1(exact)
    assert (np.abs(np64(dh) + p @ np64(w)) <= (2 * 2.0 ** -8 + off[:, None]) * size).all()


def test_more_kept_rows_than_one_pass_takes():
    """70,000 rows of a small vocabulary: kept numerators in two passes of 65,536 rows, against chunks that are formed again."""
    n, hdim, vocab = 70_000, 64, 264
    g = torch.Generator(device=DEV).manual_seed(4)
    h = torch.randn(n, hdim, generator=g, device=DEV).to(torch.bfloat16)
    w = (0.1 * torch.randn(vocab, hdim, generator=g, device=DEV)).to(torch.bfloat16)
    y = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    y[torch.rand(n, generator=g, device=DEV) < 0.02] = -100
    up = torch.randn(n, generator=g, device=DEV)
    a, b = LP.flp_fwd(h, w, y, keep=True), LP.flp_fwd(h, w, y, keep=False)
    assert torch.equal(a[0], b[0]) and int(a[1]) == int(b[1])
    dh, dw = LP.flp_bwd(h, w, y, up, saved=a[3])
    dh2, dw2 = LP.flp_bwd(h, w, y, up, chunk_tokens=4096)
    # the exact gradients in 64 bits, and what rounding may make of each (see the oracle)
    at = y >= 0
    p = torch.softmax(h.double() @ w.double().T.contiguous(), 1) * (up.double() * at)[:, None]
    dz = -p
    dz[at.nonzero()[:, 0], y[at]] += up.double()[at]
    want = dz @ w.double()
    off = 1.05 * (2.0 ** -8 * (p.abs() @ w.double().abs() + want.abs()) + 1e-4 * up.double().abs()[:, None])
    for got in (dh, dh2):
        assert bool(((got.double() - want).abs() <= off).all()) and bool((got[~at] == 0).all())
    want = dz.T.contiguous() @ h.double()
    # E and the scaled rows rounded, sums of n products in fp32 (eight at once), the label terms' weights
    label = torch.zeros_like(want).index_add_(0, y[at], (up.double().abs()[:, None] * h.double().abs())[at])
    off = (2.0 ** -7 + n / 8 * 2.0 ** -24) * (p.abs().T.contiguous() @ h.double().abs()) + 2.0 ** -8 * want.abs()
    off = 1.05 * off + (1e-4 + n / 8 * 2.0 ** -24) * label
    for got in (dw, dw2):
        assert bool(((got.double() - want).abs() <= off).all())


def test_kept_and_recomputed_agree_and_repeat():
    h, w, y, up = make(900, 256, 3008, seed=10)
    hd, wd, yd, ud = h.to(DEV), w.to(DEV), y.to(DEV), up.to(DEV)
    a = LP.flp_fwd(hd, wd, yd, keep=True)
    b = LP.flp_fwd(hd, wd, yd, keep=False)
    assert torch.equal(a[0], b[0])
    before = a[3].clone()
    first = LP.flp_bwd(hd, wd, yd, ud, saved=a[3])
    assert torch.equal(a[3], before)  # only read
    for s, chunk in ((a[3], None), (None, 1024)):
        again = LP.flp_bwd(hd, wd, yd, ud, saved=s, chunk_tokens=chunk)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    assert torch.equal(LP.flp_bwd(hd, wd, yd, ud, saved=a[3], need_dweight=False)[0], first[0])
    only_w = LP.flp_bwd(hd, wd, yd, ud, saved=a[3], need_dhidden=False)
    assert only_w[0] is None and torch.equal(only_w[1], first[1])


def test_autograd_shapes_types_frozen_and_retained():
    h, w, y, up = make(60, 128, 520, seed=11)
    hg = h.view(4, 15, 128).to(DEV).requires_grad_()
    wg, yd, ud = w.to(DEV).requires_grad_(), y.view(4, 15).to(DEV), up.view(4, 15).to(DEV)
    want = LP.flp_bwd(hg.detach().view(60, 128), wg.detach(), yd.view(-1), ud.view(-1), temperature=1.3)
    scaled = LP.fused_linear_log_probs(hg, wg, yd)
    scaled *= 2.0  # the result is no view of anything: it may be changed in place
    torch.autograd.grad(scaled.sum(), [hg])
    for keep_bytes in (1 << 30, 0):
        logp = LP.fused_linear_log_probs(hg, wg, yd, temperature=1.3, keep_bytes=keep_bytes)
        assert logp.shape == (4, 15) and logp.dtype == torch.float32
        got = torch.autograd.grad(logp, [hg, wg], ud, retain_graph=True)
        again = torch.autograd.grad(logp, [hg, wg], ud)
        assert torch.equal(got[0].view(60, 128), want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    frozen = LP.fused_linear_log_probs(hg, wg.detach(), yd, temperature=1.3)
    assert torch.equal(torch.autograd.grad(frozen, [hg], ud)[0].view(60, 128), want[0])
    head = LP.fused_linear_log_probs(hg.detach(), wg, yd, temperature=1.3)
    assert torch.equal(torch.autograd.grad(head, [wg], ud)[0], want[1])
    with torch.no_grad():
        lone = LP.fused_linear_log_probs(hg, wg, yd, temperature=1.3)
    assert lone.grad_fn is None and torch.equal(lone, logp)
    # a broadcast upstream gradient, and fp32 master copies
    g1, = torch.autograd.grad(LP.fused_linear_log_probs(hg, wg.detach(), yd).sum(), [hg])
    g2, = torch.autograd.grad(LP.fused_linear_log_probs(hg, wg.detach(), yd), [hg], torch.ones(4, 15, device=DEV))
    assert torch.equal(g1, g2)
    h32, w32 = hg.detach().float().requires_grad_(), wg.detach().float().requires_grad_()
    got = torch.autograd.grad(LP.fused_linear_log_probs(h32, w32, yd, temperature=1.3), [h32, w32], ud)
    assert got[0].dtype == torch.float32 and torch.equal(got[0].view(60, 128), want[0].float())
    assert torch.equal(got[1], want[1].float())


def test_gradient_is_a_difference():
    """One direction in ``hidden``, central differences of the fp32 log-probabilities."""
    h, w, y, up = make(64, 128, 520, seed=12, ignored=0.1)
    g = torch.Generator().manual_seed(1)
    h = (h.float() * 8).round().div(8).to(torch.bfloat16)  # steps of 1 / 8 below 16: moved by 1 / 16 exactly
    d = (torch.randint(-1, 2, h.shape, generator=g) / 16).to(torch.bfloat16)
    hd, wd, yd, ud = h.to(DEV), w.to(DEV), y.to(DEV), up.to(DEV).double()
    assert torch.equal((hd + d.to(DEV)).float(), hd.float() + d.to(DEV).float())
    up_, down = (LP.flp_fwd(hd + s * d.to(DEV), wd, yd)[0].double() for s in (1, -1))
    num = ((up_ - down) * ud / 2).cpu().numpy()
    dh, _ = LP.flp_bwd(hd, wd, yd, up.to(DEV), need_dweight=False)
    got = (dh.double() * d.to(DEV).double()).sum(1).cpu().numpy()
    ref = olp.linear_log_probs(np64(h), np64(w), y.numpy(), np64(up))
    # a row's move changes its logits by s = |w| |d| at most, typically 0.05 * 128^0.5 / 20: the third derivative of a
    # log-sum-exp is at most 2 s^3 / 6; plus what rounding makes of the gradient and of the two values
    s = np.abs(np64(d)) @ np.abs(np64(w)).T
    spread = np.linalg.norm(np64(d), axis=1) * np.linalg.norm(np64(w), axis=1).max()
    bound = np.abs(np64(up)) * (spread ** 3 / 3 + ref["logp_off"]) + (ref["dh_off"] * np.abs(np64(d))).sum(1) + 1e-9
    assert s.max() > 0 and (np.abs(num - got) <= bound).all()


def chain(kind, h, w, y, cu, mask, old, ref, adv, dtype64=False):
    """Hidden states to loss and gradients, as a training step runs it."""
    hg, wg = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    logp = LP.fused_linear_log_probs(hg, wg, y.to(DEV))
    if kind == "pref":
        loss = P.preference_loss(logp, ref, cu, mask=mask, beta=0.5).loss
    else:
        loss = P.policy_loss(logp, old, adv, cu, mask=mask, reference_logps=ref, kl_coef=0.1, aggregation="sequence").loss
    loss.backward()
    return float(loss.detach()), hg.grad, wg.grad


@pytest.mark.parametrize("kind", ["pref", "policy"])
def test_a_run_from_hidden_states_to_the_loss(kind):
    lengths = [70, 130, 1, 99, 0, 200]
    n = sum(lengths)
    h, w, y, _ = make(n, 256, 1000, seed=13, ignored=0.4)
    cu = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    base = olp.linear_log_probs(np64(h), np64(w), y.numpy())["logp"]
    rng = np.random.default_rng(3)
    old, ref = (np.float32(base + 0.2 * rng.standard_normal(n)) for _ in range(2))
    adv = np.float32(rng.standard_normal(len(lengths)))
    mask = (y != -100).numpy()
    cu_t, mask_t, old_t, ref_t, adv_t = (torch.tensor(v, device=DEV) for v in (cu, mask, old, ref, adv))
    loss, dh, dw = chain(kind, h, w, y, cu_t, mask_t, old_t, ref_t, adv_t)
    if kind == "pref":
        want, _, _, g = op.preference(base, ref, cu, mask, beta=0.5)
    else:
        want, _, _, g = op.policy(base, old, adv, cu, mask, ref, kl_coef=0.1, aggregation="sequence")
    out = olp.linear_log_probs(np64(h), np64(w), y.numpy(), g)
    # what the log-probabilities' own error does to the weights: sums of up to 200 of them in the pairs' margins
    wobble = 1 + 300 * out["logp_off"].max()
    assert abs(loss - want) <= 300 * out["logp_off"].max() * (1 + abs(want))
    assert (np.abs(np64(dh) - out["dh"]) <= wobble * out["dh_off"] + (wobble - 1) * np.abs(out["dh"])).all()
    assert (np.abs(np64(dw) - out["dw"]) <= wobble * out["dw_off"] + (wobble - 1) * np.abs(out["dw"]).max()).all()


def test_streams_and_captured_calls():
    h, w, y, up = make(500, 128, 1000, seed=14)
    hd, wd, yd, ud = h.to(DEV), w.to(DEV), y.to(DEV), up.to(DEV)

    def call(keep):
        logp, _, _, saved = LP.flp_fwd(hd, wd, yd, keep=keep)
        return (logp, *LP.flp_bwd(hd, wd, yd, ud, saved=saved, chunk_tokens=128))

    want = [call(True), call(False)]
    torch.cuda.synchronize()
    got = []
    for st in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(st):
            got.append([call(True), call(False)])
    torch.cuda.synchronize()
    for pair in got:
        for a, b in zip(pair, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [call(True), call(False)]
    for i in range(3):
        hd.copy_(torch.randn_like(hd))
        yd.copy_(yd.roll(1))
        ud.copy_(torch.randn_like(ud))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, [call(True), call(False)]):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_a_second_derivative_is_refused():
    h, w, y, _ = make(20, 64, 264)
    hg = h.to(DEV).requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(LP.fused_linear_log_probs(hg, w.to(DEV), y.to(DEV)).sum(), [hg], create_graph=True)


def test_a_preference_step_of_a_packed_model():
    """Two pairs of answers in one packed batch through a small Qwen2: the model's log-probabilities are those of its own
    logits, and the loss's gradient reaches every parameter as through the logits."""
    transformers = pytest.importorskip("transformers")
    from siq_vl_amd import attention
    from siq_vl_amd.cross_entropy import shift_labels
    from siq_vl_amd.text_model import enable_fused_cross_entropy

    attention.register()
    cfg = transformers.Qwen2Config(vocab_size=264, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                                   num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=512)
    torch.manual_seed(2)
    model = transformers.Qwen2ForCausalLM(cfg).to(DEV, torch.bfloat16).train()
    model.config._attn_implementation = "siq_varlen"
    lengths = [30, 41, 17, 50]
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device=DEV)
    ids = torch.randint(0, 264, (1, sum(lengths)), device=DEV)
    labels = ids.clone()
    for a, n in zip(cu[:-1].tolist(), lengths):
        labels[0, a:a + n // 3] = -100  # the prompt; the first label of a sequence is no target of the one before
    pos = torch.cat([torch.arange(n) for n in lengths]).to(DEV)[None]
    inputs = dict(input_ids=ids, position_ids=pos, use_cache=False, cu_seq_lens_q=cu, cu_seq_lens_k=cu,
                  max_length_q=50, max_length_k=50)
    targets = shift_labels(labels)
    mask = targets != -100
    ref = torch.randn(1, sum(lengths), device=DEV) - 5.5
    logits = model(**inputs).logits
    z = torch.log_softmax(logits.float(), -1).gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    want = torch.where(mask, z, 0.0)
    P.preference_loss(want, ref, cu, mask=mask, beta=0.1).loss.backward()
    grads = {n: p.grad.double() for n, p in model.named_parameters()}
    model.zero_grad()
    enable_fused_cross_entropy(model)
    with pytest.raises(ValueError, match="labels"):
        model(**inputs, return_log_probs=True)
    out = model(**inputs, labels=labels, return_log_probs=True)
    assert out.loss is None and out.logits is None and out.log_probs.shape == (1, sum(lengths))
    # the stock path rounds its logits to bf16: half a step of the largest of them, twice
    off = 2 * 2.0 ** -8 * float(logits.abs().max()) + 1e-4
    assert float((out.log_probs - want).abs().max()) <= off
    P.preference_loss(out.log_probs, ref, cu, mask=mask, beta=0.1).loss.backward()
    for n, p in model.named_parameters():
        # the same in bf16 activations and gradients, the logits' gradient not rounded: a few roundings of 2^-8
        rel = float((p.grad.double() - grads[n]).norm() / grads[n].norm())
        assert rel <= 0.05, (n, rel)
    with torch.no_grad():  # a reference model's pass
        lone = model(**inputs, labels=labels, return_log_probs=True).log_probs
    assert torch.equal(lone, out.log_probs)
    warm = model(**inputs, labels=labels, return_log_probs=True, temperature=2.0).log_probs
    assert not torch.equal(warm, lone)
    assert model(**inputs, labels=labels).loss is not None


def test_what_the_forward_kept_is_checked():
    h, w, y, up = (t.to(DEV) for t in make(40, 64, 1000, seed=1))
    saved = LP.flp_fwd(h, w, y, keep=True)[3]
    for other, text in ((saved.cpu(), "saved must live on"), (saved.view(torch.int32), "what the forward kept"),
                        (saved[:-64], "saved")):
        with pytest.raises(ValueError, match=text):
            LP.flp_bwd(h, w, y, up, saved=other)


@pytest.mark.parametrize("n", [50, 300])
@pytest.mark.parametrize("keep", [True, False])
def test_a_label_of_no_probability_beside_columns_of_little(n, keep):
    """The label 2^-135 of the row's largest column, another tile 2^-83: its columns' gradient is small and not zero."""
    h, w = torch.zeros(n, 64), torch.zeros(1024, 64)
    h[:, 0], w[300:400, 0], w[600:640, 0] = 1.0, 36.0, 90.0
    h[:, 1], w[:, 1] = torch.randn(n, generator=torch.Generator().manual_seed(n)), 0.25
    y = torch.arange(n) % 256
    up = 0.5 + torch.rand(n, generator=torch.Generator().manual_seed(1))
    _, _, dw = check(h.to(torch.bfloat16), w.to(torch.bfloat16), y, up, 1.0, keep, rounds=2.0)
    assert bool((dw[300:400, 0] < 0).all())


@pytest.mark.parametrize("n", [50, 300])
def test_every_call_with_bad_labels_is_judged_once(n):
    h, w, y, _ = (t.to(DEV) for t in make(n, 64, 1000, seed=2))
    bad = y.clone()
    bad[3] = 1000
    C.check_pending_labels(block=True)
    for _ in range(3):
        LP.fused_linear_log_probs(h, w, y)
    C.check_pending_labels(block=True)
    LP.fused_linear_log_probs(h, w, bad)
    torch.cuda.synchronize()
    with pytest.raises(C.LabelError, match="1 label"):  # the first call's; the second is tracked all the same
        LP.fused_linear_log_probs(h.clone().requires_grad_(), w, bad)
    with pytest.raises(C.LabelError, match="1 label"):
        C.check_pending_labels(block=True)
    C.check_pending_labels(block=True)
    LP.fused_linear_log_probs(h, w, bad, validate=False)
    C.check_pending_labels(block=True)
    with pytest.raises(C.LabelError):
        LP.fused_linear_log_probs(h, w, bad, validate="sync")


def test_a_freed_graph_is_refused_and_a_kept_one_repeats():
    h, w, y, up = (t.to(DEV) for t in make(40, 64, 1000, seed=4))
    cu = torch.tensor([0, 25, 40], dtype=torch.int32, device=DEV)
    old = torch.randn(40, device=DEV)
    h.requires_grad_()
    for last in (lambda lp: (lp * up).sum(), lambda lp: P.preference_loss(lp, old, cu).loss,
                 lambda lp: P.policy_loss(lp, old, torch.ones(2, device=DEV), cu).loss):
        loss = last(LP.fused_linear_log_probs(h, w, y))
        first, = torch.autograd.grad(loss, [h], retain_graph=True)
        again, = torch.autograd.grad(loss, [h])
        assert torch.equal(first, again)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(loss, [h])


def test_a_call_that_fails_behind_its_launch_keeps_its_counts_memory(monkeypatch):
    h, w, y, _ = (t.to(DEV) for t in make(40, 64, 1000, seed=6))
    C.check_pending_labels(block=True)
    native = LP._lib.native()
    hosts = []

    class Failing:
        def linear_log_probs(self, *args):
            hosts.append(args[-1])
            native.linear_log_probs(*args)
            raise KeyboardInterrupt

    monkeypatch.setattr(LP._lib, "_NATIVE", Failing())
    y[0] = 1000  # (a failed call's labels are not judged)
    with pytest.raises(KeyboardInterrupt):
        LP.fused_linear_log_probs(h, w, y)
    held = [call[2] for call in C._LABEL_CHECKS._pending]
    assert len(held) == 1 and held[0] is hosts[0] and held[0].is_pinned()
    C.check_pending_labels(block=True)
    assert len(C._LABEL_CHECKS) == 0 and hosts[0].tolist() == [int((y >= 0).sum()) - 1, 1]


def test_what_another_shape_kept_is_refused():
    h, w, y, up = (t.to(DEV) for t in make(40, 64, 1000, seed=1))
    more = LP.flp_fwd(h.repeat(2, 1), w, y.repeat(2), keep=True)[3]
    with pytest.raises(ValueError, match="what the forward kept"):
        LP.flp_bwd(h, w, y, up, saved=more)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", ["hidden", "weight"])
@pytest.mark.parametrize("fp32", [False, True])
def test_a_forward_mode_derivative_is_refused(fp32, which, grad):
    """The log-probabilities and the cross-entropy give no result that has lost its tangent."""
    fw = torch.autograd.forward_ad
    h, w, y, _ = (t.to(DEV) for t in make(20, 64, 264))
    if fp32:
        h, w = h.float(), w.float()
    with fw.dual_level(), torch.set_grad_enabled(grad):
        args = [fw.make_dual(h, h), w, y] if which == "hidden" else [h, fw.make_dual(w, w), y]
        for call in (LP.fused_linear_log_probs, C.fused_linear_cross_entropy):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*args)
            call(h, w, y)


@pytest.mark.parametrize("items", [300, torch.tensor(300)])
def test_a_number_of_items_on_the_host_costs_the_cross_entropy_no_synchronisation(items):
    h, w, y, _ = make(400, 64, 264, seed=3)
    hd, wd, yd = h.to(DEV), w.to(DEV), y.to(DEV)
    want = C.fused_linear_cross_entropy(hd, wd, yd, num_items_in_batch=torch.tensor(300.0, device=DEV))
    C.check_pending_labels(block=True)
    torch.cuda.set_sync_debug_mode("error")
    try:
        got = C.fused_linear_cross_entropy(hd, wd, yd, num_items_in_batch=items)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert torch.equal(got, want)


@pytest.mark.parametrize("n,hdim,need_dw", [(48, 896, False), (48, 896, True), (128, 896, True), (128, 1536, True),
                                            (129, 896, True), (1, 1536, True)])
@pytest.mark.parametrize("keep", [True, False])
def test_few_rows_of_a_real_vocabulary(n, hdim, need_dw, keep):
    """151,936 columns, against the definition in 64 bits on the GPU; bounds as the oracle's."""
    vocab, half, t = 151_936, 2.0 ** -8, 0.8
    print(f"few rows n={n} h={hdim} dw={need_dw} keep={keep}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(n + hdim)
    w = (0.05 * torch.randn(vocab, hdim, generator=g, device=DEV)).to(torch.bfloat16)
    y = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    lean = 20 * torch.rand(n, 1, generator=g, device=DEV) / (0.05 ** 2 * hdim)
    h = (torch.randn(n, hdim, generator=g, device=DEV) + lean * w[y].float()).to(torch.bfloat16)
    up = torch.randn(n, generator=g, device=DEV)
    if n > 1:
        y[::5], y[1], y[n - 1] = -100, vocab - 1, 0
        up[::5] = float("nan")  # of rows that do not count
    logp, count, bad, saved = LP.flp_fwd(h, w, y, temperature=t, keep=keep)
    dh, dw = LP.flp_bwd(h, w, y, up, temperature=t, saved=saved, need_dweight=need_dw)
    del saved
    at = (y >= 0).nonzero()[:, 0]
    assert int(count) == at.numel() and int(bad) == 0
    out = y < 0
    assert bool((logp[out] == 0).all()) and bool((dh[out] == 0).all())
    hk, wd, yk = h[at].double(), w.double(), y[at]
    rows = torch.arange(at.numel(), device=DEV)
    z = hk @ wd.T.contiguous() / t
    want = z[rows, yk] - torch.logsumexp(z, 1)
    depth = hdim / 8 + 4
    wabs = wd.abs()
    off = 2 * depth * 2.0 ** -24 * (hk.abs() @ wabs.T.contiguous()).amax(1) / t + 1e-6 + 4 * 2.0 ** -24 * want.abs()
    assert bool(((logp[at].double() - want).abs() <= off).all())
    p = torch.softmax(z, 1)
    gk = up[at].double()[:, None] / t
    dz = -gk * p
    soft = dz.abs()
    soft[rows, yk] = 0.0
    dz[rows, yk] += gk[:, 0]
    label = gk.abs() * (8 * 2.0 ** -24 + off[:, None])
    dh_want, spread = dz @ wd, soft @ wabs
    bound = 1.05 * ((half + off[:, None]) * spread + label * wabs[yk] + half * dh_want.abs()) + 1e-30
    assert bool(((dh[at].double() - dh_want).abs() <= bound).all())
    if not need_dw:
        assert dw is None
        return
    dw_want = dz.T.contiguous() @ hk
    bound = 2 * half * (soft.T.contiguous() @ hk.abs()) + half * dw_want.abs()
    bound += (off[:, None] * soft).T.contiguous() @ hk.abs()
    bound.index_add_(0, yk, label * hk.abs())
    assert bool(((dw.double() - dw_want).abs() <= 1.05 * bound + 1e-30).all())


def test_more_kept_numerators_than_32_bits_count():
    """16,390 rows of 151,936 columns: 2.5e9 numerators, and offsets of 5e9 bytes, in the weight's gradient and the rows'."""
    n, hdim, vocab, half = 16_390, 64, 151_936, 2.0 ** -8
    g = torch.Generator(device=DEV).manual_seed(6)
    h = torch.randn(n, hdim, generator=g, device=DEV).to(torch.bfloat16)
    w = (0.3 * torch.randn(vocab, hdim, generator=g, device=DEV)).to(torch.bfloat16)
    y = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    y[100:130], y[n - 1] = -100, vocab - 1
    up = torch.randn(n, generator=g, device=DEV)
    logp, count, _, saved = LP.flp_fwd(h, w, y, keep=True)
    assert int(count) == n - 30 and saved.numel() > 2 * (1 << 31)
    got = [LP.flp_bwd(h, w, y, up, saved=saved), LP.flp_bwd(h, w, y, up)]
    del saved
    wd, wabs = w.double(), w.double().abs()
    wt, wt_abs = wd.T.contiguous(), wabs.T.contiguous()
    dw, dw_off = torch.zeros(2, vocab, hdim, dtype=torch.float64, device=DEV)
    for c in range(0, n, 1024):  # bounds as the oracle's
        at = c + (y[c:c + 1024] >= 0).nonzero()[:, 0]
        rows, hk, yk = torch.arange(at.numel(), device=DEV), h[at].double(), y[at]
        z = hk @ wt
        want = z[rows, yk] - torch.logsumexp(z, 1)
        off = 2 * (hdim / 8 + 4) * 2.0 ** -24 * (hk.abs() @ wt_abs).amax(1) + 1e-6 + 4 * 2.0 ** -24 * want.abs()
        assert bool(((logp[at].double() - want).abs() <= off).all())
        gk = up[at].double()[:, None]
        dz = torch.softmax(z, 1).mul_(-gk)
        soft = dz.abs()
        soft[rows, yk] = 0.0
        dz[rows, yk] += gk[:, 0]
        label = gk.abs() * (8 * 2.0 ** -24 + off[:, None])
        dh_want = dz @ wd
        bound = 1.05 * ((half + off[:, None]) * (soft @ wabs) + label * wabs[yk] + half * dh_want.abs()) + 1e-30
        for dh, _ in got:
            assert bool(((dh[at].double() - dh_want).abs() <= bound).all())
        dw += dz.T.contiguous() @ hk
        dw_off += (soft * (2 * half + off[:, None])).T.contiguous() @ hk.abs()
        dw_off.index_add_(0, yk, label * hk.abs())
        del z, dz, soft
    # sums of n products in fp32, eight at once, beside the oracle's terms
    dw_off += half * dw.abs() + n / 8 * 2.0 ** -24 * dw_off / half
    for dh, grad in got:
        assert bool((dh[100:130] == 0).all())
        assert bool(((grad.double() - dw).abs() <= 1.05 * dw_off + 1e-30).all())
