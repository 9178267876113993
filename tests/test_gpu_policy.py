"""Preference and policy losses on the GPU against the oracle in 64 bits: lengths from none to long, masks that leave
nothing, values that must not matter, borders, aggregations, and the ways they are called."""

import threading

import numpy as np
import pytest
import torch

from oracle import policy as op
from siq_vl_amd import policy as P

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32 = 2.0 ** -24  # half a step of fp32, relative to the value
SLICE = 2048  # tokens of one slice


def np64(t):
    return t.detach().double().cpu().numpy()


LENGTHS = {
    "one token each": [1, 1],
    "short": [31, 100],
    "empty ones": [0, 5, 7, 0, 0, 0, 300, 1],
    "slices": [SLICE, SLICE - 1, 1, 2 * SLICE + 1, 3 * SLICE, 5],
    "one long": [3, 40_001, 2, 9],
    "many": [int(v) for v in np.random.default_rng(0).integers(0, 90, 3000)],
}


def batch(lengths, seed=0, tail=0, drift=0.3):
    rng = np.random.default_rng(seed)
    n = sum(lengths) + tail
    old = -rng.exponential(0.7, n)
    cu = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    mask = rng.random(n) < 0.6
    for s in range(0, len(lengths), 3):  # some sequences count nothing
        mask[cu[s]:cu[s + 1]] = False
    ref, lp = old + drift * rng.standard_normal(n), old + drift * rng.standard_normal(n)
    return cu, mask, *(np.float32(v) for v in (lp, old, ref))


def gpu(*arrays):
    return [None if a is None else torch.tensor(a, device=DEV) for a in arrays]


def poison(x, mask, value):
    """Values in masked places must not matter."""
    y = x.copy()
    y[~mask] = value
    return y


def check_scalar(name, got, want, scale):
    """fp32 rounding of a sum in 64 bits whose terms are off by ``scale`` altogether."""
    assert abs(float(got) - want) <= F32 * abs(want) + scale, (name, float(got), want)


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("kw", [
    dict(), dict(loss_type="sigmoid", label_smoothing=0.2, order="halves"), dict(loss_type="ipo", length_normalized=True),
    dict(loss_type="hinge", beta=0.7, num_items_in_batch=5), dict(length_normalized=True, order="halves", beta=2.0)])
def test_preference(lengths, kw):
    print("preference", lengths, kw, flush=True)
    cu, mask, pi, _, ref = batch(LENGTHS[lengths], tail=11)
    mask_t, cu_t, pi_t, ref_t = gpu(mask, cu, poison(pi, mask, np.nan), poison(ref, mask, -np.inf))
    pi_t.requires_grad_()
    out = P.preference_loss(pi_t, ref_t, cu_t, mask=mask_t, **kw)
    grad, = torch.autograd.grad(out.loss, [pi_t], torch.tensor(3.0, device=DEV))
    want = op.preference(pi, ref, cu, np.append(mask[:-11], np.zeros(11, bool)), beta=kw.get("beta", 0.1),
                         loss_type=kw.get("loss_type", "sigmoid"), smoothing=kw.get("label_smoothing", 0.0),
                         normalized=kw.get("length_normalized", False), order=kw.get("order", "interleaved"),
                         items=kw.get("num_items_in_batch"))
    # everything is in 64 bits (sums of T terms: T 2^-53 of their magnitudes) and rounded once
    slack = 1e-9 * (1 + np.abs(np.concatenate(want[1:3])).max())
    check_scalar("loss", out.loss, want[0], slack * (1 + abs(want[0])))
    for got, w in ((out.chosen_rewards, want[1]), (out.rejected_rewards, want[2])):
        assert (np.abs(np64(got) - w) <= F32 * np.abs(w) + slack).all()
    # coef rounded, and its products with the upstream gradient
    assert (np.abs(np64(grad) - 3 * want[3]) <= 3.01 * F32 * np.abs(3 * want[3]) + 1e-12).all()
    assert bool((grad[torch.tensor(~mask, device=DEV)] == 0).all()) and bool((grad[-11:] == 0).all())


def test_preference_without_mask_and_reference():
    cu, _, pi, _, _ = batch([100, 3, 700, 5000], seed=4)
    pi_t, cu_t = gpu(pi.reshape(1, -1), cu)
    pi_t.requires_grad_()
    out = P.preference_loss(pi_t, None, cu_t)
    want = op.preference(pi, None, cu)
    check_scalar("loss", out.loss, want[0], 1e-9 * (1 + abs(want[0])))
    grad, = torch.autograd.grad(out.loss, [pi_t])
    assert grad.shape == pi_t.shape and np.allclose(np64(grad)[0], want[3], rtol=3.01 * F32, atol=1e-12)
    with torch.no_grad():
        assert float(P.preference_loss(pi_t, None, cu_t).loss) == float(out.loss)


@pytest.mark.parametrize("score,want,slope", [(np.inf, 0.0, 0.0), (-np.inf, np.inf, -0.5), (np.nan, np.nan, np.nan),
                                              (1e30, 0.0, 0.0), (-1e30, 5e29, -0.5)])
def test_preference_of_extreme_scores(score, want, slope):
    pi, ref, cu = gpu(np.float32([score, 0.0]), np.float32([0.0, 0.0]), np.int32([0, 1, 2]))
    pi.requires_grad_()
    out = P.preference_loss(pi, ref, cu, beta=0.5)
    grad, = torch.autograd.grad(out.loss, [pi])
    assert np.isclose(float(out.loss), want, rtol=1e-6, equal_nan=True)
    assert np.isclose(float(grad[0]), slope, equal_nan=True) and np.isclose(float(grad[1]), -slope, equal_nan=True)


KINDS = [
    dict(), dict(aggregation="sequence"), dict(kl_coef=0.1), dict(kl_coef=0.1, aggregation="sequence", kl_type="k2"),
    dict(kl_coef=0.3, kl_type="k1", dual_clip=1.3), dict(clip_low=0.1, clip_high=0.3, dual_clip=3.0, num_items_in_batch=50),
    dict(clip_low=1.0, clip_high=0.0), dict(aggregation="sequence", num_items_in_batch=9, kl_coef=0.02),
]


def run_policy(cu, mask, lp, old, adv, ref, kw, upstream=1.0):
    lp, old, adv, ref, mask, cu = gpu(lp, old, adv, ref, mask, cu)
    lp.requires_grad_()
    out = P.policy_loss(lp, old, adv, cu, mask=mask, reference_logps=ref, **kw)
    grad, = torch.autograd.grad(out.loss, [lp], torch.tensor(upstream, device=DEV))
    return out, grad


def names(kw):
    new = {"clip_low": "low", "clip_high": "high", "dual_clip": "dual", "num_items_in_batch": "items"}
    return {new.get(k, k): v for k, v in kw.items()}


def check_policy(cu, mask, lp, old, adv, ref, kw, upstream=1.0, fill=np.nan):
    args = [None if v is None else poison(v, mask, fill) for v in (lp, old, ref)]
    adv_in = poison(adv, mask, fill) if adv.shape == lp.shape else adv
    out, grad = run_policy(cu, mask, args[0], args[1], adv_in, args[2], kw, upstream)
    loss, kl, cut, dlp = op.policy(lp, old, adv, cu, mask, ref, **names(kw))
    # terms: the ratio's exponent is off by 1.45 |d| half steps and a rounding of its own, then exp and two products
    d = np.abs(np.float64(lp) - old)[mask].max(initial=0)
    y = 0 if ref is None else np.abs(np.float64(ref) - lp)[mask].max(initial=0)
    off = (1.5 * max(d, y) + 12) * F32
    size = np.exp(d) * np.abs(adv).max(initial=0) + abs(kw.get("kl_coef", 0)) * (np.exp(y) + y)
    per = len(cu) if kw.get("num_items_in_batch") else 1
    check_scalar("loss", out.loss, loss, off * size * max(per, mask.sum() / kw.get("num_items_in_batch", np.inf)))
    check_scalar("kl", out.kl, kl, off * (np.exp(y) + y))
    check_scalar("cut", out.clip_fraction, cut, 0)
    # each token's gradient: relative to its two terms
    bound = np.abs(upstream) * off * size * (np.abs(dlp).max(initial=0) > 0)
    w = np.zeros(lp.size)
    for s, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        m = mask[a:b].sum()
        items = kw.get("num_items_in_batch")
        w[a:b] = 1 / (items or max(mask[:cu[-1]].sum(), 1)) if kw.get("aggregation", "token") == "token" else \
            1 / ((items or len(cu) - 1) * max(m, 1))
    assert (np.abs(np64(grad) - upstream * dlp) <= bound * w + 4 * F32 * np.abs(upstream * dlp)).all()
    assert bool((grad[torch.tensor(~mask, device=DEV)] == 0).all())
    return out, grad


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("kw", KINDS)
@pytest.mark.parametrize("per_token", [True, False])
def test_policy(lengths, kw, per_token):
    print("policy", lengths, kw, per_token, flush=True)
    cu, mask, lp, old, ref = batch(LENGTHS[lengths], seed=2, tail=5)
    mask[-5:] = False
    adv = np.float32(np.random.default_rng(3).standard_normal(lp.size if per_token else len(cu) - 1))
    adv[0] = 0.0
    check_policy(cu, mask, lp, old, adv, ref if "kl_coef" in kw else None, kw, upstream=-2.5)


def test_policy_tail_counts_nowhere_even_unmasked():
    cu, mask, lp, old, ref = batch([300, 5000], tail=70)
    adv = np.float32([1.0, -1.0])
    for kw in (dict(kl_coef=0.1), dict(aggregation="sequence")):
        mask[-70:] = True
        out, grad = run_policy(cu, mask, lp, old, adv, ref, kw)
        mask[-70:] = False
        out2, grad2 = run_policy(cu, mask, lp, old, adv, ref, kw)
        assert float(out.loss) == float(out2.loss) and torch.equal(grad, grad2) and bool((grad[-70:] == 0).all())


@pytest.mark.parametrize("kw", [dict(kl_coef=0.1), dict(aggregation="sequence", kl_coef=0.1)])
def test_policy_that_counts_nothing_is_zero(kw):
    cu, mask, lp, old, ref = batch([30, 500], tail=3)
    mask[:] = False
    out, grad = run_policy(cu, mask, lp * np.nan, old, np.float32([1, 2]), ref, kw)
    assert float(out.loss) == 0 and float(out.kl) == 0 and float(out.clip_fraction) == 0 and bool((grad == 0).all())
    out, grad = run_policy(np.int32([0, 0, 0]), mask[:0], lp[:0], old[:0], np.float32([1, 2]), ref[:0], kw)
    assert float(out.loss) == 0 and grad.shape == (0,)


def test_policy_without_offsets_is_one_sequence():
    _, mask, lp, old, ref = batch([7000], seed=8)
    mask[::2] = True
    cu = np.int32([0, 7000])
    adv = np.float32([0.7])
    a, ga = run_policy(None, mask, lp, old, adv, ref, dict(kl_coef=0.1))
    b, gb = run_policy(cu, mask, lp, old, adv, ref, dict(kl_coef=0.1))
    assert float(a.loss) == float(b.loss) and torch.equal(ga, gb)
    c, gc = run_policy(None, mask, lp, old, np.full(7000, 0.7, np.float32), ref, dict(kl_coef=0.1, aggregation="sequence"))
    assert np.isclose(float(c.loss), float(a.loss), rtol=1e-6) and torch.allclose(gc, ga, rtol=1e-6)


@pytest.mark.parametrize("low,high,dual", [(0.2, 0.25, 1.5), (0.0, 0.0, None), (0.05, 0.05, 3.0)])
def test_policy_cuts_at_the_border_exactly(low, high, dual):
    """Log-ratios on both sides of each border, one fp32 step apart: cut or not as in 64 bits, bit for bit."""
    edges = [np.log1p(high), np.log1p(-low)] + ([np.log(dual)] if dual else [])
    d = []
    for e in edges:
        x = np.float32(e)
        for _ in range(6):
            x = np.nextafter(x, np.float32(-9))
        for _ in range(13):
            d.append(x)
            x = np.nextafter(x, np.float32(9))
    d = np.repeat(np.float32(d), 2)
    for old in (0.0, -0.75):  # exact sums of the two: the difference is the one that was meant, or its rounding
        lp = np.float32(np.float32(old) + d)
        o = np.full(lp.shape, old, np.float32)
        adv = np.float32(np.tile([1.0, -1.0], d.size // 2))
        kw = dict(clip_low=low, clip_high=high, dual_clip=dual)
        out, grad = run_policy(None, np.ones(lp.size, bool), lp, o, adv, None, kw)
        dlp = op.policy(lp, o, adv, None, None, None, low=low, high=high, dual=dual)[3]
        assert np.array_equal(np64(grad) == 0, dlp == 0)
    on, _ = run_policy(None, np.ones(4, bool), np.zeros(4, np.float32), np.zeros(4, np.float32),
                       np.float32([1, -1, 2, -2]), None, dict(clip_low=0.0))
    assert float(on.clip_fraction) == 0  # on-policy tokens are never cut


def test_kl_of_close_and_far_policies_keeps_its_digits():
    """k3 cancels by e^x - 1 - x; each estimate must keep fp32 accuracy relative to itself."""
    x = np.float32(np.concatenate([[0.0], np.geomspace(1e-6, 20, 60), -np.geomspace(1e-6, 20, 60)]))
    for v in x:
        lp, ref = np.float32([-30.0]), np.float32(np.float32(-30.0) + v)
        y = np.float64(ref) - np.float64(lp[0])
        out, grad = run_policy(None, np.ones(1, bool), lp, lp, np.float32([0.0]), np.float32([ref]), dict(kl_coef=1.0))
        want = np.expm1(y) - y
        assert abs(float(out.kl) - want) <= (1.5 * abs(y) + 24) * F32 * want
        assert abs(float(grad[0]) + np.expm1(y)) <= (1.5 * abs(y) + 24) * F32 * abs(np.expm1(y))


def test_inputs_are_checked():
    lp = torch.zeros(10, device=DEV)
    cu = torch.tensor([0, 4, 10], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="even number"):
        P.preference_loss(lp, lp, torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="cu_seqlens"):
        P.preference_loss(lp, lp, cu.long())
    with pytest.raises(ValueError, match="cu_seqlens"):
        P.policy_loss(lp, lp, lp, cu.cpu())
    with pytest.raises(ValueError, match="mask"):
        P.policy_loss(lp, lp, lp, cu, mask=torch.ones(10, device=DEV))
    with pytest.raises(ValueError, match="mask"):
        P.preference_loss(lp, lp, cu, mask=torch.ones(9, dtype=torch.bool, device=DEV))
    with pytest.raises(ValueError, match="reference_logps"):
        P.preference_loss(lp, lp[:5], cu)
    with pytest.raises(ValueError, match="detach"):
        P.policy_loss(lp, torch.zeros(10, device=DEV, requires_grad=True), lp, cu)
    with pytest.raises(ValueError, match="advantages must be"):
        P.policy_loss(lp, lp, lp[:3], cu)
    with pytest.raises(ValueError, match="dual_clip"):
        P.policy_loss(lp, lp, lp, cu, dual_clip=0.9)
    with pytest.raises(ValueError, match="clip_low"):
        P.policy_loss(lp, lp, lp, cu, clip_low=1.2)
    with pytest.raises(ValueError, match="reference"):
        P.policy_loss(lp, lp, lp, cu, kl_coef=0.1)
    with pytest.raises(ValueError, match="beta"):
        P.preference_loss(lp, lp, cu, beta=-1.0)
    with pytest.raises(ValueError, match="one number"):
        P.preference_loss(lp, lp, cu, num_items_in_batch=torch.ones(2, device=DEV))


def test_bad_offsets_touch_nothing_else():
    """Offsets outside the batch, or decreasing, give wrong numbers for their sequences and no access outside."""
    _, mask, lp, old, ref = batch([5000])
    lp_t, old_t, ref_t, mask_t = gpu(lp, old, ref, mask)
    lp_t.requires_grad_()
    for bad in ([0, 4000, 100, 9999, 5000], [-7, 3, 2 ** 31 - 1, -2 ** 31, 20], [9, 9, 9, 9, 9]):
        cu = torch.tensor(bad, dtype=torch.int32, device=DEV)
        out = P.preference_loss(lp_t, ref_t, cu, mask=mask_t)
        torch.autograd.grad(out.loss, [lp_t])
        out = P.policy_loss(lp_t, old_t, torch.ones(4, device=DEV), cu, mask=mask_t, aggregation="sequence")
        torch.autograd.grad(out.loss, [lp_t])
    torch.cuda.synchronize()
    cu = torch.tensor([0, 2500, 5000], dtype=torch.int32, device=DEV)
    good = op.preference(lp, ref, [0, 2500, 5000], mask)
    assert np.isclose(float(P.preference_loss(lp_t, ref_t, cu, mask=mask_t).loss), good[0], rtol=1e-6)


def test_losses_may_be_changed_in_place():
    cu, _, pi, old, ref = batch([30, 40])
    pi_t, old_t, ref_t, cu_t = gpu(pi, old, ref, cu)
    pi_t.requires_grad_()
    for f in (lambda: P.preference_loss(pi_t, ref_t, cu_t).loss, lambda: P.policy_loss(pi_t, old_t, old_t[:2], cu_t).loss):
        want, = torch.autograd.grad(f(), [pi_t])
        loss = f()
        loss /= 4  # gradient accumulation
        got, = torch.autograd.grad(loss, [pi_t])
        assert torch.equal(got * 4, want)


def test_two_streams_a_retained_graph_and_reproducibility():
    cu, mask, lp, old, ref = batch(LENGTHS["slices"], seed=6)
    lp_t, old_t, ref_t, mask_t, cu_t = gpu(lp, old, ref, mask, cu)
    lp_t.requires_grad_()
    adv = torch.randn(len(cu) - 1, device=DEV)

    def call():
        out = P.policy_loss(lp_t, old_t, adv, cu_t, mask=mask_t, reference_logps=ref_t, kl_coef=0.1, aggregation="sequence")
        pair = P.preference_loss(lp_t, ref_t, cu_t, mask=mask_t)
        total = out.loss + 2 * pair.loss
        g1, = torch.autograd.grad(total, [lp_t], retain_graph=True)
        g2, = torch.autograd.grad(total, [lp_t])
        assert torch.equal(g1, g2)
        return total.detach(), g1

    want = call()
    torch.cuda.synchronize()
    got = []
    for st in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(st):
            got.append(call())
    torch.cuda.synchronize()
    for total, g in got:
        assert torch.equal(total, want[0]) and torch.equal(g, want[1])


def test_captured_losses_replay_on_new_values():
    cu, mask, lp, old, ref = batch([500, 2100, 0, 900], seed=9)
    lp_t, old_t, ref_t, mask_t, cu_t = gpu(lp, old, ref, mask, cu)
    adv = torch.randn(4, device=DEV)
    items = torch.tensor(7.0, device=DEV)

    def call(leaf):
        out = P.policy_loss(leaf, old_t, adv, cu_t, mask=mask_t, reference_logps=ref_t, kl_coef=0.1,
                            num_items_in_batch=items)
        pair = P.preference_loss(leaf, ref_t, cu_t, mask=mask_t, order="halves")
        return out.loss.detach(), pair.loss.detach(), *torch.autograd.grad([out.loss, pair.loss], [leaf])

    stream = torch.cuda.Stream()
    leaf = lp_t.clone().requires_grad_()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call(leaf)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(leaf)
    for i in range(3):
        with torch.no_grad():
            leaf.copy_(lp_t + 0.1 * i * torch.randn_like(lp_t))
        adv.copy_(torch.randn(4, device=DEV))
        items.fill_(3.0 + i)
        graph.replay()
        torch.cuda.synchronize()
        want = call(lp_t.clone().copy_(leaf.detach()).requires_grad_())
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_a_second_derivative_is_refused():
    cu, _, pi, old, _ = batch([4, 6])
    pi_t, old_t, cu_t = gpu(pi, old, cu)
    pi_t.requires_grad_()
    for loss in (P.preference_loss(pi_t, old_t, cu_t).loss, P.policy_loss(pi_t, old_t, torch.ones(2, device=DEV), cu_t).loss):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(loss, [pi_t], create_graph=True)


def test_what_is_reported_beside_the_loss_carries_no_graph():
    cu, mask, pi, old, ref = batch([40, 60], seed=3)
    pi_t, old_t, ref_t, mask_t, cu_t = gpu(pi, old, ref, mask, cu)
    pi_t.requires_grad_()
    pair = P.preference_loss(pi_t, ref_t, cu_t, mask=mask_t)
    out = P.policy_loss(pi_t, old_t, torch.ones(2, device=DEV), cu_t, mask=mask_t)
    assert [t.requires_grad for t in pair] == [True, False, False]
    assert [t.requires_grad for t in out] == [True, False, False]
    with torch.no_grad():
        assert not P.preference_loss(pi_t, ref_t, cu_t, mask=mask_t).loss.requires_grad


def test_saved_tensors_go_through_their_hooks():
    cu, mask, pi, old, ref = batch([40, 2500, 60, 7], seed=5)
    pi_t, old_t, ref_t, mask_t, cu_t = gpu(pi, old, ref, mask, cu)
    pi_t.requires_grad_()

    def losses():
        return [P.preference_loss(pi_t, ref_t, cu_t, mask=mask_t).loss, P.preference_loss(pi_t, None, cu_t).loss,
                P.policy_loss(pi_t, old_t, torch.ones(4, device=DEV), cu_t, aggregation="sequence").loss,
                P.policy_loss(pi_t, old_t, pi_t.detach()).loss]

    want = [torch.autograd.grad(loss, [pi_t])[0] for loss in losses()]
    with torch.autograd.graph.save_on_cpu():
        kept = losses()
    for loss, grad in zip(kept, want):
        assert torch.equal(torch.autograd.grad(loss, [pi_t])[0], grad)


def test_two_threads_on_streams_of_their_own():
    data = [batch([500 + 40 * i, 2100, 0, 900], seed=20 + i) for i in range(2)]
    torch.cuda.synchronize()

    def step(cu, mask, lp, old, ref):
        lp_t, old_t, ref_t, mask_t, cu_t = gpu(lp, old, ref, mask, cu)
        lp_t.requires_grad_()
        out = P.policy_loss(lp_t, old_t, torch.ones(4, device=DEV), cu_t, mask=mask_t, reference_logps=ref_t, kl_coef=0.1)
        pair = P.preference_loss(lp_t, ref_t, cu_t, mask=mask_t)
        return [t.cpu() for t in (out.loss.detach(), pair.loss.detach(),
                                  *torch.autograd.grad([out.loss, pair.loss], [lp_t]))]

    want, got = [step(*d) for d in data], [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(step(*data[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 20
        assert all(torch.equal(a, b) for step in got[i] for a, b in zip(step, want[i]))


@pytest.mark.parametrize("kl_type,far", [("k3", 100.0), ("k3", -np.inf), ("k2", 1e30), ("k1", np.inf)])
@pytest.mark.parametrize("tokens", [300, 5000])
def test_a_kl_estimate_that_is_only_reported_leaves_the_loss_alone(tokens, kl_type, far):
    """Coefficient 0: an infinite estimate shows in ``kl`` and nowhere else."""
    cu, mask, lp, old, ref = batch([tokens - 100, 100], seed=11)
    mask[:] = True
    ref[7] = lp[7] + np.float32(far)
    adv = np.float32([1.0, -0.5])
    for aggregation in ("token", "sequence"):
        kw = dict(kl_coef=0.0, kl_type=kl_type, aggregation=aggregation)
        out, grad = run_policy(cu, mask, lp, old, adv, ref, kw)
        lone, want = run_policy(cu, mask, lp, old, adv, None, kw)
        assert not np.isfinite(float(out.kl))
        assert float(out.loss) == float(lone.loss) and torch.equal(grad, want)


@pytest.mark.parametrize("aggregation", ["token", "sequence"])
@pytest.mark.parametrize("tokens", [300, 50_000])
def test_a_batch_that_counts_nothing_is_zero_whatever_is_divided_by(tokens, aggregation):
    """The number of items of a step in which nothing counts is 0."""
    cu, mask, lp, old, ref = batch([tokens - 100, 100])
    mask[:] = False
    for items in (0, torch.zeros((), device=DEV), 3):
        kw = dict(kl_coef=0.1, aggregation=aggregation, num_items_in_batch=items)
        out, grad = run_policy(cu, mask, lp, old, np.float32([1, 2]), ref, kw)
        assert float(out.loss) == 0 and float(out.kl) == 0 and bool((grad == 0).all())


@pytest.mark.parametrize("items", [7, 7.0, torch.tensor(7), torch.tensor([7.0])])
def test_a_number_of_items_on_the_host_costs_no_synchronisation(items):
    cu, mask, lp, old, ref = batch([500, 2100, 40, 900], seed=9)
    lp_t, old_t, ref_t, mask_t, cu_t = gpu(lp, old, ref, mask, cu)
    lp_t.requires_grad_()
    adv = torch.randn(4, device=DEV)
    on_device = torch.tensor(7.0, device=DEV)

    def calls(n):
        a = P.policy_loss(lp_t, old_t, adv, cu_t, mask=mask_t, num_items_in_batch=n).loss
        b = P.preference_loss(lp_t, ref_t, cu_t, mask=mask_t, num_items_in_batch=n).loss
        return a.detach(), b.detach()

    want = calls(on_device)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        got = calls(items)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_captured_call_with_a_number_of_items_replays():
    cu, mask, lp, old, ref = batch([500, 2100, 0, 900], seed=10)
    lp_t, old_t, mask_t, cu_t = gpu(lp, old, mask, cu)
    adv = torch.randn(4, device=DEV)

    def call():
        return P.policy_loss(lp_t, old_t, adv, cu_t, mask=mask_t, num_items_in_batch=7).loss

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(3):
        lp_t.copy_(old_t + 0.3 * torch.randn_like(old_t))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, call())
