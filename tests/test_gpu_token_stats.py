"""Token statistics on the GPU against the oracle in 64 bits: scores, alternatives, gradients kept and formed again."""

import numpy as np
import pytest
import torch

from oracle import token_stats as ots
from siq_vl_amd import cross_entropy as C
from siq_vl_amd import log_probs as LP

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
    ent = 0.3 * torch.randn(n, generator=g)
    return h.to(torch.bfloat16), w, y, up, ent


def on_grid(n, hdim, vocab, seed=0, steps=20):
    """Hidden states and a table whose sums of products are exact in fp32 in any order, so that equal logits are equal:
    multiples of 1 / 16 below 2 and of 1 / 256 below 20 / 256, sums of 320 or fewer products below 2^24 steps."""
    g = torch.Generator().manual_seed(seed)
    h = torch.randint(-31, 32, (n, hdim), generator=g) / 16
    w = torch.randint(-steps, steps + 1, (vocab, hdim), generator=g) / 256
    return h.to(torch.bfloat16), w.to(torch.bfloat16), torch.randint(0, vocab, (n,), generator=g)


def check(h, w, y, up, ent, temperature=1.0, top_k=5, keep=True, chunk=None, need_dw=True, exact_ids=False):
    hd, wd, yd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(need_dw), y.to(DEV)
    out = LP.fused_linear_token_stats(hd, wd, yd, top_k, temperature=temperature, chunk_tokens=chunk,
                                      keep_bytes=1 << 32 if keep else 0, validate=False)
    grads = torch.autograd.grad([out.log_probs, out.entropy], [hd, wd] if need_dw else [hd], [up.to(DEV), ent.to(DEV)])
    torch.cuda.synchronize()
    ref = ots.linear_token_stats(np64(h), np64(w), y.numpy(), top_k, np64(up), np64(ent), temperature, roundings=1 + keep)
    for name, got in (("logp", out.log_probs), ("entropy", out.entropy)):
        assert (np.abs(np64(got) - ref[name]) <= ref[name + "_off"]).all(), name
    if top_k:
        check_top(out, ref, y.numel(), exact_ids)
    else:
        assert out.top_ids is None and out.top_log_probs is None
    skipped = (y == -100) | (y < 0) | (y >= w.shape[0])
    assert bool((out.log_probs[skipped.to(DEV)] == 0).all()) and bool((grads[0][skipped.to(DEV)] == 0).all())
    for name, got in zip(("dh", "dw"), grads):
        assert (np.abs(np64(got) - ref[name]) <= ref[name + "_off"]).all(), name
    return out, grads


def check_top(out, ref, n, exact_ids):
    at, ids, lps = ref["at"], out.top_ids.cpu().numpy(), np64(out.top_log_probs)
    skipped = np.setdiff1d(np.arange(n), at)
    assert (ids[skipped] == -1).all() and (lps[skipped] == 0).all()
    if exact_ids:
        assert (ids == ref["top_ids"]).all()
    ids, lps, off = ids[at], lps[at], ref["off"][:, None]
    assert (ids >= 0).all() and (ids < ref["z"].shape[1]).all()
    assert all(len(set(r)) == len(r) for r in ids.tolist())
    # the logit of each rank is that rank's, but for what a logit may be off by
    best = np.take_along_axis(ref["z"], ref["top_ids"][at], 1)
    assert (np.abs(np.take_along_axis(ref["z"], ids, 1) - best) <= 2 * off).all()
    want = np.take_along_axis(ref["lp"], ids, 1)
    assert (np.abs(lps - want) <= 2 * off + ots.SUM + 4 * ots.FP32 * np.abs(want)).all()
    assert (np.diff(lps, axis=1) <= 0).all()


@pytest.mark.parametrize("keep,chunk", [(True, None), (True, 100), (False, None), (False, 128), (False, 100)])
@pytest.mark.parametrize("n,hdim,vocab,k", [(1, 64, 8, 8), (3, 64, 1000, 1), (50, 896, 520, 20), (64, 64, 2000, 128),
                                            (65, 192, 1000, 5), (128, 320, 4104, 64), (129, 320, 4104, 0), (255, 320, 264, 128),
                                            (257, 128, 2000, 33), (300, 896, 1000, 7)])
def test_against_the_oracle(n, hdim, vocab, k, keep, chunk):
    print(f"stats n={n} h={hdim} V={vocab} K={k} keep={keep} chunk={chunk}", flush=True)
    data = make(n, hdim, vocab, seed=n, ignored=0.3 if n > 1 else 0.0, lean=3.0)
    check(*data, 1.0, k, keep, chunk)
    check(*data, 0.7, k, keep, chunk, need_dw=False)


@pytest.mark.parametrize("n", [1, 40, 128, 300])
@pytest.mark.parametrize("steps", [1, 20])
@pytest.mark.parametrize("k", [1, 20, 128])
def test_equal_logits_go_by_id(n, steps, k):
    """Logits that are exact in fp32: the ids are the definition's, ties among them (with a table of -1, 0 and 1 most of
    them are)."""
    h, w, y = on_grid(n, 128, 4104, seed=n + k, steps=steps)
    w[3000], w[17] = w[5], w[4103]
    ref = ots.linear_token_stats(np64(h), np64(w), y.numpy(), k)
    out = LP.fused_linear_token_stats(h.to(DEV), w.to(DEV), y.to(DEV), k)
    check_top(out, ref, n, True)


@pytest.mark.parametrize("n", [5, 200])
@pytest.mark.parametrize("vocab", [8, 264, 4104])
def test_rows_without_a_difference(n, vocab):
    """Hidden states of zeros: every logit is equal, the first ids win and the entropy is ln V."""
    h, w = torch.zeros(n, 64, dtype=torch.bfloat16), make(1, 64, vocab)[1]
    k = min(vocab, 128)
    out = LP.fused_linear_token_stats(h.to(DEV), w.to(DEV), None, k)
    assert out.log_probs is None
    assert torch.equal(out.top_ids.cpu(), torch.arange(k).expand(n, k))
    off = ots.SUM + 4 * ots.FP32 * np.log(vocab)
    assert float((out.entropy.double() - np.log(vocab)).abs().max()) <= 2 * off
    assert float((out.top_log_probs.double() + np.log(vocab)).abs().max()) <= off


@pytest.mark.parametrize("n", [3, 100, 300])
@pytest.mark.parametrize("offset", [-2048.0, 2048.0])
@pytest.mark.parametrize("features", [2, 128])
def test_logits_with_a_large_part_in_common(n, offset, features):
    """Logits next to +-2048, exact in fp32 (steps of 2^-12): apart by less than 0.01 all of them, or by some units."""
    h, w, y = on_grid(n, 128, 4104, seed=n)
    h[:, features:] = 0
    h[:, 0], w[:, 0] = 2048.0, offset / 2048
    for k in (1, 64):
        ref = ots.linear_token_stats(np64(h), np64(w), y.numpy(), k)
        out = LP.fused_linear_token_stats(h.to(DEV), w.to(DEV), y.to(DEV), k)
        check_top(out, ref, n, True)
        for name, got in (("logp", out.log_probs), ("entropy", out.entropy)):
            assert (np.abs(np64(got) - ref[name]) <= ref[name + "_off"]).all(), name


@pytest.mark.parametrize("n", [5, 200])
def test_sorted_logits_in_either_direction(n):
    """All large logits beside one another: parts of rows that hold more than their share of the alternatives."""
    vocab = 8192
    h = torch.zeros(n, 64)
    h[:, 0] = 1.0
    for ramp in (torch.arange(vocab), torch.arange(vocab).flip(0)):
        w = torch.zeros(vocab, 64)
        w[:, 0] = (ramp // 64) / 16  # runs of 64 equal ones
        y = torch.full((n,), 1)
        h16, w16 = h.to(torch.bfloat16), w.to(torch.bfloat16)
        ref = ots.linear_token_stats(np64(h16), np64(w16), y.numpy(), 128)
        out = LP.fused_linear_token_stats(h16.to(DEV), w16.to(DEV), y.to(DEV), 128)
        check_top(out, ref, n, True)


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("n", [40, 300])
def test_far_apart_logits(n, keep):
    """Logits a hundred apart: probabilities that vanish beside others."""
    check(*make(n, 128, 1000, seed=6, wscale=2.0), 1.0, 9, keep)
    check(*make(n, 128, 1000, seed=6, wscale=2.0), 0.25, 9, keep)


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("n", [40, 300])
def test_near_certain_tokens_keep_their_digits(n, keep):
    """Log-probabilities and entropies of 1e-9: right relative to themselves."""
    g = torch.Generator().manual_seed(3)
    w = (0.05 * torch.randn(1000, 256, generator=g)).to(torch.bfloat16)
    y = torch.randint(0, 1000, (n,), generator=g)
    h = (torch.linspace(12, 32, n)[:, None] * w[y].float() / (0.05 ** 2 * 256)).to(torch.bfloat16)
    out, _ = check(h, w, y, torch.ones(n), torch.ones(n), 1.0, 3, keep)
    z = np64(h) @ np64(w).T
    off = 2 * 36 * 2.0 ** -24 * (np.abs(np64(h)) @ np.abs(np64(w)).T).max(1) + 64 * 2.0 ** -24
    gap = np.array([np.delete(r, k) - r[k] for r, k in zip(z, y.numpy())])
    rest = np.exp(gap).sum(1)
    logp, ent = -np.log1p(rest), np.log1p(rest) - (np.exp(gap) * gap).sum(1) / (1 + rest)
    assert logp.max() > -1e-8 and (np.abs(np64(out.log_probs) - logp) <= off * np.abs(logp)).all()
    # (an exponent's error weighs with the exponent there)
    assert (np.abs(np64(out.entropy) - ent) <= 2 * off * ent).all()


@pytest.mark.parametrize("keep", [True, False])
def test_nothing_counts_no_rows_and_bad_labels(keep):
    h, w, y, up, ent = make(300, 128, 1000, seed=8)
    y[:] = -100
    _, grads = check(h, w, y, up, ent, 1.0, 4, keep)
    assert bool((grads[1] == 0).all())
    hd, wd = h[:0].to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    out = LP.fused_linear_token_stats(hd, wd, y[:0].to(DEV), 4, keep_bytes=1 << 32 if keep else 0)
    assert out.log_probs.shape == out.entropy.shape == (0,) and out.top_ids.shape == (0, 4)
    dh, dw = torch.autograd.grad(out.entropy.sum(), [hd, wd])
    assert dh.shape == (0, 128) and bool((dw == 0).all())
    y[:] = 5
    y[3], y[200] = 1000, -7
    up[3], ent[200] = float("nan"), float("nan")  # of rows that do not count
    check(h, w, y, up.nan_to_num(), ent.nan_to_num(), 1.0, 4, keep)
    hd, wd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    out = LP.fused_linear_token_stats(hd, wd, y.to(DEV), 4, keep_bytes=1 << 32 if keep else 0, validate=False)
    grads = torch.autograd.grad([out.log_probs, out.entropy], [hd, wd], [up.to(DEV), ent.to(DEV)])
    assert not any(bool(x.isnan().any()) for x in grads)
    with pytest.raises(C.LabelError, match="2 label"):
        LP.fused_linear_token_stats(h.to(DEV), w.to(DEV), y.to(DEV), 4, validate="sync")
    C.check_pending_labels(block=True)
    LP.fused_linear_token_stats(h.to(DEV), w.to(DEV), y.to(DEV))
    with pytest.raises(C.LabelError, match="2 label"):
        C.check_pending_labels(block=True)


@pytest.mark.parametrize("n", [40, 300])
def test_rows_that_are_not_numbers_stay_among_themselves(n):
    h, w, y, up, ent = make(n, 128, 1000, seed=9, ignored=0.0)
    clean = LP.fused_linear_token_stats(h.to(DEV), w.to(DEV), y.to(DEV), 6)
    h[7], h[11, 5] = float("nan"), float("inf")
    out = LP.fused_linear_token_stats(h.to(DEV), w.to(DEV), y.to(DEV), 6)
    odd = torch.zeros(n, dtype=torch.bool, device=DEV)
    odd[7] = odd[11] = True
    for a, b in zip(out, clean):
        assert torch.equal(a[~odd], b[~odd])
    assert bool(out.log_probs[odd].isnan().all()) and bool(out.entropy[odd].isnan().all())
    assert bool(out.top_log_probs[odd].isnan().all())
    assert int(out.top_ids.min()) >= 0 and int(out.top_ids.max()) < 1000


def test_one_gradient_alone_and_the_log_probabilities_own():
    h, w, y, up, ent = make(300, 128, 1000, seed=10)
    hd, wd, yd, ud = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), y.to(DEV), up.to(DEV)
    zero = torch.zeros_like(ud)
    for keep in (0, 1 << 32):
        out = LP.fused_linear_token_stats(hd, wd, yd, keep_bytes=keep)
        for which, both in ((out.log_probs, [ud, zero]), (out.entropy, [zero, ud])):
            got = torch.autograd.grad(which, [hd, wd], ud, retain_graph=True)
            want = torch.autograd.grad([out.log_probs, out.entropy], [hd, wd], both, retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    # the same log-probabilities as fused_linear_log_probs, each within its bound of the exact ones
    ref = ots.linear_token_stats(np64(h), np64(w), y.numpy())
    other = LP.fused_linear_log_probs(hd, wd, yd)
    assert (np.abs(np64(out.log_probs) - np64(other)) <= 2 * ref["logp_off"]).all()


def test_autograd_shapes_types_frozen_and_retained():
    h, w, y, up, ent = make(60, 128, 520, seed=11)
    hg = h.view(4, 15, 128).to(DEV).requires_grad_()
    wg, yd, ud, ed = w.to(DEV).requires_grad_(), y.view(4, 15).to(DEV), up.view(4, 15).to(DEV), ent.view(4, 15).to(DEV)
    out = LP.fused_linear_token_stats(hg, wg, yd, 3, temperature=1.3)
    assert out.log_probs.shape == out.entropy.shape == (4, 15) and out.top_ids.shape == out.top_log_probs.shape == (4, 15, 3)
    assert out.top_ids.dtype == torch.int64 and not out.top_log_probs.requires_grad
    want = torch.autograd.grad([out.log_probs, out.entropy], [hg, wg], [ud, ed], retain_graph=True)
    again = torch.autograd.grad([out.log_probs, out.entropy], [hg, wg], [ud, ed])
    assert all(torch.equal(a, b) for a, b in zip(want, again)) and want[0].shape == hg.shape
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out.entropy.sum(), [hg])
    frozen = LP.fused_linear_token_stats(hg, wg.detach(), yd, temperature=1.3)
    assert torch.equal(torch.autograd.grad([frozen.log_probs, frozen.entropy], [hg], [ud, ed])[0], want[0])
    head = LP.fused_linear_token_stats(hg.detach(), wg, yd, temperature=1.3)
    assert torch.equal(torch.autograd.grad([head.log_probs, head.entropy], [wg], [ud, ed])[0], want[1])
    with torch.no_grad():
        lone = LP.fused_linear_token_stats(hg, wg, yd, 3, temperature=1.3)
    assert lone.entropy.grad_fn is None and all(torch.equal(a, b) for a, b in zip(lone, out))
    # strided operands, fp32 master copies, labels given or not
    wide = torch.zeros(4, 15, 256, dtype=torch.bfloat16, device=DEV)
    wide[..., :128] = hg.detach()
    strided = LP.fused_linear_token_stats(wide[..., :128], wg.detach().T.contiguous().T, yd, 3, temperature=1.3)
    assert all(torch.equal(a, b) for a, b in zip(strided, lone))
    h32, w32 = hg.detach().float().requires_grad_(), wg.detach().float().requires_grad_()
    out = LP.fused_linear_token_stats(h32, w32, yd, temperature=1.3)
    got = torch.autograd.grad([out.log_probs, out.entropy], [h32, w32], [ud, ed])
    assert got[0].dtype == torch.float32 and all(torch.equal(a, b.float()) for a, b in zip(got, want))
    free = LP.fused_linear_token_stats(hg, wg.detach(), None, 3, temperature=1.3)
    at = (yd >= 0)
    assert free.log_probs is None and torch.equal(free.top_ids[at], lone.top_ids[at])
    assert float((free.entropy.detach() - lone.entropy)[at].abs().max()) <= 1e-5
    # their gradient in a row that counts in both is the same entropy's
    g1, = torch.autograd.grad(free.entropy, [hg], torch.where(at, ed, 0.0))
    g2, = torch.autograd.grad(LP.fused_linear_token_stats(hg, wg.detach(), yd, temperature=1.3).entropy, [hg], ed)
    ref = ots.linear_token_stats(np64(h), np64(w), y.numpy(), 0, None, np64(ent), 1.3, roundings=2)
    assert (np.abs(np64(g1 - g2)).reshape(60, 128) <= 2 * ref["dh_off"]).all()


@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("n", [60, 300])
def test_results_may_be_changed_in_place(n, keep):
    h, w, y, up, ent = make(n, 128, 520, seed=16)
    hd, wd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()

    def call(change):
        out = LP.fused_linear_token_stats(hd, wd, y.to(DEV), 3, keep_bytes=1 << 32 if keep else 0)
        a, b = out.log_probs, out.entropy
        if change:
            a *= 2.0
            b += 7.0
            out.top_log_probs.zero_()
        else:
            a = 2.0 * a
        return torch.autograd.grad([a, b], [hd, wd], [up.to(DEV), ent.to(DEV)])

    assert all(torch.equal(a, b) for a, b in zip(call(True), call(False)))


@pytest.mark.parametrize("n", [2, 128, 300])
def test_one_token_for_all_rows(n):
    h, w, y, up, ent = make(n, 128, 1000, seed=17, ignored=0.0)
    y[:] = 999
    check(h, w, y, up, ent)


@pytest.mark.parametrize("n", [3, 300])
def test_more_columns_than_a_row_pass_holds(n):
    """270,336 columns: rows of more parts than are read once, scores and gradients."""
    vocab = 270_336
    h, w, y = on_grid(n, 64, vocab, seed=n)
    y[-1] = vocab - 1
    hd, wd = h.to(DEV).requires_grad_(), w.to(DEV)
    out = LP.fused_linear_token_stats(hd, wd, y.to(DEV), 40)
    z = h.to(DEV).double() @ wd.double().T.contiguous()
    key = (z * 4096).round().long() * 2 ** 19 + (vocab - 1 - torch.arange(vocab, device=DEV))
    want = vocab - 1 - key.topk(40, dim=1).values.remainder(2 ** 19)
    assert torch.equal(out.top_ids, want)
    lp = torch.log_softmax(z, 1)
    off = 2 * ots.SUM + 8 * ots.FP32 * lp.abs().amax(1)
    assert bool(((out.log_probs.double() - lp.gather(1, y.to(DEV)[:, None])[:, 0]).abs() <= off).all())
    assert bool(((out.top_log_probs.double() - lp.gather(1, want)).abs() <= off[:, None]).all())
    H = -(lp.exp() * lp).sum(1)
    assert bool(((out.entropy.double() - H).abs() <= 3 * off * (1 + H)).all())
    dh, = torch.autograd.grad(out.entropy.sum(), [hd])
    dz = -lp.exp() * (lp + H[:, None])
    want, size = dz @ wd.double(), (2 * dz.abs() + lp.exp()) @ wd.double().abs()
    assert bool(((dh.double() - want).abs() <= 2.0 ** -8 * (1.1 * size + want.abs())).all())


@pytest.mark.parametrize("k", [1, 20, 128])
@pytest.mark.parametrize("shape", ["random", "rising", "falling", "flat", "late"])
def test_bounded_alternatives_of_a_real_vocabulary(shape, k):
    """1,100 rows of 151,936 columns: an eighth of them (or more, for more alternatives) bounds what is written of the others.
    Logits are exact, so ids are the definition's: ties, sorted logits, all equal ones, and all large ones at the end."""
    n, vocab = 1100, 151_936
    print(f"stats bounded {shape} K={k}", flush=True)
    h, w, y = on_grid(n, 64, vocab, seed=k)
    if shape != "random":
        h[:], w[:] = 0, 0
        h[:, 0] = 1.0
        place = torch.arange(vocab)
        w[:, 0] = {"rising": place // 1024 / 4, "falling": (vocab - 1 - place) // 1024 / 4, "flat": torch.zeros(vocab),
                   "late": (place >= vocab - 300) * 1.0}[shape]
    y[::7] = -100
    out = LP.fused_linear_token_stats(h.to(DEV), w.to(DEV), y.to(DEV), k)
    at = (y >= 0).to(DEV)
    assert bool((out.top_ids[~at] == -1).all())
    hd, wd = h.to(DEV).double()[at], w.to(DEV).double()
    ids, lps = out.top_ids[at], out.top_log_probs[at]
    for c in range(0, ids.shape[0], 200):
        z = hd[c:c + 200] @ wd.T.contiguous()
        key = (z * 4096).round().long() * 2 ** 18 + (vocab - 1 - torch.arange(vocab, device=DEV))
        assert torch.equal(ids[c:c + 200], vocab - 1 - key.topk(k, dim=1).values.remainder(2 ** 18))
        want = torch.log_softmax(z, 1).gather(1, ids[c:c + 200])
        assert bool(((lps[c:c + 200].double() - want).abs() <= ots.SUM + 4 * ots.FP32 * want.abs()).all())


def test_gradient_is_a_difference():
    """One direction in ``hidden``, central differences of the fp32 results."""
    h, w, y, up, ent = make(64, 128, 520, seed=12, ignored=0.1)
    g = torch.Generator().manual_seed(1)
    h = (h.float() * 8).round().div(8).to(torch.bfloat16)  # steps of 1 / 8 below 16: moved by 1 / 16 exactly
    d = (torch.randint(-1, 2, h.shape, generator=g) / 16).to(torch.bfloat16)
    hd, wd, yd, dd = h.to(DEV).requires_grad_(), w.to(DEV), y.to(DEV), d.to(DEV)
    out = LP.fused_linear_token_stats(hd, wd, yd)
    dh, = torch.autograd.grad([out.log_probs, out.entropy], [hd], [up.to(DEV), ent.to(DEV)])
    val = [LP.fused_linear_token_stats(hd.detach() + s * dd, wd, yd) for s in (1, -1)]
    num = sum(g * np64(a - b) / 2 for g, a, b in ((np64(up), val[0].log_probs, val[1].log_probs),
                                                   (np64(ent), val[0].entropy, val[1].entropy)))
    got = (dh.double() * dd.double()).sum(1).cpu().numpy()
    ref = ots.linear_token_stats(np64(h), np64(w), y.numpy(), 0, np64(up), np64(ent), roundings=2)
    # with s what a row's move changes a logit by at most: the third derivative of the logsumexp is at most 2 s^3, of the
    # entropy (whose logarithms reach ln V and what the logits spread) at most 8 s^3 (1 + ln V + their spread)
    s = np.linalg.norm(np64(d), axis=1) * np.linalg.norm(np64(w), axis=1).max()
    spread = 1 + np.log(520) + np.ptp(np64(h) @ np64(w).T, axis=1)
    bound = np.abs(np64(up)) * (s ** 3 / 3 + ref["logp_off"]) + np.abs(np64(ent)) * (4 * s ** 3 / 3 * spread + ref["entropy_off"])
    assert (np.abs(num - got) <= bound + (ref["dh_off"] * np.abs(np64(d))).sum(1) + 1e-9).all()


def test_streams_devices_and_captured_calls():
    h, w, y, up, ent = (t.to(DEV) for t in make(500, 128, 4104, seed=14))

    def call(keep):
        hg, wg = h.detach().requires_grad_(), w.detach().requires_grad_()
        out = LP.fused_linear_token_stats(hg, wg, y, 9, chunk_tokens=256, keep_bytes=keep)
        return [*(x.detach() for x in out), *torch.autograd.grad([out.log_probs, out.entropy], [hg, wg], [up, ent])]

    want = [call(0), call(1 << 32)]
    torch.cuda.synchronize()
    got = []
    for st in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(st):
            got.append([call(0), call(1 << 32)])
    torch.cuda.synchronize()
    for pair in got:
        for a, b in zip(pair, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs = []
    for keep in (0, 1 << 32):  # two graphs, each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((keep, graph, call(keep)))
    for i in range(3):
        h.copy_(torch.randn_like(h))
        y.copy_(y.roll(1))
        up.copy_(torch.randn_like(up))
        for _, graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for keep, _, captured in graphs:
            assert all(torch.equal(p, q) for p, q in zip(captured, call(keep)))


def test_a_second_derivative_and_a_tangent_are_refused():
    h, w, y, _, _ = (t.to(DEV) for t in make(20, 64, 264))
    hg = h.clone().requires_grad_()
    out = LP.fused_linear_token_stats(hg, w, y)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.entropy.sum(), [hg], create_graph=True)
    fw = torch.autograd.forward_ad
    for grad in (False, True):
        with fw.dual_level(), torch.set_grad_enabled(grad):
            with pytest.raises(RuntimeError, match="forward-mode"):
                LP.fused_linear_token_stats(fw.make_dual(h, h), w, y)


def test_refusals_on_the_gpu():
    h, w, y, _, _ = (t.to(DEV) for t in make(20, 64, 264))
    for kw, text in ((dict(top_k=129), "top_k"), (dict(top_k=-1), "top_k"), (dict(temperature=0.0), "temperature"),
                     (dict(weight=w.cpu()), "weight must live on"), (dict(labels=y.cpu()), "labels must live on"),
                     (dict(labels=y.int()), "labels must be int64"), (dict(weight=w[:260 // 8 * 8 + 3]), "multiple of 8")):
        args = dict(hidden=h, weight=w, labels=y)
        args.update(kw)
        with pytest.raises(ValueError, match=text):
            LP.fused_linear_token_stats(**args)
    with pytest.raises(ValueError, match="top_k"):
        LP.fused_linear_token_stats(h, w[:8], None, 9)


@pytest.mark.parametrize("n,hdim,k,train", [(1, 896, 20, False), (48, 896, 5, True), (128, 1536, 128, True), (129, 896, 64, True),
                                            (400, 320, 0, True)])
@pytest.mark.parametrize("keep", [True, False])
def test_a_real_vocabulary(n, hdim, k, train, keep):
    """151,936 columns, against the definition in 64 bits on the GPU; bounds as the oracle's."""
    vocab, half, t, fp32 = 151_936, 2.0 ** -8, 0.8, 2.0 ** -24
    print(f"stats real n={n} h={hdim} K={k} train={train} keep={keep}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(n + hdim)
    w = (0.05 * torch.randn(vocab, hdim, generator=g, device=DEV)).to(torch.bfloat16)
    y = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    lean = 20 * torch.rand(n, 1, generator=g, device=DEV) / (0.05 ** 2 * hdim)
    h = (torch.randn(n, hdim, generator=g, device=DEV) + lean * w[y].float()).to(torch.bfloat16)
    up, ent = torch.randn(n, generator=g, device=DEV), torch.randn(n, generator=g, device=DEV)
    if n > 1:
        y[::5], y[1], y[n - 1] = -100, vocab - 1, 0
        up[::5] = float("nan")
    hg, wg = h.requires_grad_(train), w.requires_grad_(train)
    out = LP.fused_linear_token_stats(hg, wg, y, k, temperature=t, keep_bytes=1 << 36 if keep else 0)
    at = (y >= 0).nonzero()[:, 0]
    hk, wd, yk = h.detach()[at].double(), w.detach().double(), y[at]
    rows = torch.arange(at.numel(), device=DEV)
    z = hk @ wd.T.contiguous() / t
    lp = torch.log_softmax(z, 1)
    p = lp.exp()
    H = -(p * lp).sum(1)
    wabs = wd.abs()
    off = (hdim / 8 + 4) * fp32 * (hk.abs() @ wabs.T.contiguous()).amax(1) / t + 2 * fp32 * z.abs().amax(1)
    assert bool(((out.log_probs[at].double() - lp[rows, yk]).abs() <= 2 * off + ots.SUM + 4 * fp32 * lp[rows, yk].abs()).all())
    slope = (p * (lp + H[:, None])).abs()
    bound = off * slope.sum(1) + ots.SUM * (1 + 2 * (p * lp).abs().sum(1)) + 4 * fp32 * H
    assert bool(((out.entropy[at].double() - H).abs() <= bound).all())
    if k:
        ids = out.top_ids[at]
        assert bool(((z.gather(1, ids) - z.topk(k, 1).values).abs() <= 2 * off[:, None]).all())
        assert all(len(set(r)) == k for r in ids.tolist())
        want = lp.gather(1, ids)
        assert bool(((out.top_log_probs[at].double() - want).abs() <= 2 * off[:, None] + ots.SUM + 4 * fp32 * want.abs()).all())
    if not train:
        return
    dh, dw = torch.autograd.grad([out.log_probs, out.entropy], [hg, wg], [up, ent])
    gk, ek = up[at].double()[:, None] / t, ent[at].double()[:, None] / t
    dz = -p * (gk + ek * (lp + H[:, None]))
    soft = dz.abs() * (1 + keep) + (ek.abs() * p if keep else 0)
    soft[rows, yk] = 0.0
    rel = (2 * off + 2 * ots.SUM + 8 * fp32)[:, None]
    size = half * soft + rel * p * (gk.abs() + ek.abs() * ((lp + H[:, None]).abs() + 1 + H[:, None]))
    dz[rows, yk] += gk[:, 0]
    size[rows, yk] += (rel * (gk.abs() + ek.abs()))[:, 0] + 8 * fp32 * dz[rows, yk].abs()
    want = dz @ wd
    assert bool(((dh[at].double() - want).abs() <= 1.05 * (size @ wabs + half * want.abs()) + 1e-30).all())
    want = dz.T.contiguous() @ hk
    assert bool(((dw.double() - want).abs() <= 1.05 * (size.T.contiguous() @ hk.abs() + half * want.abs()) + 1e-30).all())


def test_more_kept_numerators_than_32_bits_count():
    """16,390 rows of 151,936 columns: 2.5e9 numerators and logits offsets of 1e10 bytes; kept against formed again."""
    n, hdim, vocab = 16_390, 64, 151_936
    g = torch.Generator(device=DEV).manual_seed(6)
    h = torch.randn(n, hdim, generator=g, device=DEV).to(torch.bfloat16).requires_grad_()
    w = (0.3 * torch.randn(vocab, hdim, generator=g, device=DEV)).to(torch.bfloat16).requires_grad_()
    y = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    y[100:130], y[n - 1] = -100, vocab - 1
    up, ent = torch.randn(n, generator=g, device=DEV), torch.randn(n, generator=g, device=DEV)
    got = []
    for keep in (1 << 36, 0):
        out = LP.fused_linear_token_stats(h, w, y, 3, keep_bytes=keep)
        got.append([*(x.detach() for x in out), *torch.autograd.grad([out.log_probs, out.entropy], [h, w], [up, ent])])
    assert all(torch.equal(a, b) for a, b in zip(got[0][:4], got[1][:4]))
    wd, wt = w.detach().double(), w.detach().double().T.contiguous()
    half = 2.0 ** -8
    for c in (0, n - 300):  # the first rows and the last
        at = c + (y[c:c + 300] >= 0).nonzero()[:, 0]
        z = h.detach()[at].double() @ wt
        lp = torch.log_softmax(z, 1)
        p, rows = lp.exp(), torch.arange(at.numel(), device=DEV)
        H = -(p * lp).sum(1, keepdim=True)
        off = 2 * (hdim / 8 + 4) * 2.0 ** -24 * (h.detach()[at].double().abs() @ wt.abs()).amax(1) + ots.SUM
        assert bool(((got[0][0][at].double() - lp[rows, y[at]]).abs() <= off + 4 * 2.0 ** -24 * lp[rows, y[at]].abs()).all())
        assert bool(((got[0][2][at].double() - lp.topk(3, 1).values).abs() <= 2 * off[:, None]).all())
        gk, ek = up[at].double()[:, None], ent[at].double()[:, None]
        dz = -p * (gk + ek * (lp + H))
        soft = 2 * dz.abs() + ek.abs() * p
        soft[rows, y[at]] = 0
        size = half * soft + 4 * (off[:, None] + ots.SUM) * p * (gk.abs() + ek.abs() * ((lp + H).abs() + 1 + H))
        dz[rows, y[at]] += gk[:, 0]
        size[rows, y[at]] += (4 * off[:, None] * (gk.abs() + ek.abs()))[:, 0]
        want = dz @ wd
        for r in got:
            assert bool(((r[4][at].double() - want).abs() <= 1.05 * (size @ wd.abs() + half * want.abs()) + 1e-30).all())
    # dW: each is at most one and a half roundings of E and a sum of n products away from the other
    spread = (got[0][5].double() - got[1][5].double()).norm() / got[1][5].double().norm()
    assert float(spread) <= 4 * half
    assert bool((got[0][4][100:130] == 0).all())


def test_a_model_scores_its_tokens():
    transformers = pytest.importorskip("transformers")
    from siq_vl_amd.cross_entropy import shift_labels
    from siq_vl_amd.text_model import enable_fused_cross_entropy

    cfg = transformers.Qwen2Config(vocab_size=264, hidden_size=128, intermediate_size=256, num_hidden_layers=1,
                                   num_attention_heads=4, num_key_value_heads=2)
    torch.manual_seed(2)
    model = transformers.Qwen2ForCausalLM(cfg).to(DEV, torch.bfloat16)
    ids = torch.randint(0, 264, (2, 30), device=DEV)
    labels = ids.clone()
    labels[:, :7] = -100
    logits = model(input_ids=ids, use_cache=False).logits
    enable_fused_cross_entropy(model)
    out = model(input_ids=ids, labels=labels, use_cache=False, return_log_probs=True, top_k=4)
    assert out.loss is None and out.top_ids.shape == out.top_log_probs.shape == (2, 30, 4)
    targets = shift_labels(labels)
    lp = torch.log_softmax(logits.float(), -1)
    # the stock path rounds its logits to bf16: half a step of the largest of them, twice
    off = 2 * 2.0 ** -8 * float(logits.abs().max()) + 1e-4
    at = targets != -100
    assert float((out.log_probs - lp.gather(-1, targets.clamp(min=0)[..., None])[..., 0])[at].abs().max()) <= off
    assert float((out.top_log_probs - lp.topk(4, -1).values)[at].abs().max()) <= off
    assert bool((out.top_ids[~at] == -1).all())
    alone = model(input_ids=ids, labels=labels, use_cache=False, return_log_probs=True, top_k=0)
    assert alone.top_ids is None and torch.equal(alone.entropy, out.entropy)
    alone.entropy.sum().backward()
    assert all(bool(p.grad.isfinite().all()) for p in model.parameters() if p.grad is not None)
