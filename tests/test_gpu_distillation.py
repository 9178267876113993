"""Distillation on the GPU against the oracle in 64 bits, and together with the token statistics that a teacher gives."""

import numpy as np
import pytest
import torch

from oracle import distillation as od
from siq_vl_amd import cross_entropy as C
from siq_vl_amd import distillation as D
from siq_vl_amd import log_probs as LP

pytestmark = pytest.mark.gpu
DEV = "cuda"


def np64(t):
    return t.detach().double().cpu().numpy()


def make(n, hdim, vocab, k, seed=0, ignored=0.3, wscale=0.05, lean=2.0, mass=0.9):
    """A student that leans towards its teacher's first token; labels from the teacher's tokens or any."""
    g = torch.Generator().manual_seed(seed)
    w = (wscale * torch.randn(vocab, hdim, generator=g)).to(torch.bfloat16)
    ids = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(n)])
    lt = torch.log_softmax(1.5 * torch.randn(n, k, generator=g), 1) + float(np.log(mass))
    y = torch.where(torch.rand(n, generator=g) < 0.7, ids[:, k // 2], torch.randint(0, vocab, (n,), generator=g))
    h = torch.randn(n, hdim, generator=g) + lean * torch.rand(n, 1, generator=g) * w[ids[:, 0]].float() / (wscale ** 2 * hdim)
    y[torch.rand(n, generator=g) < ignored] = -100
    return h.to(torch.bfloat16), w, y, ids, lt


def check(h, w, y, ids, lt, chunk=None, need_dw=True, redone=False, upstream=1.0, **kw):
    hd, wd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(need_dw)
    args = dict(kw)
    divisor = args.pop("divisor", None)
    out = D.fused_linear_distillation(hd, wd, y.to(DEV), ids.to(DEV), lt.to(DEV), chunk_tokens=chunk, validate=False,
                                      num_items_in_batch=divisor, **args)
    grads = torch.autograd.grad(out.loss * upstream, [hd, wd] if need_dw else [hd])
    torch.cuda.synchronize()
    ref = od.linear_distillation(np64(h), np64(w), y.numpy(), ids.numpy(), np64(lt), redone=redone, **kw)
    for name in ("loss", "divergence", "cross_entropy"):
        got = float(getattr(out, name).detach())
        assert abs(got - ref[name]) <= ref[name + "_off"], (name, got, ref[name], ref[name + "_off"])
    for name, got in zip(("dh", "dw"), grads):
        # (scaling rounds once more unless it is by 1)
        off = upstream * ref[name + "_off"] + (upstream != 1.0) * 2.0 ** -8 * np.abs(upstream * ref[name])
        assert (np.abs(np64(got) - upstream * ref[name]) <= 1.01 * off).all(), name
    with torch.no_grad():
        alone = D.fused_linear_distillation(hd, wd, y.to(DEV), ids.to(DEV), lt.to(DEV), validate=False,
                                            num_items_in_batch=divisor, **args)
    assert all(abs(float(a) - float(b)) <= 2 * ref[n + "_off"] for n, a, b in zip(out._fields, alone, out))
    return out, grads, ref


KINDS = [dict(), dict(tail=False), dict(ce_weight=0.3), dict(ce_weight=1.0), dict(temperature=1.7), dict(divergence="reverse"),
         dict(divergence="reverse", ce_weight=0.2), dict(divisor=77.0, tail=False, ce_weight=0.5)]


@pytest.mark.parametrize("kind", range(len(KINDS)))
@pytest.mark.parametrize("n,hdim,vocab,k", [(1, 64, 8, 8), (1, 64, 1000, 1), (50, 896, 520, 20), (64, 64, 2000, 128),
                                            (65, 192, 1000, 5), (128, 320, 4104, 64), (129, 320, 4104, 1), (255, 320, 264, 128),
                                            (257, 128, 2000, 33)])
def test_against_the_oracle(n, hdim, vocab, k, kind):
    print(f"distill n={n} h={hdim} V={vocab} K={k} {KINDS[kind]}", flush=True)
    check(*make(n, hdim, vocab, k, seed=n, ignored=0.3 if n > 1 else 0.0), **KINDS[kind])


@pytest.mark.parametrize("chunk", [64, 100, 128, 256, 300])
@pytest.mark.parametrize("kind", [2, 6])
def test_in_chunks(chunk, kind):
    print(f"distill chunk={chunk} {KINDS[kind]}", flush=True)
    check(*make(700, 192, 1000, 9, seed=chunk), chunk=chunk, **KINDS[kind])
    check(*make(90, 192, 1000, 9, seed=chunk), chunk=chunk, need_dw=False, **KINDS[kind])


@pytest.mark.parametrize("n", [50, 300])
@pytest.mark.parametrize("kind", range(len(KINDS)))
def test_what_a_teacher_leaves_out_or_names_twice(n, kind):
    h, w, y, ids, lt = make(n, 128, 1000, 12, seed=kind)
    ids[1] = -1                                # a row that names nothing
    ids[3, 4:], lt[5, ::2] = -1, -np.inf       # names less
    lt[7] = -np.inf
    ids[9, 1], ids[11, :] = ids[9, 0], ids[11, 3]  # names twice, and one token twelve times
    ids[13, 2], ids[15, 3], ids[17, 0] = 1000, -2, 2 ** 40
    ids[19, 0] = y[19] = 999
    for name, i in (("int64", ids), ("int32", ids.where(ids < 2 ** 31, 2 ** 31 - 1).int())):
        hd, wd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        kw = dict(KINDS[kind])
        divisor = kw.pop("divisor", None)
        out = D.fused_linear_distillation(hd, wd, y.to(DEV), i.to(DEV), lt.to(DEV), validate=False, num_items_in_batch=divisor, **kw)
        got = [x.detach() for x in out] + list(torch.autograd.grad(out.loss, [hd, wd]))
        if name == "int64":
            first = got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
    _, _, ref = check(h, w, y, ids, lt, **KINDS[kind])
    assert ref["bad_tokens"] > 0
    C.check_pending_labels(block=True)
    kw.update(num_items_in_batch=divisor)
    with pytest.raises(D.TeacherError, match=f"{ref['bad_tokens']} of the teacher's tokens"):
        D.fused_linear_distillation(h.to(DEV), w.to(DEV), y.to(DEV), ids.to(DEV), lt.to(DEV), validate="sync", **kw)
    D.fused_linear_distillation(h.to(DEV), w.to(DEV), y.to(DEV), ids.to(DEV), lt.to(DEV), **kw)
    with pytest.raises(D.TeacherError):
        C.check_pending_labels(block=True)


@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("kind", [0, 1, 2, 5])
def test_a_teacher_of_all_mass_and_of_every_token(n, kind):
    h, w, y, ids, lt = make(n, 128, 264, 6, seed=kind, mass=1.0)
    lt[::3] += 1e-3  # a little more than 1, as rounding leaves it
    check(h, w, y, ids, lt, **KINDS[kind])
    ids = torch.stack([torch.randperm(128) for _ in range(n)])
    w = w[:128]
    y = torch.where(y >= 0, y % 128, y)
    lt = torch.log_softmax(torch.randn(n, 128), 1)
    check(h, w, y, ids, lt, **KINDS[kind])


@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("kind", range(len(KINDS)))
def test_a_student_that_is_its_teacher(n, kind):
    """The teacher's tokens are the student's own: the divergence is next to nothing, and so is its gradient."""
    h, w, y, _, _ = make(n, 128, 1000, 5, seed=21)
    kw = dict(KINDS[kind])
    t = kw.get("temperature", 1.0)
    top = LP.fused_linear_token_stats(h.to(DEV), w.to(DEV), y.to(DEV), 30, temperature=t)
    check(h, w, y, top.top_ids.cpu(), top.top_log_probs.cpu(), **kw)
    if kw.get("ce_weight") or kw.get("divisor"):
        return
    out = D.fused_linear_distillation(h.to(DEV), w.to(DEV), y.to(DEV), top.top_ids, top.top_log_probs, **kw)
    if kw.get("tail", True):
        assert abs(float(out.divergence)) <= 1e-5


@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("kind", [0, 2, 5])
def test_far_apart_logits(n, kind):
    """Labels and teachers far below the student's best logits: tiles are formed again relative to their own maximum."""
    check(*make(n, 128, 1000, 12, seed=6, wscale=2.0), redone=True, **KINDS[kind])


@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("kind", [0, 1, 2, 5])
def test_a_certain_student_keeps_its_tails_digits(n, kind):
    """All but 1e-9 on the teacher's first token: what is left to the others is no difference from 1."""
    h, w, y, ids, lt = make(n, 256, 1000, 4, seed=5, lean=0.0, mass=0.999, ignored=0.0)
    h = (torch.linspace(12, 26, n)[:, None] * w[ids[:, 0]].float() / (0.05 ** 2 * 256)).to(torch.bfloat16)
    check(h, w, y, ids, lt, **KINDS[kind])


@pytest.mark.parametrize("n", [2, 128, 300])
@pytest.mark.parametrize("kind", [0, 2, 5])
def test_one_token_for_all_rows(n, kind):
    """Every teacher and every label names the same token first: its gradients meet in one row of dW."""
    h, w, y, ids, lt = make(n, 128, 1000, 3, seed=18, ignored=0.0)
    ids = torch.where(ids == 999, 5, ids)
    ids[:, 0] = y[:] = 999
    lt[:, 0] += 3.0
    lt = torch.log_softmax(lt, 1) - 0.05
    check(h, w, y, ids, lt, **KINDS[kind])


def test_nothing_counts_no_rows_and_bad_labels():
    h, w, y, ids, lt = make(300, 128, 1000, 5, seed=8)
    hd, wd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    nothing = torch.full_like(y, -100).to(DEV)
    out = D.fused_linear_distillation(hd, wd, nothing, ids.to(DEV), lt.to(DEV))
    assert bool(out.loss.isnan())  # as F.cross_entropy's mean over nothing
    out = D.fused_linear_distillation(hd, wd, nothing, ids.to(DEV), lt.to(DEV), num_items_in_batch=10)
    dh, dw = torch.autograd.grad(out.loss, [hd, wd])
    assert float(out.loss) == 0 and bool((dh == 0).all()) and bool((dw == 0).all())
    none = hd[:0].detach().requires_grad_()
    out = D.fused_linear_distillation(none, wd, nothing[:0], ids[:0].to(DEV), lt[:0].to(DEV), num_items_in_batch=10)
    dh, dw = torch.autograd.grad(out.loss, [none, wd])
    assert float(out.loss) == 0 and dh.shape == (0, 128) and bool((dw == 0).all())
    y[3], y[200] = 1000, -7
    check(h, w, y, ids, lt, ce_weight=0.2)
    C.check_pending_labels(block=True)
    with pytest.raises(C.LabelError, match="2 label"):
        D.fused_linear_distillation(hd, wd, y.to(DEV), ids.to(DEV), lt.to(DEV), validate="sync")


def test_rows_that_do_not_count_are_not_read():
    h, w, y, ids, lt = make(300, 128, 1000, 5, seed=9)
    hd, wd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()

    def call(h, ids, lt):
        out = D.fused_linear_distillation(h, wd, y.to(DEV), ids.to(DEV), lt.to(DEV), ce_weight=0.1, validate="sync")
        return [out.loss.detach(), *torch.autograd.grad(out.loss, [h, wd])]

    want = call(hd, ids, lt)
    out = y == -100
    h2, ids2, lt2 = h.clone(), ids.clone(), lt.clone()
    h2[out], ids2[out], lt2[out] = float("nan"), 10 ** 9, float("nan")
    got = call(h2.to(DEV).requires_grad_(), ids2, lt2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert bool((got[1][out.to(DEV)] == 0).all())


@pytest.mark.parametrize("n", [60, 600])
def test_autograd_shapes_types_frozen_and_retained(n):
    h, w, y, ids, lt = make(n, 128, 520, 7, seed=11)
    shape = (4, n // 4)
    hg, wg = h.view(*shape, 128).to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    rest = (y.view(shape).to(DEV), ids.view(*shape, 7).to(DEV), lt.view(*shape, 7).to(DEV))
    out = D.fused_linear_distillation(hg, wg, *rest, ce_weight=0.2)
    assert out.loss.shape == () and out.loss.requires_grad and not out.divergence.requires_grad
    loss, div, ce = (float(x.detach()) for x in out)
    assert abs(loss - (0.8 * div + 0.2 * ce)) <= 4 * 2.0 ** -24 * (abs(div) + abs(ce))
    want = torch.autograd.grad(out.loss, [hg, wg], retain_graph=True)
    twice = torch.autograd.grad(out.loss, [hg, wg], torch.tensor(2.0, device=DEV), retain_graph=True)
    again = torch.autograd.grad(out.loss, [hg, wg])
    assert all(torch.equal(a, b) and torch.equal(c, 2 * a) for a, b, c in zip(want, again, twice))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out.loss, [hg])
    frozen = D.fused_linear_distillation(hg, wg.detach(), *rest, ce_weight=0.2)
    assert torch.equal(torch.autograd.grad(frozen.loss, [hg])[0], want[0])
    head = D.fused_linear_distillation(hg.detach(), wg, *rest, ce_weight=0.2)
    assert torch.equal(torch.autograd.grad(head.loss, [wg])[0], want[1])
    with torch.no_grad():
        lone = D.fused_linear_distillation(hg, wg, *rest, ce_weight=0.2)
    assert lone.loss.grad_fn is None and abs(float(lone.loss) - loss) <= 1e-6 * abs(loss)
    # strided and narrower operands, fp32 master copies
    wide = torch.zeros(*shape, 256, dtype=torch.bfloat16, device=DEV)
    wide[..., :128] = hg.detach()
    every = torch.stack([rest[1], rest[1]], -1)[..., 0]
    strided = D.fused_linear_distillation(wide[..., :128], wg.detach(), rest[0], every, rest[2].double(), ce_weight=0.2)
    assert torch.equal(strided.loss, lone.loss)
    h32, w32 = hg.detach().float().requires_grad_(), wg.detach().float().requires_grad_()
    out = D.fused_linear_distillation(h32, w32, *rest, ce_weight=0.2)
    got = torch.autograd.grad(out.loss, [h32, w32])
    assert got[0].dtype == torch.float32 and all(torch.equal(a, b.float()) for a, b in zip(got, want))
    half = D.fused_linear_distillation(hg, wg, *rest[:2], rest[2].to(torch.bfloat16))
    assert torch.isfinite(half.loss)
    items = torch.tensor(float(n), device=DEV)
    a, b = (D.fused_linear_distillation(hg, wg, *rest, num_items_in_batch=x).loss for x in (n, items))
    assert torch.equal(a, b)


def test_without_labels_every_row_counts():
    h, w, _, ids, lt = make(200, 128, 1000, 5, seed=12)
    ids[4, 0], ids[5] = -1, -1
    out = D.fused_linear_distillation(h.to(DEV), w.to(DEV), None, ids.to(DEV), lt.to(DEV), validate="sync")
    any_label = torch.zeros(200).long()
    ref = od.linear_distillation(np64(h), np64(w), any_label.numpy(), ids.numpy(), np64(lt))
    assert out.cross_entropy is None and abs(float(out.loss) - ref["loss"]) <= ref["loss_off"]


def test_weight_one_is_the_cross_entropy():
    h, w, y, ids, lt = make(600, 320, 2000, 6, seed=13)
    hd, wd, yd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), y.to(DEV)
    out = D.fused_linear_distillation(hd, wd, yd, ids.to(DEV), lt.to(DEV), ce_weight=1.0)
    loss = C.fused_linear_cross_entropy(hd, wd, yd)
    ref = od.linear_distillation(np64(h), np64(w), y.numpy(), ids.numpy(), np64(lt), ce_weight=1.0)
    assert abs(float(out.loss) - float(loss)) <= 2 * ref["loss_off"]
    for a, b, name in zip(torch.autograd.grad(out.loss, [hd, wd]), torch.autograd.grad(loss, [hd, wd]), ("dh", "dw")):
        assert (np.abs(np64(a) - np64(b)) <= 2 * ref[name + "_off"]).all()


@pytest.mark.parametrize("kind", [0, 5])
def test_gradient_is_a_difference(kind):
    """One direction in ``hidden``, central differences of the fp32 losses, row by row."""
    h, w, y, ids, lt = make(24, 128, 520, 9, seed=14, ignored=0.0)
    g = torch.Generator().manual_seed(1)
    h = (h.float() * 8).round().div(8).clamp(-15, 15).to(torch.bfloat16)  # steps of 1 / 8 below 16: moved by 1 / 16 exactly
    d = (torch.randint(-1, 2, h.shape, generator=g) / 16).to(torch.bfloat16)
    rest = (ids.to(DEV), lt.to(DEV))
    hd = h.to(DEV).requires_grad_()
    out = D.fused_linear_distillation(hd, w.to(DEV), y.to(DEV), *rest, num_items_in_batch=1, **KINDS[kind])
    dh, = torch.autograd.grad(out.loss, [hd])
    got = (dh.double() * d.to(DEV).double()).sum(1).cpu().numpy()
    ref = od.linear_distillation(np64(h), np64(w), y.numpy(), ids.numpy(), np64(lt), divisor=1.0, **KINDS[kind])
    # what a row's move changes a logit by at most; the third derivative of a row's divergence is at most 8 s^3 times one
    # and the largest logarithm in it (a logsumexp's 2 s^3, with the weights' own derivatives in the reverse)
    s = np.linalg.norm(np64(d), axis=1) * np.linalg.norm(np64(w), axis=1).max()
    size = 8 * (2 + np.log(520) + np.ptp(np64(h) @ np64(w).T, axis=1) + np.abs(np64(lt)).max(1))
    for i in range(24):
        one = torch.full_like(y, -100)
        one[i] = y[i]
        up, down = (D.fused_linear_distillation((h + s_ * d).to(DEV), w.to(DEV), one.to(DEV), *rest, num_items_in_batch=1,
                                                **KINDS[kind]).loss.double().item() for s_ in (1, -1))
        row = od.linear_distillation(np64(h)[i:i + 1], np64(w), y.numpy()[i:i + 1], ids.numpy()[i:i + 1], np64(lt)[i:i + 1],
                                     divisor=1.0, **KINDS[kind])
        bound = size[i] * s[i] ** 3 / 6 + row["loss_off"] + (ref["dh_off"][i] * np.abs(np64(d)[i])).sum() + 1e-9
        assert abs((up - down) / 2 - got[i]) <= bound


def test_streams_and_captured_calls():
    h, w, y, ids, lt = (t.to(DEV) for t in make(500, 128, 4104, 9, seed=15))

    def call(n, kw):
        hg, wg = h[:n].detach().requires_grad_(), w.detach().requires_grad_()
        out = D.fused_linear_distillation(hg, wg, y[:n], ids[:n], lt[:n], chunk_tokens=256, **kw)
        return [*(x.detach() for x in out), *torch.autograd.grad(out.loss, [hg, wg])]

    cases = [(500, dict(ce_weight=0.2)), (100, dict(divergence="reverse"))]
    want = [call(*c) for c in cases]
    torch.cuda.synchronize()
    got = []
    for st in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(st):
            got.append([call(*c) for c in cases])
    torch.cuda.synchronize()
    for pair in got:
        for a, b in zip(pair, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs = []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((c, graph, call(*c)))
    for i in range(3):
        h.copy_(torch.randn_like(h))
        y.copy_(y.roll(1))
        ids.copy_(ids.roll(1, 0))
        for _, graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for c, _, captured in graphs:
            assert all(torch.equal(p, q) for p, q in zip(captured, call(*c)))


def test_a_second_derivative_and_a_tangent_are_refused():
    h, w, y, ids, lt = (t.to(DEV) for t in make(20, 64, 264, 3))
    hg = h.clone().requires_grad_()
    out = D.fused_linear_distillation(hg, w, y, ids, lt)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.loss, [hg], create_graph=True)
    fw = torch.autograd.forward_ad
    for grad in (False, True):
        with fw.dual_level(), torch.set_grad_enabled(grad):
            for args in ((fw.make_dual(h, h), w, y, ids, lt), (h, w, y, ids, fw.make_dual(lt, lt))):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    D.fused_linear_distillation(*args)


def test_refusals_on_the_gpu():
    h, w, y, ids, lt = (t.to(DEV) for t in make(20, 64, 264, 3))
    base = dict(hidden=h, weight=w, labels=y, top_ids=ids, top_log_probs=lt)
    for kw, text in ((dict(temperature=0.0), "temperature"), (dict(ce_weight=0.5, temperature=2.0), "temperature 1"),
                     (dict(ce_weight=1.5), "ce_weight"), (dict(divergence="reverse", tail=False), "tail"),
                     (dict(top_ids=ids.float()), "top_ids must be int64 or int32"), (dict(top_ids=ids.cpu()), "top_ids must live on"),
                     (dict(top_log_probs=lt.cpu()), "top_log_probs must live on"), (dict(top_log_probs=lt.long()), "float32"),
                     (dict(labels=y.int()), "labels must be int64"),
                     (dict(top_ids=ids[:, :0], top_log_probs=lt[:, :0]), "top_k"),
                     (dict(top_ids=ids.repeat(1, 43), top_log_probs=lt.repeat(1, 43)), "top_k")):
        with pytest.raises(ValueError, match=text):
            D.fused_linear_distillation(**{**base, **kw})


@pytest.mark.parametrize("n,hdim,k,kind", [(1, 896, 20, 0), (48, 896, 16, 2), (128, 1536, 128, 5), (129, 896, 64, 1),
                                           (400, 320, 100, 2)])
def test_a_real_vocabulary(n, hdim, k, kind):
    """151,936 columns against the definition in 64 bits on the GPU: relative errors of the losses and of the gradients as a
    whole, which roundings of 2^-8 an element, three of them in a row, cannot exceed."""
    vocab = 151_936
    kw = {x: v for x, v in KINDS[kind].items()}
    print(f"distill real n={n} h={hdim} K={k} {kw}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(n + hdim)
    w = (0.05 * torch.randn(vocab, hdim, generator=g, device=DEV)).to(torch.bfloat16).requires_grad_()
    ids = torch.rand(n, 4096, generator=g, device=DEV).argsort(1)[:, :k] * 37  # different ones
    lt = torch.log_softmax(2 * torch.randn(n, k, generator=g, device=DEV), 1) - 0.1
    y = torch.where(torch.rand(n, generator=g, device=DEV) < 0.6, ids[:, 0], torch.randint(0, vocab, (n,), generator=g, device=DEV))
    lean = 20 * torch.rand(n, 1, generator=g, device=DEV) / (0.05 ** 2 * hdim)
    h = (torch.randn(n, hdim, generator=g, device=DEV) + lean * w.detach()[ids[:, 0]].float()).to(torch.bfloat16).requires_grad_()
    if n > 1:
        y[::5] = -100
    out = D.fused_linear_distillation(h, w, y, ids, lt, **kw)
    got = torch.autograd.grad(out.loss, [h, w])
    at = (y >= 0).nonzero()[:, 0]
    hk, wd = h.detach()[at].double(), w.detach().double()
    z = (hk @ wd.T.contiguous()).requires_grad_()
    lp = torch.log_softmax(z, 1)
    ls, t, lk = lp.gather(1, ids[at]), lt[at].double().exp(), lt[at].double()
    lq = torch.logsumexp(lp.scatter(1, ids[at], -np.inf), 1)
    r = 1 - t.sum(1)
    if kw.get("divergence") == "reverse":
        div = (ls.exp() * (ls - lk)).sum(1) + lq.exp() * (lq - r.log())
    else:
        div = (t * (lk - ls)).sum(1) + (r * (r.log() - lq) if kw.get("tail", True) else 0)
    ce = -lp.gather(1, y[at][:, None])[:, 0]
    c = kw.get("ce_weight", 0.0)
    loss = ((1 - c) * div + c * ce).mean()
    for a, b in zip(out, (loss, div.mean(), ce.mean())):
        assert abs(float(a.detach()) - float(b.detach())) <= 3e-6 * max(1.0, abs(float(b.detach())))
    dz, = torch.autograd.grad(loss, [z])
    dh = torch.zeros_like(h, dtype=torch.float64)
    dh[at] = dz @ wd
    for a, b in zip(got, (dh, dz.T.contiguous() @ hk)):
        assert float((a.double() - b).norm() / b.norm()) <= 3 * 2.0 ** -8


def test_rows_past_32_bit_offsets():
    """9,000 rows of 151,936 columns in one chunk: numerators past 2^30 elements and 2^31 bytes, the last rows checked."""
    n, hdim, vocab, k = 9_000, 64, 151_936, 8
    g = torch.Generator(device=DEV).manual_seed(7)
    h = torch.randn(n, hdim, generator=g, device=DEV).to(torch.bfloat16).requires_grad_()
    w = (0.3 * torch.randn(vocab, hdim, generator=g, device=DEV)).to(torch.bfloat16)
    ids = torch.rand(n, 1024, generator=g, device=DEV).argsort(1)[:, :k] * 148
    lt = torch.log_softmax(torch.randn(n, k, generator=g, device=DEV), 1) - 0.05
    y = torch.randint(0, vocab, (n,), generator=g, device=DEV)
    out = D.fused_linear_distillation(h, w, y, ids, lt, num_items_in_batch=1, chunk_tokens=16384)
    dh, = torch.autograd.grad(out.loss, [h])
    wd = w.double()
    for c in (0, n - 200):
        hk = h.detach()[c:c + 200].double()
        z = (hk @ wd.T.contiguous()).requires_grad_()
        lp = torch.log_softmax(z, 1)
        ls, t, lk = lp.gather(1, ids[c:c + 200]), lt[c:c + 200].double().exp(), lt[c:c + 200].double()
        lq = torch.logsumexp(lp.scatter(1, ids[c:c + 200], -np.inf), 1)
        r = 1 - t.sum(1)
        dz, = torch.autograd.grad(((t * (lk - ls)).sum(1) + r * (r.log() - lq)).sum(), [z])
        want = dz @ wd
        assert float((dh[c:c + 200].double() - want).norm() / want.norm()) <= 3 * 2.0 ** -8


@pytest.mark.parametrize("n", [90, 700])
def test_a_teacher_and_its_student(n):
    """A teacher scores a batch, a student of another size learns from what it says: the whole run against 64 bits."""
    g = torch.Generator().manual_seed(n)
    vocab = 1000
    ht, wt = torch.randn(n, 256, generator=g).to(torch.bfloat16), (0.1 * torch.randn(vocab, 256, generator=g)).to(torch.bfloat16)
    hs, ws = torch.randn(n, 128, generator=g).to(torch.bfloat16), (0.1 * torch.randn(vocab, 128, generator=g)).to(torch.bfloat16)
    y = torch.randint(0, vocab, (n,), generator=g)
    y[torch.rand(n, generator=g) < 0.4] = -100
    with torch.no_grad():
        top = LP.fused_linear_token_stats(ht.to(DEV), wt.to(DEV), y.to(DEV), 16)
    out, _, ref = check(hs, ws, y, top.top_ids.cpu(), top.top_log_probs.cpu(), ce_weight=0.25, upstream=0.5)
    assert ref["bad_tokens"] == 0
    D.fused_linear_distillation(hs.to(DEV), ws.to(DEV), y.to(DEV), top.top_ids, top.top_log_probs, validate="sync")


def test_a_model_learns_from_a_model():
    transformers = pytest.importorskip("transformers")
    from siq_vl_amd.text_model import enable_fused_cross_entropy

    def build(hidden, seed):
        cfg = transformers.Qwen2Config(vocab_size=264, hidden_size=hidden, intermediate_size=2 * hidden, num_hidden_layers=1,
                                       num_attention_heads=4, num_key_value_heads=2)
        torch.manual_seed(seed)
        model = transformers.Qwen2ForCausalLM(cfg).to(DEV, torch.bfloat16)
        enable_fused_cross_entropy(model)
        return model

    teacher, student = build(256, 1), build(128, 2)
    ids = torch.randint(0, 264, (2, 30), device=DEV)
    labels = ids.clone()
    labels[:, :7] = -100
    with torch.no_grad():
        said = teacher(input_ids=ids, labels=labels, use_cache=False, return_log_probs=True, top_k=12)
    out = student(input_ids=ids, labels=labels, use_cache=False, teacher=(said.top_ids, said.top_log_probs),
                  distillation=dict(ce_weight=0.5))
    plain = student(input_ids=ids, labels=labels, use_cache=False)
    assert out.logits is None and out.loss.requires_grad
    assert abs(float(out.cross_entropy) - float(plain.loss.detach())) <= 1e-5 * float(plain.loss.detach())
    assert abs(float(out.loss.detach()) - 0.5 * (float(out.divergence) + float(out.cross_entropy))) <= 1e-5
    items = int((labels[:, 1:] != -100).sum())
    summed = student(input_ids=ids, labels=labels, use_cache=False, teacher=(said.top_ids, said.top_log_probs),
                     distillation=dict(ce_weight=0.5), num_items_in_batch=items)
    assert abs(float(summed.loss.detach()) - float(out.loss.detach())) <= 1e-6 * float(out.loss.detach())
    out.loss.backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in student.parameters())


@pytest.mark.parametrize("n", [8, 130])
@pytest.mark.parametrize("wscale", [0.05, 2.0])
def test_more_columns_than_a_row_pass_holds(n, wscale):
    """270,336 columns: more tiles than a row of few takes at once, and lists of three spans; formed again or not."""
    data = make(n, 64, 270_336, 7, seed=n, wscale=wscale)
    data[3][0, 0], data[3][1, 1] = 270_335, 131_072  # (at a span's borders)
    check(*data, redone=wscale > 1, **KINDS[2])
