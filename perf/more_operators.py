"""The operators of scoring and distillation that are timed: one pass per case, through the entry points that a script
calls.

A case is a dict of plain values.  Its ``kind`` picks the operator:

* ``stats``    ``fused_linear_token_stats``: from hidden states, without logits, the log-probabilities of given tokens, the
               entropy of every row's distribution, and its most probable tokens with their log-probabilities;
* ``distill``  ``fused_linear_distillation``: the loss of a student against a teacher's most probable tokens, and its
               gradients.

``own`` False computes the same in elementary torch operations.  Which rows count follows from the case alone
(``_counted``), values from the seed alone.
"""

from __future__ import annotations

import math
import random

import torch

own = False

VOCAB = 151936  # Qwen2.5's table
IGNORE = -100
DEV = "cuda"


# --------------------------------------------------------------------------- the cases
def _stats(name, rows, hidden, vocab, top_k, train, masked, temperature):
    """``train``: "none" (scores alone), "frozen" (gradients of the hidden states) or "full" (the head's too)."""
    return {"name": name, "kind": "stats", "rows": rows, "hidden": hidden, "vocab": vocab, "top_k": top_k, "train": train,
            "masked": masked, "temperature": temperature}


def _distill(name, rows, hidden, vocab, top_k, train, masked, temperature, ce_weight, divergence, tail):
    return {"name": name, "kind": "distill", "rows": rows, "hidden": hidden, "vocab": vocab, "top_k": top_k, "train": train,
            "masked": masked, "temperature": temperature, "ce_weight": ce_weight, "divergence": divergence, "tail": tail}


def listed():
    return [
        # one decoding step of the 0.5B model: the sampled token's log-probability and its alternatives, latency bound
        _stats("stats one token", 1, 896, VOCAB, 20, "none", 0.0, 0.7),
        # a short answer scored by the 0.5B model, an odd row count
        _stats("stats short answer", 61, 896, VOCAB, 5, "none", 0.0, 1.0),
        # the 1.5B model as a teacher: what a student's step over the same packed batch is trained on
        _stats("stats teacher", 8192, 1536, VOCAB, 64, "none", 0.3, 1.0),
        # a policy batch with an entropy bonus and a frozen lm_head (LoRA), at the temperature of its answers
        _stats("stats entropy frozen", 2048, 1536, VOCAB, 0, "frozen", 0.3, 0.7),
        # the same in full training of the 0.5B model, an odd row count
        _stats("stats entropy train", 4099, 896, VOCAB, 0, "full", 0.3, 1.0),
        # the student's answer to one prompt: the head's table is read for 48 rows
        _distill("distill short answer", 48, 896, VOCAB, 16, "full", 0.0, 1.0, 0.0, "forward", True),
        # a batch of the 0.5B student with a frozen lm_head (LoRA), softened distributions, an odd row count
        _distill("distill frozen head", 4099, 896, VOCAB, 32, "frozen", 0.3, 2.0, 0.0, "forward", True),
        # the reverse divergence over a smaller vocabulary with many alternatives
        _distill("distill reverse", 2051, 2048, 49152, 100, "full", 0.5, 1.0, 0.0, "reverse", True),
        # evaluation: the loss alone
        _distill("distill evaluation", 5000, 896, VOCAB, 64, "none", 0.3, 1.0, 0.1, "forward", True),
        # the 16k-token packed step of the 1.5B student in full training, labels mixed in: the largest
        _distill("distill train", 16384, 1536, VOCAB, 64, "full", 0.3, 1.0, 0.1, "forward", True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    hidden, vocab = rng.choice([320, 896, 1536, 2048]), rng.choice([VOCAB, VOCAB, 32008, 49152])
    rows, masked = _log_int(rng, 1, 16384), rng.choice([0.0, 0.3, 0.7])
    train = rng.choice(["none", "frozen", "full"])
    temperature = rng.choice([1.0, 1.0, 0.7, 1.5])
    if rng.random() < 0.5:
        top_k = rng.choice([0, _log_int(rng, 1, 128), _log_int(rng, 1, 128)])
        case = _stats("", rows, hidden, vocab, top_k, train, masked, temperature)
        most = 0.8e13  # (the plain form sorts its alternatives out: rows are what it takes time for)
    else:
        reverse = rng.random() < 0.3
        ce = rng.choice([0.0, 0.1, 0.5]) if temperature == 1.0 else 0.0
        case = _distill("", rows, hidden, vocab, _log_int(rng, 1, 128), train, masked, temperature, ce,
                        "reverse" if reverse else "forward", reverse or rng.random() < 0.7)
        most = 1.6e13
    while work(case)["flops"] > most:  # no dearer than the listed ones
        case["rows"] -= case["rows"] // 4
    del case["name"]
    return case


# --------------------------------------------------------------------------- sizes that follow from a case
def _counted(case):
    """Rows whose label counts: the head of each sample (prompt, image) is ignored."""
    rng, mask = random.Random(case["rows"]), []
    while len(mask) < case["rows"]:
        n = max(16, min(4096, int(400 * math.exp(0.75 * rng.gauss(0, 1)))))
        ignored = int(round(case["masked"] * n))
        mask += [False] * ignored + [True] * (n - ignored)
    mask = mask[:case["rows"]]
    mask[-1] = True
    return mask


def work(case):
    n, h, v, k, counted = case["rows"], case["hidden"], case["vocab"], case["top_k"], sum(_counted(case))
    products = {"none": 1, "frozen": 2, "full": 3}[case["train"]]
    nbytes = 2 * n * h * min(products, 2) + 2 * v * h * (2 if products == 3 else 1)  # hidden, its gradient; weight, its
    nbytes += n * (8 + 12 * k)  # labels, alternatives
    if case["kind"] == "stats":
        nbytes += n * (8 if products == 1 else 16)  # log-probability, entropy, and what comes back for them
    return {"bytes": nbytes, "flops": 2.0 * products * counted * h * v}


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _uniform(g, *shape, dtype=torch.float32):
    return torch.rand(*shape, generator=g, device=DEV, dtype=dtype)


def _grid(x, step, most):
    """To multiples of ``step`` of at most eight bits, which bf16 holds."""
    return ((x / step).round().clamp(-most, most) * step).to(torch.bfloat16)


def _zipf(g, n, vocab):
    """Token ids as text has them: the frequency of an id falls as 1 / rank."""
    u = _uniform(g, n, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab)).to(torch.int64) - 1).clamp_(0, vocab - 1)


def _alternatives(g, n, k, vocab):
    """``k`` different ids a row, low ones more often, in no order: one of each of ``k`` ranges of equal probability."""
    u = (torch.arange(k, device=DEV) + _uniform(g, n, k, dtype=torch.float64)) / k
    ids = torch.exp(u * math.log(vocab)).to(torch.int64) - 1
    place = torch.arange(k, device=DEV)
    ids = ((ids - place).cummax(1).values + place)  # (each above the one before)
    ids = torch.minimum(ids, vocab - k + place)
    return ids.gather(1, _uniform(g, n, k).argsort(1))


def prepare(case, seed):
    g = _gen(seed)
    n, h, v, k = case["rows"], case["hidden"], case["vocab"], case["top_k"]
    st = {"case": case}
    counted = torch.tensor(_counted(case), device=DEV)
    w = 0.02 * torch.randn(v, h, generator=g, device=DEV)
    noise = torch.randn(n, h, generator=g, device=DEV)
    pull = 16 / (0.02 ** 2 * h)  # of a token's row that brings its logit to 16
    if case["kind"] == "stats":
        # values on a grid on which sums of products are exact in 32 bits in any order: which of two tokens is the more
        # probable is then no matter of rounding.  Rows lean towards their token, some hardly and some strongly.
        w = _grid(w, 2.0 ** -11, 255)
        y = _zipf(g, n, v)
        hid = _grid(noise + pull * _uniform(g, n, 1) * w[y].float(), 2.0 ** -4, 255)
        y[~counted] = IGNORE
        if case["train"] != "none":
            # a loss's gradient: of either sign, small, and zero where a token was clipped
            up = torch.randn(n, generator=g, device=DEV) / n
            st["up"] = torch.where(_uniform(g, n) < 0.1, 0.0, up)
            st["up_entropy"] = torch.full((n,), -0.01 / n, device=DEV)
    else:
        w = w.to(torch.bfloat16)
        ids = _alternatives(g, n, k, v)
        # the teacher's distribution: from near certain to flat, a tail of up to a fifth behind its alternatives
        sharp = 0.5 + 2.5 * _uniform(g, n, 1)
        scores = sharp * torch.randn(n, k, generator=g, device=DEV)
        mass = torch.log1p(-0.2 * _uniform(g, n, 1) ** 2 - 1e-4)
        teacher = torch.log_softmax(scores, 1) + mass
        # the label is drawn from it, sometimes from its tail
        y = ids.gather(1, torch.multinomial(teacher.exp(), 1, generator=g))[:, 0]
        y = torch.where(_uniform(g, n) < 0.1, _zipf(g, n, v), y)
        # the student leans towards the teacher's first choices, and somewhat towards others
        best = teacher.topk(min(k, 3), dim=1).indices
        lean = noise
        for j in range(best.shape[1]):
            lean = lean + pull * (0.9 - 0.15 * j) * _uniform(g, n, 1) * w[ids.gather(1, best[:, j:j + 1])[:, 0]].float()
        lean = lean + 0.7 * pull * _uniform(g, n, 1) ** 3 * w[_zipf(g, n, v)].float()
        hid = lean.to(torch.bfloat16)
        y[~counted] = IGNORE
        st["ids"], st["teacher"] = ids, teacher
    st["hidden"] = hid.requires_grad_(case["train"] != "none")
    st["weight"] = w.requires_grad_(case["train"] == "full")
    st["labels"] = y
    return st


# --------------------------------------------------------------------------- the framework's calls
def _leaves(st):
    return [x for x in (st["hidden"], st["weight"]) if x.requires_grad]


def _run_own(st):
    case = st["case"]
    leaves = _leaves(st)
    if case["kind"] == "stats":
        from siq_vl_amd.log_probs import fused_linear_token_stats

        out = fused_linear_token_stats(st["hidden"], st["weight"], st["labels"], top_k=case["top_k"],
                                       temperature=case["temperature"])
        got = [out.log_probs.detach(), out.entropy.detach()]
        if case["top_k"]:
            got += [out.top_log_probs, out.top_ids]
        if leaves:
            got += torch.autograd.grad([out.log_probs, out.entropy], leaves, [st["up"], st["up_entropy"]])
        return got
    from siq_vl_amd.distillation import fused_linear_distillation

    out = fused_linear_distillation(st["hidden"], st["weight"], st["labels"], st["ids"], st["teacher"],
                                    temperature=case["temperature"], ce_weight=case["ce_weight"],
                                    divergence=case["divergence"], tail=case["tail"])
    got = [out.loss.detach(), out.divergence, out.cross_entropy]
    return got + list(torch.autograd.grad(out.loss, leaves)) if leaves else got


# --------------------------------------------------------------------------- the plain form
def _best(z, k):
    """The ``k`` largest of each row, ties to the lower column: by the numbers' bits, which order as they do, with the
    column behind them."""
    bits = z.contiguous().view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64)
    order = (order << 32) + torch.arange(z.shape[1] - 1, -1, -1, device=z.device)
    return order.topk(k, dim=1).indices


def _plain_stats(st):
    case, y = st["case"], st["labels"]
    n, k, t = case["rows"], case["top_k"], case["temperature"]
    hid, w = st["hidden"].detach().float(), st["weight"].detach().float()
    counted = y != IGNORE
    at = y.clamp(min=0)[:, None]
    z = hid @ w.T
    top = []
    if k:
        ids = torch.cat([_best(z[a:a + 1024], k) for a in range(0, n, 1024)])
        top = [z.gather(1, ids), ids]
    zy = z.gather(1, at)
    high = z.amax(1, keepdim=True)
    z -= high
    z /= t
    p = torch.exp(z)
    total = p.sum(1, keepdim=True)
    p /= total
    log_total = total.log()
    z -= log_total  # ln p
    entropy = torch.cat([-(p[a:a + 1024] * z[a:a + 1024]).sum(1) for a in range(0, n, 1024)])
    out = [torch.where(counted, ((zy - high) / t - log_total)[:, 0], 0.0), torch.where(counted, entropy, 0.0)]
    if k:
        out += [torch.where(counted[:, None], (top[0] - high) / t - log_total, 0.0), torch.where(counted[:, None], top[1], -1)]
    if case["train"] != "none":
        g, ge = (torch.where(counted, st[x], 0.0)[:, None] / t for x in ("up", "up_entropy"))
        z += entropy[:, None]
        z *= -ge
        z -= g
        z *= p
        z.scatter_add_(1, at, g)
        out.append((z @ w).to(torch.bfloat16))
        if case["train"] == "full":
            out.append((z.T @ hid).to(torch.bfloat16))
    return out


def _plain_distill(st):
    case, y, ids = st["case"], st["labels"], st["ids"]
    c = case["ce_weight"]
    hid, w = st["hidden"].detach().float(), st["weight"].detach().float()
    counted = y != IGNORE
    count = counted.sum()
    at = y.clamp(min=0)[:, None]
    z = hid @ w.T
    z /= case["temperature"]
    z -= z.amax(1, keepdim=True)
    zk, zy = z.gather(1, ids), z.gather(1, at)
    e = z.exp_()
    # the tokens that the teacher does not name are summed by themselves: what is left of 1 loses its digits
    ek, ey = e.gather(1, ids), e.gather(1, at)
    e.scatter_(1, ids, 0.0)
    others = e.sum(1, keepdim=True)
    e.scatter_(1, ids, ek)
    total = others + ek.sum(1, keepdim=True)
    s, q, lt = ek / total, others / total, st["teacher"]
    # the teacher's tail is what its probabilities leave of 1: in 64 bits
    t64 = lt.double().exp()
    mass64 = t64.sum(1, keepdim=True)
    r64 = (1 - mass64).clamp(min=0.0 if case["divergence"] == "forward" else 2.0 ** -24)
    t, m, r = t64.float(), mass64.float(), r64.float()
    ls, lq, lr = zk - total.log(), q.log(), r64.log().float()
    if case["divergence"] == "forward":
        div = (t * (lt - ls)).sum(1, keepdim=True)
        if case["tail"]:
            div = div + torch.where(r > 0, r * (lr - lq), 0.0)
            inner, outer = s * (mass64 + r64).float() - t, ((mass64 + r64) - r64 / q.double()).float()
        else:
            inner, outer = s * m - t, m
    else:
        # d/dz_j of the sum of s (ln s - ln t) over the tokens and the tail: s_j (ln s_j - ln t_j - the sum itself)
        div = (s * (ls - lt)).sum(1, keepdim=True) + q * (lq - lr)
        inner, outer = s * (ls - lt - div), lq - lr - div
    ce = total.log() - zy
    each = torch.where(counted[:, None], (1 - c) * div + c * ce, 0.0)
    out = [x.sum(dtype=torch.float64).div(count).float()
           for x in (each, torch.where(counted[:, None], div, 0.0), torch.where(counted[:, None], ce, 0.0))]
    if case["train"] == "none":
        return out
    scale = torch.where(counted, 1.0, 0.0)[:, None] / (count * case["temperature"])
    e *= ((1 - c) * outer + c) / total
    e.scatter_(1, ids, (1 - c) * inner + c * s)
    e.scatter_add_(1, at, torch.full_like(zy, -c))
    e *= scale
    out.append((e @ w).to(torch.bfloat16))
    if case["train"] == "full":
        out.append((e.T @ hid).to(torch.bfloat16))
    return out


def run(st):
    if own:
        return _run_own(st)
    return _plain_stats(st) if st["case"]["kind"] == "stats" else _plain_distill(st)


# --------------------------------------------------------------------------- the same in 64 bits
def _exact_stats(case, st):
    n, k, v, t = case["rows"], case["top_k"], case["vocab"], case["temperature"]
    hid, w = st["hidden"].detach().double(), st["weight"].detach().double()
    wt = w.T.contiguous()
    keep = torch.nonzero(st["labels"] != IGNORE).flatten()
    logps, entropy = (torch.zeros(n, dtype=torch.float64, device=DEV) for _ in range(2))
    top = torch.zeros(n, k, dtype=torch.float64, device=DEV)
    ids = torch.full((n, k), -1, device=DEV)
    dh, dw = torch.zeros_like(hid), torch.zeros_like(w) if case["train"] == "full" else None
    for c in range(0, keep.numel(), 1024):
        rows = keep[c:c + 1024]
        logits = hid[rows] @ wt
        if k:  # whole multiples of 2^-15 and fewer than 2^18 tokens: one whole number a token that orders them
            key = (logits * 2.0 ** 15).round().long() * 2 ** 18 + (v - 1 - torch.arange(v, device=DEV))
            ids[rows] = v - 1 - key.topk(k, dim=1).values.remainder(2 ** 18)
            del key
        lp = torch.log_softmax(logits / t, dim=1)
        del logits
        p = lp.exp()
        at = (torch.arange(rows.numel(), device=DEV), st["labels"][rows])
        logps[rows], entropy[rows] = lp[at], -(p * lp).sum(1)
        if k:
            top[rows] = lp.gather(1, ids[rows])
        if case["train"] != "none":
            g, ge = (st[x][rows].double()[:, None] for x in ("up", "up_entropy"))
            dz = -p * (g + ge * (lp + entropy[rows][:, None]))
            dz[at] += g[:, 0]
            dz /= t
            dh[rows] = dz @ w
            if dw is not None:
                dw += dz.T.contiguous() @ hid[rows]
    out = [logps, entropy] + ([top, ids] if k else [])
    return out + ([dh] if case["train"] != "none" else []) + ([dw] if dw is not None else [])


def _exact_distill(case, st):
    n, c = case["rows"], case["ce_weight"]
    hid, w = st["hidden"].detach().double(), st["weight"].detach().double()
    wt = w.T.contiguous()
    keep = torch.nonzero(st["labels"] != IGNORE).flatten()
    dh, dw = torch.zeros_like(hid), torch.zeros_like(w) if case["train"] == "full" else None
    sums = torch.zeros(3, dtype=torch.float64, device=DEV)
    for a in range(0, keep.numel(), 1024):
        rows = keep[a:a + 1024]
        ids, lt = st["ids"][rows], st["teacher"][rows].double()
        z = (hid[rows] @ wt / case["temperature"]).requires_grad_()
        lse = torch.logsumexp(z, dim=1)
        ls = z.gather(1, ids) - lse[:, None]
        lq = torch.logsumexp(z.scatter(1, ids, -math.inf), dim=1) - lse
        rest = 1 - lt.exp().sum(1)
        if case["divergence"] == "reverse":
            rest = rest.clamp(min=2.0 ** -24)
            div = (ls.exp() * (ls - lt)).sum(1) + lq.exp() * (lq - rest.log())
        else:
            div = (lt.exp() * (lt - ls)).sum(1)
            if case["tail"]:
                rest = rest.clamp(min=0)
                div = div + torch.where(rest > 0, rest * (rest.clamp(min=1e-300).log() - lq), 0.0)
        ce = lse - z.gather(1, st["labels"][rows][:, None])[:, 0]
        loss = ((1 - c) * div + c * ce).sum()
        sums += torch.stack([loss, div.sum(), ce.sum()]).detach()
        if case["train"] != "none":
            dz, = torch.autograd.grad(loss, [z])
            dz /= keep.numel() * case["temperature"]
            dh[rows] = dz @ w
            if dw is not None:
                dw += dz.T.contiguous() @ hid[rows]
    out = list(sums / keep.numel())
    return out + ([dh] if case["train"] != "none" else []) + ([dw] if dw is not None else [])


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_stats(case, st) if case["kind"] == "stats" else _exact_distill(case, st)
