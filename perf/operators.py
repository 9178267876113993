"""The operators of preference and policy training that are timed, beside what the framework did before: one pass per
case, forward and backward, through the entry points that a training script calls.

A case is a dict of plain values.  Its ``kind`` picks the operator:

* ``logp``    ``fused_linear_log_probs``: log-probabilities of the labels from hidden states, without logits;
* ``pref``    ``preference_loss``: the loss of paired sequences from their log-probabilities;
* ``policy``  ``policy_loss``: the clipped policy loss with its KL term;
* ``pack``    ``pack8`` and ``unpack8``: an activation kept in 8 bits and read back;
* ``swiglu``  ``swiglu8``: the gated activation of an MLP that keeps its inputs in 8 bits for the backward.

``own`` False computes the same in elementary torch operations.  Sequence lengths follow from the case alone
(``_lengths``), values from the seed alone.
"""

from __future__ import annotations

import math
import random

import torch

own = False

VOCAB = 151936  # Qwen2.5's table
IGNORE = -100
GROUP = 32  # elements that share a scale in 8-bit storage
DEV = "cuda"


# --------------------------------------------------------------------------- the cases
def _logp(name, rows, hidden, vocab, frozen, masked, temperature):
    return {"name": name, "kind": "logp", "rows": rows, "hidden": hidden, "vocab": vocab, "frozen": frozen,
            "masked": masked, "temperature": temperature}


def _pref(name, pairs, tokens, loss_type, smoothing, normalized, order):
    return {"name": name, "kind": "pref", "seqs": 2 * pairs, "tokens": tokens, "loss_type": loss_type,
            "smoothing": smoothing, "normalized": normalized, "order": order}


def _policy(name, seqs, tokens, aggregation, advantages, kl, kl_coef, dual):
    return {"name": name, "kind": "policy", "seqs": seqs, "tokens": tokens, "aggregation": aggregation,
            "advantages": advantages, "kl": kl, "kl_coef": kl_coef, "dual": dual}


def _pack(name, rows, cols, dtype, fmt):
    return {"name": name, "kind": "pack", "rows": rows, "cols": cols, "dtype": dtype, "format": fmt}


def _swiglu(name, rows, cols, fmt, fused):
    return {"name": name, "kind": "swiglu", "rows": rows, "cols": cols, "dtype": "bf16", "format": fmt, "fused": fused}


def listed():
    return [
        # the answer of one short prompt scored by the 0.5B model with a frozen lm_head: the table is read for 48 rows
        _logp("logp short answer", 48, 896, VOCAB, True, 0.0, 1.0),
        # a preference batch of the 0.5B model with a frozen lm_head (LoRA), prompts masked, an odd row count
        _logp("logp frozen head", 4099, 896, VOCAB, True, 0.3, 1.0),
        # a policy batch of the 1.5B model in full training, at the temperature its answers were sampled with: the largest
        _logp("logp train", 16384, 1536, VOCAB, False, 0.3, 0.7),
        # a batch of one pair of short answers: launch and latency bound
        _pref("pref one pair", 1, 131, "sigmoid", 0.0, False, "interleaved"),
        # an accumulated batch of long documents, length-normalised
        _pref("pref long", 60, 1_000_003, "ipo", 0.0, True, "halves"),
        # one question with four sampled answers, no reference model
        _policy("policy one group", 4, 517, "token", "sequence", None, 0.0, None),
        # a group batch as it follows the 16k-token packed step: per-answer advantages, averaged answer by answer
        _policy("policy groups", 64, 16384, "sequence", "sequence", "k3", 0.04, None),
        # a whole rollout buffer with per-token advantages and the second clip for negative ones
        _policy("policy buffer", 700, 2_000_003, "token", "token", "k3", 0.05, 3.0),
        # one prompt's input of one decoder layer of the 0.5B model
        _pack("pack prompt", 197, 896, "bf16", "int8"),
        # the layer inputs that a step of the 1.5B model keeps for its backward, four layers of 16384 tokens
        _pack("pack layer inputs", 65536, 1536, "bf16", "e4m3"),
        # an MLP on an odd number of tokens, gate and up as halves of one product
        _swiglu("swiglu odd batch", 1003, 3584, "int8", True),
        # the MLP of a packed training batch, four times the 1.5B model's hidden size wide
        _swiglu("swiglu train", 16384, 6144, "int8", False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["logp", "logp", "pref", "policy", "policy", "pack", "swiglu"])
    fmt = rng.choice(["int8", "e4m3"])
    if kind == "logp":
        hidden = rng.choice([320, 896, 1536, 2048])
        rows = min(_log_int(rng, 1, 16384), 16384 * 1536 // hidden)
        case = _logp("", rows, hidden, rng.choice([VOCAB, VOCAB, 32008, 49152]), rng.random() < 0.5,
                     rng.choice([0.0, 0.3, 0.7]), rng.choice([1.0, 1.0, 0.7, 1.3]))
        while work(case)["flops"] > 1.6e13:  # no dearer than the listed ones
            case["rows"] -= case["rows"] // 4
    elif kind == "pref":
        tokens = _log_int(rng, 64, 1_000_000)
        pairs = _log_int(rng, 1, max(1, min(2000, tokens // 40)))
        loss_type = rng.choice(["sigmoid", "sigmoid", "ipo", "hinge"])
        case = _pref("", pairs, tokens, loss_type, 0.1 if loss_type == "sigmoid" and rng.random() < 0.5 else 0.0,
                     loss_type == "ipo" or rng.random() < 0.2, rng.choice(["interleaved", "halves"]))
    elif kind == "policy":
        tokens = _log_int(rng, 16, 2_000_000)
        kl = rng.choice([None, "k1", "k2", "k3", "k3"])
        case = _policy("", _log_int(rng, 1, max(1, min(4000, tokens // 16))), tokens, rng.choice(["token", "sequence"]),
                       rng.choice(["token", "sequence"]), kl, 0.0 if kl is None else rng.choice([0.0, 0.04, 0.2]),
                       rng.choice([None, None, 2.5]))
    elif kind == "pack":
        rows, cols = _log_int(rng, 1, 32768), _log_int(rng, 33, 3000)
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        case = _pack("", rows if dtype == "bf16" else (rows + 1) // 2, cols, dtype, fmt)
    else:
        fused = rng.random() < 0.4
        cols = _log_int(rng, 64, 6000)
        case = _swiglu("", _log_int(rng, 1, 16384), cols - cols % 8 if fused else cols, fmt, fused)
    del case["name"]
    return case


# --------------------------------------------------------------------------- sizes that follow from a case
def _lengths(case):
    """The packed sequences' lengths, ragged as answers are (lognormal); their sum is ``tokens``, each is at least 1."""
    total, n = case["tokens"], case["seqs"]
    rng = random.Random(total * 1009 + n)
    weights = [math.exp(0.75 * rng.gauss(0, 1)) for _ in range(n)]
    lens = [max(1, int(total * w / sum(weights))) for w in weights]
    lens[lens.index(max(lens))] += total - sum(lens)
    return lens


def _label_mask(case):
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
    kind = case["kind"]
    if kind == "logp":
        n, h, v, counted = case["rows"], case["hidden"], case["vocab"], sum(_label_mask(case))
        nbytes = 4 * n * h + 2 * v * h * (1 if case["frozen"] else 2) + 16 * n  # hidden, dhidden; weight, dweight
        return {"bytes": nbytes, "flops": 2.0 * (2 if case["frozen"] else 3) * counted * h * v}
    if kind == "pref":
        return {"bytes": case["tokens"] * (4 + 4 + 1 + 4), "flops": 0.0}
    if kind == "policy":
        per = 4 + 4 + 1 + 4 + (4 if case["kl"] else 0) + (4 if case["advantages"] == "token" else 0)
        return {"bytes": case["tokens"] * per, "flops": 0.0}
    n, e = case["rows"] * case["cols"], 4 if case["dtype"] == "fp32" else 2
    packed = n + (n + GROUP - 1) // GROUP
    if kind == "pack":
        return {"bytes": 2 * e * n + 2 * packed, "flops": 0.0}
    return {"bytes": 6 * e * n + 4 * packed, "flops": 0.0}  # gate, up, h, dh, dgate, dup; both packed, written and read


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (std * torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)).to(dtype)


def _zipf(g, n, vocab):
    """Token ids as text has them: the frequency of an id falls as 1 / rank."""
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab)).to(torch.int64) - 1).clamp_(0, vocab - 1)


def _sequences(case, g):
    """Offsets, the answers' mask (the head of each sequence is its prompt), and log-probabilities of sampled tokens."""
    lens = torch.tensor(_lengths(case), device=DEV)
    cu = torch.zeros(case["seqs"] + 1, dtype=torch.int32, device=DEV)
    cu[1:] = lens.cumsum(0)
    t = case["tokens"]
    seq = torch.searchsorted(cu[1:].long(), torch.arange(t, device=DEV), right=True)
    mask = torch.arange(t, device=DEV) - cu[seq] >= (0.4 * lens[seq]).long()
    # most sampled tokens are likely ones, some are not
    sampled = -3 * torch.rand(t, generator=g, device=DEV) ** 4 - 0.01
    return cu, seq, mask, torch.where(mask, sampled, 0.0)


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    kind = case["kind"]
    if kind == "logp":
        n, h, v = case["rows"], case["hidden"], case["vocab"]
        w = _normal(g, v, h, std=0.02)
        y = _zipf(g, n, v)
        # rows lean towards their label, some hardly and some strongly
        lean = 16 * torch.rand(n, 1, generator=g, device=DEV) / (0.02 ** 2 * h)
        hid = (torch.randn(n, h, generator=g, device=DEV) + lean * w[y].float()).to(torch.bfloat16)
        y[~torch.tensor(_label_mask(case), device=DEV)] = IGNORE
        st["hidden"], st["weight"], st["labels"] = hid.requires_grad_(), w.requires_grad_(not case["frozen"]), y
        # a loss's gradient: of either sign, small, and zero where a token was clipped
        up = _normal(g, n, std=1.0 / n, dtype=torch.float32)
        st["up"] = torch.where(torch.rand(n, generator=g, device=DEV) < 0.1, 0.0, up)
    elif kind == "pref":
        cu, _, mask, ref = _sequences(case, g)
        drift = 0.05 * torch.randn(case["tokens"], generator=g, device=DEV)
        st["policy"] = torch.where(mask, ref + drift, 0.0).clamp_(max=0.0).requires_grad_()
        st["reference"], st["cu"], st["mask"] = ref, cu, mask
    elif kind == "policy":
        cu, seq, mask, old = _sequences(case, g)
        t = case["tokens"]

        def near(x, std):
            return torch.where(mask, x + std * torch.randn(t, generator=g, device=DEV), 0.0).clamp_(max=0.0)

        st["logps"], st["old"], st["cu"], st["mask"] = near(old, 0.15).requires_grad_(), old, cu, mask
        st["reference"] = near(old, 0.1) if case["kl"] else None
        adv = torch.randn(case["seqs"], generator=g, device=DEV)
        if case["advantages"] == "token":
            adv = adv[seq] + 0.3 * torch.randn(t, generator=g, device=DEV)
        st["advantages"] = adv
    else:
        dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
        rows, cols = case["rows"], case["cols"]
        if kind == "pack":
            # a residual stream: a few channels are far larger than the others
            scale = torch.where(torch.rand(cols, generator=g, device=DEV) < 0.01, 30.0, 1.0)
            st["x"] = (torch.randn(rows, cols, generator=g, device=DEV) * scale).to(dtype)
        else:
            both = _normal(g, rows, 2 * cols, std=1.5, dtype=dtype)
            gate, up = both[:, :cols], both[:, cols:]
            if not case["fused"]:
                gate, up = gate.contiguous(), up.contiguous()
            st["gate"], st["up"] = gate.detach().requires_grad_(), up.detach().requires_grad_()
            st["dh"] = _normal(g, rows, cols, std=0.01, dtype=dtype)
    return st


# --------------------------------------------------------------------------- the framework's calls
def _run_own(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "logp":
        from siq_vl_amd.log_probs import fused_linear_log_probs

        logps = fused_linear_log_probs(st["hidden"], st["weight"], st["labels"], temperature=case["temperature"])
        leaves = [st["hidden"]] if case["frozen"] else [st["hidden"], st["weight"]]
        return [logps.detach(), *torch.autograd.grad(logps, leaves, st["up"])]
    if kind == "pref":
        from siq_vl_amd.policy import preference_loss

        out = preference_loss(st["policy"], st["reference"], st["cu"], mask=st["mask"], beta=0.1,
                              loss_type=case["loss_type"], label_smoothing=case["smoothing"],
                              length_normalized=case["normalized"], order=case["order"])
        return [out.loss.detach(), out.chosen_rewards, out.rejected_rewards, *torch.autograd.grad(out.loss, [st["policy"]])]
    if kind == "policy":
        from siq_vl_amd.policy import policy_loss

        out = policy_loss(st["logps"], st["old"], st["advantages"], st["cu"], mask=st["mask"],
                          reference_logps=st["reference"], clip_low=0.2, clip_high=0.25, dual_clip=case["dual"],
                          kl_coef=case["kl_coef"], kl_type=case["kl"] or "k3", aggregation=case["aggregation"])
        return [out.loss.detach(), out.kl, out.clip_fraction, *torch.autograd.grad(out.loss, [st["logps"]])]
    from siq_vl_amd.checkpoint8 import pack8, swiglu8, unpack8

    if kind == "pack":
        return [unpack8(pack8(st["x"], case["format"]))]
    h = swiglu8(st["gate"], st["up"], case["format"])
    return [h.detach(), *torch.autograd.grad(h, [st["gate"], st["up"]], st["dh"])]


# --------------------------------------------------------------------------- the plain form
def _plain_logp(st):
    case = st["case"]
    hid, w, y = st["hidden"].detach().float(), st["weight"].detach().float(), st["labels"]
    counted = y != IGNORE
    at = y.clamp(min=0)[:, None]
    z = hid @ w.T
    z /= case["temperature"]
    top = z.amax(1, keepdim=True)
    zy = z.gather(1, at)
    z -= top
    z.exp_()
    total = z.sum(1, keepdim=True)
    logps = torch.where(counted, ((zy - top) - total.log())[:, 0], 0.0)
    g = torch.where(counted, st["up"], 0.0)[:, None] / case["temperature"]
    z *= -g / total
    z.scatter_add_(1, at, g)
    grads = [(z @ w).to(torch.bfloat16)]
    if not case["frozen"]:
        grads.append((z.T @ hid).to(torch.bfloat16))
    return [logps, *grads]


def _seq_sums(x, cu):
    """Sums over each sequence, in 64 bits."""
    total = torch.zeros(x.numel() + 1, dtype=torch.float64, device=x.device)
    torch.cumsum(x, 0, dtype=torch.float64, out=total[1:])
    return total[cu[1:]] - total[cu[:-1]]


def _seq_of(cu, n):
    return torch.searchsorted(cu[1:], torch.arange(n, dtype=cu.dtype, device=cu.device), right=True)


def _plain_pref(st):
    case, cu, mask, beta = st["case"], st["cu"].long(), st["mask"], 0.1
    pi = st["policy"].detach()
    pairs = case["seqs"] // 2
    score = _seq_sums(torch.where(mask, pi.double() - st["reference"].double(), 0.0), cu)
    per = torch.ones_like(score)
    if case["normalized"]:
        per = 1.0 / _seq_sums(mask, cu).clamp(min=1)
    score = score * per
    if case["order"] == "interleaved":
        chosen, rejected = score[0::2], score[1::2]
    else:
        chosen, rejected = score[:pairs], score[pairs:]
    x = chosen - rejected
    if case["loss_type"] == "sigmoid":
        e = case["smoothing"]
        win, lose = torch.log1p(torch.exp(-beta * x)), torch.log1p(torch.exp(beta * x))
        loss = (1 - e) * win + e * lose
        dx = beta * (e / (1 + torch.exp(-beta * x)) - (1 - e) / (1 + torch.exp(beta * x)))
    elif case["loss_type"] == "ipo":
        loss, dx = (x - 1 / (2 * beta)) ** 2, 2 * (x - 1 / (2 * beta))
    else:
        loss, dx = (1 - beta * x).clamp(min=0), torch.where(beta * x < 1, -beta, 0.0).double()
    dx = dx / pairs
    dseq = (torch.stack([dx, -dx], 1).flatten() if case["order"] == "interleaved" else torch.cat([dx, -dx])) * per
    dpi = torch.where(mask, dseq.float()[_seq_of(cu, pi.numel())], 0.0)
    return [loss.mean().float(), (beta * chosen).float(), (beta * rejected).float(), dpi]


def _plain_policy(st):
    case, cu, mask = st["case"], st["cu"].long(), st["mask"]
    lp, adv = st["logps"].detach(), st["advantages"]
    seq = _seq_of(cu, lp.numel())
    if case["advantages"] == "sequence":
        adv = adv[seq]
    # whether a token is clipped is decided in 64 bits: 32 lose it next to the border
    d = lp.double() - st["old"].double()
    cut = ((adv > 0) & (d > math.log1p(0.25))) | ((adv < 0) & (d < math.log1p(-0.2)))
    r = torch.exp(d.float())
    obj = torch.where(cut, torch.where(adv > 0, 1.25, 0.8) * adv, r * adv)
    if case["dual"]:
        low = (adv < 0) & (d > math.log(case["dual"]))
        obj, cut = torch.where(low, case["dual"] * adv, obj), cut | low
    grad = torch.where(cut, 0.0, -adv * r)
    loss = -obj
    kl = torch.zeros_like(loss)
    if case["kl"]:
        x = (st["reference"].double() - lp.double()).float()
        if case["kl"] == "k3":
            kl, dkl = torch.expm1(x) - x, -torch.expm1(x)
        elif case["kl"] == "k2":
            kl, dkl = 0.5 * x * x, -x
        else:
            kl, dkl = -x, torch.ones_like(x)
        loss = loss + case["kl_coef"] * kl
        grad = grad + case["kl_coef"] * dkl
    loss, grad = torch.where(mask, loss, 0.0), torch.where(mask, grad, 0.0)
    count = mask.sum()
    if case["aggregation"] == "token":
        total, grad = loss.sum(dtype=torch.float64) / count, grad / count
    else:
        per = 1.0 / (case["seqs"] * _seq_sums(mask, cu).clamp(min=1))
        total, grad = (_seq_sums(loss, cu) * per).sum(), grad * per.float()[seq]
    mean_kl = torch.where(mask, kl, 0.0).sum(dtype=torch.float64) / count
    return [total.float(), mean_kl.float(), ((cut & mask).sum() / count).float(), grad]


def _power_of_two(e):
    """2^e in 32 bits for whole e in [-126, 127], from its bits: pow() and ldexp() of a GPU may miss it by a rounding."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _plain_8bit(x, fmt):
    """``x`` rounded to 8-bit codes with one power-of-two step for each 32 neighbours, as the values they stand for."""
    flat = x.detach().float().reshape(-1)
    n = flat.numel()
    groups = torch.nn.functional.pad(flat, (0, -n % GROUP)).view(-1, GROUP)
    m, e = torch.frexp(groups.abs().amax(1, keepdim=True))  # m in [0.5, 1)
    if fmt == "int8":
        # the largest code is 127: one binary step more where it would round past that
        step = _power_of_two((e - 7 + (m >= 255 / 256).to(e.dtype)).clamp(min=-126))
        codes = torch.round(groups / step).clamp(-127, 127)
    else:
        step = _power_of_two((e - 9 + (m > 464 / 512).to(e.dtype)).clamp(min=-126))
        codes = (groups / step).clamp(-448, 448).to(torch.float8_e4m3fn).float()
    return (codes * step).view(-1)[:n].view(x.shape)


def _plain_swiglu(st):
    gate, up, dh = st["gate"].detach().float(), st["up"].detach().float(), st["dh"].float()
    h = gate / (1 + torch.exp(-gate)) * up
    g, u = _plain_8bit(gate, st["case"]["format"]), _plain_8bit(up, st["case"]["format"])
    s = 1 / (1 + torch.exp(-g))
    dgate, dup = dh * u * s * (1 + g * (1 - s)), dh * g * s
    return [x.to(st["gate"].dtype) for x in (h, dgate, dup)]


def run(st):
    if own:
        return _run_own(st)
    kind = st["case"]["kind"]
    if kind == "logp":
        return _plain_logp(st)
    if kind == "pref":
        return _plain_pref(st)
    if kind == "policy":
        return _plain_policy(st)
    if kind == "pack":
        return [_plain_8bit(st["x"], st["case"]["format"]).to(st["x"].dtype)]
    return _plain_swiglu(st)


# --------------------------------------------------------------------------- the same in 64 bits
def _exact_logp(case, st):
    hid, w, y = st["hidden"].detach().double(), st["weight"].detach().double(), st["labels"]
    keep = torch.nonzero(y != IGNORE).flatten()
    logps = torch.zeros(y.numel(), dtype=torch.float64, device=DEV)
    dh = torch.zeros_like(hid)
    dw = None if case["frozen"] else torch.zeros_like(w)
    wt = w.T.contiguous()
    for c in range(0, keep.numel(), 1024):
        rows = keep[c:c + 1024]
        z = hid[rows] @ wt / case["temperature"]
        at = (torch.arange(rows.numel(), device=DEV), y[rows])
        lse = torch.logsumexp(z, dim=1)
        logps[rows] = z[at] - lse
        z = z.sub_(lse[:, None]).exp_().neg_()
        z[at] += 1
        z *= (st["up"][rows].double() / case["temperature"])[:, None]
        dh[rows] = z @ w
        if dw is not None:
            dw += z.T.contiguous() @ hid[rows]
    return [logps, dh] + ([] if dw is None else [dw])


def _segments(x, seq, n):
    return torch.zeros(n, dtype=torch.float64, device=DEV).index_add_(0, seq, x.double())


def _exact_pref(case, st):
    n, mask, beta = case["seqs"], st["mask"], 0.1
    seq = torch.repeat_interleave(torch.arange(n, device=DEV), torch.tensor(_lengths(case), device=DEV))
    pi = st["policy"].detach().double().requires_grad_()
    score = _segments((pi - st["reference"].double())[mask], seq[mask], n)
    if case["normalized"]:
        score = score / _segments(mask, seq, n).clamp(min=1)
    pair = score.view(-1, 2) if case["order"] == "interleaved" else score.view(2, -1).T
    x = pair[:, 0] - pair[:, 1]
    if case["loss_type"] == "sigmoid":
        loss = -(1 - case["smoothing"]) * torch.nn.functional.logsigmoid(beta * x)
        loss = loss - case["smoothing"] * torch.nn.functional.logsigmoid(-beta * x)
    else:
        loss = (x - 0.5 / beta).square() if case["loss_type"] == "ipo" else torch.relu(1 - beta * x)
    loss = loss.mean()
    grad, = torch.autograd.grad(loss, [pi])
    return [loss.detach(), (beta * pair[:, 0]).detach(), (beta * pair[:, 1]).detach(), grad]


def _exact_policy(case, st):
    n, mask = case["seqs"], st["mask"]
    seq = torch.repeat_interleave(torch.arange(n, device=DEV), torch.tensor(_lengths(case), device=DEV))
    lp = st["logps"].detach().double().requires_grad_()
    adv = st["advantages"].double()
    adv = adv[seq] if case["advantages"] == "sequence" else adv
    r = (lp - st["old"].double()).exp()
    obj = torch.minimum(r * adv, r.clamp(1 - 0.2, 1 + 0.25) * adv)
    if case["dual"]:
        obj = torch.where(adv < 0, torch.maximum(obj, case["dual"] * adv), obj)
    slope, = torch.autograd.grad(obj.sum(), [lp], retain_graph=True)
    clipped = (slope == 0) & (adv != 0)
    x = st["reference"].double() - lp if case["kl"] else torch.zeros_like(lp)
    kl = {"k1": -x, "k2": x * x / 2, "k3": torch.expm1(x) - x}[case["kl"] or "k3"]
    loss = case["kl_coef"] * kl - obj
    if case["aggregation"] == "token":
        total = loss[mask].mean()
    else:
        total = (_segments(loss[mask], seq[mask], n) / _segments(mask, seq, n).clamp(min=1)).mean()
    grad, = torch.autograd.grad(total, [lp])
    return [total.detach(), kl[mask].mean().detach(), clipped[mask].double().mean(), grad]


def _exact_8bit(x, fmt):
    def two_to(e):  # from the bits, as pow() may miss it
        return ((e.long() + 1023) << 52).view(torch.float64)

    v = x.detach().double().flatten()
    size = v.numel()
    v = torch.cat([v, v.new_zeros(-size % GROUP)]).view(-1, GROUP)
    top = v.abs().max(1, keepdim=True).values.clamp(min=2.0 ** -140)
    bits = 6 if fmt == "int8" else 8  # the largest value of a group, in steps, lies in [2^bits, 2^(bits + 1))
    exponent = torch.frexp(top).exponent - 1 - bits
    over = torch.round(top / two_to(exponent)) > 127 if fmt == "int8" else top / two_to(exponent) > 464
    step = two_to((exponent + over.to(exponent.dtype)).clamp(min=-126))
    v = v / step
    if fmt == "int8":
        v = torch.round(v)
    else:  # four significant bits, and a multiple of 2^-9
        ulp = two_to((torch.frexp(v).exponent - 4).clamp(min=-9))
        v = torch.round(v / ulp) * ulp
    return (v * step).flatten()[:size].view(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "logp":
        return _exact_logp(case, st)
    if case["kind"] == "pref":
        return _exact_pref(case, st)
    if case["kind"] == "policy":
        return _exact_policy(case, st)
    if case["kind"] == "pack":
        return [_exact_8bit(st["x"], case["format"])]
    gate, up, dh = (st[k].detach().double() for k in ("gate", "up", "dh"))
    h = torch.nn.functional.silu(gate) * up
    g, u = (_exact_8bit(st[k], case["format"]).requires_grad_() for k in ("gate", "up"))
    dgate, dup = torch.autograd.grad(torch.nn.functional.silu(g) * u, [g, u], dh)
    return [h, dgate, dup]
