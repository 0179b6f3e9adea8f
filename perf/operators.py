"""What a training program has this library do with sampled tokens, as cases that can be timed one by one:
logprobs of given tokens with their gradient, the clipped policy loss and the preference loss.

    score       logprobs (and entropies) of given tokens: a prompt, another model's answer, a rollout's tokens
    score-grad  the same and the gradient of a loss that the caller computed from them
    policy      the clipped policy loss with a KL term and an entropy bonus, and the logits' gradient
    preference  the loss over pairs of a chosen and a rejected sequence, and the logits' gradient

A case names the operator (`op`), the block of logits (`rows` x `vocab` of `dtype`, rows `pad` elements further
apart than they are long) and the options of the call. `masked` is the share of each sequence that is its prompt,
whose rows are not trained on; `dead` is how many columns at the end are padding, -inf in every row.

Logits are 3 N(0,1) - 1.2 ln(1 + rank) with a random rank per token: a heavy head over a long noisy tail, the shape
of a language model's logit row. Tokens are drawn from the rows' own distribution, as a rollout's are.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEVICE = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
MOST_BYTES = 4096 * 151936 * 2   # of logits: no case is larger than the largest listed one
SEQUENCE = 96                    # rows of a rollout in the policy cases


def listed():
    return [
        # one candidate token of one answer: pure call latency
        dict(name="score-1x32000-fp32", op="score", rows=1, vocab=32000, dtype="fp32", entropy=False, per_row=False),
        # a prompt's tokens under a reference model, as the KL term wants them
        dict(name="score-2048x128256-bf16", op="score", rows=2048, vocab=128256, dtype="bf16", entropy=True,
             per_row=False),
        # a caller's own loss over a few answers; rows that do not start on 16-byte boundaries
        dict(name="grad-96x50257-fp16", op="score-grad", rows=96, vocab=50257, dtype="fp16", entropy=False,
             per_row=False),
        # the same with an entropy term over rollouts of requests that had their own temperatures
        dict(name="grad-1024x151936-fp32", op="score-grad", rows=1024, vocab=151936, dtype="fp32", entropy=True,
             per_row=True),
        # the last tokens of four short rollouts
        dict(name="policy-4x32000-fp32", op="policy", rows=4, vocab=32000, dtype="fp32", kl=0.05, bonus=0.0, masked=0.0),
        # a micro-batch without a reference model; a third of its rows are prompts
        dict(name="policy-288x49152-bf16", op="policy", rows=288, vocab=49152, dtype="bf16", kl=0.0, bonus=0.01,
             masked=0.34),
        # fp16 with a loss scale, a vocabulary that is no multiple of anything inside padded rows
        dict(name="policy-777x50257-fp16-padded", op="policy", rows=777, vocab=50257, dtype="fp16", kl=0.05, bonus=0.0,
             masked=0.25, pad=47, grad_scale=4096.0),
        # the widest vocabulary in fp32, its last columns padding
        dict(name="policy-384x262144-fp32", op="policy", rows=384, vocab=262144, dtype="fp32", kl=0.02, bonus=0.001,
             masked=0.0, dead=144),
        # a full micro-batch of rollouts: the largest block
        dict(name="policy-4096x151936-bf16", op="policy", rows=4096, vocab=151936, dtype="bf16", kl=0.05, bonus=0.0,
             masked=0.0),
        # one pair of one-line answers
        dict(name="pairs-1-24x32000-fp32", op="preference", rows=24, pairs=1, vocab=32000, dtype="fp32", smoothing=0.0,
             masked=0.0),
        # short ragged answers under a small vocabulary of odd size, noisy labels
        dict(name="pairs-16-600x50257-bf16", op="preference", rows=600, pairs=16, vocab=50257, dtype="bf16",
             smoothing=0.1, masked=0.3),
        # the micro-batch of a preference run: long answers
        dict(name="pairs-8-3600x128256-bf16", op="preference", rows=3600, pairs=8, vocab=128256, dtype="bf16",
             smoothing=0.0, masked=0.2),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above: any operator, vocabularies of 2000 to 262144 (odd ones among them), one row
    up to what fits the largest block."""
    op = rng.choice(["score", "score-grad", "policy", "policy", "preference", "preference"])
    dtype = rng.choice(["bf16", "bf16", "fp32", "fp16"])
    vocab = _log_int(rng, 2000, 262144)
    if rng.random() < 0.5:
        vocab = max(2048, vocab // 64 * 64)   # most models pad their vocabulary, some do not
    rows = min(_log_int(rng, 2 if op == "preference" else 1, 4096), MOST_BYTES // (vocab * SIZE[dtype]))
    case = dict(op=op, rows=rows, vocab=vocab, dtype=dtype, pad=rng.choice([0, 0, 0, 1, 64 - vocab % 64]),
                dead=rng.choice([0, 0, vocab // 50]))
    if op.startswith("score"):
        case.update(entropy=rng.random() < 0.5, per_row=rng.random() < 0.5)
    elif op == "policy":
        case.update(kl=rng.choice([0.0, 0.02, 0.1]), bonus=rng.choice([0.0, 0.0, 0.01]),
                    masked=round(rng.choice([0.0, rng.uniform(0.0, 0.8)]), 3))
    else:
        case.update(pairs=min(_log_int(rng, 1, 256), rows // 2), smoothing=rng.choice([0.0, 0.0, 0.1]),
                    masked=round(rng.choice([0.0, rng.uniform(0.0, 0.6)]), 3))
    if dtype == "fp16" and op in ("policy", "preference"):
        case["grad_scale"] = 4096.0
    return case


# ---- inputs --------------------------------------------------------------------------------------

def _lengths(case):
    """How many rows each sequence of a case has: rollouts of a policy case cut at SEQUENCE rows, the sequences of a
    preference case at random places (some of them next to each other), both the same for every seed."""
    rows = case["rows"]
    if case["op"] == "policy":
        return [min(SEQUENCE, rows - at) for at in range(0, rows, SEQUENCE)]
    rng = random.Random(rows * 1009 + case["pairs"])
    cuts = [0] + sorted(rng.randint(0, rows) for _ in range(2 * case["pairs"] - 1)) + [rows]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _trained(case):
    """1 for every row whose token is trained on, 0 for those of the prompts."""
    if case["op"] not in ("policy", "preference"):
        return [1] * case["rows"]
    on = []
    for n in _lengths(case):
        prompt = int(n * case["masked"])
        on += [0] * prompt + [1] * (n - prompt)
    return on


def _logits(case, gen):
    rows, vocab, pad = case["rows"], case["vocab"], case.get("pad", 0)
    block = torch.zeros((rows, vocab + pad), dtype=DTYPES[case["dtype"]], device=DEVICE)
    for at in range(0, rows, 512):
        n = min(512, rows - at)
        x = torch.rand((n, vocab), generator=gen, device=DEVICE).mul_(vocab).floor_().log1p_().mul_(-1.2)
        x.add_(torch.randn((n, vocab), generator=gen, device=DEVICE), alpha=3.0)
        block[at:at + n, :vocab] = x
    if case.get("dead", 0):
        block[:, vocab - case["dead"]:vocab] = -math.inf
    return block[:, :vocab]


def _rollout(logits, temperature, gen):
    """A token of every row, drawn from its distribution, and its logprob."""
    tokens, logprobs = [], []
    for at in range(0, logits.shape[0], 512):
        z = logits[at:at + 512].float() / temperature[at:at + 512, None]
        z -= torch.logsumexp(z, 1, keepdim=True)
        t = (z.exp() / torch.empty_like(z).exponential_(generator=gen)).argmax(1)
        tokens.append(t)
        logprobs.append(z.gather(1, t[:, None])[:, 0])
    return torch.cat(tokens).to(torch.int32), torch.cat(logprobs)


def _off_the_borders(ratio):
    """Log ratios, those within 1e-4 of the clip's borders moved outwards: at the border itself the last bit of a
    32-bit logprob decides which side the gradient is on, whoever computes it."""
    for b in (math.log1p(-0.2), math.log1p(0.2)):
        ratio = torch.where((ratio - b).abs() < 1e-4, b + math.copysign(3e-4, b), ratio)
    return ratio


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    rows, op = case["rows"], case["op"]
    normal = lambda n: torch.randn(n, generator=gen, device=DEVICE)
    logits = _logits(case, gen)
    temperature = torch.ones(rows, device=DEVICE)
    if case.get("per_row"):
        temperature = torch.rand(rows, generator=gen, device=DEVICE) * 0.9 + 0.6
    tokens, logprobs = _rollout(logits, temperature, gen)
    s = dict(op=op, logits=logits, tokens=tokens, temperature=temperature if case.get("per_row") else None,
             grad_scale=case.get("grad_scale", 1.0))
    on = torch.tensor(_trained(case), device=DEVICE)
    active = max(1, int(on.sum()))
    if op.startswith("score"):
        s.update(entropy=case["entropy"], g=normal(rows), h=normal(rows) * 0.1 if case["entropy"] else None)
    elif op == "policy":   # rewards above a baseline that lags behind
        s.update(old=logprobs - _off_the_borders(normal(rows) * 0.15), advantage=normal(rows) + 0.25, weight=on.float(),
                 ref=logprobs + normal(rows) * 0.2 if case["kl"] else None, kl=case["kl"], bonus=case["bonus"],
                 scale=1.0 / active)
    else:
        s["tokens"] = torch.where(on == 0, -1, tokens).to(torch.int32)
        off = [0]
        for n in _lengths(case):
            off.append(off[-1] + n)
        s.update(off=torch.tensor(off, dtype=torch.int32, device=DEVICE), ref=logprobs + normal(rows) * 0.3,
                 smoothing=case["smoothing"], scale=1.0 / case["pairs"])
    return s


# ---- one pass ------------------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    if s["op"].startswith("score"):
        return _score(s)
    return _policy(s) if s["op"] == "policy" else _preference(s)


def _run_own(s):
    from molla_b200 import losses
    if s["op"].startswith("score"):
        out = losses.token_logprobs(s["logits"], s["tokens"], temperature=s["temperature"], want_entropy=s["entropy"])
        got = dict(logprob=out["logprob"])
        if s["entropy"]:
            got["entropy"] = out["entropy"]
        if s["op"] == "score-grad":
            got["grad"] = losses.token_logprobs_backward(s["logits"], s["tokens"], out, s["g"], grad_entropy=s["h"],
                                                         temperature=s["temperature"])
        return got
    if s["op"] == "policy":
        out = losses.policy_loss(s["logits"], s["tokens"], s["old"], s["advantage"], weight=s["weight"],
                                 ref_logprob=s["ref"], clip_low=0.2, clip_high=0.2, kl_coef=s["kl"],
                                 entropy_coef=s["bonus"], scale=s["scale"], grad_scale=s["grad_scale"])
        names = ["loss", "row_loss", "logprob", "clipped", "grad_logits"]
        names += ["kl"] if s["ref"] is not None else []
        names += ["entropy"] if s["bonus"] else []
        return {k: out[k] for k in names}
    out = losses.preference_loss(s["logits"], s["tokens"], s["off"], ref_logprob=s["ref"], beta=0.1,
                                 label_smoothing=s["smoothing"], scale=s["scale"], grad_scale=s["grad_scale"])
    return {k: out[k] for k in ("loss", "pair_loss", "margin", "seq_logratio", "logprob", "grad_logits")}


# The plain forms: what belongs to a logit in 32 bits, what belongs to a row in 64.

def _softmax(logits, temperature, tokens, want_entropy):
    """(z - max z, exp of that, its sum, the tokens' logprobs, the entropies) of every row."""
    d = logits.float()
    top = d.amax(1, keepdim=True)
    at = tokens.clamp(min=0).long()[:, None]
    token = (d.gather(1, at).double() - top.double())[:, 0]   # a logprob's last bits matter next to another one
    d = d - top
    if temperature is not None:
        d, token = d / temperature[:, None], token / temperature.double()
    e = torch.exp(d)
    total = e.sum(1, dtype=torch.float64)
    logprob = token - total.log()
    entropy = None
    if want_entropy:
        entropy = total.log() - torch.where(e > 0, e * d, 0.0).sum(1, dtype=torch.float64) / total
    return d, e, total, logprob, entropy


def _gradient(d, e, total, entropy, tokens, g, h, temperature, dtype):
    """g d logprob + h d entropy with respect to the logits, rounded once; g and h are a value a row, in 64 bits."""
    inv = total.reciprocal().float()[:, None]
    if temperature is not None:
        g = g / temperature
        h = None if h is None else h / temperature
    if h is None:
        out = e * inv * -g.float()[:, None]
    else:
        u = (d - (total.log() - entropy).float()[:, None]) * h.float()[:, None] + g.float()[:, None]
        out = torch.where(e > 0, e * inv * -u, 0.0)
    at = tokens.clamp(min=0).long()[:, None]
    return out.scatter_add(1, at, g.float()[:, None]).to(dtype)


def _score(s):
    d, e, total, logprob, entropy = _softmax(s["logits"], s["temperature"], s["tokens"], s["entropy"])
    got = dict(logprob=logprob.float())
    if s["entropy"]:
        got["entropy"] = entropy.float()
    if s["op"] == "score-grad":
        got["grad"] = _gradient(d, e, total, entropy, s["tokens"], s["g"].double(), None if s["h"] is None else s["h"].double(),
                                s["temperature"], s["logits"].dtype)
    return got


def _policy(s):
    d, e, total, logprob, entropy = _softmax(s["logits"], None, s["tokens"], s["bonus"] != 0)
    on, w, a = s["weight"] != 0, s["weight"].double(), s["advantage"].double()
    ratio = torch.exp(logprob - s["old"].double())
    free, capped = ratio * a, ratio.clamp(0.8, 1.2) * a
    clipped = on & (capped < free)
    term = -torch.minimum(free, capped)
    g = torch.where(clipped, 0.0, -free)
    got = {}
    if s["ref"] is not None:
        q = s["ref"].double() - logprob
        kl = torch.expm1(q) - q
        term = term + s["kl"] * kl
        g = g - s["kl"] * torch.expm1(q)
        got["kl"] = torch.where(on, kl, 0.0).float()
    h = None
    if s["bonus"]:
        term = term - s["bonus"] * entropy
        h = -w * s["bonus"] * (s["scale"] * s["grad_scale"])
        got["entropy"] = torch.where(on, entropy, 0.0).float()
    row = torch.where(on, w * term, 0.0)
    g = w * g * (s["scale"] * s["grad_scale"])
    got.update(loss=(row.sum() * s["scale"]).float(), row_loss=row.float(), logprob=torch.where(on, logprob, 0.0).float(),
               clipped=clipped, grad_logits=_gradient(d, e, total, entropy, s["tokens"], g, h, None, s["logits"].dtype))
    return got


def _sequence_of(off, rows):
    """The sequence that each row belongs to."""
    return torch.searchsorted(off[1:].long(), torch.arange(rows, device=off.device), right=True)


def _preference(s):
    d, e, total, logprob, _ = _softmax(s["logits"], None, s["tokens"], False)
    on = s["tokens"] >= 0
    logprob = torch.where(on, logprob, 0.0)
    ratio = torch.where(on, logprob - s["ref"].double(), 0.0)
    seq, n = _sequence_of(s["off"], len(on)), len(s["off"]) - 1
    sums = torch.zeros(n, dtype=torch.float64, device=on.device).index_add_(0, seq, ratio)
    margin = 0.1 * (sums[0::2] - sums[1::2])
    soft = lambda m: torch.clamp(m, min=0.0) + torch.log1p(torch.exp(-m.abs()))
    eps = s["smoothing"]
    pair = (1 - eps) * soft(-margin) + eps * soft(margin)
    dm = eps / (1 + torch.exp(-margin)) - (1 - eps) / (1 + torch.exp(margin))
    g = 0.1 * s["scale"] * s["grad_scale"] * torch.stack([dm, -dm], 1).reshape(-1)[seq]
    grad = _gradient(d, e, total, None, s["tokens"], torch.where(on, g, 0.0), None, None, s["logits"].dtype)
    return dict(loss=(pair.sum() * s["scale"]).float(), pair_loss=pair.float(), margin=margin.float(), seq_logratio=sums.float(),
                logprob=logprob.float(), grad_logits=grad)


def work(case):
    """The logits of the rows that count read once; where a gradient is asked for, all rows of it written once; a few
    values a row. Per logit a subtraction, a scaling, an exponential and an addition, two more for the entropy; the
    gradient's exponential and two products."""
    n, v, op = case["rows"], case["vocab"], case["op"]
    on = sum(_trained(case))
    size = SIZE[case["dtype"]]
    grad = op != "score"
    entropy = bool(case.get("entropy") or case.get("bonus"))
    return dict(bytes=on * v * size + (n * v * size if grad else 0) + 32 * n,
                flops=on * v * (4 + 2 * entropy + grad * (4 + 2 * entropy)))


# ---- the definitions, in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    """log softmax and its derivatives from their definitions, a piece of the rows at a time."""
    s = prepare(case, seed)
    x, op = s["logits"], case["op"]
    rows, vocab = x.shape
    t = s["tokens"].long()
    temp = torch.ones(rows, dtype=torch.float64, device=DEVICE) if s["temperature"] is None else s["temperature"].double()
    entropy_wanted = bool(case.get("entropy") or case.get("bonus"))
    if op == "policy":
        on = s["weight"] > 0
    else:
        on = t >= 0
    live = t.clamp(min=0)

    def log_p(a, b):
        z = x[a:b].double() / temp[a:b, None]
        return z - torch.logsumexp(z, dim=1, keepdim=True)

    lp, ent = torch.zeros(rows, dtype=torch.float64, device=DEVICE), torch.zeros(rows, dtype=torch.float64, device=DEVICE)
    step = 256
    for a in range(0, rows, step):
        l = log_p(a, a + step)
        lp[a:a + step] = l[torch.arange(len(l)), live[a:a + step]]
        if entropy_wanted:
            ent[a:a + step] = torch.special.entr(l.exp()).sum(1)
    got = {}
    gh = torch.zeros(rows, dtype=torch.float64, device=DEVICE)
    if op.startswith("score"):
        got["logprob"] = lp
        gl = s["g"].double()
        if case["entropy"]:
            got["entropy"], gh = ent, s["h"].double()
        if op == "score":
            return got
        name = "grad"
    elif op == "policy":
        name = "grad_logits"
        w, adv = s["weight"].double(), s["advantage"].double()
        r = (lp - s["old"].double()).exp()
        inside = (r >= 0.8) & (r <= 1.2)
        held = ~inside & (((adv > 0) & (r > 1.2)) | ((adv < 0) & (r < 0.8)))   # where the clip takes the gradient away
        edge = torch.where(r > 1, 1.2, 0.8)
        surrogate = torch.where(held, edge * adv, r * adv)
        ell, gl = -surrogate, torch.where(held, 0.0, -r * adv)
        if s["ref"] is not None:
            back = s["ref"].double() - lp
            kl = back.exp() - 1 - back
            ell, gl = ell + s["kl"] * kl, gl + s["kl"] * (1 - back.exp())
            got["kl"] = kl * on
        if s["bonus"]:
            ell = ell - s["bonus"] * ent
            gh = -s["bonus"] * w * s["scale"] * s["grad_scale"]
            got["entropy"] = ent * on
        gl = gl * w * s["scale"] * s["grad_scale"]
        got.update(loss=(w * ell).sum() * s["scale"], row_loss=w * ell, logprob=lp * on, clipped=None)
    else:
        name = "grad_logits"
        lp = lp * on
        part = torch.cat([torch.zeros(1, dtype=torch.float64, device=DEVICE), ((lp - s["ref"].double()) * on).cumsum(0)])
        a = part[s["off"][1:].long()] - part[s["off"][:-1].long()]
        m = 0.1 * (a[0::2] - a[1::2])
        ls = torch.nn.functional.logsigmoid
        eps = s["smoothing"]
        pl = -(1 - eps) * ls(m) - eps * ls(-m)
        dm = -(1 - eps) * torch.sigmoid(-m) + eps * torch.sigmoid(m)
        per = torch.repeat_interleave(torch.stack([dm, -dm], 1).flatten(), (s["off"][1:] - s["off"][:-1]).long())
        gl = per * on * 0.1 * s["scale"] * s["grad_scale"]
        got.update(loss=pl.sum() * s["scale"], pair_loss=pl, margin=m, seq_logratio=a, logprob=lp)
    grad = torch.empty((rows, vocab), dtype=torch.float64, device=DEVICE)
    for a in range(0, rows, step):
        l = log_p(a, a + step)
        p = l.exp()
        out = -p * gl[a:a + step, None]
        if entropy_wanted:
            out += gh[a:a + step, None] * (torch.special.entr(p) - p * ent[a:a + step, None])
        out[torch.arange(len(l)), live[a:a + step]] += gl[a:a + step]
        grad[a:a + step] = out / temp[a:a + step, None]
    got[name] = grad
    return got
