"""Logprobs of given tokens, the policy loss and the preference loss against their definitions in 64 bits.

How far a result may be off. With d = (x - max)/T a term e of a row's sum is 2^(c (x - max)): the difference, c and the product are rounded
(half a step of 2^-24 each, relative to the exponent), the exponential is good to 2^-22. The sum adds at most CHAIN
terms one after the other, tree and all. So a probability is relatively off by at most
    rel_p = 2^-22 + 3 |d| 2^-24   and   rel_S = 2^-22 + 3 E|d| 2^-24 + CHAIN 2^-24
(E|d| the mean of |d| under the row's distribution), a logprob by rel_S and half a step of its own value, an entropy, ln S + sum p |d|, by
rel_S + sum p |d| (rel_p + rel_S + 2^-22) and half a step. A derivative's factor g takes its rows' logprob errors times
its own slope with it. A value in the gradient is rounded once: half a step of its type.
"""
import math

import pytest
import torch

from molla_b200 import capi, losses

pytestmark = pytest.mark.gpu

CHAIN = 128
U = 2.0**-24
HALF_STEP = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LEAST = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25}   # below: subnormal steps (an exponential is flushed)
TYPES = [torch.float32, torch.bfloat16, torch.float16]
BAD = capi.ROW_BAD_TOKEN


class Rows:
    """The definitions, in 64 bits, and how far 32-bit rows may be from them."""

    def __init__(self, x, tokens, T=None):
        self.x, self.t, self.dtype = x.double(), tokens.long(), x.dtype
        self.T = torch.ones(x.shape[0], dtype=torch.float64, device=x.device) if T is None else T.double()
        self.on = self.t >= 0
        self.at = self.t.clamp(0, x.shape[1] - 1)[:, None]
        z = self.x / self.T[:, None]
        self.d = (z - z.max(1, keepdim=True).values).abs()
        self.lnp = z - torch.logsumexp(z, 1, keepdim=True)
        self.p = self.lnp.exp()
        live = self.p > 0
        zero = torch.zeros((), dtype=torch.float64, device=x.device)
        self.pd = torch.where(live, self.p * self.d, zero)
        self.mean_d = self.pd.sum(1)
        self.plnp = torch.where(live, self.p * self.lnp, zero)
        self.l = self.lnp.gather(1, self.at)[:, 0]
        self.H = -self.plnp.sum(1)
        self.rel_p = 2.0**-22 + 3 * self.d * U
        self.rel_S = 2.0**-22 + 3 * self.mean_d * U + CHAIN * U
        d_t = self.d.gather(1, self.at)[:, 0]
        self.err_l64 = self.rel_S + 2 * d_t * 2.0**-52
        self.err_l = self.err_l64 + self.l.abs() * U
        self.err_H64 = self.rel_S + (torch.where(live, self.pd * self.rel_p, zero)).sum(1) + self.mean_d * (self.rel_S + 2.0**-22)
        self.err_H = self.err_H64 + self.H.abs() * U

    def gradient(self, g, h=None, err_g=None):
        """(g dl + h dH by the logits, how far it may be off); g, h a value a row."""
        g = torch.where(self.on, g.double(), 0.0)
        h = torch.zeros_like(g) if h is None else torch.where(self.on, h.double(), 0.0)
        err_g = torch.zeros_like(g) if err_g is None else err_g
        lnp = torch.where(self.p > 0, self.lnp, 0.0)
        inner = g[:, None] + h[:, None] * (lnp + self.H[:, None])
        out = -self.p * inner
        out.scatter_add_(1, self.at, g[:, None])
        one = torch.zeros_like(out).scatter_(1, self.at, 1.0)
        size = g.abs()[:, None] + h.abs()[:, None] * (lnp.abs() + self.H[:, None])
        rel = self.rel_p + self.rel_S[:, None] + 8 * U
        off = self.p * (size * rel + h.abs()[:, None] * (self.err_H64[:, None] + lnp.abs() * 4 * U) + err_g[:, None])
        off = off + one * (g.abs()[:, None] * 2 * U + err_g[:, None])
        out, off = out / self.T[:, None], off / self.T[:, None]
        return out, off + (out.abs() + off) * HALF_STEP[self.dtype] + LEAST[self.dtype] * (1 + size / self.T[:, None])


def close(got, want, off, what=""):
    got = got.double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= off)
    assert not bool(bad.any()), (what, int(bad.sum()), got[bad][:4], want[bad][:4], off.expand_as(want)[bad][:4])


def make(B, V, dtype, dev, seed=0, pad=0, shift=0, spread=3.0):
    """Logits with a heavy head, `pad` elements between the rows and `shift` before the first."""
    gen = torch.Generator(device=dev)
    gen.manual_seed(1000 * seed + 7 * B + V)
    buf = torch.full((shift + B * (V + pad),), math.nan, dtype=dtype, device=dev)
    x = buf[shift:].as_strided((B, V), (V + pad, 1))
    x.copy_(spread * torch.randn((B, V), generator=gen, device=dev) - 1.2 * torch.log1p(torch.randint(0, V, (B, V), generator=gen, device=dev)))
    tok = torch.randint(0, V, (B,), generator=gen, device=dev, dtype=torch.int32)
    return x, tok, gen


def normal(gen, n, dev):
    return torch.randn(n, generator=gen, device=dev)


SHAPES = [(1, 1), (3, 2), (5, 7), (2, 31), (4, 33), (700, 64), (3, 1000), (2, 1024), (3, 1025), (5, 2047), (9, 4099), (3, 8193),
          (33, 5000), (1, 32000), (160, 32000), (7, 50257), (2, 151936), (1, 262144)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,V", SHAPES)
def test_logprobs_entropies_and_their_gradient(dev, lib, B, V, dtype):
    x, tok, gen = make(B, V, dtype, dev)
    T = torch.rand(B, generator=gen, device=dev) * 1.5 + 0.4
    g, h = normal(gen, B, dev), normal(gen, B, dev)
    for temperature in (None, T):
        ref = Rows(x, tok, temperature)
        plain = losses.token_logprobs(x, tok, temperature=temperature)
        got = losses.token_logprobs(x, tok, temperature=temperature, want_entropy=True)
        assert torch.equal(plain["logprob"], got["logprob"]) and not got["row_status"].any()
        close(got["logprob"], ref.l, ref.err_l, "logprob")
        close(got["entropy"], ref.H, ref.err_H, "entropy")
        close(losses.token_logprobs_backward(x, tok, plain, g, temperature=temperature), *ref.gradient(g), "gradient")
        # its own entropies come back into the gradient: rounded once more
        both, off = ref.gradient(g, h)
        off = off + ref.p * (h.abs().double() * (ref.err_H + ref.H.abs() * U) / ref.T)[:, None]
        close(losses.token_logprobs_backward(x, tok, got, g, grad_entropy=h, temperature=temperature), both, off, "with entropies")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,shift,out_pad,out_shift", [(1, 0, 0, 0), (3, 1, 3, 1), (0, 5, 0, 5), (8, 0, 3, 0), (0, 0, 1, 3), (64, 2, 0, 0)])
@pytest.mark.parametrize("V", [29, 3001, 9000])
def test_strides_and_alignments(dev, lib, V, pad, shift, out_pad, out_shift, dtype):
    B = 11
    x, tok, gen = make(B, V, dtype, dev, pad=pad, shift=shift)
    buf = torch.full((out_shift + B * (V + out_pad) + 16,), 5.0, dtype=dtype, device=dev)
    out = buf[out_shift:].as_strided((B, V), (V + out_pad, 1))
    g = normal(gen, B, dev)
    ref = Rows(x, tok)
    got = losses.token_logprobs(x, tok)
    close(got["logprob"], ref.l, ref.err_l)
    assert losses.token_logprobs_backward(x, tok, got, g, out=out) is out
    close(out, *ref.gradient(g))
    adv = normal(gen, B, dev)
    out.fill_(7.0)
    p = losses.policy_loss(x, tok, got["logprob"], adv, out=out)
    rel = ref.err_l + ref.err_l64
    close(out, *ref.gradient(-adv, err_g=adv.abs().double() * rel * 1.01))
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep[out_shift:].as_strided((B, V), (V + out_pad, 1)).fill_(False)
    assert bool((buf[keep] == 5.0).all()), "something was written between the rows"
    assert torch.equal(p["logprob"], got["logprob"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1.0, 0.6])
def test_the_entropy_gradient_of_flat_rows(dev, lib, T, dtype):
    """-h p (ln p + H)/T is as small as the logits are close, beside an entropy of 12. The depth between them is some 40 sums in 32 bits from
    its terms: relatively off by 40^(1/2) 2^-24 / 3^(1/2) = 2.2e-7 as a standard error, and four times as large as a spread of the logits
    (4.3 at 151936); 1e-6 of the gradient's norm, and each value's own roundings 3e-7. Through the entropy, off by 2.8e-7, it was 1e-5."""
    B, V = 64, 151936
    gen = torch.Generator(device=dev)
    gen.manual_seed(71)
    x = (0.03 * torch.randn((B, V), generator=gen, device=dev)).to(dtype)
    tok = torch.randint(0, V, (B,), generator=gen, device=dev, dtype=torch.int32)
    temperature, zero, h = torch.full((B,), T, device=dev), torch.zeros(B, device=dev), torch.full((B,), 2.0**12, device=dev)
    got = losses.token_logprobs(x, tok, temperature=temperature, want_entropy=True)
    out = losses.token_logprobs_backward(x, tok, got, zero, grad_entropy=h, temperature=temperature)
    same = losses.policy_loss(x, tok, got["logprob"], zero, entropy_coef=-(2.0**12), temperature=temperature)
    assert torch.equal(out, same["grad_logits"]) and torch.equal(got["entropy"], same["entropy"])
    ref = Rows(x, tok, temperature)
    want, off = ref.gradient(zero, h)
    close(out, want, off)
    if dtype is torch.float32:
        assert float((out.double() - want).norm() / want.norm()) < 2e-6
    # callers who kept no more than the entropies
    kept = dict(stats=got["stats"], entropy=got["entropy"])
    close(losses.token_logprobs_backward(x, tok, kept, zero, grad_entropy=h, temperature=temperature), want,
          off + ref.p * (h.double() * (ref.err_H + ref.H.abs() * U) / ref.T)[:, None])


# ---- what is left of the rounding ---------------------------------------------------------------------------
#
# Beside a reference logprob that is the row's own, rounded to 32 bits, a sequence of one row has its log ratio in full: the logprob's
# error is seen to 1e-13. A term of a row's sum is off by at random up to 2^-22 (its exponential) and by half a step of its exponent, for those that count 2^-23
# or less; of many terms that is below 2^-24 of the sum as a standard error, the logarithm's 2^-25 with it. Over 2048 rows the mean
# keeps 1/45 of that, 1.3e-9. What has one sign in all rows is larger by far where it is left in: 5e-8 of the hardware's exponential, 4e-8 of the
# rounding of log2(e)/T, up to 2^-24 of a sum in 32 bits. MEAN is below these and above 3 x 1.3e-9 twice over.

MEAN, STANDARD = 2.0**-26, 2.0**-24


def logprob_errors(x, tok, T=None):
    B = len(tok)
    exact = torch.cat([Rows(x[a:a + 256], tok[a:a + 256], None if T is None else T[a:a + 256]).l for a in range(0, B, 256)])
    ref = exact.float()
    off = torch.arange(B + 1, dtype=torch.int32, device=x.device)
    got = losses.preference_loss(x, tok, off, ref_logprob=ref, temperature=T, want_grad=False)
    assert not got["row_status"].any()
    long = losses.preference_loss(x, tok, off[[0, B // 2, B]], ref_logprob=ref, temperature=T, want_grad=False)["seq_logratio"]
    left = exact - ref.double()
    return got["seq_logratio"].double() - left, long.double() - left.view(2, -1).sum(1)


def check_errors(errors, long, mean=MEAN):
    n = len(errors) // 2
    assert abs(float(errors.mean())) <= mean, float(errors.mean())
    assert float(errors.std()) <= STANDARD, float(errors.std())
    assert bool((long.abs() <= n * mean + 4 * math.sqrt(n) * STANDARD).all()), long


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,T", [(32000, None), (128256, None), (50257, 0.7), (32000, 1.3)])
def test_errors_of_logprobs_do_not_add_up(dev, lib, V, T, dtype):
    x, tok, gen = make(2048, V, dtype, dev, seed=59)
    check_errors(*logprob_errors(x, tok, None if T is None else torch.full((2048,), T, device=dev)))


@pytest.mark.parametrize("spread", [0.03, 0.3, 1.0])
def test_errors_of_flat_rows_do_not_add_up(dev, lib, spread):
    """Logits close to one another, at the temperature between 1/2 and 2 whose exponents are rounded most. Of a spread of 0.03 the exponents
    have a mean of -4 x 0.03 x 1.44 / 1.1 = -0.16 and a standard deviation of 0.04: where they all lie in a sixth of a binade the exponential's errors
    there, up to 2^-22 each, need not have the mean of a whole one, and the sum's may be as large. Of 0.3 they are spread over two binades."""
    B, V = 2048, 32000
    gen = torch.Generator(device=dev)
    gen.manual_seed(67)
    x = spread * torch.randn((B, V), generator=gen, device=dev)
    tok = torch.randint(0, V, (B,), generator=gen, device=dev, dtype=torch.int32)
    check_errors(*logprob_errors(x, tok, torch.full((B,), 1.1, device=dev)), mean=2.0**-22 if spread < 0.1 else MEAN)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("masked", [False, True])
def test_errors_of_rows_of_equal_logits_do_not_add_up(dev, lib, masked, dtype):
    """Rows of k logits that are alike, the others -inf, at the end of the row or in between: the probabilities are 1/k."""
    B, V = 2048, 9000
    gen = torch.Generator(device=dev)
    gen.manual_seed(61)
    k = torch.randint(700, V, (B, 1), generator=gen, device=dev)
    place = torch.rand((B, V), generator=gen, device=dev).argsort(1) if masked else torch.arange(V, device=dev).expand(B, V)
    x = torch.where(place < k, torch.randint(-40, 40, (B, 1), generator=gen, device=dev) / 4.0, -math.inf).to(dtype)
    check_errors(*logprob_errors(x, place.argmin(1).to(torch.int32)))


# ---- the policy loss -----------------------------------------------------------------------------------

def policy_reference(x, tok, old, adv, w=None, ref=None, lo=0.2, hi=0.2, kl=0.0, ent=0.0, T=None, scale=1.0, grad_scale=1.0):
    R = Rows(x, tok, T)
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))   # settings cross the C entry point as fp32
    lo, hi, kl, ent, gs = f32(lo), f32(hi), f32(kl), f32(ent), f32(scale) * f32(grad_scale)
    w = torch.ones_like(R.l) if w is None else w.double()
    on = R.on & (w != 0)
    r = torch.exp(R.l - old.double())
    u, c = r * adv.double(), r.clamp(1 - lo, 1 + hi) * adv.double()
    held = on & (c < u)
    term, g = -torch.minimum(u, c), torch.where(held, 0.0, -u)
    err_term = torch.where(held, 0.0, u.abs() * R.err_l64 * 1.01)
    err_g = err_term.clone()
    k = None
    if ref is not None:
        q = ref.double() - R.l
        k = torch.expm1(q) - q
        term, g = term + kl * k, g - kl * torch.expm1(q)
        err_k = torch.expm1(q).abs() * R.err_l64 + torch.exp(q) * R.err_l64**2
        err_term, err_g = err_term + kl * err_k, err_g + kl * torch.exp(q) * R.err_l64 * 1.01
    term = term - ent * R.H
    err_term = err_term + ent * R.err_H64
    row = torch.where(on, w * term, 0.0)
    err_row = torch.where(on, w.abs() * err_term, 0.0) + row.abs() * U
    z = lambda v: torch.where(on, v, 0.0)
    R.on = on
    grad = R.gradient(z(w * g) * gs, z(-w * ent) * gs, z(w.abs() * err_g) * abs(gs))
    loss = row.sum() * f32(scale)
    return dict(R=R, on=on, held=held, row=row, err_row=err_row, kl=k, err_kl=None if k is None else err_k + k.abs() * U, grad=grad,
                loss=loss, err_loss=err_row.sum() * abs(f32(scale)) + loss.abs() * U, w=w)


def check_policy(got, want):
    R, on = want["R"], want["on"]
    assert not got["row_status"].any()
    close(got["logprob"], torch.where(on, R.l, 0.0), torch.where(on, R.err_l, 0.0), "logprob")
    close(got["row_loss"], want["row"], want["err_row"], "row loss")
    close(got["loss"], want["loss"], want["err_loss"], "loss")
    assert torch.equal(got["clipped"], want["held"])
    if got["entropy"] is not None:
        close(got["entropy"], torch.where(on, R.H, 0.0), torch.where(on, R.err_H, 0.0), "entropy")
    if got["kl"] is not None:
        close(got["kl"], torch.where(on, want["kl"], 0.0), torch.where(on, want["err_kl"], 0.0), "kl")
    if got["grad_logits"] is not None:
        close(got["grad_logits"], *want["grad"], "gradient")


def rollout(x, tok, gen, dev, T=None):
    """Old and reference logprobs near the rows' own (none within 1e-3 of a clip border of 0.2), and advantages."""
    l = Rows(x, tok, T).l
    n = normal(gen, len(l), dev).double() * 0.25
    for b in (math.log(0.8), math.log(1.2)):
        n = torch.where((n - b).abs() < 1e-3, n + 3e-3, n)
    return (l - n).float(), (l + 0.2 * normal(gen, len(l), dev).double()).float(), normal(gen, len(l), dev)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,V", [(1, 1), (2, 9), (6, 1031), (40, 2500), (300, 513), (3, 32000), (170, 6007), (2, 200001)])
@pytest.mark.parametrize("terms", ["clip", "kl", "entropy", "all"])
def test_policy_loss(dev, lib, B, V, dtype, terms):
    x, tok, gen = make(B, V, dtype, dev, seed=3)
    T = torch.rand(B, generator=gen, device=dev) + 0.5 if terms == "all" else None
    old, ref, adv = rollout(x, tok, gen, dev, T)
    k = dict(T=None, ref=None, kl=0.0, ent=0.0, w=None, scale=1.0, grad_scale=1.0)
    if terms in ("kl", "all"):
        k.update(ref=ref, kl=0.07)
    if terms in ("entropy", "all"):
        k.update(ent=0.03)
    if terms == "all":
        w = torch.rand(B, generator=gen, device=dev) + 0.5
        w[::3] = 0.0
        k.update(T=T, w=w, scale=1.0 / B, grad_scale=512.0)
    want = policy_reference(x, tok, old, adv, **k)
    args = dict(weight=k["w"], ref_logprob=k["ref"], kl_coef=k["kl"], entropy_coef=k["ent"], temperature=k["T"], scale=k["scale"],
                grad_scale=k["grad_scale"])
    got = losses.policy_loss(x, tok, old, adv, **args)
    check_policy(got, want)
    # without a gradient, and in the logits' place: the same
    none = losses.policy_loss(x, tok, old, adv, want_grad=False, **args)
    assert none["grad_logits"] is None
    y = x.clone()
    place = losses.policy_loss(y, tok, old, adv, out=y, **args)
    assert place["grad_logits"] is y and torch.equal(y, got["grad_logits"])
    for n in ("loss", "row_loss", "logprob", "clipped"):
        assert torch.equal(none[n], got[n]) and torch.equal(place[n], got[n]), n


def test_old_and_reference_logprobs_far_from_the_rows_own(dev, lib):
    """Impossible tokens and infinite logprobs: what the formulas give, row by row."""
    V = 300
    x, tok, gen = make(7, V, torch.float32, dev, seed=41)
    x[5] = 0.0
    x[5, int(tok[5])] = -math.inf                      # a token that cannot be: ratio 0, KL infinite
    x[6] = 0.0
    x[6, int(tok[6])], x[6, int(tok[6]) - 1] = -3e38, 3e38   # one whose logprob is beyond 32 bits
    l = losses.token_logprobs(x, tok)["logprob"]
    assert l[5] == -math.inf and l[6] == -math.inf and bool(l[:5].isfinite().all())
    inf = math.inf
    old = torch.tensor([-inf, -inf, 0.0, 0.0, 0.0, 0.0, 0.0], device=dev)
    old[2:5] = l[2:5]
    ref = l.clone()
    ref[2], ref[3] = -inf, l[3] + 200.0
    ref[5:] = 0.0
    adv = torch.tensor([1.0, -1.0, 1.0, 1.0, 0.0, -1.0, 1.0], device=dev)
    got = losses.policy_loss(x, tok, old, adv, ref_logprob=ref, kl_coef=0.5)
    assert got["clipped"].tolist() == [True, False, False, False, False, True, False]
    row, kl, grad = got["row_loss"].tolist(), got["kl"].tolist(), got["grad_logits"]
    # the clip holds an infinite ratio; what is left is the KL term's, whose q is the rounding of the reference logprob, half a step of it
    assert abs(row[0] + 1.2) < 2e-7 and bool((grad[0].abs() <= 0.5 * 1.01 * float(l[0].abs()) * U).all())
    assert row[1] == inf and not grad[1].isfinite().all()
    assert kl[2] == inf and row[2] == inf                         # exp(q) - 1 is -1: the gradient is finite
    R = Rows(x[2:3], tok[2:3])
    close(grad[2:3], *R.gradient(torch.tensor([-1.0 + 0.5], device=dev), err_g=2 * R.err_l))
    assert kl[3] == inf and row[3] == inf
    assert abs(row[4]) < 1e-6 and not bool((grad[4].abs() > 1e-6).any())
    assert kl[5] == inf and kl[6] == inf


def test_the_clip_on_either_side(dev, lib):
    """Ratios of 1/2, 1 and 2 for advantages of either sign, one of zero, and clip ranges that are not alike."""
    V = 500
    x, tok, gen = make(7, V, torch.float32, dev, seed=5)
    l = Rows(x, tok).l
    ratio = torch.tensor([0.5, 0.5, 1.0, 1.0, 2.0, 2.0, 2.0], dtype=torch.float64, device=dev)
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 1.0, -1.0, 0.0], device=dev)
    old = (l - ratio.log()).float()
    for lo, hi, held in ((0.2, 0.2, [0, 1, 0, 0, 1, 0, 0]), (0.6, 0.2, [0, 0, 0, 0, 1, 0, 0]), (0.2, 3.0, [0, 1, 0, 0, 0, 0, 0]),
                         (0.2, math.inf, [0, 1, 0, 0, 0, 0, 0]), (2.0, 0.0, None)):
        want = policy_reference(x, tok, old, adv, lo=lo, hi=hi)
        got = losses.policy_loss(x, tok, old, adv, clip_low=lo, clip_high=hi)
        if held is not None:
            check_policy(got, want)
            assert got["clipped"].int().tolist() == held
            assert not got["grad_logits"][got["clipped"]].any()


def test_a_rollout_scored_by_the_policy_that_made_it_has_ratios_of_one(dev, lib):
    """The same rows give the same logprobs, bit for bit, from every call and in every batch: the ratio is exactly one."""
    for dtype in TYPES:
        for V in (4096, 32000, 151936):
            x, tok, gen = make(37, V, dtype, dev, seed=11)
            adv = normal(gen, 37, dev)
            all_rows = losses.token_logprobs(x, tok)
            for n in (1, 2, 5, 19, 37):
                part = losses.token_logprobs(x[:n], tok[:n], want_entropy=True)
                assert torch.equal(part["logprob"], all_rows["logprob"][:n])
                got = losses.policy_loss(x[:n], tok[:n], part["logprob"], adv[:n])
                assert torch.equal(got["logprob"], part["logprob"])
            off = torch.tensor([0, 20, 37], dtype=torch.int32, device=dev)
            assert torch.equal(losses.preference_loss(x, tok, off)["logprob"], all_rows["logprob"])
            got = losses.policy_loss(x, tok, all_rows["logprob"], adv)
            # the old logprobs are rounded to 32 bits: within half a step of one
            assert bool(((got["row_loss"] + adv).abs() <= adv.abs() * (all_rows["logprob"].abs() * U + 2 * U)).all())


@pytest.mark.parametrize("B,V,dtype", [(2400, 30001, torch.bfloat16), (2400, 9001, torch.float32), (1200, 28601, torch.float32),
                                       (1200, 57201, torch.float16), (1200, 129000, torch.bfloat16)])
def test_rows_among_many_are_what_they_are_among_few(dev, lib, B, V, dtype):
    """The same bits, whatever the number of rows makes of their way through the device; in place as well."""
    x, tok, gen = make(B, V, dtype, dev, seed=B + V)
    old, ref, adv, g, h = (normal(gen, B, dev) for _ in range(5))
    T = 0.5 + torch.rand(B, generator=gen, device=dev)
    tok[7::13] = -1

    def calls(s):
        scored = losses.token_logprobs(x[s], tok[s], T[s], want_entropy=True)
        grad = losses.token_logprobs_backward(x[s], tok[s], scored, g[s], h[s], T[s])
        plain = losses.token_logprobs(x[s], tok[s], T[s])["logprob"]
        pol = losses.policy_loss(x[s], tok[s], old[s], adv[s], ref_logprob=ref[s], kl_coef=0.1, entropy_coef=0.01, temperature=T[s])
        place = x[s].clone()
        losses.policy_loss(place, tok[s], old[s], adv[s], out=place)
        return [scored["logprob"], scored["entropy"], grad, plain, pol["row_loss"], pol["logprob"], pol["entropy"], pol["grad_logits"], place]

    many = calls(slice(0, B))
    for s in (slice(0, 24), slice(B // 2, B // 2 + 40), slice(B - 24, B)):
        for k, (a, b) in enumerate(zip(many, calls(s))):
            assert torch.equal(a[s].view(torch.uint8 if a.dim() > 1 else a.dtype), b.view(torch.uint8 if b.dim() > 1 else b.dtype)), (k, s)


# ---- the preference loss ---------------------------------------------------------------------------------

def preference_reference(x, tok, off, ref=None, w=None, beta=0.1, eps=0.0, T=None, scale=1.0, grad_scale=1.0):
    R = Rows(x, tok, T)
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))
    beta, eps, gs = f32(beta), f32(eps), f32(scale) * f32(grad_scale)
    n = (len(off) - 1) // 2
    w = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    ratio = torch.where(R.on, R.l - (0.0 if ref is None else ref.double()), 0.0)
    o = off.tolist()
    err = torch.where(R.on, R.err_l, 0.0)
    s = torch.stack([ratio[a:b].sum() for a, b in zip(o, o[1:])])
    e = torch.stack([err[a:b].sum() for a, b in zip(o, o[1:])])
    m, em = beta * (s[0::2] - s[1::2]), beta * (e[0::2] + e[1::2])
    sp = torch.nn.functional.softplus
    soft = lambda v: torch.where(v > 30, v + torch.exp(-v), sp(v))
    pair = w * ((1 - eps) * soft(-m) + eps * soft(m))
    dm = w * (eps * torch.sigmoid(m) - (1 - eps) * torch.sigmoid(-m))
    g, eg = torch.zeros_like(R.l), torch.zeros_like(R.l)
    for p in range(n):
        sig = float(torch.sigmoid(m[p]))
        slope = float(w[p].abs()) * sig * (1 - sig) * 1.01
        for a, b, sign in ((o[2 * p], o[2 * p + 1], 1.0), (o[2 * p + 1], o[2 * p + 2], -1.0)):
            g[a:b] = sign * beta * dm[p] * gs
            eg[a:b] = abs(beta * gs) * (slope * em[p] + dm[p].abs() * 2 * U)
    inside = torch.zeros_like(R.on)
    inside[o[0]:o[-1]] = True
    on = R.on
    R.on = on & inside
    grad = R.gradient(g, None, torch.where(R.on, eg, 0.0))
    return dict(l=torch.where(on, R.l, 0.0), err_l=torch.where(on, R.err_l, 0.0), s=s, err_s=e + s.abs() * U, m=m, err_m=em + m.abs() * U, pair=pair,
                err_pair=w.abs() * em + pair.abs() * 2 * U, loss=pair.sum() * f32(scale), grad=grad, scale=f32(scale))


def check_preference(got, want):
    assert not got["row_status"].any() and not got["pair_status"].any()
    close(got["logprob"], want["l"], want["err_l"], "logprob")
    close(got["seq_logratio"], want["s"], want["err_s"], "log ratios")
    close(got["margin"], want["m"], want["err_m"], "margin")
    close(got["pair_loss"], want["pair"], want["err_pair"], "pair loss")
    close(got["loss"], want["loss"], abs(want["scale"]) * want["err_pair"].sum() + want["loss"].abs() * U, "loss")
    if got["grad_logits"] is not None:
        close(got["grad_logits"], *want["grad"], "gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,off", [(5, [0, 1, 2]), (1009, [0, 3, 9, 9, 12, 40, 41]), (3000, [2, 5, 5, 5, 5, 70, 130]), (50257, [0, 9, 20]),
                                   (515, [0, 200, 333]), (70, list(range(0, 331, 5)))])
@pytest.mark.parametrize("options", ["plain", "all"])
def test_preference_loss(dev, lib, V, off, dtype, options):
    """Sequences of no row, of one, rows of no sequence before and behind, rows without a token, weights of zero."""
    B = off[-1] + (3 if options == "all" else 0)
    x, tok, gen = make(B, V, dtype, dev, seed=17)
    o = torch.tensor(off, dtype=torch.int32, device=dev)
    n = len(off) // 2
    k = dict(ref=(Rows(x, tok).l + 0.3 * normal(gen, B, dev).double()).float())
    if options == "all":
        tok[::4] = -1
        w = torch.rand(n, generator=gen, device=dev) + 0.5
        w[1::3] = 0.0
        k.update(w=w, beta=0.4, eps=0.1, T=torch.rand(B, generator=gen, device=dev) + 0.5, scale=1.0 / n, grad_scale=256.0)
    want = preference_reference(x, tok, o, **k)
    args = dict(ref_logprob=k["ref"], pair_weight=k.get("w"), beta=k.get("beta", 0.1), label_smoothing=k.get("eps", 0.0),
                temperature=k.get("T"), scale=k.get("scale", 1.0), grad_scale=k.get("grad_scale", 1.0))
    got = losses.preference_loss(x, tok, o, **args)
    check_preference(got, want)
    assert not got["grad_logits"][off[-1]:].any() and not got["grad_logits"][:off[0]].any()
    none = losses.preference_loss(x, tok, o, want_grad=False, **args)
    y = x.clone()
    place = losses.preference_loss(y, tok, o, out=y, **args)
    assert none["grad_logits"] is None and torch.equal(y, got["grad_logits"])
    for name in ("loss", "pair_loss", "margin", "seq_logratio", "logprob"):
        assert torch.equal(none[name], got[name]) and torch.equal(place[name], got[name]), name


def test_margins_far_from_zero(dev, lib):
    """Sure pairs: a loss of next to nothing on one side, of the margin on the other, gradients to match."""
    x, tok, gen = make(4, 64, torch.float32, dev)
    off = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device=dev)
    ref = torch.tensor([-900.0, 0.0, 0.0, -900.0], device=dev)
    got = losses.preference_loss(x, tok, off, ref_logprob=ref, beta=1.0)
    assert got["margin"][0] > 800 and got["margin"][1] < -800
    assert got["pair_loss"][0] == 0 and got["pair_loss"][1] == -got["margin"][1]
    assert not got["grad_logits"][:2].any()
    close(got["grad_logits"][2:], *(v[2:] for v in Rows(x, tok).gradient(torch.tensor([0.0, 0.0, -1.0, 1.0], device=dev))))


@pytest.mark.parametrize("dtype", TYPES)
def test_margins_of_tokens_that_cannot_be(dev, lib, dtype):
    """A token whose logit is -inf in the rejected sequence: the margin is +inf, -ln sigmoid of it 0, and the pair adds nothing to loss
    and gradient. In the chosen one the loss is +inf and its derivative by the margin -1. The other pair is as if alone."""
    x, tok, gen = make(6, 300, dtype, dev, seed=53)
    off = torch.tensor([0, 2, 4, 5, 6], dtype=torch.int32, device=dev)
    alone = losses.preference_loss(x[4:], tok[4:], torch.arange(3, dtype=torch.int32, device=dev))
    for row, margin, loss in ((3, math.inf, 0.0), (0, -math.inf, math.inf)):
        y = x.clone()
        y[row, int(tok[row])] = -math.inf
        got = losses.preference_loss(y, tok, off)
        assert got["margin"][0] == margin and got["pair_loss"][0] == loss and not got["pair_status"].any() and not got["row_status"].any()
        assert got["pair_loss"][1] == alone["pair_loss"][0] and got["loss"] == alone["loss"] + loss
        assert torch.equal(got["grad_logits"][4:], alone["grad_logits"])
        g = torch.zeros(4, device=dev) if loss == 0 else torch.tensor([-0.1, -0.1, 0.1, 0.1], device=dev)
        R = Rows(y[:4], tok[:4])
        R.rel_p = torch.where(R.p > 0, R.rel_p, 0.0)
        close(got["grad_logits"][:4], *R.gradient(g))
        # a label that may be wrong makes a sure pair infinitely dear; a weight of 0 none
        smooth = losses.preference_loss(y, tok, off, label_smoothing=0.1)
        assert smooth["pair_loss"][0] == math.inf and bool(smooth["grad_logits"].isfinite().all())
        w = losses.preference_loss(y, tok, off, pair_weight=torch.tensor([0.0, 1.0], device=dev))
        assert w["loss"] == alone["loss"] and not w["grad_logits"][:4].any()


@pytest.mark.parametrize("off", [[0, 3, 2], [-1, 3, 6], [0, 3, 9], [0, 2, 4, 3, 8], [0, 5, 8, 2, 3, 4, 8], [2**31 - 1, -2**31, 5]])
def test_offsets_against_the_rules(dev, lib, off):
    x, tok, _ = make(8, 100, torch.float32, dev)
    o = torch.tensor(off, dtype=torch.int32, device=dev)
    got = losses.preference_loss(x, tok, o)
    n = len(off) // 2
    ok = lambda a, b: 0 <= a <= b <= 8
    want = [0 if ok(off[2 * p], off[2 * p + 1]) and ok(off[2 * p + 1], off[2 * p + 2]) else capi.ROW_INVALID_CONFIG for p in range(n)]
    assert got["pair_status"].tolist() == want and any(want)
    for name in ("loss", "pair_loss", "margin", "seq_logratio"):
        assert bool(got[name].isnan().all()), name
    assert not got["grad_logits"].any()


# ---- rows that cannot be answered, and values that are not ordinary -----------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [8, 1500, 40000])
def test_rows_without_an_answer(dev, lib, V, dtype):
    B = 9
    x, tok, gen = make(B, V, dtype, dev, seed=23)
    T = torch.ones(B, device=dev)
    tok[1], tok[2], tok[3] = V, -2, -1
    x[4] = -math.inf
    T[5], T[6], T[7] = 0.0, math.nan, -1.0
    INV, EMPTY = capi.ROW_INVALID_CONFIG, capi.ROW_EMPTY
    status = [0, BAD, BAD, 0, EMPTY, INV, INV, INV, 0]
    fine = torch.tensor([True, False, False, True, False, False, False, False, True], device=dev)
    got = losses.token_logprobs(x, tok, temperature=T, want_entropy=True)
    assert got["row_status"].tolist() == status
    for name in ("logprob", "entropy"):
        assert torch.equal(~got[name].isnan(), fine), name
        assert got[name][3] == 0
    g = normal(gen, B, dev)
    back = losses.token_logprobs_backward(x, tok, got, g, grad_entropy=g, temperature=T)
    assert not back[1:8].any() and bool(back[0].any()) and bool(back[8].any() or V == 1)
    for w in (None, torch.ones(B, device=dev)):
        p = losses.policy_loss(x, tok, g, g, weight=w, ref_logprob=g, kl_coef=0.1, entropy_coef=0.1, temperature=T)
        assert p["row_status"].tolist() == status and bool(p["loss"].isnan())
        for name in ("row_loss", "logprob", "entropy", "kl"):
            assert torch.equal(~p[name].isnan(), fine), name
            assert p[name][3] == 0
        assert not p["grad_logits"][1:8].any() and bool(p["grad_logits"][0].any()) and not p["clipped"][1:8].any()
    # with no weight on them they are nobody's business
    w = fine.float()
    p = losses.policy_loss(x, tok, g, g, weight=w, ref_logprob=g, kl_coef=0.1, temperature=T)
    assert not p["row_status"].any() and not p["row_loss"][1:8].any() and not p["grad_logits"][1:8].any() and bool(p["loss"].isfinite())
    # pairs: the one with such a row has no loss and no gradient, the other is as if alone
    off = torch.tensor([0, 2, 3, 8, 9], dtype=torch.int32, device=dev)
    q = losses.preference_loss(x, tok, off, temperature=T)
    assert q["pair_status"].tolist() == [BAD, EMPTY | INV] and bool(q["loss"].isnan()) and not q["grad_logits"].any()
    tok[1], tok[2] = 0, 0
    q = losses.preference_loss(x, tok, off, temperature=T)
    assert q["pair_status"].tolist() == [0, EMPTY | INV] and bool(q["pair_loss"][0].isfinite()) and bool(q["grad_logits"][:3].any(1).all())
    q = losses.preference_loss(x, tok, off, temperature=T, pair_weight=torch.tensor([1.0, 0.0], device=dev))
    assert bool(q["loss"].isfinite()) and not q["grad_logits"][3:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [16, 1200, 33000])
def test_masks_inside_rows(dev, lib, V, dtype):
    """Logits of -inf and of the type's lowest value have no probability and no gradient, wherever they are; a row of nothing but
    lowest values is uniform; one where a single token is left is sure of it."""
    low = torch.finfo(dtype).min
    x, tok, gen = make(8, V, dtype, dev, seed=29)
    dead = torch.rand((8, V), generator=gen, device=dev) < 0.5
    dead[:, 3] = False
    tok[:] = 3
    x[0][dead[0]] = -math.inf
    x[1][dead[1]] = low
    x[2][V // 2:] = -math.inf
    x[3] = low
    x[4] = -math.inf
    x[4, 3] = 1.5
    x[5] = low
    x[5, 3] = -2.0
    x[6] = torch.finfo(dtype).max
    x[7][4:] = -math.inf
    g, h = normal(gen, 8, dev), normal(gen, 8, dev)
    got = losses.token_logprobs(x, tok, want_entropy=True)
    assert not got["row_status"].any()
    ref = Rows(x.double().clamp(min=-1e5, max=1e5).to(torch.float64) if dtype != torch.float16 else x, tok)   # (the same distributions, without overflows in the reference)
    ref.dtype = dtype
    ref.rel_p = torch.where(ref.p > 0, ref.rel_p, 0.0)
    close(got["logprob"], ref.l, ref.err_l)
    close(got["entropy"], ref.H, ref.err_H + 1e-300)
    out = losses.token_logprobs_backward(x, tok, got, g, grad_entropy=h)
    want, off = ref.gradient(g, h)
    close(out, want, off + ref.p * (h.abs().double() * (ref.err_H + ref.H.abs() * U))[:, None])
    gone = ref.p == 0
    assert not out[gone].any() and bool(gone.any())
    p = losses.policy_loss(x, tok, got["logprob"], g, entropy_coef=0.1)
    assert not p["grad_logits"][gone].any() and bool(p["loss"].isfinite())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,h,grad_scale", [(1e-3, 0.01, 65536.0), (0.02, 0.01, 2.0**24), (5e-5, 1.0, 1.0), (1e-19, 1.0, 1.0), (1e-25, 0.5, 64.0),
                                            (1e-36, 0.1, 1.0), (1.0, 0.0, 1.0), (1e36, 1.0, 1.0)])
def test_masked_logits_at_any_temperature_and_scale(dev, lib, T, h, grad_scale, dtype):
    """A masked logit has no gradient whatever the factor that its probability of 0 meets, and leaves the others theirs. The logits are some
    temperatures apart, so that the rows' distributions are no matter of T."""
    B, V = 4, 1500
    low = torch.finfo(dtype).min
    x, tok, gen = make(B, V, dtype, dev, seed=43)
    if dtype is torch.float16:
        T = min(T, 1000.0)
    x.copy_(2.0 * T * torch.randn((B, V), generator=gen, device=dev, dtype=torch.float64))   # (what fp16 has of them: zeros, at the lowest temperatures)
    dead = torch.rand((B, V), generator=gen, device=dev) < 0.5
    dead[2], dead[3] = True, False
    dead[:, 3] = False
    tok[:] = 3
    x[0][dead[0]] = -math.inf
    x[1][dead[1]] = low
    x[2][dead[2]] = -math.inf
    temperature = torch.full((B,), T, device=dev)
    ref = Rows(x, tok, temperature)
    ref.rel_p = torch.where(ref.p > 0, ref.rel_p, 0.0)
    got = losses.token_logprobs(x, tok, temperature=temperature, want_entropy=True)
    close(got["logprob"], ref.l, ref.err_l, "logprob")
    close(got["entropy"], ref.H, ref.err_H + 1e-300, "entropy")
    g, hs = normal(gen, B, dev) * grad_scale, torch.full((B,), h * grad_scale, device=dev)
    want, off = ref.gradient(g, hs)
    off = off + ref.p * (hs.double() * (ref.err_H + ref.H.abs() * U) / ref.T)[:, None]
    back = losses.token_logprobs_backward(x, tok, got, g, grad_entropy=hs, temperature=temperature)
    adv = g / grad_scale
    p = losses.policy_loss(x, tok, got["logprob"], adv, entropy_coef=h, temperature=temperature, grad_scale=grad_scale)["grad_logits"]
    want_p, off_p = ref.gradient(-adv * grad_scale, -hs, adv.abs().double() * grad_scale * (ref.err_l + ref.err_l64) * 1.01)
    for out, w, o in ((back, want, off), (p, want_p, off_p)):
        assert not out[dead].any()
        live = w.abs() < 0.9 * torch.finfo(dtype).max   # (fp16 ends at 65504)
        close(out[live], w[live], o[live], "gradient")


def test_masked_logits_where_the_gradient_itself_leaves_32_bits(dev, lib):
    """50 over a temperature of 1e-38: whatever the row's own logits get, those without a probability get 0."""
    x, tok, gen = make(3, 3000, torch.float32, dev, seed=47)
    x *= 1e-38
    dead = torch.rand(x.shape, generator=gen, device=dev) < 0.5
    dead[:, 7] = False
    dead[2] = True
    dead[2, 7] = False
    tok[:] = 7
    x[dead] = -math.inf
    T, g = torch.full((3,), 1.5e-38, device=dev), torch.full((3,), 50.0, device=dev)
    got = losses.token_logprobs(x, tok, temperature=T, want_entropy=True)
    for out in (losses.token_logprobs_backward(x, tok, got, g, temperature=T), losses.token_logprobs_backward(x, tok, got, g, g, temperature=T),
                losses.policy_loss(x, tok, got["logprob"], g, temperature=T)["grad_logits"],
                losses.policy_loss(x, tok, got["logprob"], g, entropy_coef=50.0, temperature=T)["grad_logits"]):
        assert not out[dead].any() and not out.isnan().any()
        assert not out[2].any()   # a row sure of its token


def test_nan_and_infinity_stay_in_their_row(dev, lib):
    for dtype in TYPES:
        x, tok, gen = make(5, 3001, dtype, dev)
        clean = losses.policy_loss(x, tok, torch.zeros(5, device=dev), normal(gen, 5, dev))
        g = torch.ones(5, device=dev)
        x[1, 1700], x[3, 5] = math.nan, math.inf
        got = losses.token_logprobs(x, tok, want_entropy=True)
        assert got["logprob"].isnan().tolist() == [False, True, False, True, False]
        back = losses.token_logprobs_backward(x, tok, got, g)
        assert back.isnan().all(1).tolist() == [False, True, False, True, False] and not back[[0, 2, 4]].isnan().any()
        p = losses.policy_loss(x, tok, g, g)
        assert p["grad_logits"].isnan().all(1).tolist() == [False, True, False, True, False] and bool(p["loss"].isnan())
        # where nothing counts on them they are not looked at
        w = torch.tensor([1.0, 0.0, 1.0, 0.0, 1.0], device=dev)
        p = losses.policy_loss(x, tok, g, g, weight=w)
        assert bool(p["loss"].isfinite()) and not p["grad_logits"][[1, 3]].any()
        assert not losses.token_logprobs_backward(x, tok, got, w)[[1, 3]].any()
        tok[1] = tok[3] = -1
        p = losses.policy_loss(x, tok, g, g)
        assert bool(p["loss"].isfinite()) and not p["grad_logits"][[1, 3]].any()
        assert clean["loss"].isfinite()


# ---- differences ----------------------------------------------------------------------------------------------

def test_gradients_against_differences(dev, lib):
    """(L(x + s v) - L(x - s v)) / 2 s against the gradient's product with v. L is of the order of 1 and rounded to 32 bits: the
    quotient is off by 2^-24 |L| / s at most, and by s^2 / 6 of the third derivative along v, which for a unit direction is below 10 |L| here."""
    B, V, s = 6, 41, 2.0**-6
    x, tok, gen = make(B, V, torch.float32, dev, spread=1.0)
    x = x.contiguous()
    old = Rows(x, tok).l.float() - 0.05
    ref, adv = (old - 0.2), torch.tensor([1.0, -0.5, 2.0, 0.3, -1.0, 0.7], device=dev)
    off = torch.tensor([0, 2, 3, 5, 6], dtype=torch.int32, device=dev)
    calls = {
        "policy": lambda y: losses.policy_loss(y, tok, old, adv, ref_logprob=ref, kl_coef=0.3, entropy_coef=0.2, scale=0.25, clip_low=0.9, clip_high=5.0),
        "preference": lambda y: losses.preference_loss(y, tok, off, ref_logprob=ref, beta=0.7, label_smoothing=0.2),
    }
    for name, f in calls.items():
        at = f(x)
        for _ in range(8):
            v = torch.randn((B, V), generator=gen, device=dev)
            v /= v.norm()
            d = (float(f(x + s * v)["loss"]) - float(f(x - s * v)["loss"])) / (2 * s)
            L = abs(float(at["loss"])) + 1
            assert abs(d - float((at["grad_logits"].double() * v.double()).sum())) < L * (2 * U / s + 10 * s * s / 6), name


def test_autograd_agrees_on_a_head(dev, lib):
    """The gradient handed to a graph that made the logits, against torch's own graph in 64 bits."""
    gen = torch.Generator(device=dev)
    gen.manual_seed(4)
    hidden = torch.randn((30, 16), generator=gen, device=dev)
    head = (torch.randn((1001, 16), generator=gen, device=dev) * 0.3).requires_grad_()
    tok = torch.randint(0, 1001, (30,), generator=gen, device=dev, dtype=torch.int32)
    off = torch.tensor([0, 10, 20, 30, 30], dtype=torch.int32, device=dev)
    logits = hidden @ head.T
    got = losses.preference_loss(logits.detach(), tok, off, beta=0.2)
    logits.backward(got["grad_logits"])
    w = head.detach().double().requires_grad_()
    lp = torch.log_softmax((hidden.double() @ w.T), 1)[torch.arange(30), tok.long()]
    m = 0.2 * torch.stack([lp[:10].sum() - lp[10:20].sum(), lp[20:].sum()])
    loss = -torch.nn.functional.logsigmoid(m).sum()
    loss.backward()
    # logits and gradient in 32 bits (and the products of either): 1001 terms of up to |hidden| = 5, rounded at 2^-24 each
    assert abs(float(got["loss"]) - loss.item()) < 1e-5 * (1 + abs(loss.item()))
    assert float((head.grad.double() - w.grad).norm() / w.grad.norm()) < 1e-4


def test_a_gradient_in_the_place_of_logits_that_a_graph_keeps(dev, lib):
    """A linear head does not need its logits again: the same gradient. A tanh does: its graph refuses instead of using what is there now."""
    gen = torch.Generator(device=dev)
    gen.manual_seed(73)
    hidden, tok = torch.randn((12, 16), generator=gen, device=dev), torch.randint(0, 1000, (12,), generator=gen, device=dev, dtype=torch.int32)
    head = (torch.randn((1000, 16), generator=gen, device=dev) * 0.3).requires_grad_()
    old, adv, off = normal(gen, 12, dev) - 7, normal(gen, 12, dev), torch.tensor([0, 5, 12], dtype=torch.int32, device=dev)
    calls = [lambda x, **k: losses.policy_loss(x, tok, old, adv, **k)["grad_logits"], lambda x, **k: losses.preference_loss(x, tok, off, **k)["grad_logits"],
             lambda x, **k: losses.token_logprobs_backward(x, tok, losses.token_logprobs(x, tok), adv, **k)]
    for call in calls:
        grads = []
        for place in (False, True):
            head.grad = None
            logits = hidden @ head.T
            logits.backward(call(logits.detach(), **(dict(out=logits.detach()) if place else {})))
            grads.append(head.grad.clone())
        assert torch.equal(*grads)
        capped = 30 * torch.tanh(hidden @ head.T / 30)
        inner = torch.tanh(hidden @ head.T)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            inner.backward(call(inner.detach(), out=inner.detach()))
        capped.backward(call(capped.detach(), out=capped.detach()))   # (tanh kept its own result, not the scaled one)
        with torch.inference_mode():
            x = torch.zeros((12, 1000), device=dev)
            call(x, out=x)


# ---- how it is called ------------------------------------------------------------------------------------------

def everything(x, tok, off, old, ref, adv):
    a = losses.token_logprobs(x, tok, want_entropy=True)
    b = losses.token_logprobs_backward(x, tok, a, adv, grad_entropy=old)
    c = losses.policy_loss(x, tok, old, adv, ref_logprob=ref, kl_coef=0.1, entropy_coef=0.01)
    d = losses.preference_loss(x, tok, off, ref_logprob=ref)
    return [a["logprob"], a["entropy"], a["stats"], b] + [t for o in (c, d) for t in o.values() if t is not None]


@pytest.mark.parametrize("V", [3000, 70000])
def test_graphs_streams_and_repeats_give_the_same_bits(dev, lib, V):
    B = 40
    off = torch.tensor([0, 10, 20, 31, 40], dtype=torch.int32, device=dev)
    sets = []
    for seed in (1, 2):
        x, tok, gen = make(B, V, torch.bfloat16, dev, seed=seed)
        sets.append((x, tok, off, *rollout(x, tok, gen, dev)))
    want = [[t.clone() for t in everything(*s)] for s in sets]
    for s, w in zip(sets, want):   # again
        assert all(torch.equal(a, b) for a, b in zip(everything(*s), w))
    # captured, and replayed with other inputs in the same places; two graphs in turn
    place = [t.clone() for t in sets[0]]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(everything(*place))
        graphs.append(g)
    for i in (1, 0, 1):
        for p, t in zip(place, sets[i]):
            p.copy_(t)
        for g, o in zip(graphs, outs):
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want[i]))
    # two streams at once
    streams = [torch.cuda.Stream(dev) for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(everything(*s))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(o, want[i % 2]))


@pytest.mark.parametrize("dtype", TYPES)
def test_the_widest_rows(dev, lib, dtype):
    """720896 logits: rows that no cluster of thread blocks holds, at least in 32 bits."""
    V, B = 720896, 3
    x, tok, gen = make(B, V, dtype, dev, seed=31)
    old, ref, adv = rollout(x, tok, gen, dev)
    want = policy_reference(x, tok, old, adv, ref=ref, kl=0.1, ent=0.01)
    y = x.clone()
    check_policy(losses.policy_loss(y, tok, old, adv, ref_logprob=ref, kl_coef=0.1, entropy_coef=0.01, out=y), want)
    assert not torch.equal(x, y)
    with pytest.raises(capi.MollaSampleError, match="too wide"):
        losses.token_logprobs(torch.zeros((1, V + 1), dtype=dtype, device=dev), tok[:1])


@pytest.mark.parametrize("B", [1, 2, 9, 24, 70, 150])
def test_the_widest_rows_for_any_number_of_rows(dev, lib, B):
    """Every layout that the number of rows chooses, at the width where least shared memory is left."""
    V = 720896
    x, tok, gen = make(1, V, torch.float32, dev, seed=37)
    x, tok = x.expand(B, V).contiguous(), tok.expand(B).contiguous()
    ref = Rows(x[:1], tok[:1])
    got = losses.token_logprobs(x, tok, want_entropy=True)
    close(got["logprob"], ref.l.expand(B), ref.err_l.expand(B))
    close(got["entropy"], ref.H.expand(B), ref.err_H.expand(B))
    adv = torch.ones(B, device=dev)
    want, off = ref.gradient(-adv[:1], err_g=2 * ref.err_l)
    back = losses.token_logprobs_backward(x, tok, got, -adv)
    p = losses.policy_loss(x, tok, got["logprob"], adv, out=x)
    for r in range(B):
        close(back[r:r + 1], want, off)
        close(p["grad_logits"][r:r + 1], want, off)


def test_rows_further_apart_than_32_bits_count(dev, lib):
    """A row that begins 2^31 + 2^20 elements into its block, for the logits and for the gradient."""
    V, step = 40000, 2**30 + 2**19
    buf = torch.empty(2 * step + V, dtype=torch.bfloat16, device=dev)
    out = torch.empty(2 * step + V, dtype=torch.bfloat16, device=dev)
    x, y = (b.as_strided((3, V), (step, 1)) for b in (buf, out))
    src, tok, gen = make(3, V, torch.bfloat16, dev)
    x.copy_(src)
    old, _, adv = rollout(src, tok, gen, dev)
    got = losses.policy_loss(x, tok, old, adv, out=y)
    check_policy(got, policy_reference(src, tok, old, adv))
    off = torch.tensor([0, 1, 3], dtype=torch.int32, device=dev)
    check_preference(losses.preference_loss(x, tok, off, out=y), preference_reference(src, tok, off))


def test_many_rows_and_none(dev, lib):
    x, tok, gen = make(20011, 40, torch.bfloat16, dev)
    old, ref, adv = rollout(x, tok, gen, dev)
    check_policy(losses.policy_loss(x, tok, old, adv, ref_logprob=ref, kl_coef=0.1, scale=1 / 20011),
                 policy_reference(x, tok, old, adv, ref=ref, kl=0.1, scale=1 / 20011))
    e = x[:0]
    no = losses.policy_loss(e, tok[:0], old[:0], adv[:0])
    assert no["loss"] == 0 and no["grad_logits"].shape == (0, 40)
    assert losses.token_logprobs(e, tok[:0])["logprob"].shape == (0,)
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    assert losses.preference_loss(e, tok[:0], zero)["loss"] == 0
    with pytest.raises(ValueError, match="need rows"):
        losses.preference_loss(e, tok[:0], torch.zeros(3, dtype=torch.int32, device=dev))
    got = losses.preference_loss(x, tok, zero)
    assert got["loss"] == 0 and not got["grad_logits"].any() and bool(got["logprob"].isfinite().all())
    # sequences of nothing: a margin of nothing
    got = losses.preference_loss(x, tok, torch.full((5,), 7, dtype=torch.int32, device=dev))
    assert not got["margin"].any() and not got["grad_logits"].any()
    assert bool(((got["pair_loss"] - math.log(2)).abs() < 2 * U).all())


def test_refusals_of_tensors(dev, lib):
    x, tok, gen = make(4, 64, torch.float32, dev)
    f = torch.zeros(4, device=dev)
    for bad in (x.double(), x[0], x.T, x.cpu(), x[:, ::2], x[:1].expand(4, 64)):
        with pytest.raises(ValueError, match="logit"):
            losses.token_logprobs(bad, tok)
    for bad in (tok.long(), tok[:3], tok.cpu(), torch.zeros(8, dtype=torch.int32, device=dev)[::2]):
        with pytest.raises(ValueError, match="tokens"):
            losses.policy_loss(x, bad, f, f)
    for name in ("weight", "ref_logprob", "temperature"):
        with pytest.raises(ValueError, match=name):
            losses.policy_loss(x, tok, f, f, **{name: f.double()})
    with pytest.raises(ValueError, match="shape, type and device"):
        losses.policy_loss(x, tok, f, f, out=x.bfloat16())
    with pytest.raises(capi.MollaSampleError, match="overlaps"):
        b = torch.zeros(5 * 64, device=dev)
        losses.policy_loss(b[:256].view(4, 64), tok, f, f, out=b[64:].view(4, 64))
    with pytest.raises(capi.MollaSampleError, match="KL term needs"):
        losses.policy_loss(x, tok, f, f, kl_coef=0.1)
    with pytest.raises(capi.MollaSampleError, match="clip range"):
        losses.policy_loss(x, tok, f, f, clip_low=-1.0)
    with pytest.raises(ValueError, match="want_entropy"):
        losses.token_logprobs_backward(x, tok, losses.token_logprobs(x, tok), f, grad_entropy=f)
    with pytest.raises(ValueError, match="stats"):
        losses.token_logprobs_backward(x, tok, losses.token_logprobs(x[:2], tok[:2]), f)
    for bad in (torch.zeros(4, dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)):
        with pytest.raises(ValueError, match="seq_off"):
            losses.preference_loss(x, tok, bad)
    # interleaved rows of one buffer are clear of each other
    b = torch.zeros((4, 128), device=dev)
    b[:, :64] = x
    got = losses.policy_loss(b[:, :64], tok, f, f + 1, out=b[:, 64:])
    assert torch.equal(b[:, :64], x) and torch.equal(got["grad_logits"], losses.policy_loss(x, tok, f, f + 1)["grad_logits"])


# ---- together ------------------------------------------------------------------------------------------------------

def test_a_rollout_from_sampling_to_both_losses(dev, lib):
    """Tokens from the sampler, their logprobs at the temperatures they were drawn at, the reference model's, and the losses."""
    from molla_b200 import sampler as S, workloads as W
    B, V = 24, 8000
    w = W.config3(seed=5, B=B, V=V, H=16)
    w["temperature"][:] = w["temperature"].clip(0.3, None)
    logits = torch.from_numpy(w["logits"]).to(dev)
    p = S.upload_params(w, dev)
    out = S.sample_batch(logits, p, want_logprob=True)
    tok, T = out["tokens"], p["temperature"]
    assert int(tok.min()) >= 0
    # the sampler's own logprobs are of the raw logits
    raw = losses.token_logprobs(logits, tok)
    R = Rows(logits, tok)
    close(out["chosen_logprob"], raw["logprob"].double(), R.err_l + 1e-5)
    old = losses.token_logprobs(logits, tok, temperature=T)["logprob"]
    later = (logits + 0.05 * torch.sin(torch.arange(V, device=dev))).bfloat16()   # the policy some steps on
    ref = losses.token_logprobs(logits.bfloat16(), tok, temperature=T)["logprob"]
    adv = torch.linspace(-1, 1, B, device=dev)
    got = losses.policy_loss(later, tok, old, adv, ref_logprob=ref, kl_coef=0.05, temperature=T, scale=1 / B)
    want = policy_reference(later, tok, old, adv, ref=ref, kl=0.05, T=T, scale=1 / B)
    near = (torch.exp(want["R"].l - old.double()) - 1).abs()
    assert not bool(((near - 0.2).abs() < 1e-4).any())
    check_policy(got, want)
    off = torch.arange(0, B + 1, 4, dtype=torch.int32, device=dev)
    off = off[: len(off) - (len(off) + 1) % 2]
    check_preference(losses.preference_loss(later, tok, off, ref_logprob=ref, temperature=T),
                     preference_reference(later, tok, off, ref=ref, T=T))


# ---- a load that never comes, as the testing build pretends ----------------------------------------------------------

@pytest.mark.parametrize("V", [3000, 151936])
def test_a_wait_that_runs_out_is_the_rows_status(dev, lib, V):
    x, tok, gen = make(6, V, torch.bfloat16, dev)
    old, ref, adv = rollout(x, tok, gen, dev)
    off = torch.tensor([0, 3, 6], dtype=torch.int32, device=dev)
    tok[2] = -1
    with capi.testing_library() as T:
        T.molla_sample_debug_knobs(16)
        try:
            a = losses.token_logprobs(x, tok, want_entropy=True)
            b = losses.policy_loss(x, tok, old, adv)
            c = losses.preference_loss(x, tok, off)
        finally:
            T.molla_sample_debug_knobs(0)
        torch.cuda.synchronize()
        late = [0 if r == 2 else capi.ROW_LOAD_TIMEOUT for r in range(6)]
        for got in (a, b, c):
            assert got["row_status"].tolist() == late
            assert got["logprob"].isnan().tolist() == [r != 2 for r in range(6)]
        assert bool(b["loss"].isnan()) and not b["grad_logits"].any()
        assert c["pair_status"].tolist() == [capi.ROW_LOAD_TIMEOUT] and not c["grad_logits"].any()
        assert not losses.token_logprobs_backward(x, tok, a, adv).any()
        again = losses.token_logprobs(x, tok)
    assert not again["row_status"].any() and bool(again["logprob"].isfinite().all())


def with_knob(knob, call):
    """The call's results in the testing build, with and without one of its switches."""
    with capi.testing_library() as T:
        clean = call()
        T.molla_sample_debug_knobs(knob)
        try:
            late = call()
            torch.cuda.synchronize()
        finally:
            T.molla_sample_debug_knobs(0)
        again = call()
    for a, b in zip(clean.values(), again.values()):
        assert a is None or torch.equal(a, b)
    return clean, late


def check_given_up(clean, late, row, alone):
    """Rows that were given up say so, have no numbers and a gradient of zeros; the others are what they are otherwise."""
    gone = late["row_status"] != 0
    assert bool(gone[row]) and (int(gone.sum()) == 1 or not alone) and not bool(gone[:row].any())
    assert bool((late["row_status"][gone] == capi.ROW_LOAD_TIMEOUT).all()) and not bool(gone.all())
    for name in ("logprob", "entropy", "row_loss", "kl"):
        if late.get(name) is not None:
            assert bool(late[name][gone].isnan().all()) and torch.equal(late[name][~gone], clean[name][~gone]), name
    if late.get("grad_logits") is not None:
        assert not late["grad_logits"][gone].any() and torch.equal(late["grad_logits"][~gone], clean["grad_logits"][~gone])
    if "loss" in late:
        assert bool(late["loss"].isnan()) and bool(clean["loss"].isfinite())


# rows that stay in one block, in a cluster, that are read twice; alone in their blocks and several of a block
LATE_SHAPES = [(6, 3000, torch.bfloat16), (6, 3001, torch.float32), (6, 40000, torch.float16), (6, 151936, torch.bfloat16), (3, 720896, torch.float32),
               (900, 120000, torch.bfloat16), (5000, 3000, torch.bfloat16)]


@pytest.mark.parametrize("B,V,dtype", LATE_SHAPES)
@pytest.mark.parametrize("knob", [256, 512], ids=["answer", "copy"])
def test_an_answer_or_a_copy_that_never_comes(dev, lib, B, V, dtype, knob):
    x, tok, gen = make(B, V, dtype, dev)
    old, adv = normal(gen, B, dev) - 9, normal(gen, B, dev)
    clean, late = with_knob(knob, lambda: losses.policy_loss(x, tok, old, adv, ref_logprob=old, kl_coef=0.01, entropy_coef=0.01))
    check_given_up(clean, late, B // 2, B < 10)
    place = lambda: (lambda y: losses.policy_loss(y, tok, old, adv, out=y))(x.clone())
    check_given_up(*with_knob(knob, place), B // 2, B < 10)
    if knob == 512:
        check_given_up(*with_knob(knob, lambda: losses.policy_loss(x, tok, old, adv, want_grad=False)), B // 2, B < 10)
        check_given_up(*with_knob(knob, lambda: losses.token_logprobs(x, tok, want_entropy=True)), B // 2, B < 10)


@pytest.mark.parametrize("B,V,dtype", [(3, 720896, torch.float32), (900, 120000, torch.bfloat16), (400, 120001, torch.float16), (300, 262144, torch.float32)])
def test_a_second_copy_that_never_comes(dev, lib, B, V, dtype):
    """Rows that are read again for their gradient: their logprobs are known by then, and are withdrawn. (Where the clip holds the row its
    gradient is zeros without another reading: it keeps its answer.)"""
    x, tok, gen = make(B, V, dtype, dev)
    old, adv = normal(gen, B, dev) - 9, normal(gen, B, dev)
    check_given_up(*with_knob(1024, lambda: losses.policy_loss(x, tok, old, adv, ref_logprob=old, kl_coef=0.01, entropy_coef=0.01)), B // 2, B < 10)
    clean, late = with_knob(1024, lambda: (lambda y: losses.policy_loss(y, tok, old, adv, out=y))(x.clone()))
    if clean["clipped"][B // 2]:
        assert late["row_status"][B // 2] == 0 and not late["grad_logits"][B // 2].any()
    else:
        check_given_up(clean, late, B // 2, B < 10)


@pytest.mark.parametrize("B,V,dtype", LATE_SHAPES)
def test_a_copy_that_never_comes_to_a_backward_pass(dev, lib, B, V, dtype):
    """No row's gradient is silently wrong: what could not be taken is NaN, and the preference loss says which rows they are."""
    x, tok, gen = make(B, V, dtype, dev)
    g = normal(gen, B, dev)
    scored = losses.token_logprobs(x, tok, want_entropy=True)
    backward = lambda: dict(grad=losses.token_logprobs_backward(x, tok, scored, g, grad_entropy=g))
    clean, late = with_knob(512, backward)
    gone = late["grad"].isnan().any(1)
    assert bool(gone[B // 2]) and not bool(gone.all()) and (int(gone.sum()) == 1 or B > 10)
    assert torch.equal(late["grad"][~gone], clean["grad"][~gone])
    off = torch.tensor([0, B // 3, B], dtype=torch.int32, device=dev)
    for ref in (None, scored["logprob"]):
        clean, late = with_knob(1024, lambda: losses.preference_loss(x, tok, off, ref_logprob=ref))
        if not clean["grad_logits"].any():   # so sure a pair that no row's gradient is read for
            assert ref is None and B > 10 and all(torch.equal(late[k], clean[k]) for k in clean)
            continue
        gone = late["grad_logits"].isnan().any(1)
        assert bool(gone[B // 2]) and not bool(gone.all())
        assert torch.equal(late["grad_logits"][~gone], clean["grad_logits"][~gone])
        assert torch.equal(late["row_status"], gone.int() * capi.ROW_LOAD_TIMEOUT) and torch.equal(late["logprob"].isnan(), gone)
        assert bool(late["loss"].isnan()) and torch.equal(late["pair_loss"], clean["pair_loss"])


@pytest.mark.parametrize("knob", [256, 512], ids=["answer", "copy"])
def test_clusters_of_several_rows_that_lose_one(dev, lib, knob):
    """Four blocks a row, four rows and more a cluster: the blocks that had all they needed withdraw the row as well."""
    B, V = 300, 262144
    x, tok, gen = make(B, V, torch.float32, dev)
    old, adv = normal(gen, B, dev) - 9, normal(gen, B, dev)
    call = lambda: losses.policy_loss(x, tok, old, adv, ref_logprob=old, kl_coef=0.01, entropy_coef=0.01)
    check_given_up(*with_knob(knob, call), B // 2, False)


def test_room_for_sums_that_never_comes(dev, lib):
    """Without a gradient a row's answer is wanted four rows later, when its place is to be used again: the row has its answer, rows
    of the same block from there on have none."""
    B, V = 20000, 3000
    x, tok, gen = make(B, V, torch.bfloat16, dev)
    clean, late = with_knob(256, lambda: losses.token_logprobs(x, tok, want_entropy=True))
    gone = late["row_status"] != 0
    assert bool(gone.any()) and not bool(gone[:B // 2 + 1].any()) and int(gone.sum()) < 40
    assert bool((late["row_status"][gone] == capi.ROW_LOAD_TIMEOUT).all())
    for name in ("logprob", "entropy"):
        assert bool(late[name][gone].isnan().all()) and torch.equal(late[name][~gone], clean[name][~gone])
    assert not losses.token_logprobs_backward(x, tok, late, torch.ones(B, device=dev))[gone].any()
