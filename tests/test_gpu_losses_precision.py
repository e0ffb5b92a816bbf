"""Rows whose values are easily lost in the operators on sampled tokens' logits:
barred targets among low logits, one likely column, confident tokens, vanishing
temperatures; and errors with a mean.  Against the 64-bit oracle, within bounds
counted from the kernels' roundings (u = 2^-24)."""
import math

import pytest
import torch

from b200_sampler import policy_loss_and_grad, preference_loss_and_grad, token_logprobs
from losses_bounds import U, close, entropy_bound, grad_bound, sum_bound
from oracle import losses_oracle as O

pytestmark = pytest.mark.gpu
INF = math.inf
HALVES = [torch.bfloat16, torch.float16]
TYPES = [torch.float32, *HALVES]
# rows of one block's first vectors, and rows that policy_kernel holds on chip
VOCABS = [1003, 32000]


def _joins(vocab):
    """Additions of a sum after its largest term has joined it, at most: 3 in the term's vector, its thread's further
    vectors (a block's 256 threads add up 2 x 2 elements a turn at the least), 4 that end the thread's part, 5 of a
    warp's lanes, 5 of a block's warps, 3 of a cluster."""
    return 3 + vocab / (256 * 4) + 4 + 13


def _normal(seed, *shape, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


# ------------------------------------------------- the offset is not the target's logit
def _barred(dtype, vocab, shift, mask):
    """Logits around `shift` whose targets are masked."""
    x = _normal(vocab, 8, vocab, scale=3.0) + shift
    targets = torch.randint(0, vocab, (8,), generator=torch.Generator().manual_seed(1))
    x[torch.arange(8), targets] = mask
    return x.to(dtype).cuda(), targets.cuda()


BARRED = [(t, -INF, s) for t in TYPES for s in (0.0, -20.0, -30.0, -40.0, -45.0, 40.0)] + \
         [(t, -1e4, s) for t in HALVES for s in (0.0, -20.0, -40.0, 40.0)]


@pytest.mark.parametrize("dtype,mask,shift", BARRED)
@pytest.mark.parametrize("vocab", VOCABS)
def test_barred_targets_among_shifted_logits(dtype, mask, shift, vocab):
    """A target without probability: the row's sums are taken around 0, and its entropy, gradient and loss are as
    exact as the distance of its logits from 0 allows."""
    x, targets = _barred(dtype, vocab, shift, mask)
    ln_p, lp, ent, alive, t = O.rows(x, targets)
    # the offset in place of the target's: as far from the largest logit as that lies from 0
    far = -x.float().nan_to_num(neginf=-INF).amax(1).abs().cpu().double()
    lp_off = sum_bound(ln_p, far) + U * (4 * lp.abs() + 4)
    a, h = _normal(2, 8).cuda(), _normal(3, 8).cuda()
    leaf = x.clone().requires_grad_()
    got_lp, got_ent = token_logprobs(leaf, targets, entropy=True)
    close(got_lp, lp, lp_off.nan_to_num(), "logprobs")
    close(got_ent, ent, entropy_bound(ln_p, far, ent), "entropy")
    (grad,) = torch.autograd.grad([got_lp, got_ent], [leaf], [a, h])
    want, zero = O.gradient(ln_p, ent, alive, t, targets, a, h), torch.zeros_like(ent)

    def off(grad, a, h, a_off=zero):
        return grad_bound(ln_p, far, t, ent, targets.cpu(), grad, a, a_off, h, dtype).nan_to_num()
    close(grad, want, off(want, a.cpu().double(), h.cpu().double()), "grad")

    # the ratio is 0: a row's loss is its clipped term less the entropy bonus
    old, adv = _normal(4, 8).cuda() - 8, _normal(5, 8).cuda()
    want = O.policy(x, targets, old, adv, entropy_coef=0.05)
    got, grad = policy_loss_and_grad(x, targets, old, adv, entropy_coef=0.05)
    row_off = 0.05 * entropy_bound(ln_p, far, ent) + 6 * U * want["row_loss"].abs()
    close(got.logprobs, lp, lp_off.nan_to_num(), "policy logprobs")
    close(got.entropy, ent, entropy_bound(ln_p, far, ent), "policy entropy")
    close(got.row_loss, want["row_loss"], row_off, "row_loss")
    close(got.loss, want["loss"], row_off.mean() + 2 * U * want["loss"].abs(), "loss")
    close(grad, want["grad"], off(want["grad"], want["a"], want["h"]), "policy grad")

    if math.isfinite(mask):
        offsets = torch.tensor([0, 2, 4, 5, 8])
        want = O.preference(x, targets, offsets, None, 0.01)
        got, grad = preference_loss_and_grad(x, targets, offsets.cuda(), beta=0.01)
        total = 0.01 * (lp_off + U * lp.abs()).sum() + 4 * U * want["rewards"].abs().max()
        close(got.rewards, want["rewards"], total, "rewards")
        close(got.loss, want["loss"], 2 * total + 4 * U * (1 + want["loss"].abs()), "preference loss")
        a_off = want["a"].abs() * 8 * U + 0.01 / 2 * 2 * total
        close(grad, want["grad"], off(want["grad"], want["a"], zero, a_off), "preference grad")


# --------------------------------------------------------------------- peaked rows
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 1003, 32000, 50257])
@pytest.mark.parametrize("rows", [1, 300])
def test_entropy_does_not_depend_on_the_target(dtype, vocab, rows):
    """One likely column and a target far below it: the entropy is a property of the row, not negative, and its error
    stays that of sums around the row's largest logit.  A target less than 8 bits away, or than 256 entropies, may
    serve as the sums' offset: U is then a sum around 8 bits or 256 H.  Through each way that rows are added up."""
    cases = [(q, d) for q in (1e-3, 1e-5, 1e-7) for d in (1.0, 2.5, 7.0, 16.0, 20.0, 40.0, 61.0, 80.0)]
    cases = cases if rows > 1 else cases[3::5]
    q, d = (torch.tensor(c)[:, None] for c in zip(*cases))
    x = _normal(vocab, len(cases), vocab, scale=0.5) + torch.log(q / vocab) + 10.0
    at = torch.randint(0, vocab, (len(cases),), generator=torch.Generator().manual_seed(2))
    here = torch.arange(len(cases))
    targets = (at + 1) % vocab
    x[here, at] = 10.0
    x[here, targets] = 10.0 - d[:, 0]
    turn = (torch.arange(rows) % len(cases)) if rows > 1 else None
    for part in ([turn] if rows > 1 else [torch.tensor([i]) for i in range(len(cases))]):
        z, tg = x[part].to(dtype).cuda(), targets[part].cuda()
        one = torch.arange(min(len(part), len(cases)))         # the rows repeat: the oracle sees each once
        ln_p, lp, ent, alive, t = O.rows(z[one], tg[one])
        # the offset's distance from the largest logit, in nats
        far = torch.minimum(lp.abs(), torch.maximum(torch.full_like(ent, 8 * math.log(2)), 256 * ent))
        zz = (ln_p - ln_p.max(1, keepdim=True).values).abs() + far[:, None]
        p = ln_p.exp()
        mean, square = (p * zz).sum(1), (p * zz * zz).sum(1)
        n = _joins(vocab)
        # S and U are off by a rounding an addition and by each term's: 4 u of the exponential, 3 u |z| of its argument
        bound = U * ((n + 8) * (1 + 2 * mean) + 3 * (mean + square) + 4 * (1 - p.max(1).values) + 4 * ent)
        bound = bound[turn % len(cases)] if rows > 1 else bound
        want = ent[turn % len(cases)] if rows > 1 else ent
        got = token_logprobs(z, tg, entropy=True)[1]
        close(got, want, bound, "entropy")
        assert (got >= 0).all()
        old, adv = torch.zeros(len(part), device="cuda"), torch.zeros(len(part), device="cuda")
        got, grad = policy_loss_and_grad(z, tg, old, adv, entropy_coef=1.0, weights=torch.ones(len(part), device="cuda"))
        close(got.entropy, want, bound, "policy entropy")
        assert (got.entropy >= 0).all()
        g = O.gradient(ln_p, ent, alive, t, tg[one], torch.zeros_like(ent), -torch.ones_like(ent))
        off = grad_bound(ln_p, -far, t, ent, tg[one].cpu(), g, torch.zeros_like(ent), torch.zeros_like(ent),
                         torch.ones_like(ent), dtype)
        off = off + p * bound[one][:, None]
        close(grad[one], g, off, "policy grad")


@pytest.mark.parametrize("rows,vocab,dtype", [
    (40, 32000, torch.bfloat16), (40, 64007, torch.float16), (500, 100003, torch.bfloat16), (420, 170000, torch.float16),
    (30, 400000, torch.bfloat16), (40, 32000, torch.float32), (30, 151936, torch.float32), (6, 600000, torch.float32)])
@pytest.mark.parametrize("entropy", [0.0, 0.01])
def test_rows_that_are_added_up_again(rows, vocab, dtype, entropy):
    """Targets 80 nats below their row's largest logit, and 16-bit logits at a temperature that puts them past 1024,
    among ordinary rows and rows without a token: on every way that policy_kernel holds a row, into a new gradient, one
    of another stride, and the logits' place."""
    alive = torch.randperm(rows, generator=torch.Generator().manual_seed(rows))[:min(rows, 9)].sort().values.cuda()
    n = len(alive)
    part = _normal(vocab, n, vocab, scale=2.0)
    targets = torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(3))
    temperature = torch.ones(n)
    for i in range(n):
        if i % 3 == 0:                  # all but impossible
            part[i, targets[i]] = -75.0
            part[i, (targets[i] + 7) % vocab] = 15.0
        elif i % 3 == 1:                # cold
            temperature[i] = 0.02
            part[i] += 30.0
            targets[i] = part[i].argmax()
    x = torch.full((rows, vocab), math.nan, dtype=dtype, device="cuda")
    x[alive] = part.to(dtype).cuda()
    every = torch.full((rows,), -1, device="cuda")
    every[alive] = targets.cuda()
    part = x[alive].clone()
    ln_p, lp, ent, _, t = O.rows(part, targets, temperature)
    old = torch.zeros(rows, device="cuda")
    # a ratio of 1.1 in an ordinary row, 1 in a cold one; one that no fp32 of either probability would hold is left out
    old[alive] = torch.where(lp > -60, lp - 0.1 * (torch.arange(n) % 3 == 2), torch.full_like(lp, -60.0)).float().cuda()
    adv, w = torch.full((rows,), -1.5, device="cuda"), torch.full((rows,), 0.25, device="cuda")
    temps = torch.ones(rows, device="cuda")
    temps[alive] = temperature.cuda()
    want = O.policy(part, targets, old[alive], adv[alive], None, w[alive], temperature, 0.2, 0.2, 0.0, entropy)

    def run(z, out):
        return policy_loss_and_grad(z, every, old, adv, weights=w, temperature=temps, entropy_coef=entropy, out=out)
    got, grad = run(x, None)
    assert (grad[every < 0] == 0).all()
    n_add = _joins(vocab) + 8
    close(got.logprobs[alive], lp, U * (n_add + 8 * lp.abs() + 3 * ent + 16), "logprobs")
    mean = (ln_p.exp() * (ln_p - ln_p.max(1, keepdim=True).values).nan_to_num(neginf=0.0).abs()).sum(1) + lp.abs().clamp(max=40)
    ent_off = U * (n_add * (1 + 2 * mean) + 8 * (mean + 1) ** 2)
    if entropy:
        close(got.entropy[alive], ent, ent_off, "entropy")
    # e^lp: relative errors of the sums and of the offset, which is at most 69 nats away
    rel = U * (n_add + 8 * lp.abs() + 3 * ent + 32)
    bound = grad_bound(ln_p, lp, t, ent, targets, want["grad"], want["a"], rel * want["a"].abs(), want["h"], dtype)
    bound = bound + ln_p.exp() * (want["h"].abs() * ent_off)[:, None] / t[:, None]
    close(grad[alive], want["grad"], bound, "grad")
    wide = torch.full((rows, vocab + 3), 5.0, dtype=dtype, device="cuda")
    moved = run(x, wide[:, 1:1 + vocab])[1]
    assert torch.equal(moved, grad) and (wide[:, 0] == 5).all() and (wide[:, 1 + vocab:] == 5).all()
    again, same = run(x, x)
    assert same.data_ptr() == x.data_ptr() and torch.equal(same, grad)
    for u, v in zip(got, again):
        assert v is None and u is None or torch.equal(u, v)


# ------------------------------------------------------------------- confident tokens
def _peaked(dtype, vocab, peaks, rest, seed=7):
    """Rows of one likely column: its logit is peaks[i], and the others share about rest[i] times its mass."""
    n = len(peaks)
    peak, rest = torch.tensor(peaks)[:, None], torch.tensor(rest)[:, None]
    x = peak + torch.log(rest / (vocab - 1)) + _normal(seed, n, vocab, scale=0.5)
    at = torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed))
    x[torch.arange(n), at] = peak[:, 0]
    return x.to(dtype).cuda(), at.cuda()


PEAKS = [20.0, 30.0, 38.5, 64.0, 90.0, 130.0, 300.0, 420.0, 640.0]
REST = [1e-3, 1e-4, 1e-5, 1e-6]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1.0, 0.7])
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_gradient_at_a_confident_token(dtype, temperature, vocab, sign):
    """a (1 - p) of a target with p near 1 keeps what S, a sum near 1, can tell of it: S is off by a rounding an
    addition and by the exponential's 2^-22 = 4 u, and the rest by its own relative error."""
    peaks = [p * s for p in PEAKS for s in (temperature, -1.0)]
    peaks, rest = [p for p in peaks for _ in REST], REST * len(peaks)
    x, targets = _peaked(dtype, vocab, peaks, rest)
    n = len(peaks)
    x = x if temperature == 1.0 else ((x.float() - torch.tensor(peaks).cuda()[:, None]) * temperature
                                      + torch.tensor(peaks).cuda()[:, None]).to(dtype)
    a = sign * (1 + torch.rand(n, generator=torch.Generator().manual_seed(1))).cuda()
    ln_p, lp, ent, alive, t = O.rows(x, targets, temperature)
    off = U * (_joins(vocab) + 4 + 2) - torch.expm1(lp) * U * 64
    info, here = torch.finfo(dtype), torch.arange(n)

    def check(grad, a, rel, what):                  # rel: the coefficient's relative error
        a = a.cpu().double()
        want = O.gradient(ln_p, ent, alive, t, targets, a)
        bound = grad_bound(ln_p, lp, t, ent, targets.cpu(), want, a, rel * a.abs(), torch.zeros_like(a), dtype)
        at = want[here, targets.cpu()]
        bound[here, targets.cpu()] = (a.abs() / t * off + at.abs() * (info.eps / 2 + rel + 4 * U)
                                      + info.smallest_normal * info.eps)
        close(grad, want, bound, what)
    leaf = x.clone().requires_grad_()
    (grad,) = torch.autograd.grad(token_logprobs(leaf, targets, temperature=temperature), [leaf], [a])
    check(grad, a, 0.0, "token_logprobs")
    # from the policy loss: without a drift the coefficient is -A w
    old, w = lp.float().cuda(), torch.ones(n, device="cuda")
    got, grad = policy_loss_and_grad(x, targets, old, -a, weights=w, temperature=temperature)
    want = O.policy(x, targets, old, -a, None, w, temperature)
    check(grad, want["a"], U * (_joins(vocab) + 16), "policy_loss_and_grad")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_entropy_gradient_at_the_peak(dtype, vocab):
    """-h p (ln p + H) at a likely column, where ln p + H cancels: as exact as H itself."""
    peaks, rest = [p * s for p in PEAKS for s in (1.0, -1.0)], [1e-3]
    x, targets = _peaked(dtype, vocab, peaks, rest * len(peaks))
    n = len(peaks)
    ln_p, lp, ent, alive, t = O.rows(x, targets)
    h, zero = torch.linspace(0.5, 2.0, n).cuda(), torch.zeros(n, dtype=torch.float64)
    leaf = x.clone().requires_grad_()
    _, got = token_logprobs(leaf, targets, entropy=True)
    (grad,) = torch.autograd.grad(got, [leaf], [h])
    hh = h.cpu().double()
    want = O.gradient(ln_p, ent, alive, t, targets, zero, hh)
    bound = grad_bound(ln_p, lp, t, ent, targets.cpu(), want, zero, zero, hh, dtype)
    # at the peak: ln p and H are off by S's error and by that of the small terms of U
    at, info = want[torch.arange(n), targets.cpu()], torch.finfo(dtype)
    off = U * (_joins(vocab) + 6) * 2 + ent * U * (_joins(vocab) + 64)
    bound[torch.arange(n), targets.cpu()] = hh * off + at.abs() * (info.eps / 2 + 4 * U) + info.smallest_normal * info.eps
    close(grad, want, bound, "grad")


# ------------------------------------------------------------------ low temperatures
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1e-30, 1e-37, 1e-39, 1e-44])
@pytest.mark.parametrize("vocab", VOCABS)
def test_gradients_at_vanishing_temperatures(dtype, temperature, vocab):
    """The distribution is the largest logit's alone; a / T may be past fp32, but a column without probability has
    no gradient, and neither has a certain target."""
    x = _normal(3, 4, vocab, scale=3.0).to(dtype).cuda()
    x[:, 5] = 40.0
    targets = torch.tensor([5, 5, 5, -1]).cuda()
    each = torch.full((4,), temperature, device="cuda")
    leaf = x.clone().requires_grad_()
    lp, ent = token_logprobs(leaf, targets, temperature=each, entropy=True)
    (grad,) = torch.autograd.grad([lp, ent], [leaf], [torch.ones_like(lp), torch.ones_like(ent)])
    assert (lp == 0).all() and (ent == 0).all() and (grad == 0).all()
    ones = torch.ones(4, device="cuda")
    for kw in (dict(), dict(entropy_coef=0.1)):
        got, grad = policy_loss_and_grad(x, targets, 0 * ones, ones, temperature=each, **kw)
        assert (got.logprobs == 0).all() and (grad == 0).all()
    # targets without probability: the gradient is a / T at them, or infinite
    targets = torch.tensor([7, 8, 9, -1]).cuda()
    (grad,) = torch.autograd.grad(token_logprobs(leaf, targets, temperature=each), [leaf], [ones * 1e-30])
    assert (grad[:3, 10:] == 0).all() and (grad[3] == 0).all() and (grad[torch.arange(3), targets[:3]] > 0).all()
    assert not torch.isnan(grad).any()


# ------------------------------------------------------------------ mean errors
@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 32000), (torch.bfloat16, 32000), (torch.bfloat16, 151936)])
def test_log_probabilities_have_no_mean_error(dtype, vocab):
    """Sequences add log-probabilities up, so an error with a mean grows with their length.  The results' own rounding
    has none: half of 2^-20 at most of values up to 16, 2.8e-7 as a standard deviation, 6e-9 for the mean of 2048 rows.
    The limit is three of those: below the exponentials' mean error, 3e-8 uncorrected, and that of sums which lose
    small terms, 8e-8."""
    rows, part = 2048, 128
    mean = 0.0
    for i in range(rows // part):
        g = torch.Generator("cuda").manual_seed(i)
        x = torch.randn(part, vocab, device="cuda", generator=g) * 2.5
        targets = (torch.empty_like(x).exponential_(generator=g).log_().neg_() + x).argmax(1)
        x = x.to(dtype)
        z = x.double()
        want = z.gather(1, targets[:, None])[:, 0] - torch.logsumexp(z, 1)
        mean += (token_logprobs(x, targets).double() - want).sum().item() / rows
    assert abs(mean) < 2e-8


# ------------------------------------------------------------------- the KL term
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 32000])
def test_kl_near_zero(dtype, vocab):
    """exp(d) - d - 1 of small d, at a column that has all of the probability (its logit 0: ln p is 0, and d is the
    reference's number).  Where the three are added up, from 1/2 on, a last place of e^d - 1 is at most 4.4 of their
    sum above 0 and 3.7 below, and d's rounding is none: 16 u in all.  Below, the series has 10 roundings."""
    d = torch.tensor([s * v for v in (1e-30, 1e-8, 1e-5, 1e-3, 0.03, 0.2, 0.4999, 0.5, 0.7, 1.5, 20.0) for s in (1, -1)])
    n = len(d)
    x = torch.full((n, vocab), -INF, dtype=dtype, device="cuda")
    targets = (torch.arange(n) * 31 % vocab).cuda()
    x[torch.arange(n), targets] = 0.0
    want = torch.expm1(d.double()) - d.double()
    series = sum(d.double() ** k / math.factorial(k) for k in range(2, 14))
    want = torch.where(d.abs() < 0.1, series, want)          # 64 bits cancel too
    zero = torch.zeros(n, device="cuda")
    got, _ = policy_loss_and_grad(x, targets, zero, zero, ref_logprobs=d.cuda(), kl_coef=1.0)
    assert (got.logprobs == 0).all() and (got.kl >= 0).all()
    close(got.kl, want, 16 * U * want + 2.0 ** -149, "kl")
    close(got.row_loss, want, 17 * U * want + 2.0 ** -149, "row_loss")


def test_more_rows_added_up_again_than_a_block_lists():
    """16500 cold rows on some 444 clusters, a few of them without a token: each cluster has over 32 to add up again,
    and finds them by their marks."""
    rows, vocab, t = 16500, 14400, 0.02
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda")
    for i in range(0, rows, 1500):
        x[i:i + 1500] = (torch.randn(1500, vocab, device="cuda", generator=g) + 30).bfloat16()
    targets = torch.where(torch.arange(rows, device="cuda") % 3 > 0, x.argmax(1), torch.arange(rows, device="cuda") % vocab)
    targets[5::97] = -1
    zero, adv = torch.zeros(rows, device="cuda"), torch.randn(rows, device="cuda", generator=g)
    lp = torch.empty(rows, dtype=torch.float64, device="cuda")
    for i in range(0, rows, 1500):
        z = x[i:i + 1500].double() / t
        lp[i:i + 1500] = z.gather(1, targets[i:i + 1500].clamp(min=0)[:, None])[:, 0] - torch.logsumexp(z, 1)
    old = torch.where(targets >= 0, lp, torch.zeros_like(lp)).clamp(min=-60).float()
    w = torch.full((rows,), 1.0, device="cuda")
    got, grad = policy_loss_and_grad(x, targets, old, adv, weights=w, temperature=t)
    alive = targets >= 0
    # S has a rounding an addition and the exponentials' 4 u; the value's own rounding and the scale's
    close(got.logprobs, torch.where(alive, lp, torch.zeros_like(lp)).cpu(), U * (_joins(vocab) + 12 + 6 * lp.abs().cpu()), "logprobs")
    pick = torch.cat([torch.arange(0, rows, 271), torch.arange(rows - 40, rows)]).cuda()
    want = O.policy(x[pick], targets[pick], old[pick], adv[pick], None, w[pick], t)
    rel = U * (_joins(vocab) + 32 + 8 * want["logprobs"].abs())
    none = torch.zeros(len(pick), dtype=torch.float64)
    bound = grad_bound(want["ln_p"], want["logprobs"], want["t"], want["entropy"], targets[pick].cpu(), want["grad"], want["a"],
                       rel * want["a"].abs(), none, x.dtype)
    close(grad[pick], want["grad"], bound, "grad")
    assert (grad[~alive] == 0).all() and torch.isfinite(got.loss)
    for i in range(0, rows, 1500):      # no row is left as its memory was: a row's gradient sums to nothing beside its parts
        part = grad[i:i + 1500].double()
        assert (part.sum(1).abs() <= part.abs().sum(1) * 2.0 ** -7 + 1e-4).all()
