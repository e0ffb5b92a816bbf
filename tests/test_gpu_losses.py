"""Token log-probabilities, policy loss and preference loss on the GPU against
the 64-bit oracle, within bounds counted from the kernels' roundings."""
import math

import pytest
import torch

from b200_sampler import (policy_loss, policy_loss_and_grad, preference_loss, preference_loss_and_grad,
                          token_logprobs)
from losses_bounds import U, close, entropy_bound, grad_bound, logprob_bound
from oracle import losses_oracle as O

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan
TYPES = [torch.float32, torch.bfloat16, torch.float16]
VOCABS = [1, 2, 7, 8, 9, 31, 33, 257, 1000, 4097, 32000, 50257, 151936]


def _logits(seed, rows, vocab, dtype, layout="plain"):
    """Logits in one of the layouts a caller has: plain rows, rows inside wider
    ones (odd stride, odd start), or the last position of [rows, 3, vocab]."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).cuda()
    if layout == "plain":
        return x
    if layout == "wide":
        wide = torch.full((rows, vocab + 5), 7.0, dtype=dtype, device="cuda")
        wide[:, 3:3 + vocab] = x
        return wide[:, 3:3 + vocab]
    if layout == "last":
        full = torch.full((rows, 3, vocab), 7.0, dtype=dtype, device="cuda")
        full[:, -1] = x
        return full[:, -1]
    if layout == "column":          # columns apart from one another
        return x.t().contiguous().t()
    raise ValueError(layout)


def _targets(seed, rows, vocab, padded=0.0):
    g = torch.Generator().manual_seed(seed + 1)
    t = torch.randint(0, vocab, (rows,), generator=g)
    t[torch.rand(rows, generator=g) < padded] = -1
    return t.cuda()


def _vector(seed, rows, scale=1.0):
    return (torch.randn(rows, generator=torch.Generator().manual_seed(seed + 2)) * scale).cuda()


def _temperature(kind, rows):
    if kind == "rows":
        t = torch.linspace(0.3, 1.7, rows)
        t[rows // 2] = 0.0                           # a greedy row
        return t.cuda()
    return kind


def _check_logprobs(x, targets, temperature, entropy=True, grads=True, seed=0, extra=0.0):
    ln_p, lp, ent, alive, t = O.rows(x, targets, temperature)
    leaf = x.detach().requires_grad_()
    got = token_logprobs(leaf, targets, temperature=temperature, entropy=entropy)
    got_lp, got_ent = got if entropy else (got, None)
    assert got_lp.dtype == torch.float32
    close(got_lp, lp, logprob_bound(ln_p, lp), "logprobs")
    if entropy:
        close(got_ent, ent, entropy_bound(ln_p, lp, ent), "entropy")
    # the call without a graph gives the same bits
    with torch.no_grad():
        again = token_logprobs(x, targets, temperature=temperature, entropy=entropy)
    assert torch.equal((again[0] if entropy else again).nan_to_num(), got_lp.nan_to_num())
    if not grads:
        return
    a, h = _vector(seed, x.shape[0]), _vector(seed + 9, x.shape[0], 0.3)
    ends, seeds = ([got_lp, got_ent], [a, h]) if entropy else ([got_lp], [a])
    grad = torch.autograd.grad(ends, [leaf], seeds)[0]
    hh = h if entropy else torch.zeros_like(h)
    want = O.gradient(ln_p, ent, alive, t, targets, a, hh)
    aa = torch.where(alive, a.cpu().double(), torch.zeros_like(lp))
    bound = grad_bound(ln_p, lp, t, ent, targets.cpu(), want, aa, torch.zeros_like(lp),
                       torch.where(alive, hh.cpu().double(), torch.zeros_like(lp)), x.dtype)
    size = aa.abs()[:, None] + hh.cpu().double().abs()[:, None] * (torch.nan_to_num(ln_p, neginf=0.0).abs() + ent[:, None])
    bound = bound + extra * torch.exp(ln_p) * size / t[:, None]
    assert grad.dtype == x.dtype and grad.shape == x.shape
    close(grad, want, torch.nan_to_num(bound), "grad")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("entropy", [False, True])
def test_logprobs_and_gradient(dtype, vocab, entropy):
    for rows in (1, 3, 37) if vocab < 50000 else (1, 5):
        x = _logits(rows + vocab, rows, vocab, dtype)
        _check_logprobs(x, _targets(vocab, rows, vocab, 0.2 if rows == 37 else 0.0), 1.0, entropy)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["wide", "last", "column"])
@pytest.mark.parametrize("vocab", [9, 1000, 4097, 32000])
def test_layouts(dtype, layout, vocab):
    x = _logits(5, 11, vocab, dtype, layout)
    _check_logprobs(x, _targets(5, 11, vocab), _temperature("rows", 11))


@pytest.mark.parametrize("rows", [1, 18, 19, 37, 74, 75, 149, 297, 700])
def test_row_counts_cross_the_blocks_per_row(rows):
    x = _logits(rows, rows, 20011, torch.bfloat16)
    _check_logprobs(x, _targets(rows, rows, 20011, 0.1), _temperature("rows", rows))


@pytest.mark.parametrize("rows,vocab,dtype", [
    (295, 8193, torch.bfloat16), (296, 8193, torch.bfloat16),       # a warp per row from 296 rows on 148 SMs
    (1544, 4121, torch.float32), (1545, 4121, torch.float32),       # from 1545 rows of 1030 vectors
    (1600, 8209, torch.float16)])
def test_row_counts_cross_a_warp_per_row(rows, vocab, dtype):
    x = _logits(rows, rows, vocab, dtype)
    _check_logprobs(x, _targets(rows, rows, vocab, 0.1), _temperature("rows", rows))


@pytest.mark.parametrize("temperature", [0.0, 0.05, 0.7, 1.0, 3.0, 1e30])
def test_temperatures(temperature):
    x = _logits(1, 7, 5003, torch.float32)
    _check_logprobs(x, _targets(1, 7, 5003), temperature)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [-900.0, -600.0, 600.0, 900.0, 40000.0])
@pytest.mark.parametrize("vocab", [1003, 32000])
def test_logits_far_from_zero(dtype, shift, vocab):
    """Distributions do not see a shift of all logits; the kernels' offsets do.
    16-bit values this far out are coarse, so the rows have few distinct ones."""
    if dtype == torch.float16 and shift > 30000:
        shift = 30000.0
    x = (_logits(9, 6, vocab, torch.float32) + shift).to(dtype)
    targets = x.float().topk(3, dim=1).indices[:, 1].contiguous()
    # 16-bit gradients: the offset c s + log2 S, below 1024 + 60 in size, is rounded to 2^-14
    _check_logprobs(x, targets, 1.0, extra=0.0 if dtype == torch.float32 else math.log(2) * 2.0 ** -13)
    _check_logprobs(x, targets, 2.0, entropy=False, extra=0.0 if dtype == torch.float32 else math.log(2) * 2.0 ** -13)


def _odd_rows(dtype, vocab):
    """Rows where a distribution has holes or does not exist."""
    x = _logits(3, 12, vocab, dtype)
    low = torch.finfo(dtype).min
    x[0] = -INF                        # nothing left
    x[1, 1:] = -INF                    # one column left
    x[2] = low                         # all at the type's lowest value: uniform
    x[3] = low
    x[3, 4] = 2.0                      # one column above a masked row
    x[4, vocab // 2:] = -INF
    x[5, ::2] = low
    x[6, vocab - 1] = INF
    x[7, 3] = NAN
    x[8] = NAN                         # a padded row holds anything
    x[9] = INF
    x[10] = torch.finfo(dtype).max     # all at the largest value
    t = torch.tensor([0, 0, 2, 4, vocab - 1, 1, 2, 3, -1, -7, 5, vocab])
    return x, t.cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 4097, 151936])
@pytest.mark.parametrize("temperature", [1.0, 0.5])
def test_masks_infinities_and_nan(dtype, vocab, temperature):
    x, targets = _odd_rows(dtype, vocab)
    _check_logprobs(x, targets, temperature)
    _check_logprobs(x, targets, temperature, entropy=False)
    lp = token_logprobs(x, targets, temperature=temperature)
    assert torch.isnan(lp[[0, 6, 7, 11]]).all() and (lp[[8, 9]] == 0).all()
    # where one column has all of the probability, S is its 2^t alone: off by the exponential's 2^-22 and by S's own
    # rounding, 2^-24; and the result is not above 0
    assert -5 * U <= lp[1] <= 0 and -5 * U <= lp[3] <= 0
    assert abs(lp[2].item() + math.log(vocab)) < 1e-5 and lp[4] == -INF


def test_temperatures_without_a_distribution_give_nan():
    x = _logits(3, 6, 300, torch.float32)
    t = torch.tensor([1.0, -1.0, NAN, INF, 0.0, 2.0], device="cuda")
    _check_logprobs(x, _targets(3, 6, 300), t)


def test_no_rows():
    x = torch.empty(0, 50, device="cuda", requires_grad=True)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    lp, ent = token_logprobs(x, none, entropy=True)
    assert lp.shape == (0,) and ent.shape == (0,)
    f = torch.empty(0, device="cuda")
    got, grad = policy_loss_and_grad(x.detach(), none, f, f)
    assert got.loss.item() == 0 and grad.shape == (0, 50)
    got, grad = preference_loss_and_grad(x.detach(), none, torch.zeros(3, dtype=torch.int64, device="cuda"))
    assert abs(got.loss.item() - math.log(2)) < 1e-6 and got.rewards.tolist() == [[0.0, 0.0]]
    got, grad = preference_loss_and_grad(x.detach(), none, torch.zeros(1, dtype=torch.int64, device="cuda"))
    assert got.loss.item() == 0 and got.pair_loss.shape == (0,)


def test_gradient_of_broadcast_rows():
    """One row's logits expanded over several tokens: the gradient is the rows' sum."""
    base = _logits(8, 1, 777, torch.float32).requires_grad_()
    targets, a = _targets(8, 6, 777), _vector(8, 6)
    (grad,) = torch.autograd.grad(token_logprobs(base.expand(6, 777), targets), [base], [a])
    ln_p, lp, ent, alive, t = O.rows(base.detach().expand(6, 777), targets)
    want = O.gradient(ln_p, ent, alive, t, targets, a)
    zero = torch.zeros_like(lp)
    bound = grad_bound(ln_p, lp, t, ent, targets.cpu(), want, a.cpu().double(), zero, zero, torch.float32)
    close(grad, want.sum(0, keepdim=True), bound.sum(0, keepdim=True) + 6 * U * want.abs().sum(0), "grad")


def test_gradient_against_differences():
    """Central differences of the 64-bit forward in random directions: the
    kernel's gradient is the derivative of what the kernel computes."""
    x = _logits(4, 5, 301, torch.float32)
    targets, a, h = _targets(4, 5, 301), _vector(4, 5), _vector(40, 5, 0.5)
    temperature = _temperature("rows", 5)
    leaf = x.clone().requires_grad_()
    lp, ent = token_logprobs(leaf, targets, temperature=temperature, entropy=True)
    (grad,) = torch.autograd.grad([lp, ent], [leaf], [a, h])

    def value(z):
        _, lp, ent, _, _ = O.rows(z, targets, temperature)
        return (a.cpu().double() * lp + h.cpu().double() * ent).sum().item()
    for seed in range(4):
        d = torch.randn(x.shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
        step = 1e-4
        base = x.cpu().double()
        slope = (value(base + step * d) - value(base - step * d)) / (2 * step)
        got = (grad.cpu().double() * d).sum().item()
        # third derivatives are below 10 |a| / T^3 per unit: step^2 / 6 of them; fp32 gradients: 2^-20 of each value
        scale = (grad.cpu().double() * d).abs().sum().item()
        assert abs(got - slope) < 1e-8 * 400 / 0.3 ** 3 + 2.0 ** -20 * scale


# ----------------------------------------------------------------- policy loss
def _policy_inputs(seed, x, targets, temperature):
    _, lp, _, _, _ = O.rows(x, targets, temperature)
    g = torch.Generator().manual_seed(seed + 5)
    n = x.shape[0]
    lp = torch.nan_to_num(lp, neginf=-30.0)
    drift = torch.randn(n, generator=g, dtype=torch.float64) * 0.25
    for edge in (math.log(0.8), math.log(1.28)):      # a ratio at the border may round to either side
        drift = torch.where((drift - edge).abs() < 1e-3, drift + 0.004, drift)
    old = (lp - drift).float().cuda()
    ref = (lp + torch.randn(n, generator=g, dtype=torch.float64) * 0.3).float().cuda()
    adv = torch.randn(n, generator=g).cuda()
    weights = torch.rand(n, generator=g)
    if n > 3:
        weights[3] = 0.0
        adv[n - 1] = 0.0
    return old, ref, adv, (weights / n).cuda()


def _check_policy(got, grad, want, x, targets, old, ref, adv, weights, kl_coef):
    ln_p, lp, ent = want["ln_p"], want["logprobs"], want["entropy"]
    w = torch.full_like(lp, 1.0 / max(len(lp), 1)) if weights is None else weights.cpu().double()
    lp_off = torch.nan_to_num(logprob_bound(ln_p, lp))
    ratio = torch.nan_to_num(torch.exp(lp - old.cpu().double()) * adv.cpu().double()).abs()
    rel = lp_off + 6 * U
    up = torch.zeros_like(lp) if ref is None else torch.nan_to_num(torch.exp(ref.cpu().double() - lp))
    ent_off = torch.nan_to_num(entropy_bound(ln_p, lp, ent)) * want["h"].abs() / w.clamp(min=1e-30)
    row_off = ratio * rel + abs(kl_coef) * (up + 1) * rel + ent_off + 6 * U * torch.nan_to_num(want["row_loss"]).abs()
    close(got.logprobs, lp, torch.nan_to_num(logprob_bound(ln_p, lp)), "logprobs")
    close(got.row_loss, want["row_loss"], row_off, "row_loss")
    if ref is not None:
        close(got.kl, want["kl"], (up + 1) * rel + 4 * U * torch.nan_to_num(want["kl"]), "kl")
    if got.entropy is not None:
        close(got.entropy, ent, torch.nan_to_num(entropy_bound(ln_p, lp, ent)), "entropy")
    close(got.loss, want["loss"], (w * row_off).sum() + 2 * U * want["loss"].abs().nan_to_num(), "loss")
    if grad is not None:
        a_off = w * (ratio + abs(kl_coef) * up) * rel
        bound = grad_bound(ln_p, lp, want["t"], ent, targets.cpu(), want["grad"], want["a"], a_off, want["h"], x.dtype)
        close(grad, want["grad"], torch.nan_to_num(bound), "grad")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 9, 1000, 4097, 32000, 50257, 151936])
@pytest.mark.parametrize("kl,entropy", [(0.0, 0.0), (0.05, 0.0), (0.05, 0.01)])
def test_policy_loss(dtype, vocab, kl, entropy):
    for rows in (1, 6, 41) if vocab < 50000 else (7,):
        x = _logits(rows, rows, vocab, dtype)
        targets = _targets(rows, rows, vocab, 0.2)
        temperature = _temperature("rows", rows) if rows > 1 else 0.8
        old, ref, adv, weights = _policy_inputs(rows, x, targets, temperature)
        ref = ref if kl else None
        want = O.policy(x, targets, old, adv, ref, weights, temperature, 0.2, 0.28, kl, entropy)
        kw = dict(ref_logprobs=ref, weights=weights, temperature=temperature, clip_high=0.28, kl_coef=kl,
                  entropy_coef=entropy)
        got, grad = policy_loss_and_grad(x, targets, old, adv, **kw)
        _check_policy(got, grad, want, x, targets, old, ref, adv, weights, kl)
        # through autograd: the same loss, the gradient times the upstream one
        leaf = x.detach().requires_grad_()
        auto = policy_loss(leaf, targets, old, adv, **kw)
        (auto.loss * 1.0).backward()
        _check_policy(auto, leaf.grad, want, x, targets, old, ref, adv, weights, kl)
        assert not auto.logprobs.requires_grad
        with torch.no_grad():
            _check_policy(policy_loss(leaf, targets, old, adv, **kw), None, want, x, targets, old, ref, adv, weights, kl)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["wide", "last", "column"])
def test_policy_layouts_and_defaults(dtype, layout):
    x = _logits(2, 19, 4099, dtype, layout)
    targets = _targets(2, 19, 4099)
    old, ref, adv, _ = _policy_inputs(2, x, targets, 1.0)
    want = O.policy(x, targets, old, adv)
    got, grad = policy_loss_and_grad(x, targets, old, adv)
    _check_policy(got, grad, want, x, targets, old, None, adv, None, 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 4097, 151936])
def test_policy_masks_infinities_and_nan(dtype, vocab):
    x, targets = _odd_rows(dtype, vocab)
    old, ref, adv, weights = _policy_inputs(7, x, targets, 1.0)
    want = O.policy(x, targets, old, adv, ref, weights, 1.0, 0.2, 0.28, 0.05, 0.01)
    got, grad = policy_loss_and_grad(x, targets, old, adv, ref_logprobs=ref, weights=weights, clip_high=0.28,
                                     kl_coef=0.05, entropy_coef=0.01)
    _check_policy(got, grad, want, x, targets, old, ref, adv, weights, 0.05)
    assert torch.isnan(got.loss)
    # the same rows padded out: the loss is whole again and their values do not matter
    bad = torch.tensor([0, 4, 6, 7, 11], device="cuda")
    targets = targets.clone()
    targets[bad] = -1
    old, ref, adv = old.clone(), ref.clone(), adv.clone()
    old[bad], ref[bad], adv[bad] = NAN, INF, NAN
    want = O.policy(x, targets, old, adv, ref, weights, 1.0, 0.2, 0.28, 0.05, 0.01)
    got, grad = policy_loss_and_grad(x, targets, old, adv, ref_logprobs=ref, weights=weights, clip_high=0.28,
                                     kl_coef=0.05, entropy_coef=0.01)
    assert torch.isfinite(got.loss) and (grad[bad] == 0).all()
    _check_policy(got, grad, want, x, targets, torch.nan_to_num(old), torch.nan_to_num(ref), torch.nan_to_num(adv),
                  weights, 0.05)


@pytest.mark.parametrize("rows,vocab,dtype", [
    (500, 100003, torch.bfloat16),      # one block per row, registers and ring
    (420, 170000, torch.float16),       # two of them per row
    (30, 400000, torch.bfloat16),       # few rows: eight smaller blocks
    (400, 400000, torch.bfloat16),
    (6, 600000, torch.float32),         # past the smaller blocks
    (5, 700000, torch.float32),         # past what a cluster holds
    (3, 1300000, torch.bfloat16),
    (40, 14400, torch.bfloat16), (40, 14392, torch.float16),       # around the shortest rows held
    (40, 32256, torch.bfloat16), (40, 32264, torch.bfloat16), (40, 64520, torch.bfloat16), (40, 64535, torch.float16),
    (40, 16128, torch.float32), (40, 16132, torch.float32), (40, 23041, torch.float32), (40, 46090, torch.float32),
    (40, 92163, torch.float32), (3000, 14403, torch.bfloat16), (2000, 8200, torch.float16)])
@pytest.mark.parametrize("entropy", [0.0, 0.01])
def test_policy_by_size(rows, vocab, dtype, entropy):
    """Sizes on both sides of each way a row is held on chip.  Most rows hold no
    token, as in a padded batch; those that do are checked."""
    g = torch.Generator().manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) * 3).to(dtype)
    alive = torch.randperm(rows, generator=g)[:min(rows, 12)].sort().values.cuda()
    targets = torch.full((rows,), -3, device="cuda")
    targets[alive] = torch.randint(0, vocab, (len(alive),), generator=g).cuda()
    part = x[alive].contiguous()
    old, ref, adv, _ = _policy_inputs(rows, part, targets[alive], 1.0)
    every = [torch.full((rows,), NAN, device="cuda") for _ in range(3)]
    for v, w in zip(every, (old, ref, adv)):
        v[alive] = w
    want = O.policy(part, targets[alive], old, adv, ref, None, 1.0, 0.2, 0.2, 0.05, entropy)
    weights = torch.full((rows,), 1.0 / len(alive), device="cuda")
    got, grad = policy_loss_and_grad(x, targets, every[0], every[2], ref_logprobs=every[1], weights=weights,
                                     kl_coef=0.05, entropy_coef=entropy)
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[alive] = False
    assert not grad[rest].any() and not got.row_loss[rest].any() and not got.kl[rest].any()
    picked = type(got)(got.loss, *(None if t is None else t[alive] for t in got[1:]))
    _check_policy(picked, grad[alive], want, part, targets[alive], old, ref, adv, torch.full_like(old, 1.0 / len(alive)), 0.05)


def test_policy_all_rows_padded():
    x = torch.full((5, 333), NAN, device="cuda", dtype=torch.bfloat16)
    t = torch.full((5,), -1, device="cuda")
    f = torch.full((5,), NAN, device="cuda")
    got, grad = policy_loss_and_grad(x, t, f, f, ref_logprobs=f, kl_coef=0.1, entropy_coef=0.1)
    assert got.loss.item() == 0 and (grad == 0).all() and (got.kl == 0).all() and (got.entropy == 0).all()


def test_policy_extreme_ratios():
    """A ratio that overflows: clipped where the advantage is positive, infinite
    loss where it is negative, and no term without an advantage."""
    x = _logits(6, 4, 64, torch.float32)
    t = _targets(6, 4, 64)
    old = torch.tensor([-300.0, -300.0, -300.0, 300.0], device="cuda")
    adv = torch.tensor([2.0, -1.0, 0.0, 1.0], device="cuda")
    got, grad = policy_loss_and_grad(x, t, old, adv)
    assert got.row_loss[0].item() == pytest.approx(-2.4) and got.row_loss[1].item() == INF
    assert got.row_loss[2].item() == 0 and got.row_loss[3].item() == 0
    assert (grad[[0, 2, 3]] == 0).all()


# ------------------------------------------------------------- preference loss
def _check_preference(got, grad, want, x, targets, ref, beta):
    ln_p, lp = want["ln_p"], want["logprobs"]
    lp_off = torch.where(want["alive"], torch.nan_to_num(logprob_bound(ln_p, lp)), torch.zeros_like(lp))
    close(got.logprobs, lp, torch.nan_to_num(logprob_bound(ln_p, lp)), "logprobs")
    # a gain is rounded once more; a pair's margin adds its rows' errors
    gain_off = lp_off + U * (lp.abs().nan_to_num() + (0 if ref is None else ref.cpu().double().abs()))
    total = abs(beta) * gain_off.sum() + 4 * U * want["rewards"].abs().max().nan_to_num()
    close(got.rewards, want["rewards"], total, "rewards")
    close(got.pair_loss, want["pair_loss"], 2 * total + 4 * U * (1 + want["pair_loss"].abs().nan_to_num()), "pair_loss")
    close(got.loss, want["loss"], 2 * total + 4 * U * (1 + want["loss"].abs().nan_to_num()), "loss")
    if grad is not None:
        pairs = len(want["pair_loss"])
        zero = torch.zeros_like(lp)
        a_off = want["a"].abs().nan_to_num() * 8 * U + torch.where(want["alive"], abs(beta) / pairs * 2 * total, zero)
        bound = grad_bound(ln_p, lp, want["t"], zero, targets.cpu(), want["grad"], want["a"], a_off, zero, x.dtype)
        close(grad, want["grad"], torch.nan_to_num(bound), "grad")


OFFSETS = {"plain": [0, 5, 9, 12, 20], "empty": [0, 0, 4, 4, 4], "tail": [0, 3, 7], "late": [2, 6, 11], "one": [0, 1, 2]}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 9, 1000, 4097, 50257])
@pytest.mark.parametrize("offsets", list(OFFSETS))
@pytest.mark.parametrize("average,smoothing", [(False, 0.0), (True, 0.1)])
def test_preference_loss(dtype, vocab, offsets, average, smoothing):
    offs = torch.tensor(OFFSETS[offsets])
    rows = int(offs[-1]) + (4 if offsets in ("tail", "late") else 0)
    x = _logits(rows, rows, vocab, dtype)
    targets = _targets(rows + 1, rows, vocab, 0.25)
    _, lp, _, _, _ = O.rows(x, targets)
    ref = (lp + torch.randn(rows, generator=torch.Generator().manual_seed(3), dtype=torch.float64) * 0.2).float().cuda()
    beta = 1.5 if average else 0.1
    want = O.preference(x, targets, offs, ref, beta, smoothing, average)
    kw = dict(ref_logprobs=ref, beta=beta, label_smoothing=smoothing, average=average)
    got, grad = preference_loss_and_grad(x, targets, offs.cuda(), **kw)
    _check_preference(got, grad, want, x, targets, ref, beta)
    leaf = x.detach().requires_grad_()
    auto = preference_loss(leaf, targets, offs.cuda(), **kw)
    auto.loss.backward()
    _check_preference(auto, leaf.grad, want, x, targets, ref, beta)


def test_preference_without_a_reference_and_with_temperatures():
    x = _logits(12, 30, 2001, torch.bfloat16, "wide")
    targets, offs = _targets(12, 30, 2001), torch.tensor([0, 8, 14, 15, 30])
    temperature = _temperature("rows", 30)
    want = O.preference(x, targets, offs, None, 0.2, 0.0, True, temperature)
    got, grad = preference_loss_and_grad(x, targets, offs.cuda(), beta=0.2, average=True, temperature=temperature)
    _check_preference(got, grad, want, x, targets, None, 0.2)


def test_preference_rows_outside_every_sequence_do_not_matter():
    x = _logits(13, 14, 515, torch.float32)
    x[9:] = NAN
    targets = _targets(13, 14, 515)
    offs = torch.tensor([0, 4, 9], device="cuda")
    got, grad = preference_loss_and_grad(x, targets, offs)
    assert torch.isfinite(got.loss) and (grad[9:] == 0).all() and (got.logprobs[9:] == 0).all()
    short = preference_loss_and_grad(x[:9], targets[:9], offs)
    assert torch.equal(short[0].loss, got.loss) and torch.equal(short[1], grad[:9])


def test_preference_one_long_pair_and_many_short():
    for lengths in ([700, 301], [1, 2, 3, 0] * 25):
        offs = torch.zeros(len(lengths) + 1, dtype=torch.int64)
        offs[1:] = torch.tensor(lengths).cumsum(0)
        rows = int(offs[-1])
        x, targets = _logits(17, rows, 129, torch.bfloat16), _targets(17, rows, 129, 0.1)
        want = O.preference(x, targets, offs, None, 0.05)
        got, grad = preference_loss_and_grad(x, targets, offs.cuda(), beta=0.05)
        _check_preference(got, grad, want, x, targets, None, 0.05)


# ------------------------------------------------------------------ their use
def _calls(x, targets, old, ref, adv, weights, offs):
    return {
        "logprobs": lambda out: token_logprobs(x, targets, entropy=True),
        "policy": lambda out: policy_loss_and_grad(x, targets, old, adv, ref_logprobs=ref, weights=weights, kl_coef=0.05,
                                                   entropy_coef=0.01, out=out),
        "preference": lambda out: preference_loss_and_grad(x, targets, offs, ref_logprobs=ref, out=out),
    }


def _flat(got):
    out = []
    for g in got if isinstance(got, tuple) else (got,):
        out += _flat(g) if isinstance(g, tuple) else [] if g is None else [g]
    return out


def _case(dtype=torch.bfloat16, rows=44, vocab=30011, layout="plain", seed=21):
    x = _logits(seed, rows, vocab, dtype, layout)
    targets = _targets(seed, rows, vocab, 0.1)
    old, ref, adv, weights = _policy_inputs(seed, x, targets, 1.0)
    return x, targets, old, ref, adv, weights, torch.tensor([0, 10, 21, 30, 40], device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["plain", "wide"])
@pytest.mark.parametrize("vocab", [30011, 32000])
@pytest.mark.parametrize("name", ["policy", "preference"])
def test_gradient_in_place_and_into_other_strides(dtype, layout, vocab, name):
    args = _case(dtype, vocab=vocab, layout=layout)
    x = args[0]
    keep = x.clone()
    want = [t.clone() for t in _flat(_calls(*args)[name](None))]
    wide = torch.full((x.shape[0], vocab + 3), 5.0, dtype=dtype, device="cuda")
    into = _flat(_calls(*args)[name](wide[:, 2:2 + vocab]))
    assert torch.equal(x, keep)                                    # the logits are only read
    assert (wide[:, :2] == 5).all() and (wide[:, 2 + vocab:] == 5).all()
    got = _flat(_calls(*args)[name](x))
    assert got[-1].data_ptr() == x.data_ptr()
    for a, b, c in zip(want, into, got):
        assert torch.equal(a, b) and torch.equal(a, c)
    if layout == "wide":                                           # the columns around them are left
        base = x._base
        assert (base[:, :3] == 7).all() and (base[:, 3 + vocab:] == 7).all()


@pytest.mark.parametrize("name", ["logprobs", "policy", "preference"])
def test_equal_inputs_give_equal_bits_on_any_stream(name):
    args = _case()
    want = [t.clone() for t in _flat(_calls(*args)[name](None))]
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        a = _flat(_calls(*args)[name](None))
    b = _flat(_calls(*args)[name](None))          # both at once
    torch.cuda.synchronize()
    for u, v, w in zip(want, a, b):
        assert torch.equal(u, v) and torch.equal(u, w)


@pytest.mark.parametrize("name", ["logprobs", "policy", "preference"])
def test_two_captured_graphs_replayed_at_once(name):
    cases = [_case(seed=31), _case(seed=32)]
    want = [[t.clone() for t in _flat(_calls(*c)[name](None))] for c in cases]
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_flat(_calls(*c)[name](None)))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for o in outs:
            for t in o:
                t.fill_(9)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            for u, v in zip(w, o):
                assert torch.equal(u, v)


@pytest.mark.parametrize("vocab", [1003, 1000003])       # two launches, and rows held on chip
def test_offsets_past_32_bits(vocab):
    """Rows whose elements lie past 2^32 (9 rows 600 M elements apart), the
    gradient in place."""
    rows, stride = 9, 600_000_000
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 20 GB of device memory")
    buf = torch.empty((rows - 1) * stride + vocab, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((rows, vocab), (stride, 1))
    x.copy_(_logits(3, rows, vocab, torch.bfloat16))
    targets = _targets(3, rows, vocab)
    old, ref, adv, _ = _policy_inputs(3, x, targets, 1.0)
    want = O.policy(x, targets, old, adv, ref, None, 1.0, 0.2, 0.2, 0.05, 0.01)
    got, grad = policy_loss_and_grad(x, targets, old, adv, ref_logprobs=ref, kl_coef=0.05, entropy_coef=0.01, out=x)
    assert grad.data_ptr() == x.data_ptr()
    _check_policy(got, grad, want, x, targets, old, ref, adv, None, 0.05)


def test_backward_twice_and_upstream_gradients():
    x, targets, old, ref, adv, weights, offs = _case(torch.float32, vocab=1001)
    leaf = x.clone().requires_grad_()
    loss = policy_loss(leaf, targets, old, adv, ref_logprobs=ref, kl_coef=0.1, entropy_coef=0.02).loss
    (one,) = torch.autograd.grad(loss, [leaf], retain_graph=True)
    (two,) = torch.autograd.grad(loss, [leaf], torch.tensor(-4.0, device="cuda"))
    assert torch.equal(one * -4, two)              # a power of two scales exactly
    lp, ent = token_logprobs(leaf, targets, entropy=True)
    (only_h,) = torch.autograd.grad(ent.sum(), [leaf], retain_graph=True)
    (only_a,) = torch.autograd.grad(lp.sum(), [leaf])
    ln_p, lp64, ent64, alive, t = O.rows(x, targets)
    one64, zero = torch.ones_like(lp64) * alive, torch.zeros_like(lp64)
    for got, a, h in ((only_h, zero, one64), (only_a, one64, zero)):
        want = O.gradient(ln_p, ent64, alive, t, targets, a, h)
        close(got, want, grad_bound(ln_p, lp64, t, ent64, targets.cpu(), want, a, zero, h, torch.float32), "grad")


def test_the_loss_may_be_changed_in_place():
    x, targets, old, _, adv, _, offs = _case(torch.float32, vocab=100)
    for f in (lambda z: policy_loss(z, targets, old, adv).loss, lambda z: preference_loss(z, targets, offs).loss,
              lambda z: token_logprobs(z, targets).sum()):
        leaf = x.clone().requires_grad_()
        f(leaf).backward()
        half = x.clone().requires_grad_()
        loss = f(half)
        loss *= 0.5
        loss.backward()
        assert torch.equal(half.grad * 2, leaf.grad)


def test_the_other_results_may_be_changed_before_the_backward_pass():
    x, targets, old, ref, adv, _, offs = _case(torch.float32, vocab=100)
    for f, names in ((lambda z: policy_loss(z, targets, old, adv, ref_logprobs=ref, kl_coef=0.1, entropy_coef=0.02),
                      ("row_loss", "logprobs", "kl")),
                     (lambda z: preference_loss(z, targets, offs), ("pair_loss", "rewards", "logprobs"))):
        leaf, again = x.clone().requires_grad_(), x.clone().requires_grad_()
        f(leaf).loss.backward()
        got = f(again)
        for name in names:
            getattr(got, name).mul_(3.0)
        got.loss.backward()
        assert torch.equal(again.grad, leaf.grad)


def test_second_derivatives_are_refused():
    """Also where a gradient is one term of what is differentiated: it is no constant."""
    x, targets, old, _, adv, _, offs = _case(torch.float32, vocab=100)
    for f in (lambda z: policy_loss(z, targets, old, adv).loss, lambda z: preference_loss(z, targets, offs).loss,
              lambda z: token_logprobs(z, targets).sum(), lambda z: token_logprobs(z, targets).square().sum()):
        leaf = x.clone().requires_grad_()
        (grad,) = torch.autograd.grad(f(leaf), [leaf], create_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            (grad.square().sum() + leaf.sum()).backward()


def test_first_calls_captured():
    """The first call of a process is captured, and a replay gives what an eager call gives."""
    import os
    import subprocess
    import sys
    code = """
import torch
from b200_sampler import policy_loss_and_grad, preference_loss_and_grad, token_logprobs
g = torch.Generator("cuda").manual_seed(1)
x = torch.randn(40, 32000, device="cuda", generator=g).bfloat16()
t = torch.randint(0, 32000, (40,), device="cuda", generator=g)
f = torch.randn(40, device="cuda", generator=g)
offs = torch.tensor([0, 10, 30], device="cuda")
def run():
    (a, ga), (b, gb) = policy_loss_and_grad(x, t, f, f), preference_loss_and_grad(x, t, offs)
    return [token_logprobs(x, t), a.loss, a.logprobs, ga, b.loss, b.rewards, gb]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
for u, v in zip(got, run()):
    assert torch.equal(u, v)
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": os.pathsep.join(sys.path)})
    assert r.returncode == 0, r.stderr


def test_changed_logits_stop_the_backward_pass():
    x, targets, old, _, adv, _, _ = _case(torch.float32, vocab=100)
    leaf = x.clone().requires_grad_()
    h = leaf * 1.0
    loss = policy_loss(h, targets, old, adv).loss
    policy_loss_and_grad(h.detach(), targets, old, adv, out=h.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_rollout_is_sampled_scored_and_learned_from():
    """The operators together, as a training step uses them: rows are sampled,
    scored as they were drawn, and the policy's and the preference's gradients
    are taken on the same rollout."""
    from b200_sampler import SamplingParams
    from b200_sampler.sampler import DeviceBatch
    B, V, T = 24, 32000, 6
    params = [SamplingParams(temperature=0.0 if b % 5 == 0 else 0.9, top_k=40) for b in range(B)]
    batch = DeviceBatch(None, params, "cuda", seed=7)
    temps = torch.tensor([p.temperature for p in params], device="cuda")
    steps, ids, scores = [], [], []
    for step in range(T):
        x = _logits(50 + step, B, V, torch.bfloat16)
        out, lp = torch.empty(B, dtype=torch.int64, device="cuda"), torch.empty(B, device="cuda")
        assert batch.launch(x, out, offset=step) == 0
        assert batch.logprobs(x, out, lp) == 0
        steps.append(x), ids.append(out), scores.append(lp)
    x, targets, old = torch.stack(steps, 1).view(B * T, V), torch.stack(ids, 1).view(-1), torch.stack(scores, 1).view(-1)
    temperature = temps.repeat_interleave(T)
    assert (targets >= 0).all()
    ln_p, lp, ent, _, _ = O.rows(x, targets, temperature)
    close(old, lp, logprob_bound(ln_p, lp), "scores of the drawn ids")
    adv = _vector(3, B * T)
    got, grad = policy_loss_and_grad(x, targets, old, adv, temperature=temperature, ref_logprobs=old, kl_coef=0.1)
    # the policy is the one that drew: every ratio is 1 and the KL is 0
    want = O.policy(x, targets, old, adv, old, None, temperature, 0.2, 0.2, 0.1)
    _check_policy(got, grad, want, x, targets, old, old, adv, None, 0.1)
    offs = torch.arange(0, B * T + 1, T, device="cuda")[:B + 1]
    if offs.numel() % 2 == 0:
        offs = offs[:-1]
    moved = (x.float() * 1.1).to(torch.bfloat16)
    want = O.preference(moved, targets, offs, old, 0.3, 0.0, False, temperature)
    got, grad = preference_loss_and_grad(moved, targets, offs, ref_logprobs=old, beta=0.3, temperature=temperature)
    _check_preference(got, grad, want, moved, targets, old, 0.3)
