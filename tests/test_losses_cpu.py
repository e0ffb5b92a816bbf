"""Refusals of the operators on sampled tokens' logits (no GPU needed): the C
entry points reject bad arguments before touching CUDA, and the Python calls
name what is wrong.  The oracle's formulas are checked against differentiation."""
import math
import os

import pytest
import torch

from b200_sampler import _lib, losses
from oracle import losses_oracle as O

needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
BAD, TYPE = _lib.NS_ERR_INVALID_ARGUMENT, _lib.NS_ERR_UNSUPPORTED_DTYPE
ROWS = dict(logits=1, dtype=0, rows=4, vocab=10, row_stride=10, targets=1, temperature=None, temperature_all=1.0)
ENTRIES = {
    "ns_token_logprobs": dict(ROWS, logprobs=1, entropy=None, stats=None, stream=None),
    "ns_token_logprobs_grad": dict(ROWS, stats=1, entropy=None, a=1, h=None, grad=2, grad_stride=10, stream=None),
    "ns_policy_loss": dict(ROWS, old=1, ref=None, adv=1, weights=None, low=0.2, high=0.2, kl_coef=0.0, entropy_coef=0.0,
                           loss=1, row_loss=1, logprobs=1, entropy=None, kl=None, stats=1, row_grad=1, grad=None,
                           grad_stride=0, stream=None),
    "ns_preference_loss": dict(ROWS, offsets=1, pairs=1, ref=None, beta=0.1, smoothing=0.0, average=0, loss=1,
                               pair_loss=1, rewards=1, logprobs=1, stats=1, row_grad=1, grad=None, grad_stride=0,
                               stream=None),
}


def _call(name, **kw):
    a = dict(ENTRIES[name])
    assert set(kw) <= set(a)
    a.update(kw)
    return getattr(_lib.load(), name)(*a.values())


@needs_lib
@pytest.mark.parametrize("name", list(ENTRIES))
def test_c_entries_refuse_bad_rows(name):
    assert _call(name, dtype=3) == TYPE and _call(name, dtype=-1) == TYPE
    for kw in (dict(rows=-1), dict(vocab=0), dict(vocab=-5), dict(row_stride=9), dict(rows=(1 << 24) + 1),
               dict(vocab=(1 << 24) + 1, row_stride=1 << 25), dict(logits=None), dict(targets=None),
               dict(temperature_all=-0.5), dict(temperature_all=math.inf), dict(temperature_all=math.nan)):
        assert _call(name, **kw) == BAD, kw


@needs_lib
def test_c_entries_refuse_missing_results_and_bad_numbers():
    assert _call("ns_token_logprobs", logprobs=None) == BAD
    for kw in (dict(stats=None), dict(grad=None), dict(grad_stride=9), dict(h=1), dict(grad=1, grad_stride=12)):
        assert _call("ns_token_logprobs_grad", **kw) == BAD, kw
    for kw in (dict(old=None), dict(adv=None), dict(loss=None), dict(row_loss=None), dict(logprobs=None), dict(stats=None),
               dict(row_grad=None), dict(kl_coef=0.1), dict(kl=1), dict(entropy_coef=0.1), dict(low=-0.1), dict(low=1.1),
               dict(low=math.nan), dict(high=-0.1), dict(high=math.inf), dict(kl_coef=math.nan), dict(entropy_coef=math.inf),
               dict(grad=2, grad_stride=9), dict(grad=1, grad_stride=12)):
        assert _call("ns_policy_loss", **kw) == BAD, kw
    for kw in (dict(offsets=None), dict(pairs=-1), dict(beta=math.inf), dict(beta=math.nan), dict(smoothing=-0.1),
               dict(smoothing=1.0), dict(smoothing=math.nan), dict(loss=None), dict(pair_loss=None), dict(rewards=None),
               dict(logprobs=None), dict(stats=None), dict(row_grad=None), dict(grad=2, grad_stride=9),
               dict(grad=1, grad_stride=12)):
        assert _call("ns_preference_loss", **kw) == BAD, kw


@needs_lib
def test_c_entries_with_no_rows_need_no_logits():
    assert _call("ns_token_logprobs", rows=0, logits=None, targets=None, logprobs=None) == _lib.NS_OK
    assert _call("ns_token_logprobs_grad", rows=0, logits=None, targets=None, grad=None) == _lib.NS_OK


def _inputs(n=4, v=10):
    return torch.zeros(n, v), torch.zeros(n, dtype=torch.int64), torch.zeros(n), torch.zeros(n)


def test_python_refusals():
    x, t, old, adv = _inputs()
    offs = torch.tensor([0, 2, 4])
    for call in (lambda x, t, **kw: losses.token_logprobs(x, t, **kw),
                 lambda x, t, **kw: losses.policy_loss(x, t, old, adv, **kw),
                 lambda x, t, **kw: losses.policy_loss_and_grad(x, t, old, adv, **kw),
                 lambda x, t, **kw: losses.preference_loss(x, t, offs, **kw),
                 lambda x, t, **kw: losses.preference_loss_and_grad(x, t, offs, **kw)):
        for bad in (x[0], x[:, :0], x[None]):
            with pytest.raises(ValueError, match="rows, vocab"):
                call(bad, t)
        with pytest.raises(TypeError, match="dtype"):
            call(x.double(), t)
        with pytest.raises(TypeError, match="int64"):
            call(x, t.int())
        for bad in (t[:3], t[:, None]):
            with pytest.raises(ValueError, match="one value per row"):
                call(x, bad)
        for bad in (-1.0, math.inf, math.nan):
            with pytest.raises(ValueError, match="temperature"):
                call(x, t, temperature=bad)
        with pytest.raises(ValueError, match="one value per row"):
            call(x, t, temperature=torch.ones(3))
        with pytest.raises(TypeError, match="floating"):
            call(x, t, temperature=torch.ones(4, dtype=torch.int64))
        with pytest.raises(ValueError, match="CUDA"):
            call(x, t)


def test_python_refusals_of_the_losses():
    x, t, old, adv = _inputs()
    f = losses.policy_loss
    for kw, word in ((dict(clip_low=1.5), "clip"), (dict(clip_high=-1.0), "clip"), (dict(clip_low=math.nan), "clip"),
                     (dict(kl_coef=math.inf), "finite"), (dict(entropy_coef=math.nan), "finite"),
                     (dict(kl_coef=0.1), "ref_logprobs"), (dict(weights=torch.ones(5)), "weights"),
                     (dict(ref_logprobs=torch.ones(4, 1)), "ref_logprobs")):
        with pytest.raises(ValueError, match=word):
            f(x, t, old, adv, **kw)
    with pytest.raises(ValueError, match="needed"):
        f(x, t, None, adv)
    g = losses.preference_loss
    offs = torch.tensor([0, 2, 4])
    for bad in (offs[:2], offs.int(), offs[None]):
        with pytest.raises(ValueError, match="seq_offsets"):
            g(x, t, bad)
    for kw in (dict(beta=math.nan), dict(label_smoothing=1.0), dict(label_smoothing=-0.1)):
        with pytest.raises(ValueError, match="beta"):
            g(x, t, offs, **kw)
    for out in (torch.zeros(4, 9), torch.zeros(4, 10).half(), torch.zeros(10, 4).t(), torch.zeros(1, 10).expand(4, 10)):
        with pytest.raises(ValueError, match="out"):
            losses.policy_loss_and_grad(x, t, old, adv, out=out)
        with pytest.raises(ValueError, match="out"):
            losses.preference_loss_and_grad(x, t, offs, out=out)
    buf = torch.zeros(4, 12)
    with pytest.raises(ValueError, match="overlap"):
        losses.policy_loss_and_grad(buf[:, :10], t, old, adv, out=buf[:, 2:])


def test_oracle_gradients_are_the_derivatives():
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(9, 23, generator=g, dtype=torch.float64) * 2)
    x[2, 5:] = -math.inf
    t = torch.randint(0, 5, (9,), generator=g)
    t[4] = -1
    temperature = torch.linspace(0.5, 1.5, 9)
    old, adv, ref = (torch.randn(9, generator=g) - 2 for _ in range(3))
    offs = torch.tensor([0, 2, 3, 5, 9])
    for f in (lambda z: O.policy(z, t, old, adv, ref, None, temperature, 0.2, 0.3, 0.1, 0.05),
              lambda z: O.preference(z, t, offs, ref, 0.4, 0.1, True, temperature)):
        grad = f(x)["grad"]
        for seed in range(3):
            d = torch.randn(x.shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
            step = 1e-5
            up, down = f(x + step * d)["loss"], f(x - step * d)["loss"]
            slope = (up - down) / (2 * step)
            # each loss is a sum whose terms carry some 60 roundings of 2^-53, and the step divides them; the
            # exponentials' third derivative along d is at most (|d| / T)^3 < 1000 of the loss: step^2 / 6 of it
            size = up.abs() + down.abs()
            assert abs(slope - (grad * d).sum()) < size * (60 * 2.0 ** -53 / (2 * step) + 1000 * step ** 2 / 6) + 1e-10
