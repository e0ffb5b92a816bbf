"""Rows whose values are easily lost in the operators on sampled tokens' logits:
barred targets among low logits.  Against the 64-bit oracle, within bounds
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
