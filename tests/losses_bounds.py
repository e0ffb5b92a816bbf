"""Error bounds of the fp32 kernels behind include/ns_losses.h, from the
roundings they make (u = 2^-24, half a step of fp32), against 64-bit values.

t = (x - c) s, c the target's logit, has three roundings (difference, scale,
product), so 2^t is off by 3 u |ln 2^t| relative and 2^-22 = 4 u of the
exponential itself; a thread adds at most V / 256 + 16 values one after another
and 30 joins follow.  z is taken from the row's largest value here: |ln 2^t| is
at most |z| of the value plus |z| of the target (1 / p of the target, when c is
the largest value itself, is not less).
"""
import torch

U = 2.0 ** -24


def _parts(ln_p):
    z = ln_p - ln_p.max(dim=1, keepdim=True).values
    z = torch.where(torch.isfinite(z), z, torch.zeros_like(z))
    p = torch.where(torch.isfinite(ln_p), ln_p.exp(), torch.zeros_like(ln_p))
    return z.abs(), p


def adds(vocab):
    return vocab / 256 + 16 + 30


def _offset(lp):
    """|z| of the target, at most |ln p| of it."""
    return torch.nan_to_num(lp, posinf=0.0, neginf=0.0).abs()


def sum_bound(ln_p, lp):
    """Relative error of S per row."""
    z, p = _parts(ln_p)
    return U * (3 * ((p * z).sum(1) + _offset(lp)) + 4 + adds(ln_p.shape[1]))


def logprob_bound(ln_p, lp):
    return sum_bound(ln_p, lp) + U * (4 * _offset(lp) + 4)


def entropy_bound(ln_p, lp, ent):
    """H = ln S - ln2 U / S, whose terms' sizes are |ln S| = |ln p| and mean |t|."""
    z, p = _parts(ln_p)
    z = z + _offset(lp)[:, None]
    mean, square = (p * z).sum(1), (p * z * z).sum(1)
    n = adds(ln_p.shape[1]) + 8
    return U * (n * (1 + 2 * mean) + 3 * (mean + 2 * square) + 4 * (torch.nan_to_num(ent).abs() + _offset(lp)))


def grad_bound(ln_p, lp, t, ent, targets, grad, a, a_off, h, dtype):
    """Per element: the output's rounding, p's error, the coefficients' errors."""
    z, p = _parts(ln_p)
    lnp = torch.where(torch.isfinite(ln_p), ln_p, torch.zeros_like(ln_p)).abs()
    a, h, a_off = (torch.nan_to_num(v).abs()[:, None] for v in (a, h, a_off))
    ent_off, ent = entropy_bound(ln_p, lp, ent)[:, None], torch.nan_to_num(ent).abs()[:, None]
    p_off = U * (3 * (z + _offset(lp)[:, None]) + 8 + lnp) + sum_bound(ln_p, lp)[:, None]
    # a probability below 2^-126 is flushed to zero (ex2.approx.ftz): all of what it carries is off, and
    # that is at most 2^-126 times its coefficient
    off = p * ((a + h * (lnp + ent)) * (p_off + 6 * U) + a_off + h * ent_off) + 2.0 ** -126 * (a + h * (lnp + ent))
    at = targets.clamp(0, ln_p.shape[1] - 1)[:, None]
    off.scatter_add_(1, at, a_off + 4 * U * a)
    info = torch.finfo(dtype)
    return (off / t[:, None] + torch.nan_to_num(grad).abs() * (info.eps / 2 + U)
            + info.smallest_normal * info.eps)


def close(got, want, bound, what):
    """Equal where want is not finite (NaN and infinities in place), within the bound elsewhere."""
    got, want = got.detach().cpu().double(), want.double()
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    bound = torch.as_tensor(bound, dtype=torch.float64).expand_as(want)
    off = torch.where(odd, torch.zeros_like(want), (got - want).abs())
    worst = (off - bound).max().item() if off.numel() else 0.0
    assert worst <= 0, (what, "over the bound by", worst, "largest difference", off.max().item())
