"""64-bit restatement of the operators on sampled tokens' logits (test
infrastructure): log-probabilities, entropies, the policy and preference
losses, and their gradients by formula.  Plain torch in float64; rows that hold
no token (negative target) give zeros, rows without a distribution NaN."""
import math

import torch


def _each(temperature, n):
    t = torch.as_tensor(temperature, dtype=torch.float64).expand(n) if not torch.is_tensor(temperature) \
        else temperature.double().cpu()
    t = torch.where(t == 0, torch.ones_like(t), t)
    return torch.where((t > 0) & torch.isfinite(t), t, torch.full_like(t, math.nan))


def rows(logits, targets, temperature=1.0):
    """(ln p [n, V], logprob [n], entropy [n], alive [n], T [n]) in float64 on the CPU."""
    x, targets = logits.detach().cpu().double(), targets.cpu()
    n, v = x.shape
    t = _each(temperature, n)
    alive = targets >= 0
    m = x.max(dim=1).values                          # NaN if the row holds one
    z = (x - m[:, None]) / t[:, None]                # -inf - -inf and inf - inf: NaN, no distribution
    ln_p = z - torch.log(torch.exp(z).sum(1))[:, None]
    lp = ln_p.gather(1, targets.clamp(0, v - 1)[:, None]).squeeze(1)
    lp = torch.where(targets >= v, torch.full_like(lp, math.nan), lp)
    ent = -torch.where(ln_p == -math.inf, torch.zeros_like(ln_p), ln_p.exp() * ln_p).sum(1)
    ent = torch.where(targets >= v, torch.full_like(ent, math.nan), ent)
    zero = torch.zeros_like(lp)
    return ln_p, torch.where(alive, lp, zero), torch.where(alive, ent, zero), alive, t


def gradient(ln_p, ent, alive, t, targets, a, h=None):
    """d/dlogits of sum a logprob + h entropy."""
    targets, a = targets.cpu(), torch.where(alive, a.double().cpu(), torch.zeros_like(t))
    h = torch.zeros_like(a) if h is None else torch.where(alive, h.double().cpu(), torch.zeros_like(t))
    p = ln_p.exp()
    plp = torch.where(ln_p == -math.inf, torch.zeros_like(p), p * ln_p)
    g = -p * a[:, None] - h[:, None] * (plp + p * ent[:, None])
    v = ln_p.shape[1]
    g.scatter_add_(1, targets.clamp(0, v - 1)[:, None], torch.where(targets < v, a, torch.full_like(a, math.nan))[:, None])
    g = g / t[:, None]
    g = torch.where(((targets >= v) & ((a != 0) | (h != 0)))[:, None], torch.full_like(g, math.nan), g)
    return torch.where(((a == 0) & (h == 0))[:, None], torch.zeros_like(g), g)


def policy(logits, targets, old, adv, ref=None, weights=None, temperature=1.0, low=0.2, high=0.2, kl_coef=0.0,
           entropy_coef=0.0):
    ln_p, lp, ent, alive, t = rows(logits, targets, temperature)
    n = lp.shape[0]
    w = torch.full((n,), 1.0 / max(n, 1), dtype=torch.float64) if weights is None else weights.double().cpu()
    alive = alive & (w != 0)
    zero = torch.zeros(n, dtype=torch.float64)
    lp, ent = torch.where(alive, lp, zero), torch.where(alive, ent, zero)
    r, adv = torch.exp(lp - old.double().cpu()), adv.double().cpu()
    inside, clipped = r * adv, r.clamp(1 - low, 1 + high) * adv
    term, a = -torch.minimum(inside, clipped), torch.where(clipped < inside, zero, -inside)
    none = (adv == 0) & ~torch.isnan(r)
    term, a = torch.where(none, zero, term), torch.where(none, zero, a)
    kl = None
    if ref is not None:
        d = ref.double().cpu() - lp
        kl = torch.where(alive, torch.expm1(d) - d, zero)
        if kl_coef:
            term, a = term + kl_coef * kl, a - kl_coef * torch.expm1(d)
    term = torch.where(alive, term - (entropy_coef * ent if entropy_coef else 0.0), zero)
    a = torch.where(alive, a * w, zero)
    h = torch.where(alive, -entropy_coef * w, zero)
    return {"loss": torch.where(alive, term * w, zero).sum(), "row_loss": term, "logprobs": lp, "entropy": ent, "kl": kl,
            "a": a, "h": h, "grad": gradient(ln_p, ent, alive, t, targets, a, h), "ln_p": ln_p, "t": t, "alive": alive}


def preference(logits, targets, offsets, ref=None, beta=0.1, smoothing=0.0, average=False, temperature=1.0):
    ln_p, lp, ent, alive, t = rows(logits, targets, temperature)
    offsets = offsets.cpu().tolist()
    n, pairs = lp.shape[0], len(offsets) // 2
    inside = torch.zeros(n, dtype=torch.bool)
    inside[offsets[0]:offsets[-1]] = True
    alive = alive & inside
    zero = torch.zeros(n, dtype=torch.float64)
    lp = torch.where(alive, lp, zero)
    gain = torch.where(alive, lp - (0.0 if ref is None else ref.double().cpu()), zero)
    a, rewards, pair_loss = zero.clone(), torch.zeros(pairs, 2, dtype=torch.float64), torch.zeros(pairs, dtype=torch.float64)
    for p in range(pairs):
        share = []
        for k in range(2):
            rng = slice(offsets[2 * p + k], offsets[2 * p + k + 1])
            share.append(1.0 / max(int(alive[rng].sum()), 1) if average else 1.0)
            rewards[p, k] = beta * gain[rng].sum() * share[k]
        h = rewards[p, 0] - rewards[p, 1]
        pair_loss[p] = (1 - smoothing) * torch.nn.functional.softplus(-h) + smoothing * torch.nn.functional.softplus(h)
        slope = (smoothing * torch.sigmoid(h) - (1 - smoothing) * torch.sigmoid(-h)) * beta / pairs
        for k in range(2):
            rng = slice(offsets[2 * p + k], offsets[2 * p + k + 1])
            a[rng] = torch.where(alive[rng], (-slope if k else slope) * share[k], zero[rng])
    return {"loss": pair_loss.mean() if pairs else torch.zeros((), dtype=torch.float64), "pair_loss": pair_loss,
            "rewards": rewards, "logprobs": lp, "a": a, "grad": gradient(ln_p, ent, alive, t, targets, a),
            "ln_p": ln_p, "t": t, "alive": alive}
