"""Cases for the operators on the logits of sampled tokens: token log-probabilities
(with entropy, and their gradient), the clipped policy loss and the preference loss.

Each case is one call that a program around the sampler makes: the log-probabilities
of the ids a decode step drew, the scoring of a whole rollout, and the loss and
gradient of a training step on rollouts.  ``run`` computes it in plain torch, or
(``own``) through ``b200_sampler``; ``exact`` gives the same from the definitions in
64 bits.  One row of logits belongs to one token; a negative target marks a row that
holds no token (padding, prompt positions, a failed draw).
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _logprob(name, rows, vocab, dtype, grad=False, entropy=False, temperature="one", padded=0.0, barred=0):
    return {"name": name, "op": "logprob", "rows": rows, "vocab": vocab, "dtype": dtype, "grad": grad,
            "entropy": entropy, "temperature": temperature, "padded": padded, "barred": barred}


def _policy(name, rows, vocab, dtype, kl=0.0, entropy=0.0, temperature="one", padded=0.0, barred=0, high=0.2):
    return {"name": name, "op": "policy", "rows": rows, "vocab": vocab, "dtype": dtype, "kl": kl, "entropy": entropy,
            "temperature": temperature, "padded": padded, "barred": barred, "low": 0.2, "high": high}


def _preference(name, pairs, length, vocab, dtype, smoothing=0.0, average=False, padded=0.3, tail=0):
    return {"name": name, "op": "preference", "pairs": pairs, "length": length, "vocab": vocab, "dtype": dtype,
            "beta": 2.0 if average else 0.1, "smoothing": smoothing, "average": average, "padded": padded, "tail": tail}


def listed():
    return [
        # one request's decode step that returns the drawn id's log-probability
        _logprob("logprob decode 1", 1, 151936, "fp32"),
        # the decode benchmark's batch, each row at its own temperature
        _logprob("logprob decode 64", 64, 151936, "bf16", temperature="rows"),
        # scoring a finished rollout under the model that drew it, with the entropies
        _logprob("logprob rollout 4096", 4096, 151936, "bf16", entropy=True, barred=267),
        # an odd vocabulary (rows that start on any 2-byte boundary), forward and backward
        _logprob("logprob train 333 odd", 333, 50257, "fp16", grad=True, padded=0.1),
        # forward and backward with the entropy, fp32 logits
        _logprob("logprob train 512", 512, 151936, "fp32", grad=True, entropy=True, temperature="rows"),
        # a short rollout of a small-vocabulary model
        _policy("policy 16", 16, 32000, "bf16", kl=0.05),
        # a micro-batch of rollouts padded to the longest, KL to the reference model
        _policy("policy 2048", 2048, 151936, "bf16", kl=0.02, padded=0.2, temperature="all", high=0.28),
        # fp32 logits, KL and an entropy bonus, columns past the tokenizer's barred
        _policy("policy 600 fp32", 600, 151936, "fp32", kl=0.05, entropy=0.01, barred=267),
        # an odd vocabulary
        _policy("policy 777 odd", 777, 64007, "fp16", entropy=0.003, padded=0.1, temperature="rows"),
        # two short pairs
        _preference("preference 2x12", 2, 12, 32000, "bf16"),
        # a micro-batch of pairs, prompt positions without a target, padding behind the last sequence
        _preference("preference 8x128", 8, 128, 151936, "bf16", tail=37),
        # an odd vocabulary in fp32, length-normalised with smoothed labels
        _preference("preference 5x70 odd", 5, 70, 32001, "fp32", smoothing=0.1, average=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logprob", "logprob", "policy", "policy", "preference"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    vocab = rng.choice([151936, 32000, _spread(rng, 1000, 152000), _spread(rng, 1000, 152000) | 1])
    most = 4096 if op == "logprob" else 2048
    most = max(2, int(most * 151936 * 2 / (vocab * _BYTES[dtype]) / (2 if dtype == "fp32" else 1)))
    rows = _spread(rng, 1, min(most, 8192))
    temperature = rng.choice(["one", "all", "rows"])
    padded = rng.choice([0.0, 0.0, round(rng.uniform(0.02, 0.5), 3)])
    barred = rng.choice([0, 0, rng.randrange(1, 300)])
    if op == "logprob":
        grad = rng.random() < 0.5
        case = _logprob("", max(1, rows // 3) if grad else rows, vocab, dtype, grad, rng.random() < 0.5, temperature, padded, barred)
    elif op == "policy":
        case = _policy("", rows, vocab, dtype, rng.choice([0.0, round(rng.uniform(0.005, 0.1), 4)]),
                       rng.choice([0.0, round(rng.uniform(0.001, 0.02), 4)]), temperature, padded, barred,
                       rng.choice([0.2, 0.28]))
    else:
        length = _spread(rng, 4, 300)
        pairs = max(1, min(64, rows // (2 * length)))
        length = max(2, min(length, most // (2 * pairs)))
        case = _preference("", pairs, length, vocab, dtype, rng.choice([0.0, 0.1]), rng.random() < 0.3, padded,
                           rng.choice([0, rng.randrange(1, 40)]))
    del case["name"]
    return case


def _lengths(case):
    """Lengths of the 2 x pairs sequences (chosen, rejected, chosen, ...): ragged, fixed by the case."""
    n, at = 2 * case["pairs"], torch.arange(2 * case["pairs"], dtype=torch.float64)
    share = 0.5 + torch.remainder(at * 0.6180339887 + 0.25, 1.0)      # 0.5 .. 1.5 of `length`
    return torch.clamp((share * case["length"]).long(), 1, None)[:n]


def _rows(case):
    return int(_lengths(case).sum()) + case["tail"] if case["op"] == "preference" else case["rows"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kw = {"generator": g, "device": "cuda"}
    rows, vocab, op = _rows(case), case["vocab"], case["op"]
    # logits of a model: a wide background and a few per cent of likely tokens
    logits = torch.randn(rows, vocab, dtype=torch.float32, **kw).mul_(2.5)
    logits += torch.rand(rows, vocab, **kw).lt_(0.001).mul_(9.0)
    if case.get("barred"):        # columns that no token owns
        logits[:, max(1, vocab - case["barred"]):] = -math.inf
    # targets drawn from that distribution (an exponential race), as a sampler draws them
    race = torch.empty_like(logits).exponential_(generator=g).log_().neg_().add_(logits)
    targets = race.argmax(dim=1)
    del race
    logits = logits.to(_TYPES[case["dtype"]])
    state = {"op": op, "case": case}
    if case.get("padded"):
        targets[torch.rand(rows, **kw) < case["padded"]] = -1
    if op == "preference":
        offsets = torch.zeros(2 * case["pairs"] + 1, dtype=torch.int64)
        offsets[1:] = _lengths(case).cumsum(0)
        targets[int(offsets[-1]):] = -1
        state["offsets"] = offsets.cuda()
    kind = case.get("temperature", "one")
    temperature = {"one": 1.0, "all": 0.7}.get(kind) or torch.rand(rows, **kw) * 0.8 + 0.6
    state.update(logits=logits, targets=targets, temperature=temperature)

    # what the policy that drew the tokens, and the reference model, gave them: near this model's values
    t = temperature.double() if torch.is_tensor(temperature) else temperature
    at = logits.gather(1, targets.clamp(min=0)[:, None]).double().squeeze(1) / t
    m = logits.amax(dim=1).float()
    each = t.float()[:, None] if torch.is_tensor(t) else t
    lp = at - m.double() / t - torch.log(((logits.float() - m[:, None]) / each).exp_().sum(1, dtype=torch.float64))
    if op == "logprob":
        state["grad_logprobs"] = torch.randn(rows, **kw) / rows
        state["grad_entropy"] = torch.randn(rows, **kw) * (0.01 / rows)
        if case["grad"]:
            logits.requires_grad_()
    elif op == "policy":
        drift = torch.randn(rows, dtype=torch.float64, **kw) * 0.2     # log of the ratio
        # a ratio within rounding of the clip's border may fall on either side of it: none is placed there
        drift = torch.where((drift.exp() - (1 + case["high"])).abs() < 1e-3, drift + 0.004, drift)
        drift = torch.where((drift.exp() - (1 - case["low"])).abs() < 1e-3, drift + 0.004, drift)
        state["old"] = (lp - drift).float()
        state["ref"] = (lp + torch.randn(rows, dtype=torch.float64, **kw) * 0.3).float() if case["kl"] else None
        state["advantages"] = torch.randn(rows, **kw) + 0.3
        alive = targets >= 0
        state["weights"] = alive.float() / alive.sum().clamp(min=1)    # the mean over the tokens
    else:
        state["ref"] = (lp + torch.randn(rows, dtype=torch.float64, **kw) * 0.2).float()
    return state


# ---------------------------------------------------------------- plain form
def _per_row(temperature):
    return temperature[:, None] if torch.is_tensor(temperature) else temperature


def _statistics(logits, targets, temperature):
    """Per row: the scaled logits less their maximum, their exponentials, and in 64 bits the sum, the target's
    log-probability and the entropy."""
    x = logits.detach().float()
    x = x - x.amax(dim=1, keepdim=True)
    at = x.gather(1, targets.clamp(min=0)[:, None]).squeeze(1).double() / temperature
    z = x / _per_row(temperature)
    e = torch.exp(z)
    total = e.sum(dim=1, dtype=torch.float64)
    alive = targets >= 0
    logprobs = torch.where(alive, at - torch.log(total), torch.zeros_like(at))
    mean = torch.where(e > 0, e * z, torch.zeros_like(e)).sum(dim=1, dtype=torch.float64) / total
    entropy = torch.where(alive, torch.log(total) - mean, torch.zeros_like(at))
    return z, e, total, logprobs, entropy


def _gradient(z, e, total, targets, temperature, a, h, entropy, dtype):
    """d/dlogits of sum(a * logprob + h * entropy); rows without a token get zero."""
    alive = targets >= 0
    each = temperature if torch.is_tensor(temperature) else torch.full_like(total, temperature)
    a = torch.where(alive, a.double(), torch.zeros_like(total)) / each
    p = e / total.float()[:, None]
    if h is None:
        grad = p * -a.float()[:, None]
    else:
        h = torch.where(alive, h.double(), torch.zeros_like(total)) / each
        shift = a + h * (entropy - torch.log(total))
        grad = -p * (shift.float()[:, None] + h.float()[:, None] * torch.where(e > 0, z, torch.zeros_like(z)))
    grad.scatter_add_(1, targets.clamp(min=0)[:, None], a.float()[:, None])
    return grad.to(dtype)


def _plain_logprob(state):
    case, targets, temperature = state["case"], state["targets"], state["temperature"]
    z, e, total, logprobs, entropy = _statistics(state["logits"], targets, temperature)
    out = {"logprobs": logprobs.float()}
    if case["entropy"]:
        out["entropy"] = entropy.float()
    if case["grad"]:
        out["grad_logits"] = _gradient(z, e, total, targets, temperature, state["grad_logprobs"],
                                       state["grad_entropy"] if case["entropy"] else None, entropy, state["logits"].dtype)
    return out


def _plain_policy(state):
    case, targets, temperature = state["case"], state["targets"], state["temperature"]
    z, e, total, logprobs, entropy = _statistics(state["logits"], targets, temperature)
    alive, weights, advantages = targets >= 0, state["weights"].double(), state["advantages"].double()
    ratio = torch.exp(logprobs - state["old"].double())
    inside = ratio * advantages
    clipped = ratio.clamp(1 - case["low"], 1 + case["high"]) * advantages
    row = -torch.minimum(inside, clipped)
    a = torch.where(inside <= clipped, -inside, torch.zeros_like(inside))
    out = {}
    if case["kl"]:
        d = state["ref"].double() - logprobs
        kl = torch.where(alive, torch.exp(d) - d - 1, torch.zeros_like(d))
        row = row + case["kl"] * kl
        a = a + case["kl"] * (1 - torch.exp(d))
        out["kl"] = kl.float()
    h = None
    if case["entropy"]:
        row = row - case["entropy"] * entropy
        h = -case["entropy"] * weights
        out["entropy"] = entropy.float()
    loss = torch.where(alive, row * weights, torch.zeros_like(row)).sum()
    grad = _gradient(z, e, total, targets, temperature, a * weights, h, entropy, state["logits"].dtype)
    out.update(loss=loss.float(), logprobs=logprobs.float(), grad_logits=grad)
    return out


def _plain_preference(state):
    case, targets, offsets = state["case"], state["targets"], state["offsets"]
    z, e, total, logprobs, _ = _statistics(state["logits"], targets, 1.0)
    n = offsets.numel() - 1
    alive = targets >= 0
    owner = torch.bucketize(torch.arange(targets.numel(), device=targets.device), offsets, right=True) - 1
    gain = torch.where(alive, logprobs - state["ref"].double(), torch.zeros_like(logprobs))
    inside = owner < n
    sums = torch.zeros(n + 1, dtype=torch.float64, device=targets.device).index_add_(0, owner, gain)[:n]
    share = torch.ones(n + 1, dtype=torch.float64, device=targets.device)
    if case["average"]:
        count = torch.zeros_like(share).index_add_(0, owner, alive.double())
        share = 1 / count.clamp(min=1)
    rewards = (case["beta"] * sums * share[:n]).view(-1, 2)
    h = rewards[:, 0] - rewards[:, 1]
    win, lose = 1 / (1 + torch.exp(-h)), 1 / (1 + torch.exp(h))
    pair = -(1 - case["smoothing"]) * torch.log(win) - case["smoothing"] * torch.log(lose)
    slope = (case["smoothing"] * win - (1 - case["smoothing"]) * lose) * (case["beta"] / h.numel())
    each = torch.cat([torch.stack([slope, -slope], dim=1).view(-1), slope.new_zeros(1)]) * share
    a = torch.where(alive & inside, each[owner], torch.zeros_like(logprobs))
    grad = _gradient(z, e, total, targets, 1.0, a, None, None, state["logits"].dtype)
    return {"loss": pair.mean().float(), "pair_loss": pair.float(), "rewards": rewards.float(),
            "logprobs": logprobs.float(), "grad_logits": grad}


# ----------------------------------------------------- the framework's calls
def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-inference_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import b200_sampler
    return b200_sampler


def _own_logprob(state):
    case, logits = state["case"], state["logits"]
    got = _framework().token_logprobs(logits, state["targets"], temperature=state["temperature"], entropy=case["entropy"])
    logprobs, entropy = got if case["entropy"] else (got, None)
    out = {"logprobs": logprobs.detach()}
    if case["entropy"]:
        out["entropy"] = entropy.detach()
    if case["grad"]:
        ends = [logprobs, entropy] if case["entropy"] else [logprobs]
        seeds = [state["grad_logprobs"], state["grad_entropy"]][:len(ends)]
        out["grad_logits"] = torch.autograd.grad(ends, [logits], seeds)[0]
    return out


def _own_policy(state):
    case = state["case"]
    got, grad = _framework().policy_loss_and_grad(
        state["logits"], state["targets"], state["old"], state["advantages"], ref_logprobs=state["ref"],
        weights=state["weights"], temperature=state["temperature"], clip_low=case["low"], clip_high=case["high"],
        kl_coef=case["kl"], entropy_coef=case["entropy"])
    out = {}
    if case["kl"]:
        out["kl"] = got.kl
    if case["entropy"]:
        out["entropy"] = got.entropy
    out.update(loss=got.loss, logprobs=got.logprobs, grad_logits=grad)
    return out


def _own_preference(state):
    case = state["case"]
    got, grad = _framework().preference_loss_and_grad(
        state["logits"], state["targets"], state["offsets"], ref_logprobs=state["ref"], beta=case["beta"],
        label_smoothing=case["smoothing"], average=case["average"])
    return {"loss": got.loss, "pair_loss": got.pair_loss, "rewards": got.rewards, "logprobs": got.logprobs,
            "grad_logits": grad}


def run(state):
    if own:
        return {"logprob": _own_logprob, "policy": _own_policy, "preference": _own_preference}[state["op"]](state)
    return {"logprob": _plain_logprob, "policy": _plain_policy, "preference": _plain_preference}[state["op"]](state)


def work(case):
    """The logits of the rows that hold a token are read once, and every row of the gradient is written once; the
    per-row numbers are added.  Operations: a scale, a shift, an exponential and a sum for each logit read, a product
    with the running sum for the entropy, and three more for each value of a gradient."""
    rows, vocab, size, op = _rows(case), case["vocab"], _BYTES[case["dtype"]], case["op"]
    held = rows - case.get("tail", 0)
    alive = held * (1 - case.get("padded", 0.0))
    grad = op != "logprob" or case["grad"]
    per_row = 8 + 4 + {"logprob": 8, "policy": 24, "preference": 4}[op]
    flops = 4 + (2 if case.get("entropy") else 0) + (3 if grad else 0)
    return {"bytes": alive * vocab * size + (rows * vocab * size if grad else 0) + rows * per_row,
            "flops": alive * vocab * flops}


# ------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The definitions in 64 bits, the gradients by differentiating them."""
    state = prepare(case, seed)
    x = state["logits"].detach().double()
    grad = case["op"] != "logprob" or case["grad"]
    x.requires_grad_(grad)
    targets, t = state["targets"], state["temperature"]
    t = t.double()[:, None] if torch.is_tensor(t) else t
    keep = targets >= 0
    z = x / t
    log_p = z - torch.logsumexp(z, dim=1, keepdim=True)
    logprobs = torch.where(keep, log_p.gather(1, targets.clamp(min=0)[:, None]).squeeze(1), 0.0)
    out, entropy = {}, None
    if case.get("entropy"):
        # a barred column has no probability and adds nothing
        entropy = torch.where(keep, -(log_p.exp() * log_p.masked_fill(log_p == -math.inf, 0.0)).sum(1), 0.0)
        out["entropy"] = entropy.detach()
    if case["op"] == "logprob":
        goal = (logprobs * state["grad_logprobs"].double()).sum()
        if entropy is not None:
            goal = goal + (entropy * state["grad_entropy"].double()).sum()
    elif case["op"] == "policy":
        ratio, advantage = (logprobs - state["old"].double()).exp(), state["advantages"].double()
        each = -torch.minimum(ratio * advantage, ratio.clamp(1 - case["low"], 1 + case["high"]) * advantage)
        if case["kl"]:
            d = state["ref"].double() - logprobs
            kl = torch.where(keep, torch.expm1(d) - d, 0.0)
            each = each + case["kl"] * kl
            out["kl"] = kl.detach()
        if entropy is not None:
            each = each - case["entropy"] * entropy
        goal = torch.where(keep, each * state["weights"].double(), 0.0).sum()
        out["loss"] = goal.detach()
    else:
        gain = torch.where(keep, logprobs - state["ref"].double(), 0.0)
        ends = state["offsets"]
        running = torch.cat([gain.new_zeros(1), gain.cumsum(0)])
        sums = running[ends[1:]] - running[ends[:-1]]
        if case["average"]:
            held = torch.cat([keep.new_zeros(1, dtype=torch.int64), keep.long().cumsum(0)])
            sums = sums / (held[ends[1:]] - held[ends[:-1]]).clamp(min=1)
        rewards = case["beta"] * sums.view(-1, 2)
        margin = rewards[:, 0] - rewards[:, 1]
        pair = (1 - case["smoothing"]) * torch.log1p((-margin).exp()) + case["smoothing"] * torch.log1p(margin.exp())
        goal = pair.mean()
        out.update(loss=goal.detach(), pair_loss=pair.detach(), rewards=rewards.detach())
    out["logprobs"] = logprobs.detach()
    if grad:
        out["grad_logits"] = torch.autograd.grad(goal, [x])[0]
    return out
