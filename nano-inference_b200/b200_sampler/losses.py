"""Scores of sampled tokens and the losses that train on them.

    token_logprobs(logits, targets)        log-probabilities (and entropies), differentiable
    policy_loss(logits, targets, ...)      clipped policy loss with a KL term, differentiable
    preference_loss(logits, targets, ...)  loss on pairs of sequences, differentiable

``policy_loss_and_grad`` and ``preference_loss_and_grad`` return the loss
together with dloss/dlogits, without a graph: the gradient may take the logits'
place (``out=logits``), and the policy loss computes both from one reading of
the logits.  They are also the calls to capture in a CUDA graph: they allocate,
launch and return, where a captured ``backward()`` has torch's own rules.

One row of ``logits`` [rows, vocab] (fp32, bf16 or fp16, any row stride) holds
one token, and ``targets`` (int64 [rows]) its id: what ``B200Sampler`` draws,
as it is.  A negative target marks a row without a token (padding, a prompt
position, the status of a failed draw): its logits are not read, its numbers
and its gradient are 0.  A target past the vocabulary, a row that holds NaN,
+inf or nothing but -inf, and a temperature that is negative or not finite give
NaN.  ``temperature`` is one number or fp32 [rows]; 0 (a greedy row) stands for
1.  Penalties, top-k and top-p do not enter: the distribution is
softmax(logits / temperature).

Everything runs asynchronously on the current stream of the logits' device, in
the kernels behind ``include/ns_losses.h``; there is no CPU fallback.  The
other inputs are constants: no gradient reaches them.  The reference has no
counterpart (its sampler returns ids alone, ``sampling/sampler.py:36-91``).
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.NS_DTYPE_F32, torch.bfloat16: _lib.NS_DTYPE_BF16,
           torch.float16: _lib.NS_DTYPE_F16}

Temperature = Union[float, torch.Tensor]
_LEAST = 2.0 ** -149      # of fp32's values above 0


class PolicyLoss(NamedTuple):
    loss: torch.Tensor                  # fp32 scalar
    row_loss: torch.Tensor              # fp32 [rows], before the weights
    logprobs: torch.Tensor              # fp32 [rows]
    entropy: Optional[torch.Tensor]     # fp32 [rows], when entropy_coef is not 0
    kl: Optional[torch.Tensor]          # fp32 [rows], when there are ref_logprobs


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor                  # fp32 scalar
    pair_loss: torch.Tensor             # fp32 [pairs]
    rewards: torch.Tensor               # fp32 [pairs, 2]: chosen, rejected
    logprobs: torch.Tensor              # fp32 [rows]


# ------------------------------------------------------------------ arguments
def _rows(logits: torch.Tensor, targets: torch.Tensor, temperature: Temperature):
    """The checked logits (rows in place when their stride allows it), targets
    and temperature: (logits, targets, temperature tensor or None, number)."""
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("expected [rows, vocab] logits")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"unsupported logits dtype {logits.dtype}")
    n, vocab = logits.shape
    if logits.stride(1) != 1 or (n > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    if targets.dtype != torch.int64:
        raise TypeError("targets must be int64")
    _check("targets", targets, n, logits.device)
    if isinstance(temperature, torch.Tensor):
        each = _vector("temperature", temperature, n, logits.device)
        if temperature.dtype is torch.float64:
            # what fp32 rounds to 0 is no greedy row: its least value stands for it
            least = torch.copysign(torch.full_like(temperature, _LEAST), temperature).float()
            each = torch.where((each == 0) & (temperature != 0), least, each)
        return logits, targets.contiguous(), each, 1.0
    temperature = float(temperature)
    rounded = ctypes.c_float(temperature).value
    if not 0.0 <= rounded < math.inf or (rounded == 0.0 and temperature != 0.0):
        raise ValueError("temperature must be finite and not negative, and 0 or at least 1e-45 (it is held in fp32)")
    return logits, targets.contiguous(), None, temperature


def _check(name: str, t: torch.Tensor, n: int, device: torch.device) -> None:
    if t.device != device:
        raise ValueError(f"{name} must be on the logits' device")
    if t.shape != (n,):
        raise ValueError(f"{name} must have one value per row")


def _vector(name: str, t: Optional[torch.Tensor], n: int, device: torch.device) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype is not torch.float32:
        if not t.is_floating_point():
            raise TypeError(f"{name} must be floating point")
        t = t.detach().float()
    _check(name, t, n, device)
    return t.contiguous()


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stride(t: torch.Tensor) -> int:
    # the stride of a single row says nothing
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _call(name: str, device: torch.device, *args) -> None:
    """One C call on the current stream of `device`, which is current meanwhile."""
    if device.type != "cuda":
        raise ValueError("the logits must be on a CUDA device (there is no CPU fallback)")
    fn = getattr(_lib.load(), name)
    index = device.index
    if index == torch._C._cuda_getDevice():
        # the stream's handle alone: torch.cuda.current_stream makes an object of it, 4 us
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != _lib.NS_OK:
        raise RuntimeError(f"{name} failed: {_lib.status_string(rc)}")


def _head(logits, targets, temperature, temperature_all):
    return (logits.data_ptr(), _DTYPES[logits.dtype], logits.shape[0], logits.shape[1], _stride(logits),
            targets.data_ptr(), _ptr(temperature), temperature_all)


def _new(logits: torch.Tensor, *shape: int) -> torch.Tensor:
    return torch.empty(shape, dtype=torch.float32, device=logits.device)


def _parts(logits: torch.Tensor, *sizes: int):
    """fp32 vectors of these sizes from one allocation."""
    return torch.empty(sum(sizes), dtype=torch.float32, device=logits.device).split_with_sizes(sizes)


def _like(logits: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


def _grad_out(logits: torch.Tensor, given: torch.Tensor, out: Optional[torch.Tensor]) -> torch.Tensor:
    """The gradient's tensor: a new one, or the caller's after its checks.
    ``given`` is the caller's logits, ``logits`` what the kernels read."""
    if out is None:
        return _like(logits)
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out must have the logits' shape, dtype and device")
    if out.stride(1) != 1 or (out.shape[0] > 1 and out.stride(0) < out.shape[1]):
        raise ValueError("out's rows must be contiguous and must not overlap")
    if not (out.data_ptr() == given.data_ptr() and _stride(out) == _stride(given)) and _overlap(out, given):
        raise ValueError("out may be the logits themselves, and must not overlap them otherwise")
    return out


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors [rows, vocab] of one type share an element.  Of
    different strides, whether their ranges do."""
    def span(t):
        if t.numel() == 0:
            return t.data_ptr(), t.data_ptr()
        last = sum((n - 1) * abs(s) for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    if not (a0 < b1 and b0 < a1):
        return False
    if a.shape[0] == 1 or a.stride() != b.stride() or a.stride(1) != 1:
        return True
    # side by side in one buffer's rows: how far the one's columns lie behind the other's
    apart = (a0 - b0) % (a.stride(0) * a.element_size())
    width = a.shape[1] * a.element_size()
    return apart < width or apart + width > a.stride(0) * a.element_size()


def _gradient(logits, targets, temperature, temperature_all, stats, entropy, a, h):
    out = _like(logits)
    _call("ns_token_logprobs_grad", logits.device, *_head(logits, targets, temperature, temperature_all),
          stats.data_ptr(), _ptr(entropy), _ptr(a), _ptr(h), out.data_ptr(), _stride(out))
    return out


# ------------------------------------------------------------ log-probabilities
def _logprobs_forward(logits, targets, temperature, temperature_all, entropy, stats):
    n = logits.shape[0]
    logprobs = _new(logits, n)
    ent = _new(logits, n) if entropy else None
    st = _new(logits, n, 2) if stats else None
    _call("ns_token_logprobs", logits.device, *_head(logits, targets, temperature, temperature_all),
          logprobs.data_ptr(), _ptr(ent), _ptr(st))
    return logprobs, ent, st


class _Last(torch.autograd.Function):
    """Its argument, whose derivative is refused."""

    @staticmethod
    def forward(ctx, grad):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("token_logprobs, policy_loss and preference_loss are differentiable once: "
                           "their gradients have no derivatives")


class _Once(torch.autograd.Function):
    """A function whose ``gradient`` is not differentiable again, and says so
    when a graph of the backward pass is asked for."""

    @classmethod
    def backward(cls, ctx, *grads):
        if not torch.is_grad_enabled():
            return cls.gradient(ctx, *grads)
        with torch.no_grad():
            out, *rest = cls.gradient(ctx, *grads)
        return (out if out is None else _Last.apply(out.requires_grad_()), *rest)


class _TokenLogprobs(_Once):
    @staticmethod
    def forward(ctx, logits, targets, temperature, temperature_all, entropy):
        ctx.set_materialize_grads(False)
        logprobs, ent, stats = _logprobs_forward(logits, targets, temperature, temperature_all, entropy, True)
        ctx.temperature_all = temperature_all
        ctx.save_for_backward(logits, targets, temperature, stats, ent)
        return (logprobs, ent) if entropy else logprobs

    @staticmethod
    def gradient(ctx, a, h=None):
        logits, targets, temperature, stats, ent = ctx.saved_tensors
        a = None if a is None else a.contiguous()
        h = None if h is None else h.contiguous()
        if a is None and h is None:
            return None, None, None, None, None
        out = _gradient(logits, targets, temperature, ctx.temperature_all, stats, ent, a, h)
        return out, None, None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, temperature: Temperature = 1.0,
                   entropy: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """ln softmax(logits / temperature)[target] of every row (fp32 [rows]) and,
    with ``entropy``, the rows' entropies in nats: ``(logprobs, entropy)``.
    Differentiable with respect to the logits; the backward pass reads them
    again (they must not have changed) and writes the gradient in their dtype."""
    logits, targets, temperature, t_all = _rows(logits, targets, temperature)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TokenLogprobs.apply(logits, targets, temperature, t_all, bool(entropy))
    logprobs, ent, _ = _logprobs_forward(logits, targets, temperature, t_all, entropy, False)
    return (logprobs, ent) if entropy else logprobs


# ----------------------------------------------------------------- policy loss
def _policy(logits, targets, old_logprobs, advantages, ref_logprobs, weights, temperature, clip_low, clip_high,
            kl_coef, entropy_coef):
    logits, targets, temperature, t_all = _rows(logits, targets, temperature)
    n, device = logits.shape[0], logits.device
    if not 0.0 <= clip_low <= 1.0 or not 0.0 <= clip_high < math.inf:
        raise ValueError("clip_low must lie in [0, 1] and clip_high must be finite and not negative")
    if not math.isfinite(kl_coef) or not math.isfinite(entropy_coef):
        raise ValueError("kl_coef and entropy_coef must be finite")
    if kl_coef != 0.0 and ref_logprobs is None:
        raise ValueError("a KL term needs ref_logprobs")
    if old_logprobs is None or advantages is None:
        raise ValueError("old_logprobs and advantages are needed")
    vectors = (_vector("old_logprobs", old_logprobs, n, device), _vector("ref_logprobs", ref_logprobs, n, device),
               _vector("advantages", advantages, n, device), _vector("weights", weights, n, device))
    return logits, targets, temperature, t_all, vectors, (clip_low, clip_high, kl_coef, entropy_coef)


def _policy_forward(logits, targets, temperature, t_all, vectors, coefs, grad):
    """(PolicyLoss, the backward pass's numbers: stats [rows, 2], coefficients [2, rows], entropies);
    writes dloss/dlogits to ``grad`` when there is one."""
    n = logits.shape[0]
    has_entropy, has_kl = coefs[3] != 0.0, vectors[1] is not None
    loss = _new(logits)              # by itself: a part of several may not be changed in place
    row_loss, logprobs, *rest = _parts(logits, n, n, *[n] * has_kl)
    kl = rest[0] if has_kl else None
    back = _new(logits, (4 + has_entropy) * n)      # by itself: the caller may change the others before the backward pass
    entropy = back[4 * n:] if has_entropy else None
    stats = back.data_ptr()
    _call("ns_policy_loss", logits.device, *_head(logits, targets, temperature, t_all), *map(_ptr, vectors),
          *coefs, loss.data_ptr(), row_loss.data_ptr(), logprobs.data_ptr(), _ptr(entropy), _ptr(kl),
          stats, stats + 8 * n, _ptr(grad), 0 if grad is None else _stride(grad))
    return PolicyLoss(loss, row_loss, logprobs, entropy, kl), back


class _PolicyLoss(_Once):
    @staticmethod
    def forward(ctx, logits, targets, temperature, t_all, vectors, coefs):
        ctx.set_materialize_grads(False)
        got, back = _policy_forward(logits, targets, temperature, t_all, vectors, coefs, None)
        ctx.t_all, ctx.has_entropy = t_all, got.entropy is not None
        ctx.save_for_backward(logits, targets, temperature, back)
        ctx.mark_non_differentiable(*(t for t in got[1:] if t is not None))
        return tuple(got)

    @staticmethod
    def gradient(ctx, g, *_):
        if g is None:
            return None, None, None, None, None, None
        logits, targets, temperature, back = ctx.saved_tensors
        n = logits.shape[0]
        coefs = back[2 * n:4 * n] * g
        entropy, h = (back[4 * n:], coefs[n:]) if ctx.has_entropy else (None, None)
        out = _gradient(logits, targets, temperature, ctx.t_all, back, entropy, coefs, h)
        return out, None, None, None, None, None


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor, *,
                ref_logprobs: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
                temperature: Temperature = 1.0, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_coef: float = 0.0, entropy_coef: float = 0.0) -> PolicyLoss:
    """Clipped policy loss: the weighted sum over the rows that hold a token of

        -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef kl - entropy_coef entropy

    with r = exp(logprob - old_logprob), A the row's advantage and kl =
    exp(ref - logprob) - (ref - logprob) - 1.  ``weights`` (fp32 [rows]; 1 /
    rows without them) say how rows are averaged; a row of weight 0 counts as
    holding no token.  ``loss`` is differentiable with respect to the logits;
    the other fields are not."""
    args = _policy(logits, targets, old_logprobs, advantages, ref_logprobs, weights, temperature, clip_low, clip_high,
                   kl_coef, entropy_coef)
    if torch.is_grad_enabled() and logits.requires_grad:
        return PolicyLoss(*_PolicyLoss.apply(*args))
    return _policy_forward(*args, None)[0]


def policy_loss_and_grad(logits: torch.Tensor, targets: torch.Tensor, old_logprobs: torch.Tensor,
                         advantages: torch.Tensor, *, ref_logprobs: Optional[torch.Tensor] = None,
                         weights: Optional[torch.Tensor] = None, temperature: Temperature = 1.0,
                         clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                         entropy_coef: float = 0.0,
                         out: Optional[torch.Tensor] = None) -> Tuple[PolicyLoss, torch.Tensor]:
    """``policy_loss`` and its gradient in one call, outside autograd:
    ``(PolicyLoss, dloss/dlogits)``.  ``out`` takes the gradient; it may be
    ``logits``, whose values are then gone."""
    args = _policy(logits, targets, old_logprobs, advantages, ref_logprobs, weights, temperature, clip_low, clip_high,
                   kl_coef, entropy_coef)
    grad = _grad_out(args[0], logits, out)
    got = _policy_forward(*args, grad)[0]
    if out is not None:
        torch.autograd.graph.increment_version(out)
    return got, grad


# ------------------------------------------------------------- preference loss
def _preference(logits, targets, seq_offsets, ref_logprobs, beta, label_smoothing, average, temperature):
    logits, targets, temperature, t_all = _rows(logits, targets, temperature)
    if seq_offsets.dtype != torch.int64 or seq_offsets.dim() != 1 or seq_offsets.shape[0] % 2 != 1:
        raise ValueError("seq_offsets must be int64 [2 * pairs + 1]")
    if seq_offsets.device != logits.device:
        raise ValueError("seq_offsets must be on the logits' device")
    if not math.isfinite(beta) or not 0.0 <= label_smoothing < 1.0:
        raise ValueError("beta must be finite and label_smoothing lie in [0, 1)")
    ref = _vector("ref_logprobs", ref_logprobs, logits.shape[0], logits.device)
    return logits, targets, temperature, t_all, seq_offsets.contiguous(), ref, (beta, label_smoothing, int(bool(average)))


def _preference_forward(logits, targets, temperature, t_all, offsets, ref, coefs, grad):
    n, pairs = logits.shape[0], offsets.shape[0] // 2
    loss = _new(logits)
    pair_loss, rewards, logprobs = _parts(logits, pairs, 2 * pairs, n)
    rewards = rewards.view(pairs, 2)
    back = _new(logits, 3 * n)
    stats = back.data_ptr()
    _call("ns_preference_loss", logits.device, *_head(logits, targets, temperature, t_all), offsets.data_ptr(), pairs,
          _ptr(ref), *coefs, loss.data_ptr(), pair_loss.data_ptr(), rewards.data_ptr(), logprobs.data_ptr(),
          stats, stats + 8 * n, _ptr(grad), 0 if grad is None else _stride(grad))
    return PreferenceLoss(loss, pair_loss, rewards, logprobs), back


class _PreferenceLoss(_Once):
    @staticmethod
    def forward(ctx, logits, targets, temperature, t_all, offsets, ref, coefs):
        ctx.set_materialize_grads(False)
        got, back = _preference_forward(logits, targets, temperature, t_all, offsets, ref, coefs, None)
        ctx.t_all = t_all
        ctx.save_for_backward(logits, targets, temperature, back)
        ctx.mark_non_differentiable(*got[1:])
        return tuple(got)

    @staticmethod
    def gradient(ctx, g, *_):
        if g is None:
            return None, None, None, None, None, None, None
        logits, targets, temperature, back = ctx.saved_tensors
        out = _gradient(logits, targets, temperature, ctx.t_all, back, None, back[2 * logits.shape[0]:] * g, None)
        return out, None, None, None, None, None, None


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, seq_offsets: torch.Tensor, *,
                    ref_logprobs: Optional[torch.Tensor] = None, beta: float = 0.1, label_smoothing: float = 0.0,
                    average: bool = False, temperature: Temperature = 1.0) -> PreferenceLoss:
    """Preference loss on pairs of sequences packed row after row: sequence s
    holds rows ``seq_offsets[s]`` to ``seq_offsets[s + 1]`` (int64 [2 pairs +
    1], ascending, on the device), 2 p is pair p's chosen sequence and 2 p + 1
    the rejected one.  A sequence's reward is beta times the sum (``average``:
    the mean) of logprob - ref_logprob over its tokens, and a pair's loss is

        -(1 - label_smoothing) ln sigmoid(h) - label_smoothing ln sigmoid(-h)

    with h the chosen reward less the rejected one.  ``ref_logprobs`` (fp32
    [rows], ``token_logprobs`` of the reference model) counts as 0 when absent.
    Rows outside every sequence count as holding no token.  ``loss``, the mean
    over the pairs, is differentiable with respect to the logits; the other
    fields are not."""
    args = _preference(logits, targets, seq_offsets, ref_logprobs, beta, label_smoothing, average, temperature)
    if torch.is_grad_enabled() and logits.requires_grad:
        return PreferenceLoss(*_PreferenceLoss.apply(*args))
    return _preference_forward(*args, None)[0]


def preference_loss_and_grad(logits: torch.Tensor, targets: torch.Tensor, seq_offsets: torch.Tensor, *,
                             ref_logprobs: Optional[torch.Tensor] = None, beta: float = 0.1,
                             label_smoothing: float = 0.0, average: bool = False, temperature: Temperature = 1.0,
                             out: Optional[torch.Tensor] = None) -> Tuple[PreferenceLoss, torch.Tensor]:
    """``preference_loss`` and its gradient in one call, outside autograd:
    ``(PreferenceLoss, dloss/dlogits)``.  ``out`` takes the gradient; it may be
    ``logits``, whose values are then gone."""
    args = _preference(logits, targets, seq_offsets, ref_logprobs, beta, label_smoothing, average, temperature)
    grad = _grad_out(args[0], logits, out)
    got = _preference_forward(*args, grad)[0]
    if out is not None:
        torch.autograd.graph.increment_version(out)
    return got, grad
