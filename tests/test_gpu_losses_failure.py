"""What a policy loss leaves behind when a wait inside its kernel runs out: NaN
in every row that its blocks had not done, and in the loss, never memory as it
was.  ns_policy_loss_debug lets one wait count as run out; the blocks that wait
for those that gave up run into the kernel's own limit (200 ms) and return."""
import time

import pytest
import torch

from b200_sampler import _lib
from b200_sampler.losses import _head

pytestmark = pytest.mark.gpu


def _args(x, targets, old, adv, out, entropy):
    n = x.shape[0]
    r = {"loss": torch.full((1,), 5.0, device="cuda"), "grad": out}
    for name, size in (("row_loss", n), ("logprobs", n), ("entropy", n), ("stats", 2 * n), ("row_grad", 2 * n)):
        r[name] = torch.full((size,), 5.0, device="cuda")
    args = (*_head(x, targets, None, 1.0), old.data_ptr(), None, adv.data_ptr(), None, 0.2, 0.2, 0.0, entropy,
            r["loss"].data_ptr(), r["row_loss"].data_ptr(), r["logprobs"].data_ptr(),
            r["entropy"].data_ptr() if entropy else None, None, r["stats"].data_ptr(), r["row_grad"].data_ptr(),
            out.data_ptr(), out.stride(0))
    return r, args


@pytest.mark.parametrize("rows,vocab,dtype", [
    (1000, 15000, torch.bfloat16),      # three blocks an SM, rows of one block
    (500, 64007, torch.float16),        # rows of two
    (90, 151936, torch.float32),        # of eight
    (400, 100003, torch.bfloat16),      # a block an SM
    (20, 170000, torch.bfloat16)])      # clusters of one row each
@pytest.mark.parametrize("entropy,in_place", [(0.0, False), (0.01, True)])
def test_rows_left_over_are_nan(rows, vocab, dtype, entropy, in_place):
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    g = torch.Generator("cuda").manual_seed(rows)
    x = (torch.randn(rows, vocab, device="cuda", generator=g) * 2).to(dtype)
    targets = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    targets[torch.rand(rows, device="cuda", generator=g) < 0.2] = -1
    old, adv = torch.full((rows,), -12.0, device="cuda"), torch.ones(rows, device="cuda")
    alive = targets >= 0
    where = int(alive.nonzero()[len(alive.nonzero()) // 2])
    want, args = _args(x, targets, old, adv, torch.full_like(x, 5.0), entropy)
    assert lib.ns_policy_loss(*args, stream) == 0
    z = x.clone()
    got, args = _args(z, targets, old, adv, z if in_place else torch.full_like(x, 5.0), entropy)
    t0 = time.monotonic()
    assert lib.ns_policy_loss_debug(*args, where, stream) == 0
    torch.cuda.synchronize()
    assert time.monotonic() - t0 < 20
    assert torch.isnan(got["loss"]).all() and torch.isfinite(want["loss"]).all()
    void = torch.isnan(got["row_loss"])
    assert void[where] and not void[~alive].any()
    assert void.sum() <= rows // 4 + 1            # the other blocks' rows are done
    assert torch.isnan(got["grad"][void]).all()
    assert torch.equal(got["grad"][~void], want["grad"][~void]) and (got["grad"][~alive] == 0).all()
    for name in ("row_loss", "logprobs") + (("entropy",) if entropy else ()):
        assert torch.isnan(got[name][void]).all() and torch.equal(got[name][~void], want[name][~void]), name
    for name in ("stats", "row_grad"):
        a, b = (r[name].view(rows, 2) if name == "stats" else r[name].view(2, rows).t() for r in (got, want))
        assert torch.isnan(a[void]).all() and torch.equal(a[~void], b[~void]), name
    # and the next call is none the worse
    again, args = _args(x, targets, old, adv, torch.full_like(x, 5.0), entropy)
    assert lib.ns_policy_loss(*args, stream) == 0
    for name in ("loss", "row_loss", "logprobs", "grad"):
        assert torch.equal(again[name], want[name]), name


def test_rows_that_are_not_held_have_no_waits():
    x = torch.randn(6, 1000, device="cuda")
    targets, f = torch.arange(6, device="cuda"), torch.full((6,), -6.0, device="cuda")
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    want, args = _args(x, targets, f, f, torch.empty_like(x), 0.0)
    assert lib.ns_policy_loss(*args, stream) == 0
    got, args = _args(x, targets, f, f, torch.empty_like(x), 0.0)
    assert lib.ns_policy_loss_debug(*args, 2, stream) == 0
    assert torch.equal(got["grad"], want["grad"]) and torch.equal(got["loss"], want["loss"])
