"""Calls of the operators on sampled tokens' logits that their documentation
allows and that are easily got wrong: where the gradient lies."""
import pytest
import torch

from b200_sampler import policy_loss_and_grad, preference_loss_and_grad

pytestmark = pytest.mark.gpu


def _normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1003, 32000])
@pytest.mark.parametrize("gap", [0, 1])
def test_gradient_beside_the_logits_in_one_buffer(dtype, vocab, gap):
    rows = 21
    x = (_normal(1, rows, vocab) * 3).to(dtype).cuda()
    targets = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(2)).cuda()
    old, adv, offsets = _normal(3, rows).cuda() - 8, _normal(4, rows).cuda(), torch.tensor([0, 8, 21], device="cuda")
    for call in (lambda z, out: policy_loss_and_grad(z, targets, old, adv, out=out),
                 lambda z, out: preference_loss_and_grad(z, targets, offsets, out=out)):
        buf = torch.full((rows, 2 * vocab + gap), 5.0, dtype=dtype, device="cuda")
        z, out = buf[:, :vocab], buf[:, vocab + gap:]
        z.copy_(x)
        # the same logits: rows on another 16-byte boundary are added up in another order
        want, got = call(z, None)[1], call(z, out)[1]
        assert got.data_ptr() == out.data_ptr() and torch.equal(out, want) and torch.equal(z, x)
        assert (buf[:, vocab:vocab + gap] == 5).all()
