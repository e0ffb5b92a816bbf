"""Arguments of the operators on sampled tokens' logits that have to be refused
or taken as they are before anything is launched (no GPU needed)."""
import pytest
import torch

from b200_sampler import losses

X, T = torch.zeros(4, 10), torch.zeros(4, dtype=torch.int64)
F, OFFSETS = torch.zeros(4), torch.tensor([0, 2, 4])
CALLS = [lambda **kw: losses.token_logprobs(X, T, **kw), lambda **kw: losses.policy_loss(X, T, F, F, **kw),
         lambda **kw: losses.policy_loss_and_grad(X, T, F, F, **kw), lambda **kw: losses.preference_loss(X, T, OFFSETS, **kw),
         lambda **kw: losses.preference_loss_and_grad(X, T, OFFSETS, **kw)]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("temperature", [1e-50, 5e-46, 1e39])
def test_a_temperature_that_fp32_does_not_hold_is_refused(call, temperature):
    """1e-50 would become 0 on its way, and 0 stands for 1."""
    with pytest.raises(ValueError, match="temperature"):
        call(temperature=temperature)


def test_a_row_of_small_temperature_is_not_greedy():
    t = torch.tensor([1e-50, 0.0, 0.7, -1e-50], dtype=torch.float64)
    each = losses._rows(X, T, t)[2]
    assert each.dtype == torch.float32
    assert each.tolist() == [2.0 ** -149, 0.0, torch.tensor(0.7).item(), -2.0 ** -149]
