"""Arguments of the operators on sampled tokens' logits that have to be refused
or taken as they are before anything is launched (no GPU needed)."""
import os

import pytest
import torch

from b200_sampler import _lib, losses

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


# ------------------------------------------------------------------------ out
GRADS = [lambda x, out: losses.policy_loss_and_grad(x, T, F, F, out=out),
         lambda x, out: losses.preference_loss_and_grad(x, T, OFFSETS, out=out)]


@pytest.mark.parametrize("call", GRADS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("at", [10, 11, 12])
def test_out_beside_the_logits_in_the_same_rows_is_taken(call, dtype, at):
    """Columns of one buffer that do not overlap: what is refused here is the CPU's tensors, after out's checks."""
    buf = torch.zeros(4, 22, dtype=dtype)
    with pytest.raises(ValueError, match="CUDA"):
        call(buf[:, :10], buf[:, at:at + 10])
    with pytest.raises(ValueError, match="CUDA"):
        call(buf[:, at:at + 10], buf[:, :10])


@pytest.mark.parametrize("call", GRADS)
@pytest.mark.parametrize("first,second", [(0, 1), (0, 9), (9, 0), (3, 12)])
def test_out_over_some_of_the_logits_is_refused(call, first, second):
    buf = torch.zeros(5, 22)
    with pytest.raises(ValueError, match="overlap"):
        call(buf[:4, first:first + 10], buf[:4, second:second + 10])
    # the columns of the next rows
    with pytest.raises(ValueError, match="overlap"):
        call(buf[:4, first:first + 10], buf[1:, second:second + 10])
    # another stride: by their ranges
    with pytest.raises(ValueError, match="overlap"):
        call(buf[:4, first:first + 10], buf.view(-1)[:80].view(4, 20)[:, 10:])
    flat = torch.zeros(200)
    with pytest.raises(ValueError, match="overlap"):
        call(flat.as_strided((4, 10), (22, 1), first), flat.as_strided((4, 10), (22, 1), second + 22))


def test_out_behind_the_logits_across_the_end_of_a_row():
    """22 apart, 15 and 7 behind: the columns 15 to 24 reach into the next row's first 3, which are not among 5 to 14."""
    flat = torch.zeros(200)
    with pytest.raises(ValueError, match="CUDA"):
        GRADS[0](flat.as_strided((4, 10), (22, 1), 5), flat.as_strided((4, 10), (22, 1), 15))
    with pytest.raises(ValueError, match="overlap"):
        GRADS[0](flat.as_strided((4, 10), (22, 1), 2), flat.as_strided((4, 10), (22, 1), 15))


def test_out_of_a_single_row():
    """One row's stride says nothing, 0 as little as any other."""
    x, one, flat = torch.zeros(1, 10), torch.zeros(1), torch.zeros(40)
    t = torch.zeros(1, dtype=torch.int64)
    for stride in (0, 5, 22):
        a, b = flat.as_strided((1, 10), (stride, 1), 0), flat.as_strided((1, 10), (stride, 1), 10)
        with pytest.raises(ValueError, match="CUDA"):
            losses.policy_loss_and_grad(a, t, one, one, out=b)
        with pytest.raises(ValueError, match="overlap"):
            losses.policy_loss_and_grad(a, t, one, one, out=flat.as_strided((1, 10), (stride, 1), 9))


# ------------------------------------------------------------------- decode loop
def test_device_batch_scores_no_host_tensors():
    """Nothing reaches the C entry: a kernel must not be given an address of the host."""
    from b200_sampler import SamplingParams
    from b200_sampler.sampler import DeviceBatch

    class Library:
        def __getattr__(self, name):
            raise RuntimeError(name + " was called")

    class Stream:
        cuda_stream = 0
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    batch = DeviceBatch(None, [SamplingParams()] * 4, "cpu")
    batch.lib = Library()
    with pytest.raises(AssertionError):
        batch.logprobs(X, T, F, stream=Stream())


def test_device_batch_scores_on_its_own_device(monkeypatch):
    """With another device current, the call is made with the tensors' device current, on that one's stream."""
    from b200_sampler.sampler import DeviceBatch
    current, calls = [0], []

    class Tensor:
        device, is_cuda, shape = torch.device("cuda", 1), True, (4, 10)

        def __init__(self, dtype):
            self.dtype = dtype

        def stride(self, i):
            return (10, 1)[i]

        def numel(self):
            return 4

        def is_contiguous(self):
            return True

        def data_ptr(self):
            return 1

    class Device:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    class Library:
        def ns_token_logprobs(self, *args):
            calls.append((current[0], args[-1]))
            return 0

    class Stream:
        cuda_stream = 7
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    batch = DeviceBatch.__new__(DeviceBatch)
    batch.batch, batch.device, batch.params, batch.lib = 4, Tensor.device, Tensor(torch.float32), Library()
    assert batch.logprobs(Tensor(torch.float32), Tensor(torch.int64), Tensor(torch.float32)) == 0
    assert calls == [(1, 7)] and current == [0]


@pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
def test_the_debug_entry_wants_a_row():
    args = [1, 0, 4, 10, 10, 1, None, 1.0, 1, None, 1, None, 0.2, 0.2, 0.0, 0.0, 1, 1, 1, None, None, 1, 1, 2, 10]
    lib = _lib.load()
    assert lib.ns_policy_loss_debug(*args, -1, None) == _lib.NS_ERR_INVALID_ARGUMENT
    args[3] = 0
    assert lib.ns_policy_loss_debug(*args, 1, None) == _lib.NS_ERR_INVALID_ARGUMENT
