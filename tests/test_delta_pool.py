"""delta.step and the tensor that holds the pool of states: what autograd and strides make of it."""
import pytest
import torch

from accelerated_scan import delta
from test_delta import token_inputs


@pytest.mark.gpu
@pytest.mark.parametrize("view", [lambda t: t, lambda t: t[1:3], lambda t: t.view(4, 2, 16, 16)])
def test_step_counts_as_a_change_in_place(cuda_device, view):
    """An operation that saved the pool, or a view of it, for its backward must not differentiate with the new contents."""
    args = token_inputs(1, 2, 1, 2, 16, 16, torch.float32, cuda_device)
    pool = torch.randn(4, 2, 16, 16, device=cuda_device)
    weight = torch.ones(4, 2, 16, 16, device=cuda_device, requires_grad=True)
    loss = (weight * pool).sum()
    before = pool._version
    with torch.no_grad():
        delta.step(*args, view(pool), torch.tensor([0, 1], device=cuda_device))
    assert pool._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
def test_step_on_inference_tensors(cuda_device):
    """They have no version to count; the results are the same."""
    results = []
    for mode in (torch.inference_mode, torch.no_grad):
        with mode():
            args = token_inputs(2, 2, 1, 2, 16, 16, torch.float32, cuda_device)
            pool = torch.ones(2, 2, 16, 16, device=cuda_device)
            results.append([delta.step(*args, pool), pool])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    with torch.no_grad():
        delta.step(*args, results[0][1])                       # a pool made in inference mode, used outside of it


@pytest.mark.gpu
def test_no_rows_change_nothing(cuda_device):
    args = [t[:0] for t in token_inputs(3, 1, 1, 2, 16, 16, torch.float32, cuda_device)]
    pool = torch.ones(2, 2, 16, 16, device=cuda_device)
    before = pool._version
    delta.step(*args, pool)
    assert pool._version == before


@pytest.mark.gpu
@pytest.mark.parametrize("view", [lambda t: t.view(2, 1, 16, 16).transpose(0, 1), lambda t: t.as_strided((1, 2, 16, 16), (0, 256, 16, 1)),
                                  lambda t: t.as_strided((1, 2, 16, 16), (7, 256, 16, 1))])
@pytest.mark.parametrize("slots", [False, True])
def test_a_pool_of_one_state_has_any_first_stride(cuda_device, view, slots):
    args = token_inputs(4, 1, 1, 2, 16, 16, torch.float32, cuda_device)
    slots = torch.zeros(1, dtype=torch.int64, device=cuda_device) if slots else None
    plain = torch.randn(1, 2, 16, 16, device=cuda_device)
    odd = view(plain.clone())
    assert odd.shape == plain.shape and odd.stride(0) < 512
    want = delta.step(*args, plain, slots)
    assert torch.equal(delta.step(*args, odd, slots), want) and torch.equal(odd, plain)


@pytest.mark.gpu
def test_a_pool_without_states(cuda_device):
    """Every slot lies behind it, or is a padded row."""
    args = token_inputs(5, 2, 1, 2, 16, 16, torch.float32, cuda_device)
    out = delta.step(*args, torch.empty(0, 2, 16, 16, device=cuda_device), torch.tensor([0, -1], device=cuda_device))
    assert torch.isnan(out[0]).all() and (out[1] == 0).all()
