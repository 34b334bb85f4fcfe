"""Forward-mode derivatives: no operator has them, and none drops a tangent."""
import pytest
import torch
from torch.autograd import forward_ad

from accelerated_scan import delta, norm
from test_delta import inputs, token_inputs

REFUSED = pytest.raises(NotImplementedError, match="forward-mode|jvp")


def duals(args):
    """The arguments with a tangent on one of them, one after the other."""
    for i, t in enumerate(args):
        if t is not None:
            yield [forward_ad.make_dual(x, torch.ones_like(x)) if j == i else x for j, x in enumerate(args)]


def norm_arguments(device):
    return [torch.randn(4, 16, device=device) for _ in range(3)] + [torch.ones(16, device=device) for _ in range(3)]


def call_norm(x, residual, gate, post, scale, pre):
    return norm.residual_norm(x, residual, post_weight=post, gate=gate, scale=scale, pre_weight=pre)


def check(device):
    with forward_ad.dual_level():
        for args in duals(inputs(0, 2, 8, 1, 2, 16, 16, torch.float32, device)):
            with REFUSED:
                delta.scan(*args)
        state = torch.zeros(2, 2, 16, 16, device=device)
        for args in duals([*token_inputs(0, 2, 1, 2, 16, 16, torch.float32, device), state]):
            with REFUSED:
                delta.step(*args)
        assert (state == 0).all()                               # refused before anything was written
        for args in duals(norm_arguments(device)):
            with REFUSED:
                call_norm(*args)
        x = norm_arguments(device)[0]
        with REFUSED:
            norm.gated_norm(x, forward_ad.make_dual(x, x), x[0])


def test_refused():
    check("cpu")                                                # before the tensors' device is looked at


@pytest.mark.gpu
def test_refused_on_the_gpu(cuda_device):
    check(cuda_device)
    args = inputs(0, 2, 8, 1, 2, 16, 16, torch.float32, cuda_device)
    args[0].requires_grad_(True)                                # the call that goes through the autograd function
    with forward_ad.dual_level():
        for dual in duals(args):
            with REFUSED:
                delta.scan(*dual)
        plain = delta.scan(*args)                               # without a tangent an open level changes nothing
    for a, b in zip(plain, delta.scan(*args)):
        assert torch.equal(a, b)
    with forward_ad.dual_level():
        h, y = call_norm(*norm_arguments(cuda_device))
    assert torch.isfinite(h).all() and torch.isfinite(y).all()
