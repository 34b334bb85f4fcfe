"""Norms whose saved tensors come back as other ones (offloaded, copied): the same bits."""
import pytest
import torch

from accelerated_scan import norm
from test_norm import call, inputs


class Columns(torch.autograd.graph.saved_tensors_hooks):
    """Saved tensors come back with another order in memory: rows as columns, vectors strided."""
    def __init__(self):
        super().__init__(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else torch.stack([t, t], -1)[..., 0])


class Odd(torch.autograd.graph.saved_tensors_hooks):
    """... at odd addresses, as slices of wider ones."""
    def __init__(self):
        def unpack(t):
            wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
            wide[..., 1:-2] = t
            return wide[..., 1:-2]
        super().__init__(lambda t: t, unpack)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(3, 40, 128), (21, 2048), (7, 1), (5, 130)])
@pytest.mark.parametrize("hooks", [torch.autograd.graph.save_on_cpu, Columns, Odd])
def test_gradients_under_saved_tensor_hooks(cuda_device, hooks, shape, dtype):
    args = inputs(5, shape, dtype, dtype, cuda_device)
    args[1] = args[1][:1].expand_as(args[1])                    # one row of residuals for all
    leaves = [t.requires_grad_(True) for t in args]
    ends = call(*args, "silu")
    d = [torch.randn_like(t) for t in ends]
    want = torch.autograd.grad(ends, leaves, d)
    with hooks():
        ends = call(*args, "silu")
    got = torch.autograd.grad(ends, leaves, d)
    for name, a, b in zip(("x", "residual", "gate", "post", "scale", "pre"), got, want):
        if hooks is Odd and shape[-1] % 8 == 0:
            # element by element the sums run in another order: each result within a rounding and 4 x 16 x 2^-24 of the exact one
            tol = torch.finfo(dtype).eps + 128 * 2.0 ** -24
            assert (a.double() - b.double()).norm() <= tol * b.double().norm(), name
        else:
            assert torch.equal(a, b), name
