"""Columns of V are independent of one another: a call gives its columns the bits that a wider call gives them, whichever way the
results take to memory (whole tiles by copies, or element by element where V is no multiple of 8)."""
import pytest
import torch

from accelerated_scan import delta
from test_delta import inputs


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V,wide", [(68, 72), (61, 64), (130, 136), (127, 128), (1, 8)])
@pytest.mark.parametrize("lengths", [None, [300, 7, 0, 393]])
def test_narrow_against_wide(cuda_device, lengths, V, wide, dtype):
    B, T, n = (2, 700, 2) if lengths is None else (1, 700, 4)
    args = inputs(V, B, T, 1, 2, 64, wide, dtype, cuda_device, n=n)
    starts = None if lengths is None else torch.tensor([0] + lengths).cumsum(0).to(cuda_device)
    d_out = torch.randn(B, T, 2, wide, device=cuda_device).to(dtype)
    d_s = torch.randn(n, 2, 64, wide, device=cuda_device)

    def train(cols):
        q, k, v, g, b, s0 = args
        leaves = [q, k, v[..., :cols].contiguous(), g, b, s0[..., :cols].contiguous()]
        leaves = [t.detach().requires_grad_(True) for t in leaves]
        out, s = delta.scan(*leaves, seq_starts=starts)
        grads = torch.autograd.grad([out, s], leaves, [d_out[..., :cols].contiguous(), d_s[..., :cols].contiguous()])
        return [t.detach() for t in (out, s, grads[2], grads[5])]

    want = train(wide)
    for _ in range(3):
        for a, b in zip(train(V), want):
            assert torch.equal(a, b[..., :V])
