"""The same inputs give the same bits while tiles are read, handed back and written over: V in many slabs, few and many heads,
and d_log_gates, whose share of the state is summed from tiles by threads beside the tensor cores, near the definition chunk by
chunk."""
import pytest
import torch

from accelerated_scan import delta, norm
from test_delta import TOL, inputs, reference

LENGTHS = [37, 1, 64, 5, 90, 66, 0, 23] * 8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hk,H,K,V", [(2, 8, 128, 520), (4, 8, 64, 300), (4, 8, 128, 136), (1, 1, 128, 200), (4, 16, 128, 128), (2, 2, 16, 1024)])
def test_scan(cuda_device, Hk, H, K, V, dtype):
    T, n = sum(LENGTHS), len(LENGTHS)
    args = inputs(V, 1, T, Hk, H, K, V, dtype, cuda_device, n=n)
    starts = torch.tensor([0] + LENGTHS).cumsum(0).to(cuda_device)
    leaves = [t.requires_grad_(True) for t in args]
    d_out, d_s = torch.randn(1, T, H, V, device=cuda_device).to(dtype), torch.randn(n, H, K, V, device=cuda_device)
    first = None
    for _ in range(25):
        got = torch.autograd.grad(delta.scan(*args, seq_starts=starts), leaves, [d_out, d_s])
        first = first or got
        for a, b in zip(got, first):
            assert torch.equal(a, b)
    want, want_s = reference(*args, lengths=LENGTHS)
    want_g, = torch.autograd.grad([want, want_s], leaves[3], [d_out.double(), d_s.double()])
    # every gate within its bound of the largest: a chunk's sum that took another tile's values is off by far more
    assert ((first[3].double() - want_g).abs() <= 2 * TOL[dtype] * want_g.abs().max()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 1024, 4096, 8192])
def test_norm(cuda_device, dtype, D):
    rows = 3000
    x, r, z, dh, dy = (torch.randn(rows, D, device=cuda_device).to(dtype) for _ in range(5))
    w = torch.rand(D, device=cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, r, z, w)]
    first = None
    for _ in range(10):
        ends = norm.residual_norm(x, r, post_weight=w, gate=z, pre_weight=w)
        got = [t.detach() for t in ends] + list(torch.autograd.grad(ends, leaves, [dh, dy]))
        first = first or got
        for a, b in zip(got, first):
            assert torch.equal(a, b)
