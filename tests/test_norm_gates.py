"""The gates of the norms, element by element, in relative error.

With u = 2^-24, for fp32: 2^t to 4 u (the instruction's 2^-22) and one rounding of its correction, 1 + 2^t one rounding and the
reciprocal 2 u (2^-23): s to 8 u.  The gate's value adds one rounding (times z), the product with the row's element one: 10 u.
The slope is s ((1 - s) c + 0 or 1) with 1 - s = s 2^t: 8 + (8 + 5 + 1) + 2 roundings, 24 u of the sum of the magnitudes of its
terms (z s (1 - s) + s cancels near z = -1.28).  16-bit results: half a step of their own, and t's rounding, |t| 2^-23 ln 2 <= 2^-16
of 2^t where |z| <= 80, so 2^-15 of the slope's terms.
"""
import pytest
import torch

from accelerated_scan import norm

U = 2.0 ** -24


def gates(dtype, device, rows, D):
    """-80 to 80, evenly, and the border values of every binade."""
    even = torch.linspace(-80, 80, rows * D - 64, dtype=torch.float64)
    steps = 2.0 ** torch.arange(-25, 7, dtype=torch.float64)
    return torch.cat([even, -steps, steps]).to(dtype).view(rows, D).to(device)


def definition(z, act):
    z = z.double()
    s = 1 / (1 + torch.exp(-z))
    r = torch.exp(-z) * s                                   # 1 - s
    if act == "sigmoid":
        return s, s * r, s * r
    return z * s, s * (1 + z * r), s * (1 + z.abs() * r)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("D", [64, 2048, 2047, 8192])       # each form of the forward and backward kernels
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gates_elementwise(cuda_device, dtype, D, act):
    rows = max(2, 40000 // D)
    z = gates(dtype, cuda_device, rows, D).requires_grad_(True)
    x = torch.ones(rows, D, dtype=dtype, device=cuda_device)
    w = torch.ones(D, dtype=dtype, device=cuda_device)
    value, slope, terms = definition(z.detach(), act)
    for pre in (None, w):                                   # the backward of one norm, and of both
        got = norm.residual_norm(x, gate=z, activation=act, pre_weight=pre)
        hidden = got if pre is None else got[0]
        d, = torch.autograd.grad(hidden, z, torch.ones_like(hidden))
        if dtype == torch.float32:
            own, fine, tiny = 0.0, (10 * U, 24 * U), 0.0
        else:
            own, fine, tiny = torch.finfo(dtype).eps / 2, (2.0 ** -16, 2.0 ** -15), torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        off = (hidden.detach().double() - value).abs() - (own + fine[0]) * value.abs() - tiny
        assert (off <= 0).all(), z.detach().flatten()[off.argmax()].item()
        off = (d.double() - slope).abs() - own * slope.abs() - fine[1] * terms - tiny
        assert (off <= 0).all(), z.detach().flatten()[off.argmax()].item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gates_at_the_ends(cuda_device, dtype):
    """Infinite gates, and finite ones whose exponential is not: closed is 0, open is 1 or the gate, NaN stays NaN."""
    inf = float("inf")
    z = torch.tensor([-inf, -30000.0, -200.0, -129.0, -100.0, 100.0, 129.0, 200.0, 30000.0, inf, float("nan"), 0.0], dtype=dtype, device=cuda_device)
    x = torch.ones(12, dtype=dtype, device=cuda_device)
    z = z[None].requires_grad_(True)
    h = norm.residual_norm(x[None], gate=z, activation="sigmoid")
    d, = torch.autograd.grad(h, z, torch.ones_like(h))
    want = torch.tensor([0.0] * 5 + [1.0] * 5 + [float("nan"), 0.5], dtype=dtype, device=cuda_device)
    assert torch.equal(h[0].nan_to_num(7), want.nan_to_num(7)) and torch.isnan(h[0, 10])
    assert (d[0, :10].double().abs() < 1e-37).all() and torch.isnan(d[0, 10]) and d[0, 11] == 0.25
    h = norm.residual_norm(x[None], gate=z, activation="silu")
    d, = torch.autograd.grad(h, z, torch.ones_like(h))
    assert (h[0, 1:5] == 0).all() and torch.equal(h[0, 5:10], z[0, 5:10]) and torch.isnan(h[0, 10]) and h[0, 11] == 0
    assert (d[0, 1:5].double().abs() < 1e-37).all() and (d[0, 5:9] == 1).all() and d[0, 11] == 0.5
