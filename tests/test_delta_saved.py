"""delta.scan whose saved tensors come back as other ones: offloaded, copied, dense where they were slices.

What the forward keeps for the backward depends on the inputs' strides and alignment only where it holds packed copies of them,
so a backward that is given equal tensors with other strides gives the same bits: the copies are of the same values, and every
kernel reads either.
"""
import ctypes

import pytest
import torch

from accelerated_scan import _native, delta
from test_delta import inputs

BF16, F16, F32 = 1, 2, 0


def arguments(dtype, strides=(8, 8, 8), aligned=True, batch=2, seqlen=130, heads_k=1, heads=2, k_dim=64, v_dim=64):
    """strides: elements beyond a dense row from token to token, of queries, keys and values."""
    a = _native.Delta()
    a.batch, a.seqlen, a.heads_k, a.heads, a.k_dim, a.v_dim = batch, seqlen, heads_k, heads, k_dim, v_dim
    a.dtype = a.log_gates_dtype = a.betas_dtype = dtype
    for name, h, d, more in (("queries", heads_k, k_dim, strides[0]), ("keys", heads_k, k_dim, strides[1]), ("values", heads, v_dim, strides[2])):
        setattr(a, name, 4096 if aligned else 4098)
        row = h * d + more
        setattr(a, name + "_stride", (ctypes.c_int64 * 3)(seqlen * row, row, d))
    return a


def size(a, keep):
    return _native.lib.ascan_delta_forward_bytes(ctypes.byref(a), keep)


def test_which_inputs_a_forward_packs():
    packed = lambda *args, **kw: _native.lib.ascan_delta_packed(ctypes.byref(arguments(*args, **kw)))
    assert packed(BF16) == 0
    assert packed(BF16, (4, 8, 8)) == 1 and packed(BF16, (8, 4, 8)) == 2 and packed(BF16, (8, 8, 4)) == 4
    assert packed(BF16, aligned=False) == 7 and packed(F16) == 7 and packed(F32) == 7
    bad = arguments(BF16, k_dim=129)
    assert _native.lib.ascan_delta_packed(ctypes.byref(bad)) == 0


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_sizes_with_and_without_packed_copies(dtype):
    """The copies come on top of what is kept anyway, and a backward that is not told of them makes its own."""
    strides = (ctypes.c_int64 * 3)(130 * 128, 128, 64)
    back = lambda a: _native.lib.ascan_delta_backward_bytes(ctypes.byref(a), 4096, strides)
    dense, odd = arguments(dtype), arguments(dtype, (4, 4, 4))
    terms = 1 if dtype == BF16 else 2
    copies = terms * 2 * 130 * (64 + 64 + 128) * 2
    assert size(odd, 1) - size(dense, 1) == (copies if dtype == BF16 else 0)
    assert back(odd) - back(dense) == (copies if dtype == BF16 else 0)
    told = arguments(dtype, (4, 4, 4))
    told.kept_packed = 7
    assert back(odd) - back(told) == copies


class Copies(torch.autograd.graph.saved_tensors_hooks):
    """Saved tensors come back as dense copies at aligned addresses."""
    def __init__(self):
        super().__init__(lambda t: t, lambda t: t.contiguous().clone())


class Slices(torch.autograd.graph.saved_tensors_hooks):
    """... as slices of wider ones at odd addresses, the last dimension strided where that is 4-dimensional."""
    def __init__(self):
        def unpack(t):
            if t.dim() != 4 or t.dtype == torch.float32:
                return t
            wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
            wide[..., 1:-2] = t
            return wide[..., 1:-2]
        super().__init__(lambda t: t, unpack)


class Columns(torch.autograd.graph.saved_tensors_hooks):
    """... with their last two dimensions exchanged in memory."""
    def __init__(self):
        super().__init__(lambda t: t, lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() == 4 else t)


def layouts(args):
    """The inputs of a call as programs hand them over: dense, slices of a projection whose width is no multiple of 8, at an odd
    address, heads of one row (strides of zero)."""
    q, k, v, g, b, s0 = args
    B, T = q.shape[:2]
    wide = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2), torch.zeros_like(g)[..., :1], torch.zeros_like(g)[..., :1]], -1)
    ends = [q[0, 0].numel(), q[0, 0].numel() + k[0, 0].numel()]
    cut = lambda t, at: wide[..., at:at + t[0, 0].numel()].unflatten(-1, t.shape[2:])
    odd = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view_as(t).copy_(t)
    return {"dense": [q, k, v], "slices": [cut(q, 0), cut(k, ends[0]), cut(v, ends[1])], "odd": [odd(q), odd(k), v],
            "values odd": [q, k, odd(v)], "expanded": [q[:, :1].expand_as(q), k, v[:, :, :1].expand_as(v)]}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["dense", "slices", "odd", "values odd", "expanded"])
@pytest.mark.parametrize("hooks", [torch.autograd.graph.save_on_cpu, Copies, Slices, Columns])
def test_gradients_under_saved_tensor_hooks(cuda_device, hooks, layout, dtype):
    args = inputs(21, 2, 150, 2, 4, 64, 64, dtype, cuda_device)
    given = layouts(args)[layout]
    rest = [t.detach().requires_grad_(True) for t in args[3:]]
    d_out = torch.randn(2, 150, 4, 64, device=cuda_device).to(dtype)
    d_s = torch.randn(2, 4, 64, 64, device=cuda_device)

    def gradients():
        leaves = [t.detach().requires_grad_(True) for t in given]
        assert [t.stride() for t in leaves] == [t.stride() for t in given]
        out, s = delta.scan(*leaves, *rest)
        return [out, s], leaves

    ends, leaves = gradients()
    want = torch.autograd.grad(ends, leaves + rest, [d_out, d_s])
    with hooks():
        ends, leaves = gradients()
    got = torch.autograd.grad(ends, leaves + rest, [d_out, d_s])
    for name, a, b in zip("queries keys values log_gates betas state".split(), got, want):
        assert torch.equal(a, b), name


@pytest.mark.gpu
def test_gradients_of_a_packed_row_that_was_offloaded(cuda_device):
    """Slices of one projection, as a layer makes them, several sequences in a row, V beyond one share of 128 columns."""
    args = inputs(22, 1, 333, 2, 4, 128, 136, torch.bfloat16, cuda_device, n=4)
    starts = torch.tensor([3, 70, 70, 300, 330], device=cuda_device)
    given = layouts(args)["slices"]
    grads = []
    for hooks in (torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t), torch.autograd.graph.save_on_cpu(pin_memory=True)):
        leaves = [t.detach().requires_grad_(True) for t in (*given, *args[3:])]
        with hooks:
            out, s = delta.scan(*leaves, seq_starts=starts)
        grads.append(torch.autograd.grad([out, s], leaves, [torch.ones_like(out), torch.ones_like(s)]))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_recomputed_in_the_backward(cuda_device, dtype):
    from torch.utils.checkpoint import checkpoint
    args = inputs(23, 2, 100, 1, 2, 64, 64, dtype, cuda_device)
    given = layouts(args)["slices"]
    grads = []
    for call in (delta.scan, lambda *a: checkpoint(delta.scan, *a, use_reentrant=False)):
        leaves = [t.detach().requires_grad_(True) for t in (*given, *args[3:])]
        out, s = call(*leaves)
        grads.append(torch.autograd.grad([out, s], leaves, [torch.ones_like(out), torch.ones_like(s)]))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_backward_that_is_not_told_of_the_copies(cuda_device, dtype):
    """The C entry with kept_packed left at zero packs the inputs again."""
    args = inputs(24, 2, 90, 1, 2, 64, 64, dtype, cuda_device)
    q, k, v = layouts(args)["slices"]
    g, b, s0 = args[3:]
    out, s = torch.empty_like(v, memory_format=torch.contiguous_format), torch.empty_like(s0)
    d_out = torch.randn_like(out)
    results = []
    for told in (True, False):
        a = _native.delta_args(q, k, v, g, b, s0, 0.125, None)
        kept, packed = _native.delta_forward(a, q.device, out, s, True)
        assert packed == 7
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v, g, b)]
        d_s0 = torch.empty_like(s0)
        a = _native.delta_args(q, k, v, g, b, s0, 0.125, None, packed if told else 0)
        _native.delta_backward(a, q.device, d_out, None, grads, d_s0, kept)
        results.append([*grads, d_s0])
    for x, y in zip(*results):
        assert torch.equal(x, y)
