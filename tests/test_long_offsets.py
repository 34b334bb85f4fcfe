"""Arrays of more than 2^31 elements.  A call on all of them gives the bits of calls on parts of them: sequences are cut at a
multiple of the chunk, states and their gradients handed on in fp32; rows of the norms and slots of a pool do not know of one
another."""
import pytest
import torch

from accelerated_scan import delta, norm

BIG = 1 << 31


@pytest.fixture(autouse=True)
def memory():
    free, _ = torch.cuda.mem_get_info() if torch.cuda.is_available() else (0, 0)
    if free < 100 << 30:
        pytest.skip("needs 100 GB of free GPU memory")
    yield
    torch.cuda.empty_cache()


def draw(device, dtype, *shape):
    return torch.randn(*shape, device=device, dtype=torch.bfloat16).to(dtype)


@pytest.mark.gpu
def test_scan(cuda_device):
    T, cut, H, K, V = 1 << 17, 65600, 130, 64, 128
    assert T * H * V > BIG and cut % 64 == 0
    torch.manual_seed(0)
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)
    q, k = (unit(draw(cuda_device, torch.bfloat16, 1, T, 1, K)) for _ in range(2))
    v = draw(cuda_device, torch.bfloat16, 1, T, H, V)
    g, b = -torch.rand(1, T, H, device=cuda_device), torch.rand(1, T, H, device=cuda_device)
    leaves = [t.requires_grad_(True) for t in (q, k, v, g, b)]
    d_out, d_s = draw(cuda_device, torch.bfloat16, 1, T, H, V), torch.randn(1, H, K, V, device=cuda_device)
    out, s = delta.scan(*leaves)
    grads = torch.autograd.grad([out, s], leaves, [d_out, d_s])
    out = out.detach()
    first = [t.detach()[:, :cut].requires_grad_(True) for t in leaves]
    second = [t.detach()[:, cut:].requires_grad_(True) for t in leaves]
    a, middle = delta.scan(*first)
    start = middle.detach().requires_grad_(True)
    c, last = delta.scan(*second, start)
    assert torch.equal(last, s) and torch.equal(a, out[:, :cut]) and torch.equal(c, out[:, cut:])
    *got, d_middle = torch.autograd.grad([c, last], [*second, start], [d_out[:, cut:], d_s])
    for x, y in zip(got, grads):
        assert torch.equal(x, y[:, cut:])
    for x, y in zip(torch.autograd.grad([a, middle], first, [d_out[:, :cut], d_middle]), grads):
        assert torch.equal(x, y[:, :cut])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_scan_of_other_types(cuda_device, dtype):
    T, cut, H, K, V = 1 << 15, 16448, 129, 16, 520
    assert T * H * V > BIG and cut % 64 == 0
    torch.manual_seed(1)
    q, k = (draw(cuda_device, dtype, 1, T, 1, K) * 0.25 for _ in range(2))
    v = draw(cuda_device, dtype, 1, T, H, V)
    g, b = -torch.rand(1, T, H, device=cuda_device), torch.rand(1, T, H, device=cuda_device)
    out, s = delta.scan(q, k, v, g, b)
    a, middle = delta.scan(*(t[:, :cut] for t in (q, k, v, g, b)))
    assert torch.equal(a, out[:, :cut])
    del a
    c, last = delta.scan(*(t[:, cut:] for t in (q, k, v, g, b)), middle)
    assert torch.equal(last, s) and torch.equal(c, out[:, cut:])


@pytest.mark.gpu
@pytest.mark.parametrize("V", [64, 128])               # without and with the ring
def test_step(cuda_device, V):
    H, K = 32, 128
    pool = BIG // (H * K * V) + 20
    torch.manual_seed(2)
    state = torch.zeros(pool, H, K, V, device=cuda_device)
    slots = torch.tensor([pool - 1 - 3 * i for i in range(6)] * 4, device=cuda_device)
    slots = slots - torch.arange(4, device=cuda_device).repeat_interleave(6) * 20
    B = slots.numel()
    assert len(set(slots.tolist())) == B and state.numel() > BIG
    q, k = (draw(cuda_device, torch.bfloat16, B, H, K) * 0.1 for _ in range(2))
    v, g, b = draw(cuda_device, torch.bfloat16, B, H, V), -torch.rand(B, H, device=cuda_device), torch.rand(B, H, device=cuda_device)
    few = torch.randn(B, H, K, V, device=cuda_device)
    state[slots] = few
    assert torch.equal(delta.step(q, k, v, g, b, state, slots), delta.step(q, k, v, g, b, few))
    assert torch.equal(state[slots], few)
    state[slots] = 0
    assert not state.any()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [1024, 8192])
def test_norm(cuda_device, D):
    rows = BIG // D + 1000
    torch.manual_seed(3)
    x, gate = draw(cuda_device, torch.bfloat16, rows, D), draw(cuda_device, torch.bfloat16, rows, D)
    w = torch.rand(D, device=cuda_device)
    d = draw(cuda_device, torch.bfloat16, rows, D)

    def train(part):
        leaves = [t[part].detach().requires_grad_(True) for t in (x, gate)]
        ends = norm.residual_norm(*leaves, gate=leaves[1], post_weight=w, pre_weight=w)
        return [*(t.detach() for t in ends), *torch.autograd.grad(ends, leaves, [d[part], d[part]])]

    whole = train(slice(None))
    tail = slice(rows - 1500, rows)
    for a, b in zip(train(tail), whole):
        assert torch.equal(a, b[tail])
    head = slice(0, 1500)
    for a, b in zip(train(head), whole):
        assert torch.equal(a, b[head])
