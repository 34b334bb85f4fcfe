"""Gated delta rule (delta.scan, delta.step) against the definition, token by token in 64 bits.

Tolerances, as 2-norm of the error over 2-norm of the result.  A value rounded to bf16 is off by at most 2^-8 of itself
(fp16 2^-11, fp32 2^-24).  The kernels' products take fp32 operands as two bf16 terms, hi + lo, off by at most 2^-16.
  * fp32 values that are carried (final_state, d_initial_state, and everything for fp32 inputs) pass a handful of such
    products, each with two operands and one dropped term: 8 * 2^-16.
  * bf16 outputs: the output's own rounding and those of the one-term operands: out takes S, u and P, the gradients S0 or
    dS1, e, z, D or F; four roundings at most of 2^-8 each.
  * fp16 outputs: their own rounding, 2^-11, and the above for fp32.
"""
import pytest
import torch

from accelerated_scan import delta

CARRIED = 8 * 2.0 ** -16
TOL = {torch.bfloat16: 4 * 2.0 ** -8, torch.float16: 2.0 ** -11 + CARRIED, torch.float32: CARRIED}


def inputs(seed, B, T, Hk, H, K, V, dtype, device="cpu", state=True, gate_dtype=None, n=None):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)
    q, k, v = unit(rand(B, T, Hk, K)), unit(rand(B, T, Hk, K)), rand(B, T, H, V)
    lg = -torch.exp(7.0 * (torch.rand(B, T, H, generator=g) - 1.0))
    be = torch.sigmoid(rand(B, T, H))
    s0 = 0.3 * rand(n or B, H, K, V) if state else None
    gate_dtype = gate_dtype or dtype
    out = [q.to(dtype), k.to(dtype), v.to(dtype), lg.to(gate_dtype), be.to(gate_dtype), s0]
    return [None if t is None else t.to(device) for t in out]


def reference(q, k, v, lg, be, s0=None, scale=None, lengths=None):
    """The definition in 64 bits, differentiable."""
    q, k, v, lg, be = (t.double() for t in (q, k, v, lg, be))
    B, T, Hk, K = q.shape
    H, V = v.shape[2:]
    scale = K ** -0.5 if scale is None else scale
    q, k = q.repeat_interleave(H // Hk, 2), k.repeat_interleave(H // Hk, 2)
    if lengths is None:
        lengths, rows = [T], slice(None)
    outs, states, t0 = [], [], 0
    for i, n in enumerate(lengths):
        if s0 is None:
            s = torch.zeros(B, H, K, V, dtype=torch.float64, device=q.device)
        else:
            s = s0.double() if len(lengths) == 1 and s0.shape[0] == B else s0[i:i + 1].double()
        for t in range(t0, t0 + n):
            s = torch.exp(lg[:, t])[..., None, None] * s
            e = v[:, t] - torch.einsum("bhkv,bhk->bhv", s, k[:, t])
            s = s + k[:, t][..., None] * (be[:, t][..., None] * e)[..., None, :]
            outs.append(scale * torch.einsum("bhkv,bhk->bhv", s, q[:, t]))
        states.append(s)
        t0 += n
    out = torch.stack(outs, 1) if outs else v[:, :0]
    if out.shape[1] < T:
        out = torch.cat([out, torch.zeros_like(v[:, out.shape[1]:])], 1)
    return out, torch.cat(states, 0)


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


def off(got, want):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    norm = want.norm().item()
    return (got - want).norm().item() / norm if norm else got.norm().item()


def poison(device):
    """Memory that the allocator hands out next holds NaN: whatever a kernel reads before it is written shows."""
    torch.full((1 << 26,), float("nan"), device=device)
    torch.full((1 << 18,), float("nan"), device=device)


SHAPES = [  # B, T, Hk, H, K, V
    (1, 1, 1, 1, 128, 128),
    (2, 63, 2, 2, 64, 64),
    (1, 64, 1, 2, 128, 128),
    (3, 65, 2, 4, 128, 64),
    (1, 200, 1, 3, 61, 20),
    (2, 130, 1, 1, 16, 136),
    (1, 129, 2, 2, 1, 1),
    (2, 257, 4, 8, 128, 128),
    (1, 300, 1, 1, 100, 1024),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("state", [False, True])
def test_scan_forward_and_gradients(cuda_device, shape, dtype, state):
    args = inputs(sum(shape), *shape, dtype, cuda_device, state)
    leaves = [t.requires_grad_(True) for t in args if t is not None]
    want, want_s = reference(*args)
    g = torch.Generator().manual_seed(1)
    d_out = torch.randn(want.shape, generator=g).to(dtype).to(cuda_device)
    d_s = 0.3 * torch.randn(want_s.shape, generator=g).to(cuda_device)
    poison(cuda_device)
    out, s = delta.scan(*args)
    assert out.dtype == dtype and s.dtype == torch.float32
    assert off(out, want) <= TOL[dtype] and off(s, want_s) <= CARRIED
    ends = (([want, want_s], [out, s], [d_out, d_s]) if state else ([want], [out], [d_out]))
    want_g = torch.autograd.grad(ends[0], leaves, [d.double() for d in ends[2]])
    poison(cuda_device)
    got_g = torch.autograd.grad(ends[1], leaves, ends[2])
    for name, a, b, x in zip("queries keys values log_gates betas state".split(), got_g, want_g, leaves):
        assert a.dtype == x.dtype and a.shape == x.shape
        tol = CARRIED if name == "state" else TOL[dtype]
        if name == "log_gates":      # sums of q.dq and k.dk that cancel: 4 more such terms
            tol *= 2
        assert off(a, b) <= tol, name


@pytest.mark.gpu
def test_scan_without_gradient_is_the_same(cuda_device):
    args = inputs(3, 2, 200, 2, 4, 128, 128, torch.bfloat16, cuda_device)
    with torch.no_grad():
        a, s = delta.scan(*args)
    b, r = delta.scan(args[0].clone().requires_grad_(True), *args[1:])
    assert torch.equal(a, b) and torch.equal(s, r)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths", [[1], [64, 64], [63, 1, 65], [0, 70, 0, 0, 130, 3, 0], [200, 1, 1, 1, 1]])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_packed_sequences(cuda_device, lengths, dtype, index):
    """Sequences of any length, empty ones too, and tokens behind the last one."""
    T, n = sum(lengths) + 5, len(lengths)
    args = inputs(T, 1, T, 2, 4, 64, 48, dtype, cuda_device, n=n)
    leaves = [t.requires_grad_(True) for t in args]
    starts = torch.tensor([0] + lengths, dtype=index).cumsum(0).to(index).to(cuda_device)
    want, want_s = reference(*args, lengths=lengths)
    poison(cuda_device)
    out, s = delta.scan(*args, seq_starts=starts)
    assert off(out, want) <= TOL[dtype] and off(s, want_s) <= CARRIED
    assert (out[:, sum(lengths):] == 0).all()
    d_out, d_s = torch.randn_like(out), torch.randn_like(s)
    want_g = torch.autograd.grad([want, want_s], leaves, [d_out.double(), d_s.double()])
    poison(cuda_device)
    got_g = torch.autograd.grad([out, s], leaves, [d_out, d_s])
    for i, (a, b) in enumerate(zip(got_g, want_g)):
        assert off(a, b) <= (CARRIED if i == 5 else TOL[dtype]) * (2 if i == 3 else 1), i
        if i < 5:
            assert (a[:, sum(lengths):] == 0).all()


@pytest.mark.gpu
def test_packed_sequences_that_start_late(cuda_device):
    args = inputs(8, 1, 150, 1, 2, 64, 64, torch.float32, cuda_device, n=2)
    leaves = [t.requires_grad_(True) for t in args]
    starts = torch.tensor([7, 90, 120], dtype=torch.int32, device=cuda_device)
    poison(cuda_device)
    out, s = delta.scan(*args, seq_starts=starts)
    grads = torch.autograd.grad([out, s], leaves, [torch.ones_like(out), torch.ones_like(s)])
    want, want_s = reference(*(t[:, 7:120] for t in args[:5]), args[5], lengths=[83, 30])
    assert off(out[:, 7:120], want) <= CARRIED and off(s, want_s) <= CARRIED
    for t in (out, *grads[:5]):
        assert (t[:, :7] == 0).all() and (t[:, 120:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_padding_tokens_zero_gates_and_zero_rates(cuda_device, dtype):
    """beta = 0 writes nothing, gate 0 (log gate -inf, or far below) starts anew, both anywhere in a chunk."""
    args = inputs(5, 2, 190, 1, 2, 64, 64, dtype, cuda_device)
    with torch.no_grad():
        args[4][:, ::3] = 0
        args[3][:, 5, 0] = float("-inf")
        args[3][:, 64] = float("-inf")
        args[3][:, 100:103] = -200.0
        args[3][:, 127, 1] = float("-inf")
        args[3][0, 150:] = 0
        args[4][0, 150:] = 0
    leaves = [t.requires_grad_(True) for t in args]
    want, want_s = reference(*args)
    out, s = delta.scan(*args)
    assert off(out, want) <= TOL[dtype] and off(s, want_s) <= CARRIED
    assert torch.equal(s[0], delta.scan(*(t[:1, :150].detach() for t in args[:5]), args[5][:1].detach())[1][0])
    d_out, d_s = torch.randn_like(out), torch.randn_like(s)
    got_g = torch.autograd.grad([out, s], leaves, [d_out, d_s])
    zero = args[3] <= -104
    # the reference's gradient of a zero gate is 0 * x = 0, of -inf exp'(-inf) * x = 0
    want_g = torch.autograd.grad([want, want_s], leaves, [d_out.double(), d_s.double()])
    for i, (a, b) in enumerate(zip(got_g, want_g)):
        b = torch.where(zero, torch.zeros_like(b), b) if i == 3 else b
        assert off(a, b) <= (CARRIED if i == 5 else TOL[dtype]) * (2 if i == 3 else 1), i
    assert (got_g[3][zero] == 0).all()


@pytest.mark.gpu
def test_strong_decay_far_into_a_chunk(cuda_device):
    """Differences of running sums of log gates: a strong gate early in a chunk costs the later ones nothing."""
    args = inputs(6, 1, 128, 1, 1, 64, 64, torch.float32, cuda_device)
    args[3][:, 3] = -100.0
    args[3][:, 70] = -90.0
    out, s = delta.scan(*args)
    want, want_s = reference(*args)
    assert off(out, want) <= CARRIED and off(s, want_s) <= CARRIED


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_float32_gates_beside_16_bit_tensors(cuda_device, dtype):
    args = inputs(9, 2, 100, 2, 2, 64, 64, dtype, cuda_device, gate_dtype=torch.float32)
    leaves = [t.requires_grad_(True) for t in args]
    out, s = delta.scan(*args)
    want, want_s = reference(*args)
    assert off(out, want) <= TOL[dtype] and off(s, want_s) <= CARRIED
    d_out = torch.randn_like(out)
    got_g, want_g = torch.autograd.grad(out, leaves, d_out), torch.autograd.grad(want, leaves, d_out.double())
    for i, (a, b) in enumerate(zip(got_g, want_g)):
        assert a.dtype == leaves[i].dtype
        assert off(a, b) <= (CARRIED if i == 5 else TOL[dtype]) * (2 if i == 3 else 1), i


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_offsets(cuda_device, dtype):
    """Slices of one projection, transposed heads, odd offsets, an expanded gradient."""
    B, T, H, K, V = 2, 90, 2, 64, 64
    plain = inputs(10, B, T, H, H, K, V, dtype, cuda_device)
    wide = torch.cat([plain[0].flatten(2), plain[1].flatten(2), plain[2].flatten(2)], -1)
    cut = lambda i: wide[..., i * H * K:(i + 1) * H * K].view(B, T, H, K)
    want = delta.scan(*plain)
    for a, b in zip(delta.scan(cut(0), cut(1), cut(2), *plain[3:]), want):
        assert torch.equal(a, b)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in plain[:5]]
    for a, b in zip(delta.scan(*heads_first, plain[5]), want):
        assert torch.equal(a, b)
    odd = torch.empty(plain[0].numel() + 1, dtype=dtype, device=cuda_device)[1:].view_as(plain[0])
    odd.copy_(plain[0])
    last_strided = torch.stack([plain[1], plain[1]], -1)[..., 0]
    for a, b in zip(delta.scan(odd, last_strided, *plain[2:]), want):
        assert torch.equal(a, b)
    leaves = [t.requires_grad_(True) for t in plain]
    one = torch.autograd.grad(delta.scan(*plain)[0].sum(), leaves)
    other = torch.autograd.grad(delta.scan(*plain)[0], leaves, torch.ones(B, T, H, V, dtype=dtype, device=cuda_device))
    for a, b in zip(one, other):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_sequence_in_two_calls(cuda_device):
    args = inputs(11, 2, 300, 2, 4, 128, 64, torch.float32, cuda_device)
    want, want_s = delta.scan(*args)
    a, s = delta.scan(*(t[:, :170] for t in args[:5]), args[5])
    b, s = delta.scan(*(t[:, 170:] for t in args[:5]), s)
    assert off(torch.cat([a, b], 1), want) <= CARRIED and off(s, want_s) <= CARRIED


@pytest.mark.gpu
def test_unused_outputs_and_inputs_without_gradient(cuda_device):
    args = inputs(12, 1, 70, 1, 2, 64, 64, torch.float32, cuda_device)
    args[2].requires_grad_(True)
    out, s = delta.scan(*args)
    want, want_s = reference(*args)
    d_s = torch.randn_like(s)
    assert off(torch.autograd.grad(s, args[2], d_s)[0], torch.autograd.grad(want_s, args[2], d_s.double())[0]) <= CARRIED
    args[2].requires_grad_(False)
    args[5].requires_grad_(True)
    out, s = delta.scan(*args)
    want, want_s = reference(*args)
    assert off(torch.autograd.grad(out.sum(), args[5])[0], torch.autograd.grad(want.sum(), args[5])[0]) <= CARRIED


@pytest.mark.gpu
def test_gradients_against_differences(cuda_device):
    """fp32, a directional derivative; step h, error of the difference h^2 and 2^-16 / h of the outputs."""
    args = inputs(13, 1, 100, 1, 1, 32, 32, torch.float32, cuda_device)
    leaves = [t.requires_grad_(True) for t in args]
    weight = torch.randn(1, 100, 1, 32, device=cuda_device)
    loss = lambda xs: (delta.scan(*xs)[0].double() * weight).sum()
    grads = torch.autograd.grad(loss(leaves), leaves)
    h = 1e-2
    for i, x in enumerate(leaves):
        direction = torch.randn_like(x)
        direction /= direction.norm()
        moved = lambda f: [t.detach() + f * direction if j == i else t.detach() for j, t in enumerate(leaves)]
        slope = (loss(moved(h)) - loss(moved(-h))) / (2 * h)
        got = (grads[i].double() * direction).sum()
        scale = grads[i].double().norm()
        assert abs(slope - got) <= 5e-3 * scale, i


@pytest.mark.gpu
def test_results_repeat_bit_for_bit(cuda_device):
    args = inputs(14, 2, 500, 2, 8, 128, 128, torch.bfloat16, cuda_device)
    leaves = [t.requires_grad_(True) for t in args]
    runs = []
    for _ in range(3):
        out, s = delta.scan(*args)
        runs.append([out, s, *torch.autograd.grad([out, s], leaves, [torch.ones_like(out), torch.ones_like(s)])])
    for run in runs[1:]:
        for a, b in zip(run, runs[0]):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_empty_calls(cuda_device):
    for B, T in ((0, 5), (2, 0)):
        args = inputs(15, B, T, 1, 2, 64, 64, torch.bfloat16, cuda_device)
        leaves = [t.requires_grad_(True) for t in args]
        out, s = delta.scan(*args)
        assert out.shape == (B, T, 2, 64) and torch.equal(s, args[5])
        g = torch.autograd.grad([out, s], leaves, [torch.ones_like(out), torch.ones_like(s)])
        assert torch.equal(g[5], torch.ones_like(s))
    out, s = delta.scan(*inputs(15, 1, 0, 1, 2, 64, 64, torch.bfloat16, cuda_device, state=False))
    assert (s == 0).all()
    assert delta.step(*(t[:, 0] for t in inputs(15, 0, 1, 1, 2, 64, 64, torch.bfloat16, cuda_device)[:5]),
                      torch.zeros(3, 2, 64, 64, device=cuda_device)).shape == (0, 2, 64)


@pytest.mark.gpu
def test_another_stream_and_a_captured_graph(cuda_device):
    args = inputs(16, 2, 200, 2, 4, 128, 64, torch.bfloat16, cuda_device)
    leaves = [t.requires_grad_(True) for t in args]
    d_out = torch.randn(2, 200, 4, 64, device=cuda_device).to(torch.bfloat16)

    def train():
        out, s = delta.scan(*args)
        got = [out, s, *torch.autograd.grad(out, leaves, d_out)]
        return [t.detach() for t in got]       # no graph of these leaves is left when the backward is captured

    want = train()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    results = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            results.append(train())
    for _ in range(2):
        with torch.no_grad():
            d_out.mul_(2)                  # exact: gradients double
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for got in results:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for a, b in zip(got[2:], want[2:]):
            assert torch.equal(a.float(), 4 * b.float())


# ---- single tokens ----------------------------------------------------------------------------------------------------

def token_inputs(seed, B, Hk, H, K, V, dtype, device):
    return [t[:, 0] for t in inputs(seed, B, 1, Hk, H, K, V, dtype, device, state=False)[:5]]


def step_reference(q, k, v, lg, be, state):
    out, s = reference(*(t[:, None] for t in (q, k, v, lg, be)), state)
    return out[:, 0], s


def state_off(got, want, before, values):
    """Of a state after one token.  S' + beta k (v - S'^T k) may cancel, S' against the rest, so the error is held against what
    goes in: with |k| <= 1 and beta, e^g <= 1 every term is at most |S| or |v|, and each of the sums over K and of the
    product with k adds its 2^-24 of them, a handful in the 2-norm."""
    return (got.double() - want).norm().item() / (before.double().norm().item() + values.double().norm().item())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1, 1, 128, 128), (3, 2, 4, 64, 64), (5, 1, 3, 61, 20), (2, 1, 1, 1, 1), (4, 2, 2, 128, 33),
                                   (70, 2, 8, 128, 128), (2, 1, 2, 100, 1000), (40, 4, 16, 72, 80), (1030, 1, 1, 16, 16)])
def test_step(cuda_device, shape, dtype):
    """out: its own rounding, and like the state fp32 sums over K of up to 128 terms: 8 * 2^-24 of what goes in."""
    B, Hk, H, K, V = shape
    args = token_inputs(sum(shape), *shape, dtype, cuda_device)
    pool = torch.randn(B + 3, H, K, V, device=cuda_device)
    for slots in (None, torch.randperm(B + 3)[:B].to(torch.int32).to(cuda_device), torch.randperm(B + 3)[:B].to(cuda_device)):
        state = pool.clone()
        at = torch.arange(B, device=cuda_device) if slots is None else slots.long()
        want, want_s = step_reference(*args, pool[at])
        out = delta.step(*args, state, slots)
        assert out.dtype == dtype
        # out is scale S^T q with |q| = 1: what the state is off, and its own rounding
        into = K ** -0.5 * (pool[at].double().norm().item() + args[2].double().norm().item())
        assert (out.double() - want).norm().item() <= torch.finfo(dtype).eps / 2 * want.norm().item() + 16 * 2.0 ** -24 * into
        assert state_off(state[at], want_s, pool[at], args[2]) <= 8 * 2.0 ** -24
        rest = torch.ones(B + 3, dtype=torch.bool, device=cuda_device)
        rest[at] = False
        assert torch.equal(state[rest], pool[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("H,V", [(2, 64), (128, 64), (128, 96)])     # few states, and more than the SMs hold at once
def test_step_padded_rows_and_bad_slots(cuda_device, H, V):
    B = 6
    args = token_inputs(1, B, 1, H, 64, V, torch.bfloat16, cuda_device)
    pool = torch.randn(4, H, 64, V, device=cuda_device)
    state = pool.clone()
    slots = torch.tensor([2, -1, 0, 2, 4, 1 << 30], dtype=torch.int32, device=cuda_device)
    out = delta.step(*args, state, slots)
    want, want_s = step_reference(*args, pool[slots.clamp(0, 3).long()])
    for row in (0, 2):
        assert off(out[row], want[row]) <= 2.0 ** -8 + 8 * 2.0 ** -24
        assert state_off(state[slots[row]], want_s[row], pool[slots[row]], args[2][row]) <= 8 * 2.0 ** -24
    assert (out[1] == 0).all()
    assert torch.isnan(out[3:]).all()                      # a slot taken by an earlier row, slots behind the pool
    assert torch.equal(state[[1, 3]], pool[[1, 3]])


@pytest.mark.gpu
def test_step_pool_that_is_a_layer_of_a_larger_one_and_strided_inputs(cuda_device):
    B, H, K, V = 4, 2, 64, 64
    args = token_inputs(2, B, 2, H, K, V, torch.bfloat16, cuda_device)
    every = torch.randn(B, 3, H, K, V, device=cuda_device)
    want_pool = every.clone()
    want = delta.step(*args, want_pool[:, 1].contiguous())
    wide = torch.cat([t.flatten(1) for t in args[:3]], -1)
    cut = [wide[:, i * H * K:(i + 1) * H * K].view(B, H, K) for i in range(3)]
    gates = torch.stack([args[3], args[4]], -1)
    before = every.clone()
    out = delta.step(*cut, gates[..., 0], gates[..., 1], every[:, 1])
    assert torch.equal(out, want)
    assert torch.equal(every[:, 0], before[:, 0]) and torch.equal(every[:, 2], before[:, 2])
    assert not torch.equal(every[:, 1], before[:, 1])
    odd = torch.empty(B * H * K * V + 1, device=cuda_device)[1:].view(B, H, K, V)
    odd.copy_(before[:, 1])
    # element by element the sums over K run in another order: each within 8 * 2^-24 of the exact one
    assert off(delta.step(*args, odd), want) <= 2 * (2.0 ** -8 + 8 * 2.0 ** -24) and off(odd, every[:, 1]) <= 16 * 2.0 ** -24


@pytest.mark.gpu
def test_step_zero_gate(cuda_device):
    args = token_inputs(3, 2, 1, 1, 64, 64, torch.float32, cuda_device)
    args[3][0] = float("-inf")
    state = torch.randn(2, 1, 64, 64, device=cuda_device)
    start = state.clone()
    want, want_s = step_reference(*args, state)
    out = delta.step(*args, state)
    assert off(out, want) <= 16 * 2.0 ** -24 and state_off(state, want_s, start, args[2]) <= 8 * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_then_tokens(cuda_device, dtype):
    """A prompt by scan, its state handed to a pool, tokens by step: what scan answers for the whole sequence."""
    T, P = 75, 70
    args = inputs(17, 2, T, 2, 4, 128, 128, dtype, cuda_device, state=False)
    whole, last = delta.scan(*args)
    _, s = delta.scan(*(t[:, :P] for t in args[:5]))
    pool = torch.zeros(5, 4, 128, 128, device=cuda_device)
    slots = torch.tensor([3, 1], dtype=torch.int32, device=cuda_device)
    pool[slots.long()] = s
    for t in range(P, T):
        out = delta.step(*(x[:, t] for x in args[:5]), pool, slots)
        assert off(out, whole[:, t]) <= 2 * TOL[dtype]
    assert off(pool[slots.long()], last) <= 2 * CARRIED


@pytest.mark.gpu
def test_step_in_a_captured_graph(cuda_device):
    args = token_inputs(4, 3, 1, 2, 64, 64, torch.bfloat16, cuda_device)
    start = torch.randn(3, 2, 64, 64, device=cuda_device)
    state, want_state = start.clone(), start.clone()
    want = [delta.step(*args, want_state).clone() for _ in range(3)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = delta.step(*args, state)
    state.copy_(start)
    for w in want:
        graph.replay()
        assert torch.equal(out, w)
    assert torch.equal(state, want_state)


# ---- refusals (no GPU) ------------------------------------------------------------------------------------------------

def refused(error, args, **kw):
    with pytest.raises(error):
        delta.scan(*args, **kw)


def test_scan_refuses():
    good = inputs(0, 2, 8, 2, 4, 16, 16, torch.float32)
    change = lambda i, t: [t if j == i else x for j, x in enumerate(good)]
    refused(RuntimeError, good)                                                 # no CPU path
    refused(AssertionError, change(1, good[1][:, :7]))
    refused(AssertionError, change(2, good[2][:, :7]))
    refused(AssertionError, change(2, good[2][:, :, :3]))                       # 3 heads over 2 key heads
    refused(AssertionError, change(3, good[3][:, :, :2]))
    refused(AssertionError, change(4, good[4][..., None]))
    refused(AssertionError, change(0, good[0][0]))
    refused(RuntimeError, change(1, good[1].bfloat16()))
    refused(RuntimeError, change(3, good[3].bfloat16()))                        # gates narrower than the rest
    refused(RuntimeError, [t.double() for t in good])
    refused(RuntimeError, [t.to(torch.complex64) for t in good])
    refused(RuntimeError, inputs(0, 1, 4, 1, 1, 129, 16, torch.float32))
    refused(RuntimeError, inputs(0, 1, 4, 1, 1, 16, 1025, torch.float32))


def test_step_refuses():
    good = token_inputs(0, 2, 2, 4, 16, 16, torch.float32, "cpu")
    state = torch.zeros(3, 4, 16, 16)
    for args in ([good[0][:1], *good[1:]], [*good[:3], good[3][:, :3], good[4]], [good[0][0], *good[1:]]):
        with pytest.raises(AssertionError):
            delta.step(*args, state)
    with pytest.raises(RuntimeError):
        delta.step(*good, state)


@pytest.mark.gpu
def test_refusals_on_the_gpu(cuda_device):
    good = inputs(0, 1, 8, 2, 4, 16, 16, torch.float32, cuda_device)
    starts = torch.tensor([0, 8], dtype=torch.int32, device=cuda_device)
    refused(AssertionError, [torch.cat([t, t]) for t in good], seq_starts=starts)       # packed needs B == 1
    refused(RuntimeError, good, seq_starts=starts.cpu())
    refused(RuntimeError, good, seq_starts=starts.float())
    refused(AssertionError, good, seq_starts=starts[:1])
    refused(AssertionError, [*good[:5], good[5][:, :2]])
    refused(RuntimeError, [*good[:5], good[5].long()])
    refused(RuntimeError, [*good[:5], good[5].cpu()])
    token = token_inputs(0, 2, 2, 4, 16, 16, torch.float32, cuda_device)
    state = torch.zeros(3, 4, 16, 16, device=cuda_device)
    slots = torch.tensor([0, 1], dtype=torch.int32, device=cuda_device)
    for kw, error in (({"state": state.bfloat16()}, RuntimeError), ({"state": state.cpu()}, RuntimeError),
                      ({"state": state[:1]}, AssertionError), ({"state": state.transpose(2, 3)}, RuntimeError),
                      ({"state": state[:1].expand(3, 4, 16, 16)}, RuntimeError), ({"state": state[:, :2]}, AssertionError),
                      ({"state": state, "slots": slots[:1]}, AssertionError), ({"state": state, "slots": slots.cpu()}, RuntimeError),
                      ({"state": state, "slots": slots.float()}, RuntimeError)):
        with pytest.raises(error):
            delta.step(*token, **kw)
    token[0].requires_grad_(True)
    with pytest.raises(RuntimeError):
        delta.step(*token, state)


def test_bad_arguments_of_the_c_entries():
    import ctypes
    from accelerated_scan import _native

    a = _native.Delta()
    a.batch, a.seqlen, a.heads_k, a.heads, a.k_dim, a.v_dim = 1, 64, 1, 2, 64, 64
    size = lambda: _native.lib.ascan_delta_forward_bytes(ctypes.byref(a), 0)
    fake = ctypes.c_void_p(256)                        # never dereferenced
    forward = lambda: _native.lib.ascan_delta_forward(ctypes.byref(a), fake, fake, 0, fake, 1 << 40, None)
    assert size() > 2 * 2 * 4096 * 2 and size() < _native.lib.ascan_delta_forward_bytes(ctypes.byref(a), 1)
    assert forward() == 1                              # null inputs
    for name, value in (("batch", -1), ("seqlen", -1), ("heads", 0), ("heads_k", 3), ("k_dim", 0), ("v_dim", 0), ("dtype", 3),
                        ("log_gates_dtype", 1), ("betas_dtype", 2), ("n_seqs", -1), ("k_dim", 129), ("v_dim", 1025),
                        ("heads", 65536)):
        before = getattr(a, name)
        setattr(a, name, value)
        assert size() == 0 and forward() in (1, 2), name
        setattr(a, name, before)
    for name in ("queries", "keys", "values", "log_gates", "betas"):
        setattr(a, name, 256)
    assert _native.lib.ascan_delta_forward(ctypes.byref(a), fake, fake, 0, fake, size() - 1, None) == 5
    assert _native.lib.ascan_delta_forward(ctypes.byref(a), fake, fake, 0, ctypes.c_void_p(128), 1 << 40, None) == 5
    assert _native.lib.ascan_delta_forward(ctypes.byref(a), fake, None, 0, fake, 1 << 40, None) == 1
    a.batch = 0
    assert forward() == 0
    t = _native.DeltaToken()
    assert _native.lib.ascan_delta_step(ctypes.byref(t), fake, fake, 1, 1, None, 0, None) == 1
    t.batch, t.heads_k, t.heads, t.k_dim, t.v_dim = 2, 1, 1, 16, 16
    for name in ("queries", "keys", "values", "log_gates", "betas"):
        setattr(t, name, 256)
    assert _native.lib.ascan_delta_step(ctypes.byref(t), fake, fake, 1, 256, None, 0, None) == 1       # pool of one for two rows
    assert _native.lib.ascan_delta_step(ctypes.byref(t), fake, fake, 2, 255, None, 0, None) == 1       # states overlap


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(8, 650, 4, 8, 72, 200), (4, 700, 4, 4, 128, 64), (3, 600, 6, 18, 64, 128)])
def test_more_chunks_than_the_gpu_holds(cuda_device, shape, dtype):
    """Chunks times key heads beyond the number of SMs, with one, two and four slabs of V and one to three value heads."""
    args = inputs(sum(shape), *shape, dtype, cuda_device)
    leaves = [t.requires_grad_(True) for t in args]
    want, want_s = reference(*args)
    d_out, d_s = torch.randn_like(want).to(dtype), torch.randn_like(want_s).float()
    out, s = delta.scan(*args)
    assert off(out, want) <= TOL[dtype] and off(s, want_s) <= CARRIED
    want_g = torch.autograd.grad([want, want_s], leaves, [d_out.double(), d_s.double()])
    got_g = torch.autograd.grad([out, s], leaves, [d_out, d_s])
    for i, (a, b) in enumerate(zip(got_g, want_g)):
        assert off(a, b) <= (CARRIED if i == 5 else TOL[dtype]) * (2 if i == 3 else 1), i


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_short_sequences_beside_tokens_that_are_not_finite(cuda_device, dtype):
    """Every chunk ends inside the row; what stands in no sequence is infinite or NaN."""
    lengths = [37, 1, 64, 5, 90, 66, 0, 23] * 8
    T, n, front = sum(lengths) + 11, len(lengths), 6
    args = inputs(T, 1, T, 4, 8, 128, 136, dtype, cuda_device, n=n)
    starts = (torch.tensor([0] + lengths).cumsum(0) + front).to(torch.int32).to(cuda_device)
    inside = slice(front, front + sum(lengths))
    clean = [t[:, inside].clone().requires_grad_(True) for t in args[:5]] + [args[5].clone().requires_grad_(True)]
    want, want_s = reference(*clean, lengths=lengths)
    for i, t in enumerate(args[:5]):
        t[:, :front] = float("nan") if i % 2 else float("inf")
        t[:, front + sum(lengths):] = float("inf") if i % 2 else float("nan")
    leaves = [t.requires_grad_(True) for t in args]
    out, s = delta.scan(*args, seq_starts=starts)
    assert off(out[:, inside], want) <= TOL[dtype] and off(s, want_s) <= CARRIED
    d_out, d_s = torch.randn_like(out), torch.randn_like(s)
    want_g = torch.autograd.grad([want, want_s], clean, [d_out[:, inside].double(), d_s.double()])
    d_out[:, :front] = d_out[:, front + sum(lengths):] = float("nan")
    got_g = torch.autograd.grad([out, s], leaves, [d_out, d_s])
    for i, (a, b) in enumerate(zip(got_g, want_g)):
        tol = (CARRIED if i == 5 else TOL[dtype]) * (2 if i == 3 else 1)
        assert off(a[:, inside] if i < 5 else a, b) <= tol, i
        if i < 5:
            assert (a[:, :front] == 0).all() and (a[:, front + sum(lengths):] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_boundaries_outside_of_the_row_are_cut_off(cuda_device, dtype):
    args = inputs(9, 1, 150, 1, 2, 64, 64, dtype, cuda_device, n=3)
    leaves = [t.requires_grad_(True) for t in args]
    results = []
    for bounds in ([-5, 30, 150, 9000], [0, 30, 150, 150]):
        starts = torch.tensor(bounds, device=cuda_device)
        out, s = delta.scan(*args, seq_starts=starts)
        results.append((out, s, *torch.autograd.grad([out, s], leaves, [torch.ones_like(out), torch.ones_like(s)])))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hk,H,V", [(4, 8, 136), (4, 4, 192), (4, 16, 128), (8, 8, 64)])
def test_many_chunks_repeat_bit_for_bit(cuda_device, Hk, H, V, dtype):
    """Chunks of many short sequences, which CTAs take in any order: the same bits every time."""
    lengths = [37, 1, 64, 5, 90, 66, 0, 23] * 8
    args = inputs(V, 1, sum(lengths), Hk, H, 128, V, dtype, cuda_device, n=len(lengths))
    starts = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(cuda_device)
    leaves = [t.requires_grad_(True) for t in args]
    first = None
    for _ in range(12):
        out, s = delta.scan(*args, seq_starts=starts)
        if first is None:
            d_out, d_s = torch.randn_like(out), torch.randn_like(s)
        got = (out, s, *torch.autograd.grad([out, s], leaves, [d_out, d_s]))
        first = first or got
        for a, b in zip(got, first):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_training_steps_on_two_streams_at_once(cuda_device, dtype):
    """Kernels of two calls share the GPU: neither waits for the other, and each has its own scratch."""
    calls = [inputs(40 + i, 4, 700, 4, 8, 128, 128, dtype, cuda_device) for i in range(2)]
    leaves = [[t.requires_grad_(True) for t in args] for args in calls]
    d = [torch.randn(4, 700, 8, 128, device=cuda_device).to(dtype) for _ in calls]
    want = [torch.autograd.grad(delta.scan(*args)[0], own, g) for args, own, g in zip(calls, leaves, d)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(torch.autograd.grad(delta.scan(*calls[i])[0], leaves[i], d[i]))
    torch.cuda.synchronize()
    for own, expected in zip(got, want):
        for grads in own:
            for a, b in zip(grads, expected):
                assert torch.equal(a, b)


def test_an_expired_wait_is_reported_once(monkeypatch):
    """The word that a kernel sets when it gives up is read, and cleared, by the next call on its device."""
    from accelerated_scan import _native
    word = torch.zeros(4, dtype=torch.int32)
    monkeypatch.setattr(_native, "_sinks", {0: (word, word.numpy(), word.data_ptr())})
    device = torch.device("cuda", 0)
    assert _native._sink(device) == word.data_ptr()
    word[0] = 1
    with pytest.raises(RuntimeError, match="wait expired"):
        _native._sink(device)
    assert _native._sink(device) == word.data_ptr()
