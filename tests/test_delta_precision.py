"""How far the gated delta rule's results may be off, where test_delta.py asks for less.

With h = 2^-8, the most that a rounding to bf16 takes from a value, and C = 8 * 2^-16, what fp32 values are off that pass a
handful of products of two bf16 terms an operand (test_delta.py):

  * bf16 results whose operands are all two terms (d_values, d_betas): a result off by r of its norm rounds to another value
    than the exact one where a step's border lies between, so by one step in |error| / step of all cases; the squares are
    |error| * step <= |error| * 2 h |x|, so the rounded results differ by sqrt(2 h r), with r <= C.
  * Independent roundings of at most h have a root mean square of h / sqrt(3) at most, and their squares add.  d_queries and
    d_keys read the kept states in one term: two, their own one and the states', h sqrt(2 / 3).  out reads the state and P
    in one term: three, h.
  * d_log_gates sums such products over a chunk, and they cancel: twice that.
  * a row (a token of a head) by itself: the roundings at their most, of what the row holds and of what rows hold in the mean,
    since terms that cancel in one row are of that size.  Elements of d_betas and d_log_gates likewise; a running sum of up to 64
    normal errors stays within four times its root mean square.
  * float32 gates beside bf16 tensors: d_betas is not rounded, C.
"""
import pytest
import torch

from accelerated_scan import delta
from test_delta import CARRIED, inputs, off, reference

H = 2.0 ** -8
ROUNDED = (2 * H * CARRIED) ** 0.5
TWO, THREE = H * (2 / 3) ** 0.5 + CARRIED, H + CARRIED
NAMES = "queries keys values log_gates betas state".split()
SHAPES = [(2, 200, 2, 4, 128, 128), (2, 130, 1, 2, 64, 72), (1, 190, 2, 2, 100, 200)]


def rows_off(got, want, roundings):
    """The worst row's error over its bound."""
    got, want = got.double(), want.double()
    norm = want.norm(dim=-1)
    return ((got - want).norm(dim=-1) / (roundings * H * (norm + norm.square().mean().sqrt()))).max().item()


def run(args, seed=3):
    leaves = [t.requires_grad_(True) for t in args if t is not None]
    want = reference(*args)
    g = torch.Generator().manual_seed(seed)
    d = [torch.randn(t.shape, generator=g).to(x).to(t.device) for t, x in zip(want, (args[2].dtype, torch.float32))]
    got = delta.scan(*args)
    return got, want, torch.autograd.grad(got, leaves, d), torch.autograd.grad(want, leaves, [t.double() for t in d])


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_bf16(cuda_device, shape):
    got, want, got_g, want_g = run(inputs(sum(shape), *shape, torch.bfloat16, cuda_device))
    assert off(got[0], want[0]) <= THREE and rows_off(got[0], want[0], 3) <= 1
    assert off(got[1], want[1]) <= CARRIED
    for name, a, b in zip(NAMES, got_g, want_g):
        if name in ("values", "betas"):
            assert off(a, b.bfloat16()) <= ROUNDED, name
        elif name != "state":
            assert off(a, b) <= TWO * (2 if name == "log_gates" else 1), name
        else:
            assert off(a, b) <= CARRIED
        if name in ("queries", "keys", "values"):
            assert rows_off(a, b, 1 if name == "values" else 2) <= 1, name
        elif name in ("betas", "log_gates"):
            bound = (1 if name == "betas" else 4 * 2) * H * (b.abs() + b.square().mean().sqrt())
            assert ((a.double() - b).abs() <= bound).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_float32_gates(cuda_device, shape, dtype):
    got, want, got_g, want_g = run(inputs(sum(shape) + 1, *shape, dtype, cuda_device, gate_dtype=torch.float32))
    assert off(got_g[4], want_g[4]) <= CARRIED
    assert off(got_g[3], want_g[3]) <= (2 * H / 3 ** 0.5 if dtype == torch.bfloat16 else 2 * CARRIED)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_every_row(cuda_device, shape, dtype):
    """fp32 and fp16: what test_delta.py asks of the whole, of every row against the rows' mean."""
    tol = CARRIED + (2.0 ** -11 if dtype == torch.float16 else 0)
    got, want, got_g, want_g = run(inputs(sum(shape) + 2, *shape, dtype, cuda_device))
    for name, a, b in zip(["out", *NAMES], [got[0], *got_g], [want[0], *want_g]):
        if name in ("out", "queries", "keys", "values"):
            assert rows_off(a, b, tol / H) <= 1, name


def scan_off(args, tol_out, tol_state):
    out, s = delta.scan(*args)
    want, want_s = reference(*args)
    assert off(out, want) <= tol_out and off(s, want_s) <= tol_state


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_log_gates_above_zero(cuda_device, dtype):
    """States that grow and shrink by factors of e^0.3 a token, forward and backward."""
    args = inputs(31, 2, 200, 1, 2, 64, 64, dtype, cuda_device)
    args[3] = 0.3 * torch.randn(args[3].shape, generator=torch.Generator().manual_seed(5)).to(dtype).to(cuda_device)
    got, want, got_g, want_g = run(args)
    tol = {torch.bfloat16: THREE, torch.float16: 2.0 ** -11 + CARRIED, torch.float32: CARRIED}[dtype]
    assert off(got[0], want[0]) <= tol and off(got[1], want[1]) <= CARRIED
    for name, a, b in zip(NAMES, got_g, want_g):
        assert off(a, b) <= (CARRIED if name == "state" else tol) * (2 if name == "log_gates" else 1), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fall,rise", [(10, 20), (18, 30), (3, 60), (50, 70)])
def test_a_fall_and_a_rise(cuda_device, dtype, fall, rise):
    """A log gate of -70, one of 70 later on, nothing written between: the state is what it was, in one block of 16 tokens, over
    several, and over a chunk's end."""
    args = inputs(32, 1, 100, 1, 2, 64, 64, dtype, cuda_device)
    args[3][:, fall], args[3][:, rise] = -70.0, 70.0
    args[4][:, fall:rise] = 0
    scan_off(args, THREE if dtype == torch.bfloat16 else CARRIED, CARRIED)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("beta", [0.5, 1.0, 1.5, 2.0])
def test_keys_that_are_alike(cuda_device, dtype, beta):
    """The same key over and over, without decay, as padding or repeated text gives.  N = L' (I + L')^-1 for L' = beta below the
    diagonal has the entries beta (1 - beta)^(i - j - 1); a product with it is off by C of |N| |x|, and a row of |N| over a chunk
    of 64 sums to at most beta / (1 - |1 - beta|), 64 * 2 for a rate of 2: 1, 1, 3 and 128."""
    args = inputs(33, 1, 150, 1, 2, 64, 64, dtype, cuda_device)
    args[1] = args[1][:, :1].expand_as(args[1]).contiguous()
    args[1].div_(args[1].float().norm(dim=-1, keepdim=True))
    args[3].zero_()
    args[4].fill_(beta)
    carried = CARRIED * {0.5: 1, 1.0: 1, 1.5: 3, 2.0: 128}[beta]
    scan_off(args, {torch.bfloat16: H, torch.float16: 2.0 ** -11, torch.float32: 0.0}[dtype] + carried, carried)
