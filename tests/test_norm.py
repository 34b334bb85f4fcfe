"""Norms around a block (norm.residual_norm, norm.gated_norm) against 64 bits.

Tolerances, as 2-norm of the error over 2-norm of the result: the output's own rounding, half of finfo.eps, and sums of
at most 2^13 terms in fp32, by halves: 16 * 2^-24.
"""
import pytest
import torch

from accelerated_scan import norm

SUMS = 16 * 2.0 ** -24


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


def tol(dtype):
    return torch.finfo(dtype).eps / 2 + SUMS


def reference(x, residual, gate, post, scale, pre, act, eps=1e-6):
    up = lambda t: t.double() if isinstance(t, torch.Tensor) else t
    x, residual, gate, post, scale, pre = map(up, (x, residual, gate, post, scale, pre))
    rms = lambda t: t * (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x if post is None else rms(x) * post
    if gate is not None:
        s = torch.sigmoid(gate)
        n = n * {"sigmoid": s, "silu": gate * s, None: gate}[act]
    h = n * (1.0 if scale is None else scale) + (0 if residual is None else residual)
    return h if pre is None else (h, rms(h) * pre)


def inputs(seed, shape, dtype, weights, device, residual=True, gate=True, post=True, scale=True, pre=True):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)
    D = shape[-1]
    row = lambda use: rand(*shape).to(dtype).to(device) if use else None
    vec = lambda use: (1 + 0.1 * rand(D)).to(weights).to(device) if use else None
    return [row(True), row(residual), row(gate), vec(post), vec(scale), vec(pre)]


def call(x, residual, gate, post, scale, pre, act, **kw):
    return norm.residual_norm(x, residual, post_weight=post, gate=gate, scale=scale, pre_weight=pre, activation=act, **kw)


def off(got, want):
    assert got.shape == want.shape and torch.isfinite(got).all()
    n = want.double().norm().item()
    return (got.double() - want.double()).norm().item() / n if n else got.double().norm().item()


SHAPES = [(1, 1), (3, 7), (2, 5, 8), (17, 64), (1000, 128), (9, 130), (33, 256), (7, 520), (5, 1537), (300, 2048), (3, 4096), (4, 4104),
          (2, 4099), (5, 8192), (2, 8191)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,weights", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                           (torch.float16, torch.float16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(cuda_device, shape, dtype, weights):
    args = inputs(sum(shape), shape, dtype, weights, cuda_device)
    leaves = [t.requires_grad_(True) for t in args]
    hidden, normed = call(*args, "silu")
    want_h, want_y = reference(*args, "silu")
    assert hidden.dtype == normed.dtype == dtype
    assert off(hidden, want_h) <= tol(dtype) and off(normed, want_y) <= tol(dtype)
    dh, dy = torch.randn_like(hidden), torch.randn_like(normed)
    got = torch.autograd.grad([hidden, normed], leaves, [dh, dy])
    want = torch.autograd.grad([want_h, want_y], leaves, [dh.double(), dy.double()])
    for name, a, b, x in zip(("x", "residual", "gate", "post", "scale", "pre"), got, want, leaves):
        assert a.dtype == x.dtype and a.shape == x.shape
        # differences of two sums in the gradients of a norm, and rows that cancel in the weights': 4 times the sums
        if shape[-1] == 1:
            # A row of one element: the gradient of h r(h) is r (1 - h^2 r^2), and 1 - h^2 r^2 = eps r^2 is the difference of
            # two numbers near 1, each off by a few 2^-24.  So the error is held against the terms of the difference: dh + 2
            # dy w / |h| for hidden, then the factors that lead from hidden to the input (|n| <= |w|, slope of silu <= 1.1)
            z, w, c, q = (args[i].detach().double().abs() for i in (2, 3, 4, 5))
            terms = dh.double().abs() + 2 * dy.double().abs() * q / want_h.detach().double().abs()
            terms = terms * {"x": 2 * z * c * w / args[0].detach().double().abs(), "residual": 1, "gate": 1.1 * c * w, "post": z * c,
                             "scale": z * w, "pre": 1}[name]
            assert ((a.double() - b).abs() <= 4 * SUMS * terms.view_as(b) + torch.finfo(x.dtype).eps / 2 * b.abs()).all(), name
            continue
        assert off(a, b) <= torch.finfo(x.dtype).eps / 2 + 4 * SUMS, name


@pytest.mark.gpu
@pytest.mark.parametrize("use", range(32))
@pytest.mark.parametrize("act", ["sigmoid", "silu", None])
def test_every_choice_of_parts(cuda_device, use, act):
    parts = dict(zip(("residual", "gate", "post", "scale", "pre"), (bool(use >> i & 1) for i in range(5))))
    args = inputs(use, (37, 200), torch.float32, torch.float32, cuda_device, **parts)
    leaves = [t.requires_grad_(True) for t in args if t is not None]
    got, want = call(*args, act), reference(*args, act)
    got, want = (got, want) if parts["pre"] else ((got,), (want,))
    d = [torch.randn_like(t) for t in got]
    for a, b in zip(got, want):
        assert off(a, b) <= tol(torch.float32)
    for a, b in zip(torch.autograd.grad(got, leaves, d), torch.autograd.grad(want, leaves, [t.double() for t in d])):
        assert off(a, b) <= 2.0 ** -24 + 4 * SUMS


@pytest.mark.gpu
def test_one_gradient_at_a_time_and_a_number_as_scale(cuda_device):
    args = inputs(1, (21, 96), torch.float32, torch.float32, cuda_device)
    args[4] = 0.37
    want = reference(*args, "sigmoid")
    for which in range(2):
        for i in (0, 1, 2, 3, 5):
            x = args[i].detach().requires_grad_(True)
            moved = [x if j == i else t for j, t in enumerate(args)]
            got = call(*moved, "sigmoid")
            assert off(got[0], want[0]) <= tol(torch.float32)
            if which == 0 and i == 5:
                continue                                      # hidden does not depend on pre_weight
            d = torch.randn_like(got[which])
            a, = torch.autograd.grad(got[which], x, d)
            b, = torch.autograd.grad(reference(*moved, "sigmoid")[which], x, d.double())
            assert off(a, b) <= 2.0 ** -24 + 4 * SUMS


@pytest.mark.gpu
def test_strides(cuda_device):
    """Slices of a projection, odd offsets, transposed rows, an expanded gradient."""
    wide = torch.randn(50, 3 * 128, device=cuda_device).bfloat16()
    x, gate, res = (wide[:, i * 128:(i + 1) * 128] for i in range(3))
    w = torch.rand(128, device=cuda_device).bfloat16()
    want = norm.residual_norm(x.contiguous(), res.contiguous(), post_weight=w, gate=gate.contiguous(), pre_weight=w)
    got = norm.residual_norm(x, res, post_weight=w, gate=gate, pre_weight=w)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    heads = wide[:, :256].view(50, 2, 128)
    assert torch.equal(norm.gated_norm(heads, heads, w), norm.gated_norm(heads.contiguous(), heads.contiguous(), w))
    t = x.t().contiguous().t()
    assert torch.equal(norm.gated_norm(t, gate, w), norm.gated_norm(x.contiguous(), gate.contiguous(), w))
    odd = torch.empty(50 * 128 + 1, dtype=torch.bfloat16, device=cuda_device)[1:].view(50, 128)
    odd.copy_(x)
    got = norm.residual_norm(odd, res, post_weight=w, gate=gate, pre_weight=w)
    for a, b in zip(got, want):                               # another order of the sums: both within a rounding
        assert off(a, b) <= 2 * tol(torch.bfloat16)
    leaf = x.contiguous().requires_grad_(True)
    a, = torch.autograd.grad(norm.gated_norm(leaf, gate, w).sum(), leaf)
    b, = torch.autograd.grad(norm.gated_norm(leaf, gate, w), leaf, torch.ones_like(leaf))
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_extreme_values(cuda_device):
    x = torch.zeros(4, 64, device=cuda_device)
    x[1] = 1e18
    x[2] = 1e-18
    gate = torch.full_like(x, float("-inf"))
    w = torch.ones(64, device=cuda_device)
    res = torch.randn_like(x)
    h, y = norm.residual_norm(x, res, post_weight=w, gate=gate, pre_weight=w, activation="sigmoid")
    assert torch.equal(h, res) and torch.isfinite(y).all()     # a closed gate adds nothing
    assert (norm.residual_norm(x[:1], post_weight=w) == 0).all()
    x[3, 5] = float("nan")
    got = norm.residual_norm(x, res, post_weight=w)
    assert torch.isnan(got[3]).all() and torch.isfinite(got[:3]).all()


@pytest.mark.gpu
def test_results_repeat_and_captured_graph(cuda_device):
    args = inputs(2, (4000, 256), torch.bfloat16, torch.float32, cuda_device)
    leaves = [t.requires_grad_(True) for t in args]

    def train():
        h, y = call(*args, "sigmoid")
        got = [h, y, *torch.autograd.grad([h, y], leaves, [torch.ones_like(h), torch.ones_like(y)])]
        return [t.detach() for t in got]       # no graph of these leaves is left when the backward is captured

    want = train()
    assert all(torch.equal(a, b) for a, b in zip(train(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = train()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_no_rows(cuda_device):
    args = inputs(3, (0, 64), torch.float32, torch.float32, cuda_device)
    leaves = [t.requires_grad_(True) for t in args]
    h, y = call(*args, "silu")
    assert h.shape == y.shape == (0, 64)
    grads = torch.autograd.grad([h, y], leaves, [torch.ones_like(h), torch.ones_like(y)])
    assert all((g == 0).all() and g.shape == t.shape for g, t in zip(grads, leaves))


@pytest.mark.gpu
def test_a_recurrent_layer(cuda_device):
    """The operators as a layer uses them: norm, projections, the delta rule, each head's gated norm, projection, residual and the
    next norm; outputs and gradients against 64 bits.  Nine roundings to bf16 lie between input and result."""
    from accelerated_scan import delta
    from test_delta import reference as delta_reference

    B, T, E, Hk, H, K, V = 2, 100, 96, 1, 2, 64, 64
    g = torch.Generator().manual_seed(4)
    rand = lambda *s: (torch.randn(*s, generator=g) * s[0] ** -0.5)
    sizes = [Hk * K, Hk * K, H * V, H * V, H, H]
    values = {"x": torch.randn(B, T, E, generator=g), "residual": torch.randn(B, T, E, generator=g), "w_in": rand(E, sum(sizes)),
              "w_out": rand(H * V, E), "n1": 1 + 0.1 * torch.randn(E, generator=g), "n2": 1 + 0.1 * torch.randn(E, generator=g),
              "n3": 1 + 0.1 * torch.randn(V, generator=g), "c": 0.5 + 0.1 * torch.randn(E, generator=g)}
    leaves = {n: t.to(torch.bfloat16).to(cuda_device).requires_grad_(True) for n, t in values.items()}

    def layer(p, ours):
        rn = (lambda x, r, **k: norm.residual_norm(x, r, **k)) if ours else (
            lambda x, r, post_weight=None, gate=None, scale=None, pre_weight=None, activation="sigmoid":
            reference(x, r, gate, post_weight, scale, pre_weight, activation))
        h, y = rn(p["x"], p["residual"], scale=p["c"], pre_weight=p["n1"])
        q, k, v, z, a, b = (y @ p["w_in"]).split(sizes, -1)
        unit = lambda t: torch.nn.functional.normalize(t.unflatten(-1, (Hk, K)), dim=-1)
        gates = -torch.nn.functional.softplus(a.float() if ours else a) * 0.1
        v, z = v.unflatten(-1, (H, V)), z.unflatten(-1, (H, V))
        beta = torch.sigmoid(b)
        o = (delta.scan if ours else delta_reference)(unit(q), unit(k), v, gates, beta)[0]
        o = norm.gated_norm(o, z, p["n3"]) if ours else reference(o, None, z, p["n3"], None, None, "silu")
        return rn(o.flatten(2) @ p["w_out"], h, post_weight=p["n2"], scale=p["c"], pre_weight=p["n1"])

    got = layer(leaves, True)
    want = layer({n: t.double() for n, t in leaves.items()}, False)
    d = [torch.randn_like(t) for t in got]
    for a, b in zip(got, want):
        assert off(a, b) <= 9 * 2.0 ** -8
    got_g = torch.autograd.grad(got, list(leaves.values()), d)
    want_g = torch.autograd.grad(want, list(leaves.values()), [t.double() for t in d])
    for n, a, b in zip(leaves, got_g, want_g):
        assert off(a, b) <= 18 * 2.0 ** -8, n                 # forward and backward


def test_refusals():
    x = torch.randn(4, 16)
    w = torch.ones(16)
    with pytest.raises(RuntimeError):
        norm.residual_norm(x, pre_weight=w)                   # no CPU path
    for kw in ({"residual": x[:3]}, {"gate": x[:, :8]}, {"pre_weight": w[:8]}, {"scale": x}):
        with pytest.raises(AssertionError):
            norm.residual_norm(x, **kw)
    for kw in ({"residual": x.bfloat16()}, {"pre_weight": w.bfloat16()}, {"post_weight": w, "pre_weight": w.double()}):
        with pytest.raises(RuntimeError):
            norm.residual_norm(x, **kw)
    with pytest.raises(RuntimeError):
        norm.residual_norm(x.double())
    with pytest.raises(RuntimeError):
        norm.residual_norm(torch.zeros(1, 8193))
    with pytest.raises(RuntimeError):
        norm.residual_norm(torch.zeros(1, 0))
    with pytest.raises(ValueError):
        norm.residual_norm(x, gate=x, activation="tanh")


def test_bad_arguments_of_the_c_entries():
    import ctypes
    from accelerated_scan import _native

    a = _native.Norm()
    fake = ctypes.c_void_p(256)
    forward = lambda: _native.lib.ascan_norm_forward(ctypes.byref(a), fake, fake, None)
    a.rows, a.dim, a.x = 4, 16, 256
    for name, value, rc in (("rows", -1, 1), ("dim", 0, 1), ("dim", 8193, 2), ("dtype", 3, 1), ("weights_dtype", 1, 1),
                            ("activation", 3, 1), ("x", None, 1)):
        before = getattr(a, name)
        setattr(a, name, value)
        assert forward() == rc, name
        setattr(a, name, before)
    a.pre_weight = 256
    assert _native.lib.ascan_norm_forward(ctypes.byref(a), fake, None, None) == 1
    need = _native.lib.ascan_norm_backward_bytes(ctypes.byref(a))
    assert need > 0
    back = lambda ws, n: _native.lib.ascan_norm_backward(ctypes.byref(a), fake, 16, fake, 16, fake, None, None, None, None, fake, ws, n,
                                                         None)
    assert back(None, need) == 5 and back(fake, need - 1) == 5
    a.rows = 0
    assert forward() == 0
