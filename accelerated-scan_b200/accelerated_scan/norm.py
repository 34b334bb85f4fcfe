"""Norms before and after a block, fused with the block's gate and residual scale.

    hidden, normed = norm.residual_norm(block_out, residual, post_weight=..., gate=..., scale=..., pre_weight=...)
    y = norm.gated_norm(x, gate, weight)

A block of a recurrent model reads rms_norm(hidden) and adds its output to `hidden`; around the scan itself a model
norms each head's output and multiplies it by an activated gate.  As separate operations each of these is a pass over
the (..., D) tensors; here one kernel reads the inputs once and writes the results once, and one kernel computes all
gradients (a second, small one adds up those of the weights).  Sums are held in float32.
"""
import torch

from . import _native

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_ACTIVATIONS = {None: 0, "sigmoid": 1, "silu": 2}
MAX_DIM = 8192


def _rows(t, D):
    """(rows, D) with dense rows; a view where the strides allow one."""
    if t is None:
        return None
    if t.dim() == 2 and (t.stride(1) == 1 or D == 1):
        return t
    try:
        r = t.view(-1, D) if t.numel() else t.reshape(-1, D)
    except RuntimeError:
        r = t.reshape(-1, D)
    return r if r.stride(1) == 1 or D == 1 else r.contiguous()


def _forward(rows, vectors, shape, activation, eps):
    """rows: block_out, residual, gate; vectors: post_weight, scale, pre_weight."""
    x = rows[0]
    hidden = torch.empty(shape, dtype=x.dtype, device=x.device)
    normed = None if vectors[2] is None else torch.empty(shape, dtype=x.dtype, device=x.device)
    if x.shape[0]:
        _native.norm_forward(_native.norm_args(*rows, *vectors, activation, eps), x.device, hidden, normed)
    return (hidden, normed) if normed is not None else hidden


def _dense(x, residual, gate, post_weight, scale, pre_weight):
    D = x.shape[-1]
    return ((_rows(x, D), _rows(residual, D), _rows(gate, D)),
            tuple(w.contiguous() if isinstance(w, torch.Tensor) else w for w in (post_weight, scale, pre_weight)))


class ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gate, post_weight, scale, pre_weight, activation, eps):
        rows, vectors = _dense(x, residual, gate, post_weight, scale, pre_weight)
        ctx.save_for_backward(*rows, vectors[0], vectors[1] if isinstance(scale, torch.Tensor) else None, vectors[2])
        ctx.scale_value = None if isinstance(scale, torch.Tensor) else scale
        ctx.activation, ctx.eps, ctx.shape = activation, eps, x.shape
        ctx.set_materialize_grads(False)
        return _forward(rows, vectors, x.shape, activation, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_hidden, d_normed=None):
        x, residual, gate, post_weight, scale, pre_weight = ctx.saved_tensors
        if d_hidden is None and d_normed is None:
            return (None,) * 8
        D = x.shape[-1]
        # saved-tensor hooks may hand back equal tensors that lie in memory in another way
        x, residual, gate = _rows(x, D), _rows(residual, D), _rows(gate, D)
        post_weight, scale, pre_weight = (None if w is None else w.contiguous() for w in (post_weight, scale, pre_weight))
        need = ctx.needs_input_grad
        new = lambda t: torch.empty(ctx.shape, dtype=t.dtype, device=t.device)
        d_x = new(x)
        d_residual = new(residual) if need[1] else None
        d_gate = new(gate) if need[2] else None
        d_vectors = [torch.empty_like(w) if n else None for w, n in zip((post_weight, scale, pre_weight), need[3:6])]
        a = _native.norm_args(x, residual, gate, post_weight, scale if ctx.scale_value is None else ctx.scale_value, pre_weight,
                              ctx.activation, ctx.eps)
        _native.norm_backward(a, x.device, _rows(d_hidden, D), _rows(d_normed, D), d_x, d_residual, d_gate, *d_vectors)
        return d_x, d_residual, d_gate, *d_vectors, None, None


def residual_norm(block_out, residual=None, *, post_weight=None, gate=None, scale=None, pre_weight=None, activation="sigmoid",
                  eps=1e-6):
    """hidden = residual + scale * act(gate) * rms_norm(block_out) * post_weight;  normed = rms_norm(hidden) * pre_weight.

    Arguments:
        block_out (torch.Tensor): (..., D), CUDA; float32, bfloat16 or float16; D up to 8192.
        residual, gate (torch.Tensor, optional): same shape and dtype.
        post_weight, pre_weight (torch.Tensor, optional): (D,), of that dtype or float32 (the vectors all alike).  Without
            post_weight block_out is not normed; without pre_weight only `hidden` is computed.
        scale (float or torch.Tensor, optional): factor of the block's contribution, 1 if None; a (D,) tensor is a learned one
            per channel.
        activation (str, optional): "sigmoid", "silu" (gate * sigmoid(gate)), or None for the gate as it is.

    Differentiable in reverse mode, once; a forward-mode tangent is refused.

    Returns:
        hidden, or (hidden, normed) where pre_weight is given; normed is computed from hidden before its rounding.
    """
    x = block_out
    assert x.dim() >= 1, "block_out must have shape (..., D)"
    D = x.shape[-1]
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"unsupported dtype {x.dtype}: expected float32, bfloat16 or float16")
    if not 1 <= D <= MAX_DIM:
        raise RuntimeError(f"rows of {D} elements: expected 1 to {MAX_DIM}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}: expected 'sigmoid', 'silu' or None")
    for t in (residual, gate):
        if t is not None:
            assert t.shape == x.shape, "residual and gate must have the shape of block_out"
            if t.dtype != x.dtype:
                raise RuntimeError("block_out, residual and gate must have the same dtype")
    vectors = [w for w in (post_weight, scale, pre_weight) if isinstance(w, torch.Tensor)]
    for w in vectors:
        assert w.shape == (D,), "weights and a scale per channel must have shape (D,)"
        if w.dtype not in (x.dtype, torch.float32) or w.dtype != vectors[0].dtype:
            raise RuntimeError("weights and scale must all be of block_out's dtype or all float32")
    _native.refuse_tangents("residual_norm", x, residual, gate, *vectors)
    if not x.is_cuda:
        raise RuntimeError("tensors must be CUDA tensors")
    for t in (residual, gate, *vectors):
        if t is not None and t.device != x.device:
            raise RuntimeError("all tensors must be on the same device")
    if not isinstance(scale, torch.Tensor):
        scale = 1.0 if scale is None else float(scale)
    act, eps = _ACTIVATIONS[activation], float(eps)
    if torch.is_grad_enabled() and any([isinstance(t, torch.Tensor) and t.requires_grad
                                        for t in (x, residual, gate, post_weight, scale, pre_weight)]):
        return ResidualNorm.apply(x, residual, gate, post_weight, scale, pre_weight, act, eps)
    return _forward(*_dense(x, residual, gate, post_weight, scale, pre_weight), x.shape, act, eps)


def gated_norm(x, gate, weight, activation="silu", eps=1e-6):
    """rms_norm(x) * weight * act(gate) over the last dimension: the output norm of a head with its gate."""
    return residual_norm(x, post_weight=weight, gate=gate, activation=activation, eps=eps)
