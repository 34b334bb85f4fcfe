"""Gated delta rule: a recurrence with a matrix-valued state.

    out, state = delta.scan(queries, keys, values, log_gates, betas, initial_state)      # whole sequences, in chunks
    out = delta.step(queries, keys, values, log_gates, betas, state, slots)              # one token, states in place

Per token, with the K x V state S of a head (float32):

    S = exp(log_gate) * S                      # the gate, as in `warp.scan`, here for a whole matrix
    e = value - S^T key                        # what the state does not yet answer for this key
    S = S + beta * key e^T
    out = scale * S^T query

The reference's recurrence carries one number per channel (warp.py:68-83); this one carries a K x V matrix per head and
writes to it by a rank-one correction.  `scan` is differentiable in every input and in the initial state, and takes
sequences of different lengths packed into one row; `step` is its form for serving, where the states of all requests lie
in one pool.
"""
import torch

from . import _native

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
MAX_KEY_DIM, MAX_VALUE_DIM = 128, 1024


def _check_inputs(lead, queries, keys, values, log_gates, betas, state):
    """lead: names of the dimensions before the heads."""
    n = len(lead)
    assert queries.dim() == n + 2, f"queries must have shape ({', '.join(lead)}, key heads, K)"
    assert keys.shape == queries.shape, "queries and keys must have the same shape"
    assert values.dim() == n + 2 and values.shape[:n] == queries.shape[:n], f"values must have shape ({', '.join(lead)}, heads, V)"
    heads_k, K = queries.shape[n:]
    heads, V = values.shape[n:]
    _native.refuse_tangents("the gated delta rule", queries, keys, values, log_gates, betas, state)
    assert heads_k > 0 and heads > 0 and heads % heads_k == 0, "the value heads must be a multiple of the key heads"
    assert log_gates.shape == values.shape[:n + 1], f"log_gates must have shape ({', '.join(lead)}, heads)"
    assert betas.shape == values.shape[:n + 1], f"betas must have shape ({', '.join(lead)}, heads)"
    if not 1 <= K <= MAX_KEY_DIM or not 1 <= V <= MAX_VALUE_DIM:
        raise RuntimeError(f"key dimension {K} and value dimension {V}: expected 1 to {MAX_KEY_DIM} and 1 to {MAX_VALUE_DIM}")
    if queries.dtype not in _DTYPES:
        raise RuntimeError(f"unsupported dtype {queries.dtype}: expected float32, bfloat16 or float16")
    dtype, device = queries.dtype, queries.device
    if keys.dtype != dtype or values.dtype != dtype:
        raise RuntimeError("queries, keys and values must have the same dtype")
    if log_gates.dtype not in (dtype, torch.float32) or betas.dtype not in (dtype, torch.float32):
        raise RuntimeError("log_gates and betas must be float32 or of the queries' dtype")
    if not queries.is_cuda:
        raise RuntimeError("tensors must be CUDA tensors")
    if keys.device != device or values.device != device or log_gates.device != device or betas.device != device:
        raise RuntimeError("all tensors must be on the same device")


def _dense_last(t):
    """Rows of the last dimension as they lie in memory; other strides are free."""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _forward(queries, keys, values, log_gates, betas, initial_state, scale, seq_starts, keep):
    B, T, _, K = queries.shape
    H, V = values.shape[2:]
    n = B if seq_starts is None else seq_starts.shape[0] - 1
    out = torch.empty(B, T, H, V, dtype=values.dtype, device=values.device)
    state = torch.empty(n, H, K, V, dtype=torch.float32, device=values.device)
    kept, packed = None, 0
    if n:
        args = _native.delta_args(queries, keys, values, log_gates, betas, initial_state, scale, seq_starts)
        kept, packed = _native.delta_forward(args, values.device, out, state, keep)
    return out, state, kept, packed


class DeltaScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, queries, keys, values, log_gates, betas, initial_state, scale, seq_starts):
        queries, keys, values = _dense_last(queries), _dense_last(keys), _dense_last(values)
        s0 = None if initial_state is None else initial_state.float().contiguous()
        out, state, kept, packed = _forward(queries, keys, values, log_gates, betas, s0, scale, seq_starts, True)
        ctx.save_for_backward(queries, keys, values, log_gates, betas, s0, seq_starts, kept)
        ctx.scale, ctx.packed = scale, packed
        ctx.state_dtype = None if initial_state is None else initial_state.dtype
        ctx.set_materialize_grads(False)
        return out, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out, d_state):
        queries, keys, values, log_gates, betas, s0, seq_starts, kept = ctx.saved_tensors
        # saved-tensor hooks may hand back equal tensors that lie in memory in another way
        queries, keys, values = _dense_last(queries), _dense_last(keys), _dense_last(values)
        s0 = None if s0 is None else s0.contiguous()
        if d_out is None:
            d_out = torch.zeros((), dtype=values.dtype, device=values.device).expand(values.shape)
        d_out = _dense_last(d_out)
        d_state = None if d_state is None else d_state.contiguous()
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (queries, keys, values, log_gates, betas)]
        d_s0 = None
        if s0 is not None and ctx.needs_input_grad[5]:
            d_s0 = torch.empty_like(s0)
        if kept is not None:
            args = _native.delta_args(queries, keys, values, log_gates, betas, s0, ctx.scale, seq_starts, ctx.packed)
            _native.delta_backward(args, values.device, d_out, d_state, grads, d_s0, kept)
        if d_s0 is not None:
            d_s0 = d_s0.to(ctx.state_dtype)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), d_s0, None, None)


def scan(queries, keys, values, log_gates, betas, initial_state=None, scale=None, seq_starts=None):
    """The gated delta rule over whole sequences.

    Arguments:
        queries, keys (torch.Tensor): (B, T, key heads, K), CUDA; float32, bfloat16 or float16; K up to 128.  Keys are
            used as they are (normalise them before the call).
        values (torch.Tensor): (B, T, heads, V), same dtype; heads is a multiple of the key heads, value head h reads key
            head h // (heads // key heads); V up to 1024.
        log_gates, betas (torch.Tensor): (B, T, heads), of that dtype or float32.  A log gate of -104 or less (-inf too)
            is a gate of zero: the state starts anew.  A token with log gate 0 and beta 0 leaves the state as it is.
        initial_state (torch.Tensor, optional): (sequences, heads, K, V), any real dtype; zeros if None.
        scale (float, optional): factor of the outputs; K ** -0.5 if None.
        seq_starts (torch.Tensor, optional): (N + 1,) int32 or int64 on the GPU, ascending.  B must be 1; sequence i holds
            the tokens seq_starts[i] to seq_starts[i + 1] - 1 and may be empty.  Tokens outside of all sequences get
            zeros in `out`.  The values are read on the device only and are not checked.

    Strides are free but for the last dimension of queries, keys and values, which has to be dense (it is copied if not).

    Precision, as 2-norm of the error over that of the result.  The products are taken on bf16 tensor cores with fp32 sums, and
    operands that are not bf16 as two terms, 2^-16 of each: states and fp32 results are 5e-6 to 1e-5 off (elementary fp32
    operations: 2e-7), fp16 results little more than their rounding, bf16 ones likewise but for `out`, which reads the
    state and the weights within a chunk in one term: 2.4e-3, of which 1.7e-3 is its own rounding.  That is for unit keys and
    rates up to 1.  A rate of 2 reflects the state along its key; the same key over and over, undecayed, then lets the errors
    of a chunk add up (states 4e-3 off from bf16 inputs, 8e-4 from others).

    Log gates above zero let the state grow; where they rise by more than 88 in all, fp32 overflows.  What is not finite makes
    NaN of its whole chunk of 64 tokens, the ones before it too, and of what follows, also behind a beta or a gate of zero:
    padding within a sequence has to hold finite numbers.  Tokens outside of all sequences may hold anything.

    Differentiable in reverse mode, once; a forward-mode tangent is refused.

    Returns:
        out (torch.Tensor): (B, T, heads, V) in the dtype of values
        final_state (torch.Tensor): (sequences, heads, K, V) float32, to hand to the next call
    """
    _check_inputs(("B", "T"), queries, keys, values, log_gates, betas, initial_state)
    B, _, _, K = queries.shape
    H, V = values.shape[2:]
    n = B
    if seq_starts is not None:
        assert B == 1, "packed sequences need B == 1"
        assert seq_starts.dim() == 1 and seq_starts.numel() >= 2, "seq_starts must have shape (sequences + 1,)"
        if seq_starts.dtype not in (torch.int32, torch.int64):
            raise RuntimeError("seq_starts must be int32 or int64")
        if seq_starts.device != queries.device:
            raise RuntimeError("all tensors must be on the same device")
        seq_starts = seq_starts.contiguous()
        n = seq_starts.numel() - 1
    if initial_state is not None:
        assert initial_state.shape == (n, H, K, V), "initial_state must have shape (sequences, heads, K, V)"
        if not initial_state.is_floating_point():
            raise RuntimeError(f"unsupported dtype {initial_state.dtype} of initial_state")
        if initial_state.device != queries.device:
            raise RuntimeError("all tensors must be on the same device")
    scale = K ** -0.5 if scale is None else float(scale)
    if torch.is_grad_enabled() and (queries.requires_grad or keys.requires_grad or values.requires_grad or log_gates.requires_grad
                                    or betas.requires_grad or (initial_state is not None and initial_state.requires_grad)):
        return DeltaScan.apply(queries, keys, values, log_gates, betas, initial_state, scale, seq_starts)
    s0 = None if initial_state is None else initial_state.detach().float().contiguous()
    return _forward(_dense_last(queries), _dense_last(keys), _dense_last(values), log_gates, betas, s0, scale, seq_starts, False)[:2]


def step(queries, keys, values, log_gates, betas, state, slots=None, scale=None):
    """One token of the gated delta rule for a batch of sequences; their states are updated in place.

    Arguments:
        queries, keys (torch.Tensor): (B, key heads, K); values: (B, heads, V); log_gates, betas: (B, heads), as in `scan`.
        state (torch.Tensor): (pool, heads, K, V) float32; dense but for its first stride.
        slots (torch.Tensor, optional): (B,) int32 or int64 on the GPU: row b continues state[slots[b]].  None means
            slot b for row b.  A negative slot is a padded row: its output is zero.  A slot behind the pool, and a slot
            that an earlier row of the batch has, change nothing and answer NaN.
        scale (float, optional): factor of the outputs; K ** -0.5 if None.

    Returns:
        out (torch.Tensor): (B, heads, V).  Not differentiable; use `scan` to train.
    """
    _check_inputs(("B",), queries, keys, values, log_gates, betas, state)
    B, _, K = queries.shape
    H, V = values.shape[1:]
    assert state.dim() == 4 and state.shape[1:] == (H, K, V), "state must have shape (pool, heads, K, V)"
    if state.dtype != torch.float32:
        raise RuntimeError("state must be float32")
    if state.device != queries.device:
        raise RuntimeError("all tensors must be on the same device")
    if not state.is_contiguous() and state.shape[0] and (
            not state[0].is_contiguous() or (state.shape[0] > 1 and state.stride(0) < H * K * V)):
        raise RuntimeError("the states of the pool must be contiguous")
    if slots is None:
        assert state.shape[0] >= B, "without slots the pool needs a state for each row"
    else:
        assert slots.shape == (B,), "slots must have shape (B,)"
        if slots.dtype not in (torch.int32, torch.int64):
            raise RuntimeError("slots must be int32 or int64")
        if slots.device != queries.device:
            raise RuntimeError("all tensors must be on the same device")
        slots = slots.contiguous()
    if torch.is_grad_enabled() and (queries.requires_grad or keys.requires_grad or values.requires_grad or log_gates.requires_grad
                                    or betas.requires_grad or state.requires_grad):
        raise RuntimeError("step is not differentiable: call it under torch.no_grad()")
    out = torch.empty(B, H, V, dtype=values.dtype, device=values.device)
    if B:
        queries, keys, values = _dense_last(queries), _dense_last(keys), _dense_last(values)
        _native.delta_step(queries, keys, values, log_gates, betas, out, state, slots, K ** -0.5 if scale is None else float(scale))
        torch.autograd.graph.increment_version(state)       # written through its pointer: whoever saved it for a backward hears of it
    return out
