"""Timed cases of the operators around a recurrent layer with a matrix-valued state.

`delta.scan`           the gated delta rule over whole sequences, in chunks; forward, and forward + backward
`delta.step`           one token of it for a batch of requests whose states live in a pool
`norm.residual_norm`   h = residual + scale * act(gate) * rms_norm(x) and y = rms_norm(h); forward, and forward + backward

`run` computes them in plain 32-bit torch operations, or through the package where `own` is set.  `exact` computes the
same outputs in 64 bits, token by token.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
CHUNK = 64


def _package():
    """The package lies one folder below the repository's root."""
    path = os.path.join(os.getcwd(), "accelerated-scan_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from accelerated_scan import delta, norm
    return delta, norm


# ---- cases ------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one request decoding by itself: latency
        {"name": "step_one_request", "kind": "step", "type": "bf16", "batch": 1, "pool": 4, "heads_k": 8, "heads": 16,
         "K": 128, "V": 128},
        # a full serving batch, some rows padded: the states' bytes
        {"name": "step_serving_batch", "kind": "step", "type": "bf16", "batch": 128, "pool": 160, "heads_k": 16, "heads": 32,
         "K": 128, "V": 128},
        # a short prompt of one request
        {"name": "scan_short_prompt", "kind": "scan", "type": "bf16", "batch": 1, "T": 77, "seqs": 0, "heads_k": 8,
         "heads": 16, "K": 128, "V": 128, "state": False},
        # prompts of different lengths packed into one row, each continuing from a state
        {"name": "scan_packed_prompts", "kind": "scan", "type": "bf16", "batch": 1, "T": 8192, "seqs": 9, "heads_k": 16,
         "heads": 32, "K": 128, "V": 128, "state": True},
        # full precision, odd sizes: validation of a model
        {"name": "scan_fp32_odd", "kind": "scan", "type": "fp32", "batch": 2, "T": 1001, "seqs": 0, "heads_k": 8, "heads": 8,
         "K": 64, "V": 96, "state": True},
        # a batch of long documents
        {"name": "scan_long_batch", "kind": "scan", "type": "bf16", "batch": 4, "T": 16384, "seqs": 0, "heads_k": 16,
         "heads": 32, "K": 128, "V": 128, "state": False},
        # truncated backpropagation of a small model: state in, gradient of the state out
        {"name": "train_small_model", "kind": "train", "type": "fp16", "batch": 2, "T": 511, "seqs": 0, "heads_k": 4,
         "heads": 4, "K": 64, "V": 64, "state": True},
        # a training micro-batch
        {"name": "train_micro_batch", "kind": "train", "type": "bf16", "batch": 4, "T": 4096, "seqs": 0, "heads_k": 8,
         "heads": 16, "K": 128, "V": 128, "state": False},
        # the residual stream of a few decoding requests: latency
        {"name": "norm_decode", "kind": "norm", "type": "bf16", "weights": "bf16", "rows": 4, "D": 2048, "residual": True,
         "post": True, "gate": False, "scale": True, "pre": True, "act": "sigmoid"},
        # between two blocks of a long prompt: both norms, the gate and the residual
        {"name": "norm_prefill", "kind": "norm", "type": "bf16", "weights": "fp32", "rows": 32768, "D": 4096,
         "residual": True, "post": True, "gate": True, "scale": True, "pre": True, "act": "sigmoid"},
        # full precision, odd sizes, every gradient
        {"name": "norm_train_fp32_odd", "kind": "norm_train", "type": "fp32", "weights": "fp32", "rows": 1023, "D": 1537,
         "residual": True, "post": True, "gate": True, "scale": True, "pre": True, "act": "silu"},
        # the output norm of each head with its gate, over a training micro-batch
        {"name": "norm_train_heads", "kind": "norm_train", "type": "bf16", "weights": "bf16", "rows": 262144, "D": 128,
         "residual": False, "post": True, "gate": True, "scale": False, "pre": False, "act": "silu"},
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["step", "scan", "scan", "train", "train", "norm", "norm_train"])
    kind_type = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind in ("norm", "norm_train"):
        D = rng.choice([_between(rng, 64, 8192), 8 * _between(rng, 8, 1024)])
        rows = max(1, min(_between(rng, 1, 262144), (1 << 25) // D))
        pre = rng.random() < 0.6
        post = rng.random() < 0.7 or not pre
        return {"kind": kind, "type": kind_type, "weights": rng.choice([kind_type, "fp32"]), "rows": rows, "D": D,
                "residual": pre or rng.random() < 0.5, "post": post, "gate": rng.random() < 0.6,
                "scale": rng.random() < 0.5, "pre": pre, "act": rng.choice(["silu", "sigmoid"])}
    K = rng.choice([64, 128, 128, 8 * rng.randint(2, 16), rng.randint(16, 128)])
    V = rng.choice([64, 128, 128, 8 * rng.randint(2, 24), rng.randint(16, 192)])
    heads_k = rng.choice([1, 2, 3, 4, 8, 16])
    heads = heads_k * rng.choice([1, 1, 2, 4] if heads_k < 16 else [1, 2])
    case = {"kind": kind, "type": kind_type, "heads_k": heads_k, "heads": heads, "K": K, "V": V}
    if kind == "step":
        batch = min(_between(rng, 1, 160), max(1, 4096 // heads))
        case.update(batch=batch, pool=batch + rng.randint(0, 16))
        return case
    batch = rng.choice([1, 1, 2, 3, 4])
    most = 1 << (18 if kind == "scan" else 17)          # tokens times heads
    T = max(1, min(_between(rng, 1, 16384), most // (batch * heads)))
    seqs = rng.randint(2, 12) if batch == 1 and T >= 64 and rng.random() < 0.5 else 0
    case.update(batch=batch, T=T, seqs=seqs, state=rng.random() < 0.5)
    return case


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True)


def _gates(g, *shape):
    """log gates between about -1 and -0.001, write rates in (0, 1)"""
    rate = torch.rand(*shape, generator=g, device="cuda")
    return -torch.exp(7.0 * (rate - 1.0)), torch.sigmoid(_normal(g, *shape))


def _lengths(case, seed):
    """Ragged lengths that fill the row, known to the program that packed them; a function of sizes and seed."""
    import random
    T, n = case["T"], case["seqs"]
    cuts = sorted(random.Random(seed).sample(range(1, T), n - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [T])]


def prepare(case, seed):
    g = _generator(seed)
    t = TYPES[case["type"]]
    st = {"case": case}
    if case["kind"] in ("norm", "norm_train"):
        rows, D, w = case["rows"], case["D"], TYPES[case["weights"]]
        st["x"] = _normal(g, rows, D).to(t)
        st["residual"] = (2.0 * _normal(g, rows, D)).to(t) if case["residual"] else None
        st["gate"] = _normal(g, rows, D).to(t) if case["gate"] else None
        st["post_weight"] = (1.0 + 0.1 * _normal(g, D)).to(w) if case["post"] else None
        st["pre_weight"] = (1.0 + 0.1 * _normal(g, D)).to(w) if case["pre"] else None
        st["scale"] = (0.5 + 0.1 * _normal(g, D)).to(w) if case["scale"] else None
        if case["kind"] == "norm_train":
            st["d_hidden"] = _normal(g, rows, D).to(t)
            st["d_normed"] = _normal(g, rows, D).to(t) if case["pre"] else None
            for name in NORM_LEAVES:
                if st[name] is not None:
                    st[name].requires_grad_(True)
        return st
    B, Hk, H, K, V = (case[n] for n in ("batch", "heads_k", "heads", "K", "V"))
    if case["kind"] == "step":
        st["queries"] = _unit(_normal(g, B, Hk, K)).to(t)
        st["keys"] = _unit(_normal(g, B, Hk, K)).to(t)
        st["values"] = _normal(g, B, H, V).to(t)
        log_gates, betas = _gates(g, B, H)
        st["log_gates"], st["betas"] = log_gates.to(t), betas.to(t)
        st["state"] = 0.3 * _normal(g, case["pool"], H, K, V)
        slots = torch.randperm(case["pool"], generator=g, device="cuda")[:B].to(torch.int32)
        if B > 4:
            slots[torch.rand(B, generator=g, device="cuda") < 0.1] = -1          # padded rows of the batch
        st["slots"] = slots
        return st
    T = case["T"]
    st["queries"] = _unit(_normal(g, B, T, Hk, K)).to(t)
    st["keys"] = _unit(_normal(g, B, T, Hk, K)).to(t)
    st["values"] = _normal(g, B, T, H, V).to(t)
    log_gates, betas = _gates(g, B, T, H)
    st["log_gates"], st["betas"] = log_gates.to(t), betas.to(t)
    st["lengths"], st["seq_starts"], n = None, None, B
    if case["seqs"]:
        st["lengths"] = _lengths(case, seed)
        starts = [0]
        for x in st["lengths"]:
            starts.append(starts[-1] + x)
        st["seq_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        n = case["seqs"]
    st["initial_state"] = 0.3 * _normal(g, n, H, K, V) if case["state"] else None
    if case["kind"] == "train":
        st["d_out"] = _normal(g, B, T, H, V).to(t)
        st["d_state"] = 0.3 * _normal(g, n, H, K, V) if case["state"] else None
        for name in DELTA_LEAVES:
            if st[name] is not None:
                st[name].requires_grad_(True)
    return st


DELTA_LEAVES = ("queries", "keys", "values", "log_gates", "betas", "initial_state")
NORM_LEAVES = ("x", "residual", "gate", "post_weight", "scale", "pre_weight")


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(st):
    kind = st["case"]["kind"]
    if kind == "step":
        if own:
            delta, _ = _package()
            out = delta.step(st["queries"], st["keys"], st["values"], st["log_gates"], st["betas"], st["state"],
                             slots=st["slots"])
        else:
            out = _plain_step(st)
        return {"out": out, "state": st["state"]}
    if kind in ("scan", "train"):
        if own:
            delta, _ = _package()
            out, state = delta.scan(st["queries"], st["keys"], st["values"], st["log_gates"], st["betas"],
                                    st["initial_state"], seq_starts=st["seq_starts"])
        else:
            out, state = _plain_scan(st)
        got = {"out": out, "state": state}
        if kind == "train":
            leaves = [n for n in DELTA_LEAVES if st[n] is not None]
            ends, grads = ([out, state], [st["d_out"], st["d_state"]]) if st["d_state"] is not None else ([out], [st["d_out"]])
            got.update(zip(["d_" + n for n in leaves], torch.autograd.grad(ends, [st[n] for n in leaves], grads)))
        return got
    case = st["case"]
    if own:
        _, norm = _package()
        got = norm.residual_norm(st["x"], st["residual"], post_weight=st["post_weight"], gate=st["gate"],
                                 scale=st["scale"], pre_weight=st["pre_weight"], activation=case["act"])
        hidden, normed = got if case["pre"] else (got, None)
    else:
        hidden, normed = _plain_norm(st)
    got = {"hidden": hidden}
    if normed is not None:
        got["normed"] = normed
    if kind == "norm_train":
        leaves = [n for n in NORM_LEAVES if st[n] is not None]
        ends, grads = ([hidden, normed], [st["d_hidden"], st["d_normed"]]) if case["pre"] else ([hidden], [st["d_hidden"]])
        got.update(zip(["d_" + n for n in leaves], torch.autograd.grad(ends, [st[n] for n in leaves], grads)))
    return got


# ---- plain forms: 32 bits, elementary operations ----------------------------------------------------------------------

def _plain_norm(st):
    case = st["case"]
    x = st["x"].float()
    if st["post_weight"] is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * st["post_weight"].float()
    if st["gate"] is not None:
        z = st["gate"].float()
        s = 1.0 / (1.0 + torch.exp(-z))
        x = x * (z * s if case["act"] == "silu" else s)
    if st["scale"] is not None:
        x = x * st["scale"].float()
    h = x if st["residual"] is None else st["residual"].float() + x
    t = st["x"].dtype
    if st["pre_weight"] is None:
        return h.to(t), None
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * st["pre_weight"].float()
    return h.to(t), y.to(t)


def _plain_step(st):
    q, k, v, g, b = (st[n].float() for n in ("queries", "keys", "values", "log_gates", "betas"))
    group = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    live = st["slots"] >= 0
    at = st["slots"].clamp(min=0).long()
    s = st["state"][at] * torch.exp(g)[..., None, None]
    e = v - (s * k[..., None]).sum(-2)
    s = s + k[..., None] * (b[..., None] * e)[..., None, :]
    out = (s * q[..., None]).sum(-2) * q.shape[-1] ** -0.5
    st["state"].index_copy_(0, at[live], s[live])
    return torch.where(live[:, None, None], out, torch.zeros_like(out)).to(st["values"].dtype)


def _unit_lower_inverse(a):
    """Inverse of unit lower triangular matrices, from blocks of one to blocks of two to ... to the whole."""
    n = a.shape[-1]
    inv = torch.eye(n, device=a.device, dtype=a.dtype).expand(a.shape)
    size = 1
    while size < n:
        blocks = n // (2 * size)
        cut = lambda m: m.reshape(*m.shape[:-2], blocks, 2 * size, blocks, 2 * size).diagonal(dim1=-4, dim2=-2).movedim(-1, -3)
        low, done = cut(a)[..., size:, :size], cut(inv)
        first, second = done[..., :size, :size], done[..., size:, size:]
        corner = -second @ (low @ first)
        whole = torch.cat([torch.cat([first, torch.zeros_like(first)], -1), torch.cat([corner, second], -1)], -2)
        if blocks == 1:
            return whole.squeeze(-3)
        inv = torch.diag_embed(whole.movedim(-3, -1), dim1=-4, dim2=-2).reshape(a.shape)
        size *= 2
    return inv


def _plain_sequence(q, k, v, g, b, s, scale):
    """(B, T, H, ...) in 32 bits, g in 64; s (B, H, K, V)."""
    B, T, H, K = q.shape
    V = v.shape[-1]
    pad = -T % CHUNK
    n = (T + pad) // CHUNK
    def chunks(x):
        x = x.transpose(1, 2)
        if pad:
            x = torch.cat([x, x.new_zeros(B, H, pad, *x.shape[3:])], 2)
        return x.reshape(B, H, n, CHUNK, *x.shape[3:])
    q, k, v, b = chunks(q) * scale, chunks(k), chunks(v), chunks(b)
    G = chunks(g).cumsum(-1)                                              # 64 bits: differences of sums
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~low, -math.inf)).float()
    since, until, whole = torch.exp(G).float(), torch.exp(G[..., -1:] - G).float(), torch.exp(G[..., -1]).float()
    eye = torch.eye(CHUNK, device=q.device)
    T_inv = _unit_lower_inverse(eye + (k @ k.transpose(-1, -2) * decay).tril(-1) * b[..., None, :])
    P = q @ k.transpose(-1, -2) * decay
    U, W = T_inv @ v, T_inv @ (since[..., None] * k)
    q, kt = since[..., None] * q, (until[..., None] * k).transpose(-1, -2)
    outs = []
    for c in range(n):
        u = b[:, :, c, :, None] * (U[:, :, c] - W[:, :, c] @ s)
        outs.append(q[:, :, c] @ s + P[:, :, c] @ u)
        s = whole[:, :, c, None, None] * s + kt[:, :, c] @ u
    out = torch.stack(outs, 2).reshape(B, H, n * CHUNK, V)[:, :, :T]
    return out.transpose(1, 2), s


def _plain_scan(st):
    q, k, v, b = (st[n].float() for n in ("queries", "keys", "values", "betas"))
    g = st["log_gates"].double()
    group = v.shape[2] // q.shape[2]
    q, k = q.repeat_interleave(group, 2), k.repeat_interleave(group, 2)
    s0, scale = st["initial_state"], q.shape[-1] ** -0.5
    zeros = lambda B: torch.zeros(B, v.shape[2], q.shape[3], v.shape[3], device=v.device)
    if st["lengths"] is None:
        out, s = _plain_sequence(q, k, v, g, b, zeros(v.shape[0]) if s0 is None else s0, scale)
        return out.to(st["values"].dtype), s
    parts = [x.split(st["lengths"], 1) for x in (q, k, v, g, b)]
    got = [_plain_sequence(*(p[i] for p in parts), zeros(1) if s0 is None else s0[i:i + 1], scale)
           for i in range(len(st["lengths"]))]
    return torch.cat([o for o, _ in got], 1).to(st["values"].dtype), torch.cat([s for _, s in got], 0)


# ---- the definition in 64 bits, token by token ------------------------------------------------------------------------

def _exact_tokens(q, k, v, g, b, s, scale, d_out=None, d_s=None):
    """Tokens first: q, k (T, N, K), v (T, N, V), g, b (T, N), s (N, K, V).  Returns (out, s) or with gradients."""
    T = q.shape[0]
    out, kept = torch.empty_like(v), []
    every = max(1, int(math.isqrt(max(T, 1))))
    def token(s, t):
        s1 = torch.exp(g[t])[:, None, None] * s
        e = v[t] - torch.einsum("nk,nkv->nv", k[t], s1)
        return s1, e, s1 + k[t][:, :, None] * (b[t][:, None] * e)[:, None, :]
    for t in range(T):
        if d_out is not None and t % every == 0:
            kept.append(s)
        _, _, s = token(s, t)
        out[t] = scale * torch.einsum("nk,nkv->nv", q[t], s)
    if d_out is None:
        return out, s
    dq, dk, dv, dg, db = (torch.empty_like(x) for x in (q, k, v, g, b))
    ds = torch.zeros_like(s) if d_s is None else d_s
    for at in range((T - 1) // every * every, -1, -every):
        run_, x = [], kept.pop()
        for t in range(at, min(at + every, T)):
            got = token(x, t)
            run_.append(got)
            x = got[2]
        for t in range(min(at + every, T) - 1, at - 1, -1):
            s1, e, s2 = run_.pop()
            do = scale * d_out[t]
            dq[t] = torch.einsum("nkv,nv->nk", s2, do)
            ds = ds + q[t][:, :, None] * do[:, None, :]
            du = torch.einsum("nk,nkv->nv", k[t], ds)
            db[t] = (e * du).sum(-1)
            de = b[t][:, None] * du
            dv[t] = de
            dk[t] = torch.einsum("nkv,nv->nk", ds, b[t][:, None] * e) - torch.einsum("nkv,nv->nk", s1, de)
            ds = ds - k[t][:, :, None] * de[:, None, :]
            dg[t] = (ds * s1).sum((-1, -2))
            ds = torch.exp(g[t])[:, None, None] * ds
    return out, s, dq, dk, dv, dg, db, ds


def _exact_delta(st, train):
    q, k, v, g, b = (st[n].detach().double() for n in ("queries", "keys", "values", "log_gates", "betas"))
    B, T, Hk, K = q.shape
    H, V = v.shape[2:]
    group, scale = H // Hk, K ** -0.5
    lengths = st["lengths"] or [T]
    d_out = st["d_out"].double() if train else None
    got = []
    start = 0
    for i, n in enumerate(lengths):
        cut = lambda x: x[:, start:start + n].transpose(0, 1)
        flat = lambda x: cut(x).reshape(n, B * H, *x.shape[3:])
        wide = lambda x: cut(x).repeat_interleave(group, 2).reshape(n, B * H, K)
        rows = slice(0, B) if st["lengths"] is None else slice(i, i + 1)
        of_state = lambda x: x.detach()[rows].double().reshape(B * H, K, V)
        s = torch.zeros(B * H, K, V, dtype=torch.float64, device=v.device) if st["initial_state"] is None else of_state(st["initial_state"])
        ds = of_state(st["d_state"]) if train and st["d_state"] is not None else None
        parts = _exact_tokens(wide(q), wide(k), flat(v), flat(g), flat(b), s, scale, flat(d_out) if train else None, ds)
        got.append(parts)
        start += n
    def tokens(j):
        return torch.cat([p[j].reshape(p[j].shape[0], B, H, *p[j].shape[2:]).transpose(0, 1) for p in got], 1)
    def states(j):
        return torch.cat([p[j].reshape(B, H, K, V) for p in got], 0)
    res = {"out": tokens(0), "state": states(1)}
    if train:
        for j, name in ((2, "d_queries"), (3, "d_keys")):
            res[name] = tokens(j).reshape(B, T, Hk, group, K).sum(3)
        for j, name in ((4, "d_values"), (5, "d_log_gates"), (6, "d_betas")):
            res[name] = tokens(j)
        if st["initial_state"] is not None:
            res["d_initial_state"] = states(7)
    return res


def _exact_step(st):
    q, k, v, g, b = (st[n].double() for n in ("queries", "keys", "values", "log_gates", "betas"))
    state, out = st["state"].double(), torch.zeros_like(v)
    group = v.shape[1] // q.shape[1]
    for i, slot in enumerate(st["slots"].tolist()):
        if slot < 0:
            continue
        qi, ki = q[i].repeat_interleave(group, 0), k[i].repeat_interleave(group, 0)
        o, s = _exact_tokens(qi[None], ki[None], v[i][None], g[i][None], b[i][None], state[slot], q.shape[-1] ** -0.5)
        out[i], state[slot] = o[0], s
    return {"out": out, "state": state}


def _exact_norm(st, train):
    case, D = st["case"], st["x"].shape[-1]
    val = {n: None if st[n] is None else st[n].detach().double() for n in NORM_LEAVES}
    x, z = val["x"], val["gate"]
    one = torch.ones((), dtype=torch.float64, device=x.device)
    r = ((x.square().sum(-1, keepdim=True) / D) + 1e-6).pow(-0.5)
    w = val["post_weight"]
    n = x if w is None else x * r * w
    sig = None if z is None else torch.sigmoid(z)
    a = one if z is None else (sig * z if case["act"] == "silu" else sig)
    c = one if val["scale"] is None else val["scale"]
    h = n * a * c + (0 if val["residual"] is None else val["residual"])
    res = {"hidden": h}
    rh = ((h.square().sum(-1, keepdim=True) / D) + 1e-6).pow(-0.5)
    if case["pre"]:
        res["normed"] = h * rh * val["pre_weight"]
    if not train:
        return res
    dh = st["d_hidden"].double()
    if case["pre"]:
        dy = st["d_normed"].double()
        t = dy * val["pre_weight"]
        dh = dh + rh * (t - h * rh.square() * (t * h).sum(-1, keepdim=True) / D)
        res["d_pre_weight"] = (dy * h * rh).sum(0)
    if val["residual"] is not None:
        res["d_residual"] = dh
    if val["scale"] is not None:
        res["d_scale"] = (dh * a * n).sum(0)
    if z is not None:
        res["d_gate"] = dh * c * n * (sig * (1 + z * (1 - sig)) if case["act"] == "silu" else sig * (1 - sig))
    dn = dh * a * c
    if w is None:
        res["d_x"] = dn
    else:
        t = dn * w
        res["d_x"] = r * (t - x * r.square() * (t * x).sum(-1, keepdim=True) / D)
        res["d_post_weight"] = (dn * x * r).sum(0)
    return res


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] in ("norm", "norm_train"):
            return _exact_norm(st, case["kind"] == "norm_train")
        if case["kind"] == "step":
            return _exact_step(st)
        return _exact_delta(st, case["kind"] == "train")


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    size = SIZE[case["type"]]
    if case["kind"] in ("norm", "norm_train"):
        vectors = SIZE[case["weights"]] * case["D"] * sum(bool(case[n]) for n in ("post", "pre", "scale"))
        inputs = 1 + sum(bool(case[n]) for n in ("residual", "gate"))
        outputs = 1 + bool(case["pre"])
        tensors, flops = inputs + outputs, 12
        if case["kind"] == "norm_train":
            tensors, flops, vectors = tensors + outputs + inputs, 40, 2 * vectors      # gradients in, gradients out
        return {"bytes": tensors * case["rows"] * case["D"] * size + vectors, "flops": flops * case["rows"] * case["D"]}
    B, Hk, H, K, V = (case[n] for n in ("batch", "heads_k", "heads", "K", "V"))
    if case["kind"] == "step":
        return {"bytes": B * (H * (8 * K * V + size * (2 * V + 2)) + 2 * size * Hk * K), "flops": 6 * B * H * K * V}
    tokens, states = B * case["T"], (case["seqs"] or B) * H * K * V * 4
    inputs = size * tokens * (2 * Hk * K + H * (V + 2))
    outputs = size * tokens * H * V
    if case["kind"] == "scan":
        return {"bytes": inputs + outputs + states * (2 if case["state"] else 1), "flops": 6 * tokens * H * K * V}
    return {"bytes": 2 * inputs + 2 * outputs + states * (4 if case["state"] else 1), "flops": 20 * tokens * H * K * V}
