"""The measured cases of the layer operators between the linear projections:
rotary positions, the block norms, and the gated delta rule (whole sequences
and single tokens).

A decoder layer's forward pass runs three times per conversion (Hessian
capture, re-forward, evaluation), so the cases are its shapes: hidden size
4096, 32 query and 8 key/value heads of 128, calibration batches of
2048-token sequences, and the single-token steps of a generation check.
Where ``own`` is false ``run`` computes the operators in elementary torch
operations in 32 bits, rounded once at the end; where it is true it calls the
package.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one generated token: launch latency
        dict(name="rotary_token", op="rotary", batch=1, seq=1, heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, scaled=False, start=1777, dtype="fp16", heads_first=False),
        # a calibration batch in the attention's own (batch, heads, seq, dim) view of the projections
        dict(name="rotary_batch", op="rotary", batch=8, seq=2048, heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, scaled=False, start=0, dtype="fp16", heads_first=True),
        # part of a wide head, interleaved pairs, frequencies scaled for a long context, an odd length
        dict(name="rotary_partial_long", op="rotary", batch=1, seq=20001, heads=16, kv_heads=4, dim=256, rot=64,
             interleaved=True, scaled=True, start=100000, dtype="bf16", heads_first=False),
        # one generated token through residual add and the next block's norm
        dict(name="norm_token", op="norm", rows=1, d=4096, post=False, gate="", residual=True, scale=1.0,
             next=True, dtype="fp16"),
        # a calibration batch: norm after the block, scaled residual, norm before the next block
        dict(name="norm_batch", op="norm", rows=16384, d=4096, post=True, gate="", residual=True, scale=0.5,
             next=True, dtype="bf16"),
        # linear attention's output: norm per head of 128, gated by silu(z)
        dict(name="norm_gated_heads", op="norm", rows=4096 * 32, d=128, post=True, gate="silu", residual=False,
             scale=1.0, next=False, dtype="fp16"),
        # everything at once on rows of odd length
        dict(name="norm_odd", op="norm", rows=3001, d=4095, post=True, gate="sigmoid", residual=True, scale=0.7,
             next=True, dtype="fp16"),
        # one generated token of one sequence
        dict(name="delta_token", op="step", n=1, key_heads=16, heads=32, dk=128, dv=128, dtype="fp16"),
        # one generated token of each of many sequences
        dict(name="delta_tokens", op="step", n=128, key_heads=16, heads=32, dk=128, dv=128, dtype="bf16"),
        # one calibration sequence
        dict(name="delta_sequence", op="delta", seqs=1, tokens=2048, ragged=False, key_heads=16, heads=32, dk=128,
             dv=128, state=False, dtype="fp16"),
        # a calibration batch
        dict(name="delta_batch", op="delta", seqs=8, tokens=16384, ragged=False, key_heads=16, heads=32, dk=128,
             dv=128, state=False, dtype="bf16"),
        # packed sequences of all lengths, continued from their states
        dict(name="delta_ragged", op="delta", seqs=7, tokens=4099, ragged=True, key_heads=8, heads=8, dk=64,
             dv=128, state=True, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "step", "delta", "delta"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 192, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 7])
        batch = rng.choice([1, 1, 2, 5])
        most = max(1, 150_000_000 // (batch * (heads + kv) * dim))
        return dict(op=op, batch=batch, seq=_log_int(rng, 1, min(20000, most)), heads=heads, kv_heads=kv, dim=dim,
                    rot=rot, interleaved=rng.random() < 0.5, scaled=rng.random() < 0.5,
                    start=_log_int(rng, 1, 100000), dtype=dtype, heads_first=rng.random() < 0.5)
    if op == "norm":
        d = rng.choice([64, 128, 256, 1000, 2048, 2304, 4095, 4096, 5120, 8192, 14336])
        return dict(op=op, rows=_log_int(rng, 1, min(50000, 60_000_000 // d)), d=d, post=rng.random() < 0.6,
                    gate=rng.choice(["", "", "silu", "sigmoid"]), residual=rng.random() < 0.6,
                    scale=round(rng.uniform(0.25, 1.0), 2), next=rng.random() < 0.6, dtype=dtype)
    kh = rng.choice([1, 2, 4, 8, 16])
    heads = kh * rng.choice([1, 2, 2, 4])
    dk, dv = rng.choice([64, 96, 128, 128]), rng.choice([64, 128, 128, 192])
    if op == "step":
        return dict(op=op, n=_log_int(rng, 1, min(300, 2 ** 26 // (heads * dk * dv))), key_heads=kh, heads=heads,
                    dk=dk, dv=dv, dtype=dtype)
    ragged = rng.random() < 0.6
    seqs = rng.choice([1, 1, 2, 3, 6, 12])
    tokens = _log_int(rng, 13 * seqs, min(20000, max(2000, 2 ** 28 // (heads * max(dk, dv)) // (4 if ragged else 1))))
    if not ragged:
        tokens = tokens // seqs * seqs
    return dict(op=op, seqs=seqs, tokens=tokens, ragged=ragged, key_heads=kh, heads=heads, dk=dk, dv=dv,
                state=rng.random() < 0.5, dtype=dtype)


def _lengths(case):
    """Lengths of the packed sequences: equal, or from one token to most of the pack."""
    n, total = case["seqs"], case["tokens"]
    if not case["ragged"]:
        return [total // n] * n
    left, out = total, []
    for i in range(n - 1):
        most = left - (n - 1 - i)
        take = 1 if i % 3 == 1 else max(1, min(most, (left * (7 + 13 * i % 31)) // 61))
        out.append(take)
        left -= take
    return out + [left]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _frequencies(rot, scaled):
    """inv_freq in float32 and the attention factor; scaled: a factor 8 beyond
    8192 positions, interpolated for long wavelengths only."""
    half = rot // 2
    j = torch.arange(half, dtype=torch.float64)
    inv = 500000.0 ** (-j / half)
    factor = 1.0
    if scaled:
        turns = 8192 * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        inv = inv * keep + inv / 8.0 * (1 - keep)
        factor = 0.1 * math.log(8.0) + 1.0
    return inv.to(torch.float32), factor


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 9973 + 17)
    op, dt = case["op"], TYPES[case["dtype"]]

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)

    s = dict(case=case)
    if op == "rotary":
        b, t, d = case["batch"], case["seq"], case["dim"]
        s["q"], s["k"] = randn(b, t, case["heads"], d), randn(b, t, case["kv_heads"], d)
        s["positions"] = case["start"] + torch.arange(t, device=DEV)
        inv, s["factor"] = _frequencies(case["rot"], case["scaled"])
        s["inv_freq"] = inv.to(DEV)
        return s
    if op == "norm":
        r, d = case["rows"], case["d"]
        s["x"] = randn(r, d, scale=1.5)
        s["weight"] = 1 + 0.1 * randn(d) if case["post"] else None
        s["gate"] = randn(r, d) if case["gate"] else None
        s["residual"] = randn(r, d, scale=2.0) if case["residual"] else None
        s["next_weight"] = 1 + 0.1 * randn(d) if case["next"] or not (case["post"] or case["gate"] or case["residual"]) else None
        return s
    hk, h, dk, dv = case["key_heads"], case["heads"], case["dk"], case["dv"]
    n = case["n"] if op == "step" else case["tokens"]
    # q, k and v are the slices of one convolved projection, as a layer has them
    mix = torch.nn.functional.silu(randn(n, 2 * hk * dk + h * dv, dtype=torch.float32)).to(dt)
    s["q"], s["k"], v = mix.split([hk * dk, hk * dk, h * dv], dim=-1)
    s["q"], s["k"], s["v"] = s["q"].view(n, hk, dk), s["k"].view(n, hk, dk), v.view(n, h, dv)
    a = torch.rand(h, generator=gen, device=DEV) * 16 + 0.01          # decay rate of a head
    step = torch.exp(torch.rand(h, generator=gen, device=DEV) * 4.6 - 6.9)  # its time step, 0.001 .. 0.1
    bias = step + torch.log(-torch.expm1(-step))
    s["g"] = -a * torch.nn.functional.softplus(randn(n, h, dtype=torch.float32) * 0.5 + bias)
    s["beta"] = torch.sigmoid(randn(n, h, dtype=torch.float32))
    if op == "step":
        s["state"] = randn(n, h, dk, dv, scale=0.1, dtype=torch.float32)
        return s
    lens = _lengths(case)
    s["cu"] = torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)
    s["lens"] = lens
    s["state"] = randn(len(lens), h, dk, dv, scale=0.1, dtype=torch.float32) if case["state"] else None
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "norm": _own_norm, "step": _own_step, "delta": _own_delta}[op](s)
    return {"rotary": _plain_rotary, "norm": _plain_norm, "step": _plain_step, "delta": _plain_delta}[op](s)


def _own_rotary(s):
    from exl3_intel_arc_quantizer_b200.rotary import apply_rotary

    c = s["case"]
    q, k = s["q"], s["k"]
    if c["heads_first"]:
        q, k = q.transpose(1, 2), k.transpose(1, 2)
    return apply_rotary(q, k, s["positions"], s["inv_freq"], attention_factor=s["factor"],
                        interleaved=c["interleaved"], heads_first=c["heads_first"])


def _own_norm(s):
    from exl3_intel_arc_quantizer_b200.norms import block_norm

    c = s["case"]
    return block_norm(s["x"], weight=s["weight"], gate=s["gate"], gate_activation=c["gate"] or "silu",
                      residual=s["residual"], residual_scale=c["scale"], next_weight=s["next_weight"])


def _own_step(s):
    from exl3_intel_arc_quantizer_b200.delta_rule import gated_delta_step_

    o = gated_delta_step_(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], normalize_qk=True)
    return o, s["state"]


def _own_delta(s):
    from exl3_intel_arc_quantizer_b200.delta_rule import gated_delta_rule

    return gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], cu_seqlens=s["cu"],
                            initial_state=s["state"], normalize_qk=True)


def _plain_rotary(s):
    c = s["case"]
    angle = s["positions"].float()[:, None] * s["inv_freq"]
    cos, sin = (angle.cos() * s["factor"])[:, None], (angle.sin() * s["factor"])[:, None]
    r, half = c["rot"], c["rot"] // 2

    def turn(x):
        y = x.float()
        if c["interleaved"]:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            z = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        else:
            a, b = y[..., :half], y[..., half:r]
            z = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        z = torch.cat((z, y[..., r:]), dim=-1).to(x.dtype)
        return z.transpose(1, 2) if c["heads_first"] else z

    return turn(s["q"]), turn(s["k"])


def _plain_norm(s):
    c = s["case"]
    x = s["x"].float()
    changed = False
    if s["weight"] is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
        changed = True
    if s["gate"] is not None:
        z = s["gate"].float()
        x = x * (torch.sigmoid(z) if c["gate"] == "sigmoid" else z * torch.sigmoid(z))
        changed = True
    if s["residual"] is not None:
        x = s["residual"].float() + c["scale"] * x
        changed = True
    n = None
    if s["next_weight"] is not None:
        n = (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * s["next_weight"].float()).to(s["x"].dtype)
    return (x.to(s["x"].dtype) if changed else s["x"]), n


def _unit(x):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def _plain_step(s):
    c = s["case"]
    rep = c["heads"] // c["key_heads"]
    q = _unit(s["q"].float()).repeat_interleave(rep, 1) * c["dk"] ** -0.5
    k = _unit(s["k"].float()).repeat_interleave(rep, 1)
    S = s["state"] * s["g"].exp()[..., None, None]
    u = s["beta"][..., None] * (s["v"].float() - (S * k[..., None]).sum(-2))
    S = S + k[..., None] * u[..., None, :]
    s["state"].copy_(S)
    return (S * q[..., None]).sum(-2).to(s["v"].dtype), s["state"]


def _plain_delta(s):
    """Chunks of 64 tokens of padded sequences: the chunk's triangular system
    inverted by halves, then one step of the state per chunk."""
    c = s["case"]
    C, h, dk, dv = 64, c["heads"], c["dk"], c["dv"]
    rep, lens = h // c["key_heads"], s["lens"]
    n, nc = len(lens), -(-max(lens) // C)
    at = torch.arange(nc * C, device=DEV)
    cu = s["cu"].long()
    inside = at < (cu[1:] - cu[:-1])[:, None]
    index = torch.where(inside, cu[:-1, None] + at, 0)

    def chunks(x):  # (tokens, heads, ...) -> (n, heads, chunk, C, ...), zero past each end
        y = x.float()[index] * inside.view(n, nc * C, *[1] * (x.dim() - 1))
        return y.view(n, nc, C, *x.shape[1:]).movedim(3, 1)

    q = chunks(_unit(s["q"].float())).repeat_interleave(rep, 1) * dk ** -0.5
    k = chunks(_unit(s["k"].float())).repeat_interleave(rep, 1)
    v, g, beta = chunks(s["v"]), chunks(s["g"]), chunks(s["beta"])
    G = g.cumsum(-1)
    i = torch.arange(C, device=DEV)
    decay = torch.where(i[:, None] >= i, G[..., :, None] - G[..., None, :], -math.inf).exp()
    M = (beta[..., None] * (k @ k.mT) * decay).tril(-1)
    P = (q @ k.mT) * decay
    inv = torch.ones(*M.shape[:-2], C, 1, 1, device=DEV)  # diagonal blocks of the inverse, doubled in size
    size = 1
    while size < C:
        b = M.unflatten(-2, (C // (2 * size), 2, size)).unflatten(-1, (C // (2 * size), 2, size))
        low = torch.diagonal(b[..., 1, :, :, 0, :], dim1=-4, dim2=-2).movedim(-1, -3)
        A, D = inv[..., 0::2, :, :], inv[..., 1::2, :, :]
        inv = torch.cat((torch.cat((A, torch.zeros_like(A)), -1), torch.cat((-D @ low @ A, D), -1)), -2)
        size *= 2
    T = inv[..., 0, :, :] * beta[..., None, :]
    S = s["state"].clone() if s["state"] is not None else torch.zeros(n, h, dk, dv, device=DEV)
    o = torch.empty(n, h, nc, C, dv, device=DEV)
    grow, last = G.exp()[..., None], G[..., -1:]
    for t in range(nc):
        U = T[:, :, t] @ (v[:, :, t] - grow[:, :, t] * (k[:, :, t] @ S))
        o[:, :, t] = grow[:, :, t] * (q[:, :, t] @ S) + P[:, :, t] @ U
        S = last[:, :, t, :, None].exp() * S + (k[:, :, t] * (last[:, :, t] - G[:, :, t]).exp()[..., None]).mT @ U
    return o.movedim(1, 3).reshape(n, nc * C, h, dv)[inside].to(s["v"].dtype), S


# ---------------------------------------------------------------------------
# what a pass needs, and its outputs in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "rotary":
        x = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 4 * x * case["dim"] + 8 * case["seq"], "flops": 3 * x * case["rot"]}
    if op == "norm":
        e, vec = case["rows"] * case["d"], case["d"] * (bool(case["post"]) + bool(case["next"]))
        changed = case["post"] or bool(case["gate"]) or case["residual"]
        parts = 1 + bool(case["gate"]) + case["residual"] + changed + (case["next"] or not changed)
        return {"bytes": 2 * (e * parts + vec), "flops": e * (4 * case["post"] + 4 * bool(case["gate"]) + 2 * case["residual"] + 4 * case["next"])}
    hk, h, dk, dv = case["key_heads"], case["heads"], case["dk"], case["dv"]
    n = case["n"] if op == "step" else case["tokens"]
    io = n * (2 * (2 * hk * dk + 2 * h * dv) + 8 * h)
    states = 2 * case["n"] if op == "step" else case["seqs"] * (1 + case["state"])
    return {"bytes": io + 4 * states * h * dk * dv, "flops": 6 * n * h * dk * dv}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        phi = s["positions"].double()[:, None] * s["inv_freq"].double()
        turn = torch.polar(torch.full_like(phi, s["factor"]), phi)[:, None]
        r = case["rot"]
        out = []
        for x in (s["q"].double(), s["k"].double()):
            y = x.clone()
            first, second = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
            z = torch.complex(x[..., first], x[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            out.append(y.transpose(1, 2) if case["heads_first"] else y)
        return tuple(out)
    if op == "norm":
        def rms(t, w):
            return t / torch.sqrt(torch.linalg.vecdot(t, t)[:, None] / t.shape[-1] + 1e-6) * w.double()

        y = s["x"].double()
        if s["weight"] is not None:
            y = rms(y, s["weight"])
        if s["gate"] is not None:
            z = s["gate"].double()
            y = y / (1 + torch.exp(-z)) * (1 if case["gate"] == "sigmoid" else z)
        if s["residual"] is not None:
            y = torch.add(s["residual"].double(), y, alpha=case["scale"])
        return y, None if s["next_weight"] is None else rms(y, s["next_weight"])

    h, dk, dv = case["heads"], case["dk"], case["dv"]
    rep = h // case["key_heads"]

    def unit(x):
        x = x.double()
        return (x / torch.sqrt(torch.linalg.vecdot(x, x)[..., None] + 1e-6)).repeat_interleave(rep, 1)

    q, k, v = unit(s["q"]) / math.sqrt(dk), unit(s["k"]), s["v"].double()
    keep, beta = s["g"].double().exp(), s["beta"].double()

    def token(S, t):  # S (rows, h, dk, dv), t: the rows' tokens
        S = S * keep[t, :, None, None]
        kt = k[t].unsqueeze(-2)
        S = S + kt.mT @ (beta[t, :, None, None] * (v[t].unsqueeze(-2) - kt @ S))
        return S, (q[t].unsqueeze(-2) @ S).squeeze(-2)

    if op == "step":
        S, o = token(s["state"].double(), torch.arange(case["n"], device=DEV))
        return o, S
    lens = s["lens"]
    n = len(lens)
    order = sorted(range(n), key=lambda i: -lens[i])
    rows = torch.tensor(order, device=DEV)
    begin = s["cu"].long()[rows]
    S = torch.zeros(n, h, dk, dv, dtype=torch.float64, device=DEV) if s["state"] is None else s["state"].double()[rows]
    o = torch.empty(case["tokens"], h, dv, dtype=torch.float64, device=DEV)
    for t in range(max(lens)):
        live = sum(1 for i in order if lens[i] > t)  # the longest sequences come first
        if live == n:
            S, o[begin + t] = token(S, begin + t)
        else:
            at = begin[:live] + t
            S[:live], o[at] = token(S[:live], at)
    back = torch.empty_like(S)
    back[rows] = S
    return o, back
