"""The gated delta rule against its recurrence in 64 bits.

Tolerances, as the 2-norm of the difference over the 2-norm of the result.
States: the operands of the chunked form's products are held to 2^-17 of
their size (two 8-bit parts), three products follow one another in a chunk and
beta <= 1 with unit keys does not let an error grow: 2^-15. Outputs: one
rounding to the type, and for bf16 one operand rounding of the same size
before it, each at most half an ulp: 2^-11 for fp16, 2^-8 for bf16, on top of
the states'."""

from __future__ import annotations

import pytest
import torch

from exl3_intel_arc_quantizer_b200.delta_rule import delta_fault_count, gated_delta_rule, gated_delta_step_

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]
OUT_TOL = {torch.float16: 2.0 ** -11 + 2.0 ** -15, torch.bfloat16: 2.0 ** -8 + 2.0 ** -15}
STATE_TOL = 2.0 ** -15


def recurrence(q, k, v, g, beta, S=None, scale=None, normalize=False):
    """One sequence in float64: (tokens, heads, dv), (heads, dk, dv)."""
    rep = v.shape[1] // k.shape[1]
    q, k, v, g, beta = (t.double() for t in (q, k, v, g, beta))
    if normalize:
        q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    S = torch.zeros(v.shape[1], k.shape[-1], v.shape[-1], dtype=torch.float64, device=v.device) if S is None \
        else S.double().clone()
    out = []
    for t in range(q.shape[0]):
        S = S * g[t].exp()[:, None, None]
        u = beta[t][:, None] * (v[t] - torch.einsum("hkv,hk->hv", S, k[t]))
        S = S + k[t][:, :, None] * u[:, None, :]
        out.append(scale * torch.einsum("hkv,hk->hv", S, q[t]))
    return (torch.stack(out) if out else torch.zeros_like(v)), S


def inputs(tokens, hk, h, dk, dv, dtype, seed=0, decay=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*s):
        return torch.randn(s, generator=gen, device=DEV)

    q, k, v = randn(tokens, hk, dk).to(dtype), randn(tokens, hk, dk).to(dtype), randn(tokens, h, dv).to(dtype)
    g = -decay * torch.nn.functional.softplus(randn(tokens, h) - 2)
    return q, k, v, g, torch.sigmoid(randn(tokens, h))


def off(got, want):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    norm = float(want.norm())
    return float((got - want).norm()) / norm if norm else float(got.norm())


def cu_of(lens):
    return torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)


def check(q, k, v, g, beta, lens, state=None, **kw):
    o, S = gated_delta_rule(q, k, v, g, beta, cu_seqlens=cu_of(lens), initial_state=state, **kw)
    assert o.dtype == v.dtype and o.shape == v.shape and S.dtype == torch.float32
    at = 0
    for s, n in enumerate(lens):
        sl = slice(at, at + n)
        wo, wS = recurrence(q[sl], k[sl], v[sl], g[sl], beta[sl], None if state is None else state[s],
                            kw.get("scale"), kw.get("normalize_qk", False))
        if n:
            assert off(o[sl], wo) <= OUT_TOL[v.dtype], (s, n, off(o[sl], wo))
        assert off(S[s], wS) <= STATE_TOL, (s, n, off(S[s], wS))
        at += n
    return o, S


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 321])
def test_lengths(dtype, tokens):
    check(*inputs(tokens, 2, 4, 128, 128, dtype, tokens), [tokens], normalize_qk=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hk,h,dk,dv", [(1, 1, 8, 8), (2, 2, 16, 40), (1, 3, 64, 64), (2, 4, 72, 96), (1, 2, 96, 192),
                                        (4, 4, 128, 64), (1, 2, 128, 256), (1, 1, 136, 32), (1, 2, 256, 128),
                                        (3, 6, 64, 128), (1, 8, 128, 128)])
def test_head_layouts(dtype, hk, h, dk, dv):
    x = inputs(150, hk, h, dk, dv, dtype, dk + dv)
    state = torch.randn(2, h, dk, dv, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV) * 0.3
    check(*x, [70, 80], state, normalize_qk=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_ragged_sequences_with_empty_ones_and_states(dtype):
    lens = [0, 1, 130, 0, 63, 64, 65, 2, 0]
    x = inputs(sum(lens), 2, 4, 64, 128, dtype, 5)
    state = torch.randn(len(lens), 4, 64, 128, device=DEV, generator=torch.Generator(device=DEV).manual_seed(4))
    _, S = check(*x, lens, state, normalize_qk=True)
    for s, n in enumerate(lens):
        if n == 0:
            assert torch.equal(S[s], state[s])
    _, S = check(*x, lens, normalize_qk=True)
    assert not S[0].any() and not S[-1].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_without_normalization_and_with_scale(dtype):
    q, k, v, g, beta = inputs(100, 2, 2, 64, 64, dtype, 6)
    k = (k.float() / k.float().norm(dim=-1, keepdim=True)).to(dtype)
    check(q, k, v, g, beta, [100], scale=0.37)


@pytest.mark.parametrize("dtype", TYPES)
def test_gates_at_their_ends(dtype):
    """Decay 0 (g = -inf), far below any float's exponent, none (g = 0), and
    beta 0 and 1, alone and mixed in one chunk."""
    q, k, v, g, beta = inputs(192, 2, 4, 64, 64, dtype, 7)
    g[10:12, 0] = -float("inf")
    g[40, 0], g[41:100, 0] = -float("inf"), 0.0
    g[:, 1] = 0.0
    g[5::7, 2] = -1e30
    g[:, 3] = -80.0
    beta[20:60, 0], beta[60:80, 0] = 0.0, 1.0
    beta[:, 1] = 1.0
    check(q, k, v, g, beta, [192], normalize_qk=True)
    check(q, k, v, torch.full_like(g, -float("inf")), beta, [100, 92], normalize_qk=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_keys(dtype):
    """The chunk's triangular system at its densest: one key for all tokens,
    no decay, beta 1: each token replaces the one before."""
    q, k, v, g, beta = inputs(130, 1, 2, 64, 64, dtype, 8)
    k = k[:1].expand_as(k)
    check(q, k, v, torch.zeros_like(g), torch.ones_like(beta), [130], normalize_qk=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_zero_rows_and_large_values(dtype):
    q, k, v, g, beta = inputs(90, 1, 2, 64, 64, dtype, 9)
    k[3:40] = 0
    q[50] = 0
    check(q, k, v * 1000, g, beta, [90], normalize_qk=True)
    check(q * 100, k * 100, v * 1e-2, g, beta, [90], normalize_qk=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_sequence(dtype):
    check(*inputs(1500, 1, 2, 128, 128, dtype, 10, decay=0.1), [1500], normalize_qk=True)
    assert delta_fault_count() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_many_chains(dtype):
    """More chains than the narrow slices are used for: two column groups per CTA."""
    lens = [65, 130, 1, 64, 90, 3, 128, 70, 200, 63]
    check(*inputs(sum(lens), 4, 16, 64, 128, dtype, 30), lens, normalize_qk=True)
    x = inputs(200, 4, 16, 128, 192, dtype, 31)
    state = torch.randn(8, 16, 128, 192, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5))
    check(*x, [25] * 8, state, normalize_qk=True)
    assert delta_fault_count() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_growing_states(dtype):
    """Positive log decays: the state grows by e^6 in the sequence."""
    q, k, v, g, beta = inputs(300, 1, 2, 64, 64, dtype, 32)
    check(q, k, v, g * 0 + 0.02, beta, [300], normalize_qk=True)


def test_slices_of_one_projection_and_unaligned_ones():
    hk, h, dk, dv, n = 2, 4, 64, 64, 100
    mix = torch.randn(n, 2 * hk * dk + h * dv + 8, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).half()
    _, _, _, g, beta = inputs(n, hk, h, dk, dv, torch.float16, 2)
    for o in (0, 1, 8):
        q, k, v = mix[:, o:o + 2 * hk * dk + h * dv].split([hk * dk, hk * dk, h * dv], dim=-1)
        check(q.unflatten(-1, (hk, dk)), k.unflatten(-1, (hk, dk)), v.unflatten(-1, (h, dv)), g, beta, [40, 60],
              normalize_qk=True)
    q = mix[:, :2 * hk * dk:2].unflatten(-1, (hk, dk))
    gg = g.t().contiguous().t()
    check(q, q, mix[:, -h * dv:].unflatten(-1, (h, dv)), gg, beta, [100], normalize_qk=True)


def test_batched_equals_packed():
    x = inputs(3 * 70, 2, 2, 64, 64, torch.bfloat16, 11)
    o, S = gated_delta_rule(*x, cu_seqlens=cu_of([70] * 3), normalize_qk=True)
    ob, Sb = gated_delta_rule(*(t.unflatten(0, (3, 70)) for t in x), normalize_qk=True)
    assert torch.equal(o, ob.flatten(0, 1)) and torch.equal(S, Sb)
    o1, S1 = gated_delta_rule(*(t[:70] for t in x), normalize_qk=True)
    assert torch.equal(o1, o[:70]) and torch.equal(S1[0], S[0])


def test_a_sequence_does_not_depend_on_its_neighbours():
    x = inputs(300, 2, 4, 128, 128, torch.float16, 12)
    o, S = gated_delta_rule(*x, cu_seqlens=cu_of([100, 150, 50]), normalize_qk=True)
    y = [t.clone() for t in x]
    for t in y:
        t[:100], t[250:] = float("nan"), float("nan")
    o2, S2 = gated_delta_rule(*y, cu_seqlens=cu_of([100, 150, 50]), normalize_qk=True)
    assert torch.equal(o[100:250], o2[100:250]) and torch.equal(S[1], S2[1])


def test_tokens_outside_the_sequences_are_zero_and_not_read():
    x = [t.clone() for t in inputs(200, 1, 2, 64, 64, torch.float16, 13)]
    for t in x:
        t[:30], t[150:] = float("nan"), float("nan")
    cu = torch.tensor([30, 100, 150], dtype=torch.int32, device=DEV)
    o, S = gated_delta_rule(*x, cu_seqlens=cu, normalize_qk=True)
    assert not o[:30].any() and not o[150:].any() and S.isfinite().all() and o.isfinite().all()
    wo, wS = recurrence(*(t[30:100] for t in x), normalize=True)
    assert off(o[30:100], wo) <= OUT_TOL[torch.float16] and off(S[0], wS) <= STATE_TOL


def test_offsets_out_of_range_are_clamped():
    x = inputs(64, 1, 1, 64, 64, torch.float16, 14)
    cu = torch.tensor([-5, 40, 1000], dtype=torch.int32, device=DEV)
    o, S = gated_delta_rule(*x, cu_seqlens=cu, normalize_qk=True)
    o2, S2 = gated_delta_rule(*x, cu_seqlens=cu_of([40, 24]), normalize_qk=True)
    assert torch.equal(o, o2) and torch.equal(S, S2)


def test_continued_in_pieces():
    x = inputs(230, 2, 4, 128, 128, torch.float16, 15)
    want_o, want_S = recurrence(*x, normalize=True)
    S, parts = None, []
    for a, b in ((0, 100), (100, 101), (101, 230)):
        o, S = gated_delta_rule(*(t[a:b] for t in x), initial_state=S, normalize_qk=True)
        parts.append(o)
    assert off(torch.cat(parts), want_o) <= OUT_TOL[torch.float16] and off(S[0], want_S) <= STATE_TOL


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,hk,h,dk,dv", [(1, 16, 32, 128, 128), (5, 1, 1, 8, 8), (3, 2, 4, 72, 40), (2, 1, 2, 256, 128),
                                          (40, 2, 2, 64, 192), (7, 4, 8, 128, 64)])
def test_steps(dtype, n, hk, h, dk, dv):
    """Three steps, states in place, against the recurrence."""
    x = inputs(3 * n, hk, h, dk, dv, dtype, 16)
    state = torch.randn(n, h, dk, dv, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)) * 0.2
    first = state.clone()
    outs = [gated_delta_step_(*(t[i::3] for t in x), state, normalize_qk=True) for i in range(3)]
    for s in range(n):
        wo, wS = recurrence(*(t[3 * s:3 * s + 3] for t in x), first[s], normalize=True)
        assert off(torch.stack([o[s] for o in outs]), wo) <= OUT_TOL[dtype]
        assert off(state[s], wS) <= STATE_TOL


def test_step_equals_sequence_of_one():
    x = inputs(4, 2, 4, 128, 128, torch.bfloat16, 17)
    state = torch.randn(4, 4, 128, 128, device=DEV)
    o, S = gated_delta_rule(*x, cu_seqlens=cu_of([1] * 4), initial_state=state, normalize_qk=True)
    got = gated_delta_step_(*x, state, normalize_qk=True)
    assert off(got, o) <= OUT_TOL[torch.bfloat16] and off(state, S) <= STATE_TOL


def test_step_slots():
    x = inputs(5, 1, 2, 64, 64, torch.float16, 18)
    pool = torch.randn(6, 2, 64, 64, device=DEV)
    first = pool.clone()
    slots = torch.tensor([3, -1, 0, 6, 5], dtype=torch.int32, device=DEV)
    o = gated_delta_step_(*x, pool, slots=slots, normalize_qk=True)
    assert not o[1].any() and not o[3].any()
    for s in (1, 2, 4):
        assert torch.equal(pool[s], first[s])
    for i, s in ((0, 3), (2, 0), (4, 5)):
        wo, wS = recurrence(*(t[i:i + 1] for t in x), first[s], normalize=True)
        assert off(o[i:i + 1], wo) <= OUT_TOL[torch.float16] and off(pool[s], wS) <= STATE_TOL


def test_step_offsets_past_32_bits():
    """The last states of a pool of more than 2^32 elements."""
    n = 2 ** 32 // (32 * 128 * 128) + 3
    pool = torch.zeros(n, 32, 128, 128, device=DEV)
    x = inputs(2, 16, 32, 128, 128, torch.float16, 19)
    slots = torch.tensor([n - 1, 1], dtype=torch.int32, device=DEV)
    o = gated_delta_step_(*x, pool, slots=slots, normalize_qk=True)
    for i, s in ((0, n - 1), (1, 1)):
        wo, wS = recurrence(*(t[i:i + 1] for t in x), normalize=True)
        assert off(o[i:i + 1], wo) <= OUT_TOL[torch.float16] and off(pool[s], wS) <= STATE_TOL
    assert not pool[2].any() and not pool[n - 2].any() and not pool[0].any()


def test_repeated_calls_are_bit_identical_and_streams_agree():
    x = inputs(500, 2, 4, 128, 128, torch.float16, 20)
    o, S = gated_delta_rule(*x, normalize_qk=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, S2 = gated_delta_rule(*x, normalize_qk=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, o2) and torch.equal(S, S2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hk,h,dk,dv", [(1, 1, 8, 8), (2, 4, 72, 40), (2, 2, 64, 192), (4, 8, 128, 128)])
def test_short_sequences_alone_and_among_long_ones(dtype, hk, h, dk, dv):
    lens = [1, 23, 130, 24, 0, 25, 2, 64, 16]
    x = inputs(sum(lens), hk, h, dk, dv, dtype, 21)
    state = torch.randn(len(lens), h, dk, dv, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)) * 0.2
    check(*x, lens, state, normalize_qk=True)
    for n in (9, 23, 24, 25):
        check(*(t[:n] for t in x), [n], normalize_qk=True)


def test_many_short_sequences_and_a_long_one():
    lens = [1] * 90 + [300] + [7] * 60
    x = inputs(sum(lens), 2, 4, 128, 128, torch.bfloat16, 22)
    y = (*(torch.cat([t, t[..., :1]], -1)[..., :-1] for t in x[:3]), *x[3:])  # rows 129 elements apart
    state = torch.randn(len(lens), 4, 128, 128, device=DEV, generator=torch.Generator(device=DEV).manual_seed(4)) * 0.2
    check(*x, lens, state, normalize_qk=True)
    o, S = gated_delta_rule(*x, cu_seqlens=cu_of(lens), initial_state=state, normalize_qk=True)
    o2, S2 = gated_delta_rule(*y, cu_seqlens=cu_of(lens), initial_state=state, normalize_qk=True)
    assert torch.equal(o, o2) and torch.equal(S, S2)


def test_nothing_to_do():
    q, k, v, g, beta = inputs(0, 1, 2, 64, 64, torch.float16)
    o, S = gated_delta_rule(q, k, v, g, beta)
    assert o.shape == (0, 2, 64) and S.shape == (1, 2, 64, 64) and not S.any()
    assert gated_delta_step_(q, k, v, g, beta, torch.zeros(0, 2, 64, 64, device=DEV)).shape == (0, 2, 64)


def test_refusals():
    q, k, v, g, beta = inputs(6, 2, 4, 64, 64, torch.float16)
    cu = cu_of([6])
    good = dict(q=q, k=k, v=v, g=g, beta=beta)
    for change, match in (({"k": k[:, :1]}, "q's shape"), ({"v": v[:5]}, "tokens"), ({"v": v[:, :3]}, "multiple of the key"),
                          ({"k": k.bfloat16()}, "like q"), ({"g": g.half()}, "float32"), ({"beta": beta[:, :2]}, "must be .tokens"),
                          ({"q": q[..., :60], "k": k[..., :60]}, "multiple of 8"), ({"v": v[..., :4]}, "multiple of 8"),
                          ({"q": q.float(), "k": k.float(), "v": v.float()}, "float16 or bfloat16"),
                          ({"cu_seqlens": cu.long()}, "int32"), ({"initial_state": torch.zeros(2, 4, 64, 64, device=DEV)}, "1 states"),
                          ({"initial_state": torch.zeros(1, 4, 64, 32, device=DEV)}, "must be"),
                          ({"initial_state": torch.zeros(1, 4, 64, 64, device=DEV).half()}, "float32")):
        with pytest.raises(ValueError, match=match):
            gated_delta_rule(**{**good, "cu_seqlens": cu, **change})
    wide = torch.zeros(6, 1, 264, device=DEV, dtype=torch.float16)
    with pytest.raises(ValueError, match="up to 256"):
        gated_delta_rule(wide, wide, v, g, beta)
    state = torch.zeros(6, 4, 64, 64, device=DEV)
    for s, kw, match in ((state[:5], {}, "one state per token"), (state.transpose(2, 3), {}, "contiguous"),
                         (state.half(), {}, "float32"), (state, {"slots": torch.zeros(6, device=DEV)}, "int32"),
                         (state[:0], {"slots": torch.zeros(6, dtype=torch.int32, device=DEV)}, "no slots")):
        with pytest.raises(ValueError, match=match):
            gated_delta_step_(q, k, v, g, beta, s, **kw)
    with pytest.raises(RuntimeError, match="no_grad"):
        gated_delta_rule(q.clone().requires_grad_(), k, v, g, beta)
    with pytest.raises(ValueError, match="batch"):
        gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], cu_seqlens=cu)
