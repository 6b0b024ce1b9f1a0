"""Rotary positions against the rotation written as a complex product in 64
bits: both layouts, part of the head, strides, positions past 2^31, types.

Tolerance: an output is rounded once (half an ulp of its type) after fp32
products of values and of a sine and cosine that are each within 2^-22 of
exact; two products and a sum of pair elements (a, b) then err by less than
2^-20 (|a| + |b|)."""

from __future__ import annotations

import math

import pytest
import torch

from exl3_intel_arc_quantizer_b200.rotary import apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}


def turned(x, positions, inv_freq, factor, interleaved, transposed=False):
    """x (batch, tokens, heads, dim) in float64, and |a| + |b| of each element's pair."""
    r = 2 * inv_freq.numel()
    x = x.double()
    # the turn's fraction in Python integers: exact for any int64 position
    frac = torch.tensor([[math.fmod(int(p) * f, 2 * math.pi) if abs(int(p)) < 2 ** 20 else _reduced(int(p), f)
                          for f in inv_freq.double().tolist()] for p in positions.flatten().tolist()],
                        dtype=torch.float64, device=x.device)
    phi = frac.view(*positions.shape, 1, r // 2)
    if transposed:
        phi = -phi
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    z = torch.complex(a, b) * torch.polar(torch.full_like(phi, factor), phi)
    y, size = x.clone(), torch.zeros_like(x)
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y[..., first], y[..., second] = z.real, z.imag
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(factor)
    return y, size


def _reduced(p, f):
    from fractions import Fraction

    # 2 pi to 60 digits: p * f < 2^64 radians lose less than 1e-38 of a turn
    two_pi = Fraction(628318530717958647692528676655900576839433879875021164194988, 10 ** 59)
    turns = Fraction(f) * p / two_pi
    return float((turns - math.floor(turns)) * two_pi)


def check(got, want, size):
    tol = HALF_ULP[got.dtype] * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -20 * size + SMALLEST[got.dtype]
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst " \
                          f"{float(((got.double() - want).abs() - tol).max())}"


def rand(shape, dtype, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=gen, device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch,tokens,heads,kv,dim,rot", [
    (1, 1, 32, 8, 128, 128), (2, 37, 4, 4, 64, 64), (1, 5, 3, 1, 256, 64), (3, 11, 2, 1, 80, 40),
    (1, 7, 1, 1, 6, 2), (2, 3, 5, 2, 18, 14), (1, 700, 14, 2, 96, 96), (1, 2, 2, 2, 512, 512)])
def test_matches_the_rotation(dtype, interleaved, batch, tokens, heads, kv, dim, rot):
    q, k = rand((batch, tokens, heads, dim), dtype, 1), rand((batch, tokens, kv, dim), dtype, 2)
    inv, _ = rotary_frequencies(rot, device=DEV)
    pos = 1000 + 3 * torch.arange(tokens, device=DEV, dtype=torch.int32)
    qo, ko = apply_rotary(q, k, pos, inv, attention_factor=1.25, interleaved=interleaved)
    for got, x in ((qo, q), (ko, k)):
        assert got.shape == x.shape and got.dtype == dtype
        check(got, *turned(x, pos, inv, 1.25, interleaved))


@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_are_exact_far_out_and_per_batch(interleaved):
    q = rand((2, 6, 2, 64), torch.float32, 3)
    inv, _ = rotary_frequencies(64, device=DEV)
    pos = torch.tensor([[0, 1, -1, 131071, 2 ** 31 + 5, 2 ** 40 + 3],
                        [7, -2 ** 33, 2 ** 24 + 1, 10 ** 6, 2 ** 45, 999]], device=DEV)
    got, none = apply_rotary(q, None, pos, inv, interleaved=interleaved)
    assert none is None
    # the fixed-point step is within 2^-62 turns: 2^45 positions are off by
    # less than 2^-14 radians, 2^33 by less than 2^-26
    want, size = turned(q, pos, inv, 1.0, interleaved)
    far = (pos.abs() > 2 ** 33)[..., None, None]
    err = (got.double() - want).abs()
    assert not (err > 2.0 ** -20 * size + 2.0 ** -23 * want.abs()).masked_fill(far, False).any()
    assert not (err > 2.0 ** -13 * size).any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["heads_first", "sliced", "unaligned", "step", "flat", "expanded"])
def test_strides(dtype, layout):
    b, t, h, d = 2, 9, 4, 32
    inv, _ = rotary_frequencies(d, device=DEV)
    pos = torch.arange(t, device=DEV)
    if layout == "heads_first":
        q = rand((b, t, h, d), dtype, 4).transpose(1, 2)
        got, _ = apply_rotary(q, None, pos, inv, heads_first=True)
        check(got.transpose(1, 2), *turned(q.transpose(1, 2), pos, inv, 1.0, False))
        return
    if layout == "flat":
        q = rand((t, h, d), dtype, 4)
        got, _ = apply_rotary(q, None, pos, inv)
        check(got[None], *turned(q[None], pos, inv, 1.0, False))
        return
    base = rand((b, t, 3 * h * d + 8), dtype, 4)
    if layout == "sliced":
        q = base[..., :h * d].view(b, t, h, d)
    elif layout == "unaligned":
        q = base[..., 1:1 + h * d].unflatten(-1, (h, d))
    elif layout == "step":
        q = base[..., :2 * h * d:2].unflatten(-1, (h, d))
    else:
        q = base[:, :1, :h * d].unflatten(-1, (h, d)).expand(b, t, h, d)
    for kw in ({}, {"interleaved": True}):
        got, _ = apply_rotary(q, None, pos, inv, **kw)
        check(got, *turned(q, pos, inv, 1.0, bool(kw)))


def test_in_place_equals_out_of_place():
    base = rand((3, 10, 6 * 64), torch.bfloat16, 5)
    inv, _ = rotary_frequencies(32, device=DEV)
    pos = torch.arange(10, device=DEV, dtype=torch.int32)
    q, k = base[..., :4 * 64].unflatten(-1, (4, 64)), base[..., 4 * 64:].unflatten(-1, (2, 64))
    want = [x.clone() for x in apply_rotary(q, k, pos, inv)]
    got = apply_rotary(q, k, pos, inv, inplace=True)
    for w, g, x in zip(want, got, (q, k)):
        assert torch.equal(w, g) and torch.equal(x, g) and g.data_ptr() == x.data_ptr()


@pytest.mark.parametrize("interleaved", [False, True])
def test_transposed_is_the_gradient(interleaved):
    """The gradient of sum(w * rotate(x)) is the transposed map of w: against
    autograd of the formula in 64 bits, and against differences."""
    x, w = rand((1, 5, 2, 24), torch.float32, 6), rand((1, 5, 2, 24), torch.float32, 7)
    inv, _ = rotary_frequencies(16, device=DEV)
    pos = torch.arange(5, device=DEV) + 11
    got, _ = apply_rotary(w, None, pos, inv, attention_factor=1.5, interleaved=interleaved, transposed=True)
    want, size = turned(w, pos, inv, 1.5, interleaved, transposed=True)
    check(got, want, size)
    leaf = x.double().requires_grad_()
    (turned(leaf, pos, inv, 1.5, interleaved)[0] * w.double()).sum().backward()
    check(got, leaf.grad, size)
    # the map is linear: a difference quotient is exact up to rounding; 30
    # products of values below 8 in fp32, summed in 64 bits
    for at in ((0, 0, 0, 0), (0, 2, 1, 9), (0, 4, 0, 20)):
        d = torch.zeros_like(x)
        d[at] = 1.0
        diff = [apply_rotary(x + s * d, None, pos, inv, attention_factor=1.5, interleaved=interleaved)[0].double()
                for s in (1.0, -1.0)]
        quotient = ((diff[0] - diff[1]) / 2 * w.double()).sum()
        assert abs(float(quotient - got[at])) < 240 * 2.0 ** -22 * 8


def test_empty_and_other_stream():
    inv, _ = rotary_frequencies(16, device=DEV)
    q = rand((2, 0, 4, 16), torch.float16, 8)
    got, _ = apply_rotary(q, None, torch.arange(0, device=DEV), inv)
    assert got.shape == q.shape
    q = rand((1, 300, 4, 16), torch.float16, 8)
    pos = torch.arange(300, device=DEV)
    want, _ = apply_rotary(q, None, pos, inv)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = apply_rotary(q, None, pos, inv)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_refusals():
    q, k = rand((1, 4, 2, 16), torch.float16, 9), rand((1, 4, 1, 16), torch.float16, 9)
    inv, _ = rotary_frequencies(16, device=DEV)
    pos = torch.arange(4, device=DEV)
    for args, kw, match in (
            ((q, k.float(), pos, inv), {}, "k must be"),
            ((q, k[:, :3], pos, inv), {}, "k must have q's"),
            ((q, k, pos[:3], inv), {}, "positions must be"),
            ((q, k, pos.float(), inv), {}, "int32 or int64"),
            ((q, k, pos, inv.double()), {}, "float32"),
            ((q, k, pos, inv[:0]), {}, "frequencies"),
            ((q, k, pos, rotary_frequencies(18, device=DEV)[0]), {}, "frequencies"),
            ((q.long(), None, pos, inv), {}, "must be float16"),
            ((q[0, 0], None, pos, inv), {}, "4-D"),
            ((q[..., ::2], None, pos, inv[:2]), {"inplace": True}, "contiguous")):
        with pytest.raises(ValueError, match=match):
            apply_rotary(*args, **kw)
    with pytest.raises(RuntimeError, match="no_grad"):
        apply_rotary(q.clone().requires_grad_(), k, pos, inv)
    with torch.no_grad():
        apply_rotary(q.clone().requires_grad_(), k, pos, inv)
    with pytest.raises(RuntimeError):
        apply_rotary(q[:, :1].expand(1, 4, 2, 16), None, pos, inv, inplace=True)
