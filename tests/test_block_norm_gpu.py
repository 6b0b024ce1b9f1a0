"""Norms around a block against the formulas in 64 bits.

Tolerance: a sum of d squares in fp32 (at most 128 terms in a row, then a
tree) is within 2^-16 of exact, its root within 2^-17; the exponential of a
gate |z| < 16 within 2^-19; the products add a few 2^-24. So y is within
2^-16 |y|, hidden within 2^-16 (|residual| + |s y|), normed the same relative
to those terms times its factor, and each output is rounded once more (half
an ulp)."""

from __future__ import annotations

import pytest
import torch

from exl3_intel_arc_quantizer_b200.norms import block_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}


def formula(x, weight=None, gate=None, gate_activation="silu", residual=None, residual_scale=1.0,
            scale=None, next_weight=None, eps=1e-6, weight_offset=0.0):
    """(hidden, size of its terms, normed, size of its terms) in float64."""
    def rms(t):
        return torch.rsqrt((t * t).mean(-1, keepdim=True) + eps)

    y = x.double()
    if weight is not None:
        y = y * rms(y) * (weight_offset + weight.double())
    if gate is not None:
        z = gate.double()
        y = y * torch.sigmoid(z) * (1 if gate_activation == "sigmoid" else z)
    size = y.abs()
    if residual is not None:
        y = residual_scale * (1 if scale is None else scale.double()) * y
        size = residual.double().abs() + y.abs()
        y = residual.double() + y
    if next_weight is None:
        return y, size, None, None
    f = rms(y) * (weight_offset + next_weight.double())
    return y, size, y * f, size * f.abs()


def check(got, want, size):
    tol = HALF_ULP[got.dtype] * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -16 * size + SMALLEST[got.dtype]
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off"


def rand(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def inputs(rows, d, dtype, param, parts, seed=0):
    kw = {}
    if "w" in parts:
        kw["weight"] = rand(d, param, seed + 1)
    if "g" in parts or "G" in parts:
        kw["gate"] = rand((rows, d), dtype, seed + 2, 2.0)
        kw["gate_activation"] = "silu" if "g" in parts else "sigmoid"
    if "r" in parts:
        kw["residual"], kw["residual_scale"] = rand((rows, d), dtype, seed + 3, 2.0), 0.7
    if "s" in parts:
        kw["scale"] = rand(d, param, seed + 4)
    if "n" in parts:
        kw["next_weight"] = rand(d, param, seed + 5)
    return rand((rows, d), dtype, seed, 1.5), kw


def run_and_check(x, kw):
    h, n = block_norm(x, **kw)
    want = formula(x, **kw)
    assert h.shape == x.shape and h.dtype == x.dtype
    check(h, *want[:2])
    assert (n is None) == (kw.get("next_weight") is None)
    if n is not None:
        assert n.shape == x.shape and n.dtype == x.dtype
        check(n, *want[2:])
    return h, n


@pytest.mark.parametrize("dtype,param", [(torch.float16, torch.float16), (torch.float16, torch.float32),
                                         (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                         (torch.float32, torch.float32)])
@pytest.mark.parametrize("parts", ["n", "w", "g", "r", "wg", "rn", "wrn", "wGrsn", "wgrsn"])
def test_every_part(dtype, param, parts):
    run_and_check(*inputs(5, 256, dtype, param, parts))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (7, 8), (9, 31), (300, 64), (33, 128), (2, 130), (1, 1000),
                                    (5, 1024), (4, 1032), (1, 4096), (200, 4096), (3, 4095), (2, 5120),
                                    (2, 8190), (2, 14336), (2, 20000), (1, 33000), (1, 50001)])
def test_row_lengths(dtype, rows, d):
    run_and_check(*inputs(rows, d, dtype, dtype, "wgrn"))
    run_and_check(*inputs(rows, d, dtype, dtype, "n"))


@pytest.mark.parametrize("d", [4095, 4093, 130, 1001])
def test_odd_rows_many(d):
    run_and_check(*inputs(700, d, torch.float16, torch.float16, "wGrn"))
    run_and_check(*inputs(700, d, torch.bfloat16, torch.float32, "wGrsn"))


def test_strides_and_leading_dimensions():
    base = rand((6, 3 * 96 + 5), torch.float16, 1)
    w = rand(96, torch.float16, 2)
    for off in (0, 5, 8):
        x, res = base[:, off:off + 96], base[:, 96 + off:192 + off]
        run_and_check(x, dict(weight=w, residual=res, next_weight=w))
    x = rand((2, 3, 4, 96), torch.float16, 3)
    run_and_check(x, dict(weight=w, gate=rand((2, 3, 4, 96), torch.float16, 4)))
    run_and_check(x.transpose(1, 2), dict(next_weight=w))
    run_and_check(x[0, 0, 0], dict(next_weight=w))
    wide = rand((4, 192), torch.float16, 5)[:, ::2]
    run_and_check(wide, dict(weight=w, residual=wide))
    # x on a 16-byte boundary, the residual and the weight off it
    odd = rand(6 * 96 + 3, torch.float16, 6)[3:].view(6, 96)
    run_and_check(base[:, :96].contiguous(), dict(residual=odd, next_weight=rand(97, torch.float16, 7)[1:]))


def test_norm_alone_leaves_x():
    x, kw = inputs(4, 64, torch.float16, torch.float16, "n")
    h, n = block_norm(x, **kw)
    assert h is x or h.data_ptr() == x.data_ptr()


def test_offset_and_eps():
    x, kw = inputs(4, 64, torch.float32, torch.float32, "wrn")
    run_and_check(x * 1e-3, dict(kw, weight_offset=1.0, eps=1e-2))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_zeros_infinities_and_nan_stay_in_their_rows(dtype):
    x, kw = inputs(6, 96, dtype, dtype, "wgrn")
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    kw["gate"][3, 9] = -float("inf")   # silu(-inf) = -inf * 0
    kw["gate"][4, 0] = -300.0          # exp(300) overflows: the gate is 0
    kw["gate"][4, 1] = 300.0
    h, n = block_norm(x, **kw)
    want = formula(x, **kw)
    assert torch.equal(h.isnan(), want[0].isnan()) and torch.equal(n.isnan(), want[2].isnan())
    for got, w, s in ((h, want[0], want[1]), (n, want[2], want[3])):
        ok = torch.tensor([0, 4, 5], device=DEV)
        check(got[ok], w[ok], s[ok])


def test_many_rows_than_a_grid_and_offsets_past_32_bits():
    d = 65536
    x = torch.zeros((40000, d), dtype=torch.float16, device=DEV)  # 2.6e9 elements
    x[0], x[-1] = 1.0, 2.0
    w = torch.full((d,), 3.0, dtype=torch.float16, device=DEV)
    _, n = block_norm(x, next_weight=w)
    assert float(n[0, 0]) == 3.0 and float(n[-1, -1]) == 3.0
    assert not n[1:-1:997].any()


def test_refusals():
    x = rand((4, 64), torch.float16, 1)
    w = rand(64, torch.float16, 2)
    for kw, match in (({}, "nothing to do"), ({"weight": w[:32]}, "vector of 64"),
                      ({"weight": w.bfloat16()}, "float32"), ({"weight": w, "next_weight": w.float()}, "one type"),
                      ({"gate": x[:2]}, "x's shape"), ({"residual": x.float()}, "like x"),
                      ({"weight": w, "scale": w}, "needs a residual"), ({"gate": x, "gate_activation": "relu"}, "gate_activation"),
                      ({"weight": w[::2]}, "vector of 64"), ({"weight": w.cpu()}, "must be on")):
        with pytest.raises(ValueError, match=match):
            block_norm(x, **kw)
    with pytest.raises(ValueError, match="float16"):
        block_norm(x.double(), next_weight=w)
    with pytest.raises(RuntimeError, match="no_grad"):
        block_norm(x, next_weight=torch.nn.Parameter(w))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [8, 24, 64, 128, 136, 256, 264, 520, 1024, 2048, 4096, 8192])
def test_many_rows(dtype, d):
    """Enough rows for the tiles: whole ones, a last one that is not full."""
    rows = 1501 if d <= 1024 else 701
    run_and_check(*inputs(rows, d, dtype, dtype, "wgrn"))
    run_and_check(*inputs(rows, d, dtype, torch.float32, "wGrsn"))
    run_and_check(*inputs(rows, d, dtype, dtype, "n"))


@pytest.mark.parametrize("d", [33, 63, 129, 250, 517, 1023, 2047, 4093, 4095])
def test_many_odd_rows(d):
    for dtype in (torch.float16, torch.float32):
        run_and_check(*inputs(1203, d, dtype, dtype, "wgrn"))
        run_and_check(*inputs(1203, d, dtype, torch.float32, "rsn"))
    # all tensors equally far past a boundary, and not
    for shifts in ((1, 1, 1), (3, 3, 3), (1, 2, 3)):
        flat = [rand(700 * d + 8, torch.float16, i) for i in range(3)]
        x, gate, res = (f[s:s + 700 * d].view(700, d) for f, s in zip(flat, shifts))
        run_and_check(x, dict(gate=gate, residual=res, weight=rand(d, torch.float16, 9), next_weight=rand(d, torch.float16, 8)))


def test_many_strided_rows():
    base = rand((900, 3 * 256), torch.bfloat16, 1)
    x, gate, res = base.split(256, dim=1)
    w = rand(256, torch.bfloat16, 2)
    run_and_check(x, dict(weight=w, gate=gate, residual=res, next_weight=w))
    run_and_check(x, dict(weight=w, residual=res.contiguous()))
    wide = rand((900, 4096 + 64), torch.float16, 3)
    run_and_check(wide[:, :4096], dict(residual=wide[:, 64:], next_weight=rand(4096, torch.float32, 4)))


@pytest.mark.parametrize("dtype,param", [(torch.float16, torch.float16), (torch.bfloat16, torch.float32),
                                         (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,d", [(1, 333), (3, 1001), (900, 77), (700, 4095), (460, 4610), (300, 9001), (9, 18003)])
def test_rows_off_a_boundary(dtype, param, rows, d):
    """What stands beside a row is not part of it, and every length keeps its own parameters."""
    x, kw = inputs(rows, d, dtype, param, "wGrsn")
    want = run_and_check(x, kw)
    beside = torch.full((rows, d + 8), float("nan"), dtype=dtype, device=DEV)[:, :d]
    beside.copy_(x)
    got = block_norm(beside, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_overlapping_rows_off_a_boundary():
    d = 1001
    x = rand(40 * d, torch.float16, 1).as_strided((37, d), (d - 8, 1))
    _, kw = inputs(37, d, torch.float16, torch.float16, "wrn")
    run_and_check(x, kw)


@pytest.mark.parametrize("d", [16, 128, 77, 250])
def test_many_short_rows(d):
    run_and_check(*inputs(160_000 if d < 100 else 40_000, d, torch.float16, torch.float16, "wgrn"))
