"""Host side of the layer operators: frequencies, argument checks of the C
entry points (no device work is issued), and no CPU path."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from exl3_intel_arc_quantizer_b200 import _ext
from exl3_intel_arc_quantizer_b200.calibration import make_rotary_embeddings
from exl3_intel_arc_quantizer_b200.delta_rule import gated_delta_rule, gated_delta_step_
from exl3_intel_arc_quantizer_b200.norms import block_norm
from exl3_intel_arc_quantizer_b200.rotary import apply_rotary, rotary_frequencies

EINVAL = -22
P, I64, I32, F32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float


def test_plain_frequencies_are_the_calibration_models():
    inv, factor = rotary_frequencies(128)
    assert factor == 1.0 and inv.dtype == torch.float32 and inv.shape == (64,)
    cos, sin = make_rotary_embeddings(50, 128, dtype=torch.float32)
    phi = torch.outer(torch.arange(50.0), inv)
    # two fp32 roundings of the frequency and one of the product: 3 * 2^-24 * 50 radians
    assert float((phi.cos() - cos[0, 0, :, :64]).abs().max()) < 50 * 2.0 ** -22
    assert float((phi.sin() - sin[0, 0, :, 64:]).abs().max()) < 50 * 2.0 ** -22


def test_scaled_frequencies():
    d, base, f, length = 64, 10000.0, 4.0, 4096
    plain = torch.tensor([base ** (-2 * j / d) for j in range(d // 2)], dtype=torch.float64)
    turns = length * plain / (2 * math.pi)

    def ratio(**kw):
        inv, factor = rotary_frequencies(d, base, factor=f, original_length=length, **kw)
        return inv.double() / plain, factor

    r, a = ratio(scaling="linear")
    assert torch.allclose(r, torch.full_like(r, 1 / f), rtol=1e-6) and a == 1.0
    r, a = ratio(scaling="ntk")
    assert abs(float(r[0]) - 1) < 1e-6 and abs(float(r[-1]) - 1 / f) < 1e-6 and a == 1.0
    assert bool((r[1:] < r[:-1]).all())
    r, a = ratio(scaling="yarn")
    assert torch.allclose(r[turns > 33.5], torch.ones(1, dtype=torch.float64), rtol=1e-6)
    assert torch.allclose(r[turns < 0.7], torch.full((1,), 1 / f, dtype=torch.float64), rtol=1e-6)
    assert bool((r[1:] <= r[:-1] + 1e-7).all()) and abs(a - (0.1 * math.log(f) + 1)) < 1e-12
    r, a = ratio(scaling="banded")
    assert torch.allclose(r[turns > 4], torch.ones(1, dtype=torch.float64), rtol=1e-6) and a == 1.0
    assert torch.allclose(r[turns < 1], torch.full((1,), 1 / f, dtype=torch.float64), rtol=1e-6)
    mid = (turns > 1) & (turns < 4)
    keep = (turns[mid] - 1) / 3
    assert mid.any() and torch.allclose(r[mid], keep + (1 - keep) / f, rtol=1e-6)
    each = [1 + j / 7 for j in range(d // 2)]
    r, a = ratio(scaling="per_frequency", frequency_factors=each)
    assert torch.allclose(r, 1 / torch.tensor(each, dtype=torch.float64), rtol=1e-6)
    assert abs(a - math.sqrt(1 + math.log(f) / math.log(length))) < 1e-12


@pytest.mark.parametrize("kw,match", [
    (dict(rotary_dim=7), "even"), (dict(rotary_dim=0), "even"), (dict(rotary_dim=8, scaling="other"), "scaling"),
    (dict(rotary_dim=8, factor=0.5), "factor"), (dict(rotary_dim=8, base=1.0), "base"),
    (dict(rotary_dim=8, base=float("nan")), "base"), (dict(rotary_dim=8, original_length=0), "original_length"),
    (dict(rotary_dim=2, scaling="ntk", factor=2.0), "ntk"), (dict(rotary_dim=8, scaling="per_frequency"), "frequency_factors"),
    (dict(rotary_dim=8, scaling="yarn", factor=2.0, beta_slow=40.0), "beta_fast"),
    (dict(rotary_dim=8, scaling="banded", factor=2.0, high_freq_factor=1.0), "high_freq")])
def test_frequency_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        rotary_frequencies(**kw)


class RotaryArgs(ctypes.Structure):
    _fields_ = [("q", P), ("k", P), ("q_out", P), ("k_out", P), ("positions", P), ("inv_freq", P),
                ("batch", I64), ("tokens", I64), ("q_strides", I64 * 3), ("k_strides", I64 * 3),
                ("q_out_strides", I64 * 3), ("k_out_strides", I64 * 3), ("position_strides", I64 * 2),
                ("q_heads", I32), ("k_heads", I32), ("dim", I32), ("rotary_dim", I32), ("dtype", I32),
                ("positions_64", I32), ("interleaved", I32), ("transposed", I32), ("factor", F32)]


class NormArgs(ctypes.Structure):
    _fields_ = [(n, P) for n in ("x", "gate", "residual", "weight", "next_weight", "scale", "hidden", "normed")] + \
        [(n, I64) for n in ("rows", "d", "x_stride", "gate_stride", "residual_stride", "hidden_stride", "normed_stride")] + \
        [(n, I32) for n in ("dtype", "param_dtype", "gate_activation")] + \
        [(n, F32) for n in ("eps", "weight_offset", "residual_scale")]


class DeltaArgs(ctypes.Structure):
    _fields_ = [(n, P) for n in ("q", "k", "v", "g", "beta", "state_in", "state_out", "out", "cu_seqlens", "slots")] + \
        [(n, I64) for n in ("tokens", "seqs", "num_slots")] + [(n, I64 * 2) for n in ("q_strides", "k_strides", "v_strides")] + \
        [("g_stride", I64), ("beta_stride", I64)] + \
        [(n, I32) for n in ("key_heads", "heads", "dk", "dv", "dtype", "normalize_qk")] + [("scale", F32)]


def refused(f, args, match, *more):
    lib = _ext.lib()
    assert f(ctypes.byref(args), *more, None) == EINVAL
    assert match in lib.exl3_last_error(), lib.exl3_last_error()


def test_rotary_entry_point_refuses():
    f = _ext.lib().exl3_rotary
    f.argtypes = [P, P]
    good = dict(q=256, k=256, q_out=256, k_out=256, positions=256, inv_freq=256, batch=1, tokens=4, q_heads=2,
                k_heads=1, dim=64, rotary_dim=64, factor=1.0)
    assert f(None, None) == EINVAL
    for change, match in (({"dtype": 3}, b"dtype"), ({"rotary_dim": 66}, b"rotary_dim"), ({"rotary_dim": 3}, b"rotary_dim"),
                          ({"q_heads": 0}, b"q_heads"), ({"q": None}, b"NULL"), ({"k": None}, b"NULL"),
                          ({"tokens": -1}, b"non-negative"), ({"positions": None}, b"NULL"), ({"dim": 10000}, b"dim")):
        refused(f, RotaryArgs(**{**good, **change}), match)
    assert f(ctypes.byref(RotaryArgs(**{**good, "tokens": 0})), None) == 0


def test_norm_entry_point_refuses():
    f = _ext.lib().exl3_block_norm
    f.argtypes = [P, P]
    good = dict(x=256, hidden=256, normed=256, weight=256, next_weight=256, rows=3, d=64, dtype=1, param_dtype=1)
    assert f(None, None) == EINVAL
    for change, match in (({"dtype": -1}, b"dtype"), ({"param_dtype": 0}, b"param_dtype"), ({"d": 0}, b"d positive"),
                          ({"gate": 256}, b"activation"), ({"gate_activation": 3}, b"gate_activation"), ({"x": None}, b"NULL"),
                          ({"normed": None}, b"go together"), ({"next_weight": None}, b"go together"),
                          ({"hidden": None, "normed": None, "next_weight": None}, b"no output")):
        refused(f, NormArgs(**{**good, **change}), match)
    assert f(ctypes.byref(NormArgs(**{**good, "rows": 0})), None) == 0


def test_delta_entry_points_refuse():
    lib = _ext.lib()
    step, rule, size = lib.exl3_delta_step, lib.exl3_delta_rule, lib.exl3_delta_rule_ws_bytes
    step.argtypes, rule.argtypes = [P, P], [P, P, ctypes.c_size_t, P]
    size.argtypes, size.restype = [P], ctypes.c_size_t
    good = dict(q=256, k=256, v=256, g=256, beta=256, state_out=256, out=256, cu_seqlens=256, tokens=4, seqs=4,
                num_slots=4, key_heads=2, heads=4, dk=64, dv=64)
    assert step(None, None) == EINVAL and size(None) == 0
    shared = (({"dtype": 2}, b"dtype"), ({"heads": 3}, b"multiple"), ({"key_heads": 0}, b"multiple"), ({"dk": 264}, b"dk"),
              ({"dk": 12}, b"dk"), ({"dv": 4}, b"dv"), ({"tokens": -1}, b"non-negative"), ({"state_out": None}, b"states"),
              ({"state_out": 260}, b"states"), ({"q": None}, b"NULL"), ({"out": 264}, b"aligned"))
    for change, match in shared + (({"seqs": 3}, b"one token"), ({"num_slots": 3}, b"num_slots")):
        refused(step, DeltaArgs(**{**good, **change}), match)
    for change, match in shared + (({"cu_seqlens": None}, b"cu_seqlens"),):
        refused(rule, DeltaArgs(**{**good, **change}), match, 256, 1 << 40)
    args = DeltaArgs(**good)
    assert size(ctypes.byref(args)) > 0
    assert rule(ctypes.byref(args), 256, size(ctypes.byref(args)) - 1, None) == EINVAL
    assert b"smaller than" in lib.exl3_last_error()
    empty = DeltaArgs(**{**good, "tokens": 0, "seqs": 0, "num_slots": 0})
    assert step(ctypes.byref(empty), None) == 0


def test_no_cpu_path():
    x = torch.zeros(1, 1, 8, dtype=torch.float16)
    g = torch.zeros(1, 1)
    for call in (lambda: apply_rotary(x, None, torch.zeros(1, dtype=torch.int64), torch.ones(4)),
                 lambda: block_norm(x, next_weight=x[0, 0]),
                 lambda: gated_delta_rule(x, x, x, g, g),
                 lambda: gated_delta_step_(x, x, x, g, g, torch.zeros(1, 1, 8, 8))):
        with pytest.raises(_ext.NativeUnavailable, match="CUDA"):
            call()


def test_hybrid_layer_names_its_projections():
    """The Hessian groups of both kinds of layer, and what the quantizer takes."""
    from exl3_intel_arc_quantizer_b200.calibration import hessian_groups
    from exl3_intel_arc_quantizer_b200.hybrid import HybridDecoderLayer

    layer = HybridDecoderLayer(256, 512, linear=True, key_heads=2, heads=4, key_dim=64, value_dim=64)
    groups = hessian_groups(layer)
    assert groups["linear_attn.input"] == ["linear_attn.in_proj_qkv", "linear_attn.in_proj_z",
                                           "linear_attn.in_proj_b", "linear_attn.in_proj_a"]
    assert groups["linear_attn.out_proj"] == ["linear_attn.out_proj"]
    assert layer.quantizable() == ["linear_attn.in_proj_qkv", "linear_attn.in_proj_z", "linear_attn.out_proj",
                                   "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj"]
    full = HybridDecoderLayer(256, 512, linear=False, heads=4, kv_heads=2, head_dim=64)
    assert hessian_groups(full)["self_attn.input"] == ["self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"]
