"""Hybrid layers on the kernels: against the layer written out in 64 bits, step
by step against the whole sequence, and through the conversion of a layer.

Tolerance: a layer rounds about ten times to fp16 one after the other
(projections, convolution, attention, gated norm, MLP), each by at most half an
ulp (2^-11) of values that enter sums; 2-norms are compared within 2^-7."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from exl3_intel_arc_quantizer_b200.converter import convert_layer
from exl3_intel_arc_quantizer_b200.hybrid import HybridDecoderLayer, run_layer

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 2.0 ** -7


def make(linear, seed=0, **kw):
    torch.manual_seed(seed)
    kw = dict(dict(key_heads=2, heads=4, key_dim=64, value_dim=64) if linear
              else dict(heads=4, kv_heads=2, head_dim=64, rotary_dim=32), **kw)
    return HybridDecoderLayer(256, 512, linear=linear, **kw).to(DEV, torch.float16).eval()


def rms(x, w, eps):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w


def written_out(layer, x):
    """The layer in float64."""
    p = {n: t.double() for n, t in layer.named_parameters()}
    x = x.double()
    b, s, _ = x.shape
    n = rms(x, p["input_norm"], layer.eps)
    if hasattr(layer, "linear_attn"):
        m = layer.linear_attn
        w = {k[len("linear_attn."):]: v for k, v in p.items() if k.startswith("linear_attn.")}
        raw = F.pad((n @ w["in_proj_qkv.weight"].T).transpose(1, 2), (m.conv_weight.shape[-1] - 1, 0))
        mixed = F.silu(F.conv1d(raw, w["conv_weight"], groups=raw.shape[1])).transpose(1, 2)
        q, k, v = m._heads(mixed)
        q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6) for t in (q, k))
        rep = m.heads // m.key_heads
        q, k = q.repeat_interleave(rep, 2), k.repeat_interleave(rep, 2)
        g = -w["A_log"].exp() * F.softplus(n @ w["in_proj_a.weight"].T + w["dt_bias"])
        beta = torch.sigmoid(n @ w["in_proj_b.weight"].T)
        S = torch.zeros(b, m.heads, m.key_dim, m.value_dim, dtype=torch.float64, device=x.device)
        out = []
        for t in range(s):
            S = S * g[:, t, :, None, None].exp()
            u = beta[:, t, :, None] * (v[:, t] - torch.einsum("bhkv,bhk->bhv", S, k[:, t]))
            S = S + k[:, t, :, :, None] * u[:, :, None, :]
            out.append(torch.einsum("bhkv,bhk->bhv", S, q[:, t]) * m.key_dim ** -0.5)
        z = (n @ w["in_proj_z.weight"].T).unflatten(-1, (m.heads, m.value_dim))
        y = rms(torch.stack(out, 1), w["norm_weight"], m.eps) * F.silu(z)
        mixed = y.flatten(-2) @ w["out_proj.weight"].T
    else:
        m = layer.self_attn
        w = {k[len("self_attn."):]: v for k, v in p.items() if k.startswith("self_attn.")}
        q = (n @ w["q_proj.weight"].T).view(b, s, m.heads, m.head_dim).transpose(1, 2)
        k = (n @ w["k_proj.weight"].T).view(b, s, m.kv_heads, m.head_dim).transpose(1, 2)
        v = (n @ w["v_proj.weight"].T).view(b, s, m.kv_heads, m.head_dim).transpose(1, 2)
        phi = torch.arange(s, device=x.device).double()[:, None] * m.inv_freq.to(x.device).double()
        r = 2 * phi.shape[1]

        def turn(t):
            a, c = (t[..., 0:r:2], t[..., 1:r:2]) if m.interleaved else (t[..., :r // 2], t[..., r // 2:r])
            a, c = a * phi.cos() - c * phi.sin(), c * phi.cos() + a * phi.sin()
            head = torch.stack((a, c), -1).flatten(-2) if m.interleaved else torch.cat((a, c), -1)
            return torch.cat((head, t[..., r:]), -1) * 1.0

        rep = m.heads // m.kv_heads
        q, k, v = turn(q), turn(k).repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
        att = (q @ k.mT) * m.head_dim ** -0.5
        att = att.masked_fill(torch.ones(s, s, dtype=torch.bool, device=x.device).triu(1), -torch.inf).softmax(-1)
        mixed = (att @ v).transpose(1, 2).reshape(b, s, -1) @ w["o_proj.weight"].T
    h = x + mixed
    n = rms(h, p["post_attention_norm"], layer.eps)
    up = F.silu(n @ p["mlp.gate_proj.weight"].T) * (n @ p["mlp.up_proj.weight"].T)
    return h + up @ p["mlp.down_proj.weight"].T


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("linear,kw", [(True, {}), (True, dict(key_dim=128, value_dim=128)), (False, {}),
                                       (False, dict(interleaved=True, rotary_dim=64))])
def test_layer_matches_the_formulas(linear, kw):
    layer = make(linear, **kw)
    x = torch.randn(2, 90, 256, device=DEV).half()
    with torch.no_grad():
        y, cache = layer(x)
    assert off(y, written_out(layer, x)) <= TOL
    assert (cache is not None) == linear


def test_steps_continue_a_sequence():
    layer = make(True, 1)
    x = torch.randn(3, 40, 256, device=DEV).half()
    with torch.no_grad():
        whole, last = layer(x)
        y, cache = layer(x[:, :33])
        assert off(y, whole[:, :33].double()) <= TOL
        for t in range(33, 36):
            assert off(layer.step(x[:, t], cache), whole[:, t].double()) <= TOL
        y, cache = layer(x[:, 36:], cache)
    assert off(y, whole[:, 36:].double()) <= TOL
    assert off(cache.state, last.state.double()) <= TOL and off(cache.conv, last.conv.double()) <= TOL


@pytest.mark.parametrize("linear", [True, False])
def test_conversion_of_a_layer(linear):
    """Hessians, quantization, reload and re-forward of a hybrid layer."""
    layer = make(linear, 2)
    x = [torch.randn(1, 64, 256, device=DEV).half() for _ in range(2)]
    with torch.no_grad():
        before = run_layer(layer, x[0])
    names = layer.quantizable()
    assert ("linear_attn.in_proj_qkv" if linear else "self_attn.q_proj") in names
    assert not any(n.endswith(("in_proj_a", "in_proj_b")) for n in names)
    results, nxt, _ = convert_layer(layer, x, K=4, layer_runner=run_layer, module_names=names)
    assert set(results) == set(names)
    for name in names:
        w = layer.get_submodule(name).weight
        assert torch.equal(w, results[name].w_hat.T.to(w.dtype))
    with torch.no_grad():
        after = run_layer(layer, x[0])
    assert torch.equal(after, nxt[0]) and after.isfinite().all()
    # the converted layer is a quantized version of the one before
    assert 0 < off(after, before.double()) < 0.5


def test_refusals():
    layer = make(False, 3)
    x = torch.randn(1, 4, 256, device=DEV).half()
    with torch.no_grad(), pytest.raises(ValueError, match="linear layers"):
        layer.step(x[:, 0], None)
    with pytest.raises(RuntimeError, match="no_grad"):
        layer(x)
    with pytest.raises(ValueError, match="multiple of key_heads"):
        HybridDecoderLayer(256, 512, linear=True, heads=3, key_heads=2)
