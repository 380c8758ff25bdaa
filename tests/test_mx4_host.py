"""CPU checks of the 4-bit weights' host side and of the router's configuration."""
import math

import pytest
import torch

import _mx4 as ref
from smaulnative_amd import FP8Linear, MoEConfig, MX4Experts, MX4Linear, SwiFFN_MoE, mx4
from smaulnative_amd.fp8_tile import decode_block


@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (2, 33), (5, 100), (2, 3, 64)])
def test_host_quantizer_and_decoder(shape):
    gen = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(*shape, generator=gen) * torch.pow(2.0, torch.randint(-60, 60, (*shape[:-1], 1), generator=gen).float())
    flat = x.view(-1, shape[-1])
    flat[0] = 0.0
    for dtype in (torch.float32, torch.bfloat16):
        codes, scales = mx4.quantize(x.to(dtype))
        wc, ws = ref.quantize(x.to(dtype))
        assert torch.equal(codes, wc) and torch.equal(scales, ws)
        assert torch.equal(mx4.decode(codes, scales, shape[-1]).double(), ref.values(wc, ws, shape[-1]))


def test_host_quantizer_edges():
    borders = torch.tensor([b for b, _ in ref.BORDERS] + [5.999, 7.0, 7.99, 4.0])
    row = torch.cat([borders, -borders, torch.nextafter(borders, torch.tensor(9.0))[:10]])
    x = torch.stack([row[:32] * 2.0 ** e for e in (-148, -126, -125, -1, 0, 100, 125)])
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    c, s = mx4.quantize(x)
    wc, ws = ref.quantize(x)
    assert torch.equal(c, wc) and torch.equal(s, ws)
    bad = torch.ones(3, 64)
    bad[0, 3], bad[1, 40] = math.nan, math.inf
    c, s = mx4.quantize(bad)
    assert s.tolist() == [[255, 125], [125, 255], [125, 125]]
    v = mx4.decode(c, s, 64)
    assert torch.isnan(v[0, :32]).all() and torch.isnan(v[1, 32:]).all() and (v[2] == 1.0).all()


def test_modules_hold_the_quantized_weights():
    gen = torch.Generator().manual_seed(2)
    lin = torch.nn.Linear(70, 24)
    m = MX4Linear.from_float(lin)
    assert torch.equal(mx4.decode(m.w4, m.ws, 70).double(), ref.rounded(lin.weight.detach()))
    assert torch.equal(m.bias, lin.bias)
    f = FP8Linear(128, 16)
    m = MX4Linear.from_fp8(f, act="mx4")
    want = ref.rounded(decode_block(f.w8, f.sc, 0, 16, 128, 64))
    assert torch.equal(mx4.decode(m.w4, m.ws, 128).double(), want) and m.act == "mx4"
    other = MX4Linear(70, 24, bias=True)
    other.load_state_dict(MX4Linear.from_float(lin).state_dict())
    assert torch.equal(other.bias, lin.bias)
    moe = SwiFFN_MoE(MoEConfig(d_model=64, num_experts=3, num_experts_per_tok=2))
    ex = MX4Experts.from_experts(moe.experts)
    assert len(ex) == 3 and ex.gate_w.shape == (3, 160, 32) and ex.down_s.shape == (3, 64, 5)
    up = moe.experts[1].up
    assert torch.equal(mx4.decode(ex.up_w[1], ex.up_s[1], 64).double(),
                       ref.rounded(decode_block(up.w8, up.sc, 0, 160, 64, 64)))
    with pytest.raises(IndexError):
        ex[3]


def test_router_configuration():
    base = dict(d_model=64, num_experts=8, num_experts_per_tok=2)
    assert SwiFFN_MoE(MoEConfig(**base)).route_args is None  # the softmax router runs as it did
    m = SwiFFN_MoE(MoEConfig(**base, router_score="sigmoid", router_groups=4, router_top_groups=2, router_scale=2.5,
                             router_bias=True))
    assert m.route_args == dict(score="sigmoid", groups=4, top_groups=2, group_best=2, renorm=True, scale=2.5)
    assert "balance_bias" in m.state_dict() and m.balance_bias.shape == (8,)
    assert "balance_bias" not in SwiFFN_MoE(MoEConfig(**base)).state_dict()
    m.expert_token_counts = [4, 0, 1, 1, 1, 1, 0, 0]
    m.balance_step(0.5)
    assert m.balance_bias.tolist() == [-0.5, 0.5, 0.0, 0.0, 0.0, 0.0, 0.5, 0.5]
    with pytest.raises(RuntimeError):
        SwiFFN_MoE(MoEConfig(**base)).balance_step(0.1)
    for bad in (dict(router_score="max"), dict(router_groups=3), dict(router_groups=8, router_top_groups=1),
                dict(router_top_groups=2), dict(router_group_best=0)):
        with pytest.raises(ValueError):
            SwiFFN_MoE(MoEConfig(**base, **bad))
    with pytest.raises(ValueError):
        SwiFFN_MoE(MoEConfig(**base, precision="mx4", expert_act="fp8"))
    with pytest.raises(ValueError):
        SwiFFN_MoE(MoEConfig(**base, precision="fp32"))


def test_no_fallback_on_host_tensors():
    m = SwiFFN_MoE(MoEConfig(d_model=64, num_experts=2, precision="mx4"))
    with pytest.raises(RuntimeError, match="HIP device tensors"):
        with torch.no_grad():
            m(torch.zeros(3, 64))
    with pytest.raises(RuntimeError, match="HIP device tensors"):
        MX4Linear(64, 8)(torch.zeros(3, 64))
    with pytest.raises(ValueError):
        MX4Linear(64, 8, act="int8")
    with pytest.raises(ValueError):
        mx4.quantize(torch.zeros(3, 4, dtype=torch.int32))


def test_balance_bias_stays_fp32():
    """A cast of the layer leaves the bias' small steps in place; load_state_dict still writes it."""
    layer = SwiFFN_MoE(MoEConfig(d_model=64, tile=64, num_experts=4, num_experts_per_tok=2, precision="mx4",
                                 router_bias=True))
    layer._counts_host = [4, 0, 1, 3]
    for _ in range(3):
        layer.balance_step(1e-3)
    want = torch.tensor([-3e-3, 3e-3, 3e-3, -3e-3])
    layer.bfloat16()
    assert layer.gate.weight.dtype == torch.bfloat16 and layer.balance_bias.dtype == torch.float32
    assert torch.allclose(layer.balance_bias, want, rtol=0, atol=1e-8)  # three sums' half steps
    other = SwiFFN_MoE(MoEConfig(d_model=64, tile=64, num_experts=4, num_experts_per_tok=2, precision="mx4",
                                 router_bias=True)).half()
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other.balance_bias, layer.balance_bias)


def test_router_limits_are_checked_at_construction():
    """What no forward could run does not construct: moe_route's limits, and a scale that
    leaves no weight above 0."""
    def layer(E, k, **kw):
        return SwiFFN_MoE(MoEConfig(d_model=8, ffn_mult=1.0, tile=8, num_experts=E, num_experts_per_tok=k, **kw))

    for precision in ("fp8", "mx4"):
        for scale in (0.0, -1.0, math.inf, math.nan):
            with pytest.raises(ValueError, match="router_scale"):
                layer(4, 2, precision=precision, router_scale=scale)
    with pytest.raises(ValueError, match="512"):
        layer(513, 2, precision="mx4")
    with pytest.raises(ValueError, match="512"):
        layer(520, 2, router_score="sigmoid")
    with pytest.raises(ValueError, match="16"):
        layer(20, 17, router_score="sigmoid")
    with pytest.raises(ValueError, match="64"):
        layer(130, 2, router_groups=65, router_top_groups=3)
    assert layer(512, 16, precision="mx4", router_groups=64, router_top_groups=9).num_experts == 512
    assert layer(20, 17).route_args is None  # the softmax router's own limits are its entry's


def test_layers_pickled_before_the_router_fields():
    """A whole layer saved when it had no router fields loads, moves and casts as it did."""
    import copy
    import pickle
    layer = SwiFFN_MoE(MoEConfig(d_model=64, num_experts=2, num_experts_per_tok=1))
    old = copy.copy(layer)
    old.__dict__ = {k: v for k, v in layer.__dict__.items() if k not in ("route_args", "balance_bias")}
    again = pickle.loads(pickle.dumps(old))
    assert again.route_args is None and again.balance_bias is None
    assert again.to(torch.bfloat16).gate.weight.dtype == torch.bfloat16
    assert copy.deepcopy(again).route_args is None
    with pytest.raises(RuntimeError, match="HIP device tensors"):
        with torch.no_grad():
            again(torch.zeros(3, 64, dtype=torch.bfloat16))  # as a new one: no host fallback
    wide = pickle.loads(pickle.dumps(SwiFFN_MoE(MoEConfig(d_model=64, num_experts=2, router_bias=True))))
    assert wide.route_args["score"] == "softmax" and "balance_bias" in wide.state_dict()
