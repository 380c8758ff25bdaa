"""Routing, 4-bit experts, products and gradients side by side: captured, replayed, on several streams."""
import pytest
import torch

import _mx4 as ref
from smaulnative_amd import MoEConfig, SwiFFN_MoE
from smaulnative_amd.compute import get_backend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _calls(T, d, act):
    """Three calls on one set of inputs, which the test overwrites: a layer, a product, a gradient."""
    gen = torch.Generator().manual_seed(T + d)
    layer = SwiFFN_MoE(MoEConfig(d_model=d, tile=64, num_experts=8, num_experts_per_tok=2, precision="mx4",
                                 router_score="sigmoid", router_groups=4, router_top_groups=2, router_bias=True,
                                 router_scale=2.5, expert_act=act)).to(DEV).eval().requires_grad_(False)
    w, s = (t.to(DEV) for t in ref.weight(d + 32, d, gen))
    be = get_backend("rocm")
    x = torch.randn(T, d, generator=gen).bfloat16().to(DEV)
    g = torch.randn(T, d + 32, generator=gen).bfloat16().to(DEV)
    return x, g, [lambda: layer(x), lambda: be.mx4_forward(x, w, s, d, d + 32, act),
                  lambda: be.mx4_backward_input(g, w, s, d, d + 32)]


@pytest.mark.parametrize("T", [1, 64, 300])
@pytest.mark.parametrize("act", ["keep", "mx4"])
def test_graphs_replay_between_eager_calls(T, act):
    x, g, calls = _calls(T, 192, act)
    graphs = []
    for f in calls:
        f()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        graphs.append((graph, out))
    gen = torch.Generator().manual_seed(7)
    for _ in range(4):
        x.copy_(torch.randn(x.shape, generator=gen))
        g.copy_(torch.randn(g.shape, generator=gen))
        for graph, _ in graphs:
            graph.replay()
        for f, (_, out) in zip(calls, graphs):
            assert torch.equal(out, f())


@pytest.mark.parametrize("T", [5, 300])
def test_streams_side_by_side(T):
    x, g, calls = _calls(T, 256, "keep")
    want = [f() for f in calls]
    streams = [torch.cuda.Stream(DEV) for _ in calls]
    for _ in range(3):
        outs = []
        for f, stream in zip(calls, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                outs.append(f())
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_long_rows_past_32_bit_offsets():
    """The last rows of operands of more than 2^32 values come out as they do alone."""
    be = get_backend("rocm")
    gen = torch.Generator().manual_seed(3)
    K, N, rows = 1024, 1032, 4300003
    w, s = (t.to(DEV) for t in ref.weight(N, K, gen))
    x = torch.empty(rows, K, dtype=torch.bfloat16, device=DEV).normal_()
    for act in ("keep", "mx4"):
        y = be.mx4_forward(x, w, s, K, N, act)
        assert torch.equal(y[-700:], be.mx4_forward(x[-700:].clone(), w, s, K, N, act))
    codes, scales = be.mx4_quantize(x)
    wc, ws = be.mx4_quantize(x[-300:].clone())
    assert torch.equal(codes[-300:], wc) and torch.equal(scales[-300:], ws)
    assert torch.equal(be.mx4_dequantize(codes, scales, K, torch.bfloat16)[-300:],
                       be.mx4_dequantize(wc, ws, K, torch.bfloat16))
    del x, codes, scales
    dx = be.mx4_backward_input(y, w, s, K, N)
    assert torch.equal(dx[-700:], be.mx4_backward_input(y[-700:].clone(), w, s, K, N))


@pytest.mark.parametrize("precision", ["mx4", "fp8"])
@pytest.mark.parametrize("T", [3, 100])
def test_layer_of_many_experts_replays(precision, T):
    """More experts than one call takes: captured, replayed between eager calls on another stream."""
    E, k, d = 130, 6, 64
    torch.manual_seed(T)
    layer = SwiFFN_MoE(MoEConfig(d_model=d, tile=64, num_experts=E, num_experts_per_tok=k, precision=precision,
                                 router_score="sigmoid", router_groups=10, router_top_groups=4, router_bias=True,
                                 router_scale=2.5)).to(DEV).eval().requires_grad_(False)
    gen = torch.Generator().manual_seed(T)
    x = torch.randn(T, d, generator=gen).bfloat16().to(DEV)
    layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x)
        counts = layer._counts_dev
    side = torch.cuda.Stream(DEV)
    for _ in range(3):
        x.copy_(torch.randn(T, d, generator=gen))
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = layer(x)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, eager) and torch.equal(counts, layer._counts_dev) and int(counts.sum()) == T * k


def test_layer_of_other_types():
    """fp16 and fp64 rows run through fp32 experts in 4 bits, with and without gradients."""
    torch.manual_seed(0)
    layer = SwiFFN_MoE(MoEConfig(d_model=64, tile=64, num_experts=4, num_experts_per_tok=2, precision="mx4")).to(DEV)
    x = torch.randn(20, 64, generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        want = layer(x.half().float().to(DEV))
    for dtype in (torch.float16, torch.float64):
        for train in (False, True):
            with torch.set_grad_enabled(train):
                got = layer(x.half().to(dtype).to(DEV))
            assert got.dtype == dtype and layer.last_topi.shape == (20, 2)
            # fp16 rounds the expert's products, its hidden rows and outputs, half a step each
            assert float((got.detach().float() - want).norm() / want.norm()) <= (2e-3 if dtype == torch.float16 else 1e-5)
