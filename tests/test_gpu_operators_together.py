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
