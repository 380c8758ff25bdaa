"""The MoE layer with the wider router and with 4-bit experts, and ``MX4Linear``: the
modules against plain 64-bit forms, forwards and gradients."""
import pytest
import torch

import _mx4 as ref
from smaulnative_amd import MoEConfig, MX4Experts, MX4Linear, SwiFFN_MoE, mx4
from smaulnative_amd.compute import get_backend
from smaulnative_amd.fp8_tile import decode_block

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
WIDE = dict(router_score="sigmoid", router_groups=4, router_top_groups=2, router_scale=2.5, router_bias=True)


def _layer(seed, **kw):
    torch.manual_seed(seed)
    m = SwiFFN_MoE(MoEConfig(d_model=kw.pop("d", 128), ffn_mult=2.5, num_experts=kw.pop("E", 8),
                             num_experts_per_tok=kw.pop("k", 2), **kw))
    with torch.no_grad():
        m.gate.weight.mul_(3.0)
        if m.balance_bias is not None:
            m.balance_bias.normal_(std=0.05)
    return m.to(DEV)


def _rel(a, b):
    return float((a.double().cpu() - b).norm() / b.norm())


def _weights(m):
    """(gate, up, down) [E] of float64 matrices."""
    if isinstance(m.experts, MX4Experts):
        b = [t.cpu() for t in m.experts.buffers6()]
        d, h = m.experts.d, m.experts.h
        return [[ref.values(b[i][e], b[i + 1][e], n) for e in range(len(m.experts))] for i, n in ((0, d), (2, d), (4, h))]
    out = []
    for name in ("gate", "up", "down"):
        lins = [getattr(ex, name) for ex in m.experts]
        out.append([decode_block(l.w8.cpu(), l.sc.cpu(), 0, l.out_f, l.in_f, l.tile).double() for l in lins])
    return out


def _plain(m, x, topi, topw, act="keep"):
    """The layer's output in float64 on a given routing, differentiable in x and topw."""
    gate, up, down = _weights(m)
    out = torch.zeros(x.shape, dtype=torch.float64)
    xv = ref.rounded(x.detach()) if act == "mx4" else x
    for e in range(m.num_experts):
        tok, slot = (topi == e).nonzero(as_tuple=True)
        if tok.numel():
            hid = ref.swiglu(xv[tok] @ gate[e].t(), xv[tok] @ up[e].t())
            if act == "mx4":
                hid = ref.rounded(hid.detach())
            out = out.index_add(0, tok, (hid @ down[e].t()) * topw[tok, slot].unsqueeze(1))
    return out


@pytest.mark.parametrize("precision,act,dtype", [("mx4", "keep", BF), ("mx4", "keep", F32), ("mx4", "mx4", BF),
                                                 ("fp8", "keep", BF), ("fp8", "keep", F32)])
@pytest.mark.parametrize("T", [1, 40, 300])
def test_layer_with_the_wider_router(precision, act, dtype, T):
    m = _layer(T, precision=precision, expert_act=act, **WIDE)
    x = torch.randn(T, 128, generator=torch.Generator().manual_seed(T)).to(dtype).to(DEV)
    with torch.no_grad():
        out = m(x)
    logits = (x.float() @ m.gate.weight.t()).cpu()
    # the module's own logits are a library product: the choice is checked on its scores
    topi = m.last_topi.cpu()
    s = torch.sigmoid(m._logits(x).detach().double().cpu())
    want = ref.route(m._logits(x).detach().cpu(), 2, "sigmoid", m.balance_bias.cpu(), 4, 2, 2, True, 2.5)
    assert torch.equal(topi, want[1]) and logits.shape == s.shape
    assert _rel(m.last_prob, s) <= 1e-6
    # rel-L2: the bars of the FP8 layer's own tests (bf16 2e-3 times the two more
    # roundings here, of the hidden rows and the slots' outputs; fp32 1e-5)
    bar = 1e-5 if dtype == F32 else 6e-3
    assert _rel(out, _plain(m, x.double().cpu(), topi, want[2], act)) <= bar
    assert sum(m.expert_token_counts) == 2 * T
    stats = m.routing_stats()
    assert stats["top_k"] == 2 and len(stats["usage_frac"]) == 8
    # leading dimensions
    with torch.no_grad():
        wide = m(x.view(1, T, 128))
    assert wide.shape == (1, T, 128) and torch.equal(wide.view(T, 128), out)
    assert m.last_topi.shape == (1, T, 2) and m.last_prob.shape == (1, T, 8)


@pytest.mark.parametrize("T", [6, 64, 65, 200])
def test_fp8_layer_on_a_given_routing(T):
    """moe_forward(routing=) equals the layer's own run on the softmax router's outputs,
    and drops empty slots."""
    be = get_backend("rocm")
    m = _layer(3)
    x = torch.randn(T, 128, generator=torch.Generator().manual_seed(T)).to(BF).to(DEV)
    experts = [ex.buffers6() for ex in m.experts]
    want = be.moe_forward(x, m.gate.weight, None, experts, 2, 64)
    prob, topi, topw = be.moe_router(x, m.gate.weight, None, 2)
    got = be.moe_forward(x, m.gate.weight, None, experts, 2, 64, routing=(prob, topi, topw))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    topi[::3, 1], topw[::3, 1] = -1, 0.0
    topi[0], topw[0] = -1, 0.0
    out, _, ti, counts = be.moe_forward(x, m.gate.weight, None, experts, 2, 64, routing=(prob, topi, topw))
    assert ti is topi or torch.equal(ti, topi)
    assert int(counts.sum()) == int((topi >= 0).sum()) and (out[0] == 0).all()
    plain = _plain(m, x.double().cpu(), topi.cpu(), topw.double().cpu())
    assert _rel(out[1:], plain[1:]) <= 6e-3


def test_plain_router_is_untouched():
    """A layer without router fields runs the softmax router's own path, bit for bit."""
    m = _layer(4)
    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    with torch.no_grad():
        out = m(x)
    ref_out = get_backend("rocm").moe_forward(x, m.gate.weight, None, [ex.buffers6() for ex in m.experts], 2, 64)
    assert torch.equal(out, ref_out[0]) and torch.equal(m.last_topi, ref_out[2])


@pytest.mark.parametrize("precision", ["mx4", "fp8"])
@pytest.mark.parametrize("score,renorm,groups", [("sigmoid", True, 4), ("softmax", False, 1)])
def test_training_gradients(precision, score, renorm, groups):
    """x's and the router's gradients of a loss on the output and the scores."""
    m = _layer(5, precision=precision, router_score=score, router_renorm=renorm, router_groups=groups,
               router_top_groups=max(1, groups // 2), router_scale=1.5, router_bias=True).train()
    T = 90
    gen = torch.Generator().manual_seed(6)
    x0 = torch.randn(T, 128, generator=gen)
    g = torch.randn(T, 128, generator=gen)
    gp = torch.randn(T, 8, generator=gen) * 0.1
    x = x0.to(DEV).requires_grad_()
    out = m(x)
    ((out * g.to(DEV)).sum() + (m.last_prob * gp.to(DEV)).sum()).backward()
    topi = m.last_topi.cpu()
    xd = x0.double().requires_grad_()
    wd = m.gate.weight.detach().double().cpu().requires_grad_()
    z = xd @ wd.t()
    s = ref.scores(z, score)
    w = s.gather(1, topi)
    w = (w / w.sum(1, keepdim=True) if renorm else w) * 1.5
    plain = _plain(m, xd, topi, w)
    ((plain * g.double()).sum() + (s * gp.double()).sum()).backward()
    # fp32 layers: 1e-5 a product (the FP8 kernels' own bar), four in a row and back
    assert _rel(out.detach(), plain.detach()) <= 1e-5
    assert _rel(x.grad, xd.grad) <= 4e-5
    assert _rel(m.gate.weight.grad, wd.grad) <= 4e-5
    # the same in eval mode with the fused entries, without a graph
    with torch.no_grad():
        assert _rel(m(x), plain.detach()) <= 1e-5


def test_training_step_moves_the_balance():
    m = _layer(7, precision="mx4", **WIDE).train()
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(2)).to(DEV)
    out = m(x)
    loss = out.square().mean() + m.balance_loss(m.last_prob.view(-1, 8))
    loss.backward()
    assert torch.isfinite(m.gate.weight.grad).all() and float(m.gate.weight.grad.abs().sum()) > 0
    before, counts = m.balance_bias.clone(), list(m.expert_token_counts)
    m.balance_step(0.01)
    mean = sum(counts) / 8
    want = [0.01 * ((mean > c) - (mean < c)) for c in counts]
    assert torch.allclose((m.balance_bias - before).cpu(), torch.tensor(want), atol=1e-7)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("act", ["keep", "mx4"])
def test_linear_module(dtype, act):
    torch.manual_seed(8)
    m = MX4Linear(100, 48, act=act, bias=True).to(DEV)
    with torch.no_grad():
        m.bias.normal_()
    x0 = torch.randn(3, 30, 100).to(dtype)
    x = x0.to(DEV).requires_grad_()
    y = m(x)
    w = ref.values(m.w4.cpu(), m.ws.cpu(), 100)
    xv = ref.rounded(x0) if act == "mx4" else x0.double()
    want = xv @ w.t()
    half = 2.0 ** -8 if dtype == BF else 2.0 ** -24
    tol = (xv.abs() @ w.abs().t()) * 100 * 2.0 ** -24 + half * want.abs()
    got = (y.detach().double().cpu() - m.bias.detach().double().cpu())
    # the bias is added to the rounded product, in fp32
    assert ((got - want).abs() <= tol + 2.0 ** -23 * y.detach().double().cpu().abs()).all()
    g = torch.randn(3, 30, 48).to(y.dtype)
    y.backward(g.to(DEV))
    gq = g.to(dtype).double()
    dx = gq @ w  # the rounding of the activations taken as the identity
    tol = (gq.abs() @ w.abs()) * (48 * 2.0 ** -24) + half * dx.abs()
    assert x.grad.dtype == dtype and ((x.grad.double().cpu() - dx).abs() <= tol + 1e-30).all()
    assert torch.allclose(m.bias.grad.cpu().double(), g.double().sum((0, 1)), rtol=1e-5, atol=1e-4)
    assert torch.equal(mx4.decode(m.w4, m.ws, 100).double().cpu(), w)


def test_experts_are_callable():
    m = _layer(9, precision="mx4")
    x = torch.randn(20, 128, generator=torch.Generator().manual_seed(3)).to(DEV)
    gate, up, down = _weights(m)
    for e in (0, 7):
        want = ref.swiglu(x.double().cpu() @ gate[e].t(), x.double().cpu() @ up[e].t()) @ down[e].t()
        assert _rel(m.experts[e](x), want) <= 1e-5


def _plain_by_expert(m, x, topi, topw):
    """``_plain`` with act "mx4" as it runs expert by expert: gate's and up's products and
    the hidden rows are of x's type (bf16) before they are rounded to the format."""
    gate, up, down = _weights(m)
    out = torch.zeros(x.shape, dtype=torch.float64)
    xv = ref.rounded(x)
    for e in range(m.num_experts):
        tok, slot = (topi == e).nonzero(as_tuple=True)
        if tok.numel():
            g, u = ((xv[tok] @ w[e].t()).to(x.dtype).double() for w in (gate, up))
            hid = ref.rounded(ref.swiglu(g, u).to(x.dtype))
            out = out.index_add(0, tok, (hid @ down[e].t()) * topw[tok, slot].unsqueeze(1))
    return out


@pytest.mark.parametrize("precision,act,dtype,E,k,d", [
    ("mx4", "keep", F32, 80, 4, 64), ("mx4", "keep", BF, 160, 6, 64), ("mx4", "mx4", BF, 65, 2, 64), ("fp8", "keep", F32, 80, 4, 64),
    ("fp8", "keep", BF, 130, 8, 64),                                        # more experts than one call takes
    ("mx4", "keep", F32, 20, 10, 64), ("fp8", "keep", F32, 80, 10, 64),     # more slots
    ("mx4", "keep", F32, 8, 2, 36), ("mx4", "mx4", F32, 8, 2, 64)])         # widths and types that it does not take
@pytest.mark.parametrize("T", [7, 90])
def test_layers_past_one_call(precision, act, dtype, E, k, d, T):
    """What a layer takes in training it takes without gradients, and means the same."""
    groups = 5 if E % 5 == 0 else 2 if E % 2 == 0 else 1
    m = _layer(T + E, precision=precision, expert_act=act, E=E, k=k, d=d, tile=4 if d == 36 else 64, router_score="sigmoid",
               router_groups=groups, router_top_groups=max(1, groups - 1), router_scale=2.5, router_bias=True)
    x = torch.randn(T, d, generator=torch.Generator().manual_seed(T)).to(dtype).to(DEV)
    with torch.no_grad():
        out = m(x)
    topi = m.last_topi.cpu()
    want = ref.route(m._logits(x).detach().cpu(), k, "sigmoid", m.balance_bias.cpu(), groups, max(1, groups - 1), 2, True, 2.5)
    assert torch.equal(topi, want[1]) and out.dtype == dtype and out.shape == x.shape
    counts = m.expert_token_counts
    assert counts == torch.bincount(topi.flatten(), minlength=E).tolist()
    plain = _plain(m, x.double().cpu(), topi, want[2], act)
    # as test_layer_with_the_wider_router; rounded rows whose fp32 values differ in their last
    # bits may round to other codes, a step of 2^-2 of few values
    bar = 1e-5 if dtype == F32 and act == "keep" else 6e-3
    assert _rel(out, plain) <= bar
    trained = m(x.clone().requires_grad_())
    if act == "mx4" and dtype == BF:
        plain = _plain_by_expert(m, x.cpu(), topi, want[2])
    # in training bf16 also rounds gate's and up's products and each expert's output
    assert _rel(trained.detach(), plain) <= 2 * bar and m.expert_token_counts == counts
    with torch.no_grad():
        wide = m(x.view(1, T, d))
    assert wide.shape == (1, T, d) and torch.equal(wide.view(T, d), out) and m.last_topi.shape == (1, T, k)


@pytest.mark.parametrize("precision", ["mx4", "fp8"])
def test_router_scores_with_a_gate_bias(precision):
    """The layer's scores against x . W^T + b formed here in 64 bits."""
    m = _layer(21, precision=precision, **WIDE)
    T, d = 70, 128
    gen = torch.Generator().manual_seed(21)
    m.gate.bias = torch.nn.Parameter(torch.randn(8, generator=gen).to(DEV))
    x = torch.randn(T, d, generator=gen)
    w, b = m.gate.weight.detach().double().cpu(), m.gate.bias.detach().double().cpu()
    z = x.double() @ w.t() + b
    want = torch.sigmoid(z)
    # fp32 sums of d + 1 terms, each rounding at most 2^-24 of their magnitudes; sigmoid's
    # slope is s (1 - s), and its own arithmetic |z| + 16 steps of 2^-24
    dz = (x.double().abs() @ w.abs().t() + b.abs()) * (d + 1) * 2.0 ** -24
    tol = want * ((1 - want) * dz * 1.01 + (z.abs() + 16) * 2.0 ** -24)
    for train in (False, True):
        with torch.set_grad_enabled(train):
            m(x.to(DEV))
        assert ((m.last_prob.detach().cpu().double() - want).abs() <= tol).all()
