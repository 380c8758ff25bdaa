"""Routing from logits (``moe_route``) and its gradient against plain 64-bit forms."""
import math

import pytest
import torch

import _mx4 as ref
from smaulnative_amd.compute import get_backend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def _logits(T, E, dtype, seed, std=0.64):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(T, E, generator=gen) * std).to(dtype), gen


def _tol(logits, E):
    """Relative error of an fp32 score: E / 16 + 4 roundings of the sum, a rounding of
    z - m (which the exponential turns into |z - m| 2^-24), and 8 for exp and the rest."""
    z = logits.float()
    z = z[torch.isfinite(z)]
    span = min(104.0, float(z.max().double() - z.min().double())) if z.numel() else 0.0  # past it a score is 0
    return (E / 16 + 12 + span) * 2.0 ** -24


def _check(logits, k, bias=None, score="softmax", groups=1, top_groups=None, best=2, renorm=True, scale=1.0):
    be = get_backend("rocm")
    tg = groups if top_groups is None else top_groups
    prob, topi, topw = be.moe_route(logits.to(DEV), k, score=score, bias=None if bias is None else bias.to(DEV),
                                    groups=groups, top_groups=top_groups, group_best=best, renorm=renorm, scale=scale)
    s, ti, tw = ref.route(logits, k, score, bias, groups, tg, best, renorm, scale)
    assert prob.dtype == F32 and topi.dtype == torch.int64 and topw.dtype == F32
    assert torch.equal(topi.cpu(), ti)
    tol = _tol(logits, logits.shape[1])
    assert torch.equal(torch.isnan(prob.cpu()), torch.isnan(s))
    fin = ~torch.isnan(s)
    assert ((prob.cpu().double() - s).abs()[fin] <= tol * s[fin] + 1e-37).all()
    assert ((topw.cpu().double() - tw).abs() <= 3 * tol * tw + 1e-37).all()  # a score, the sum and the quotient
    none, ti2, tw2 = be.moe_route(logits.to(DEV), k, score=score, bias=None if bias is None else bias.to(DEV),
                                  groups=groups, top_groups=top_groups, group_best=best, renorm=renorm, scale=scale,
                                  need_prob=False)
    assert none is None and torch.equal(ti2, topi) and torch.equal(tw2, topw)


@pytest.mark.parametrize("T,E,k,groups,top_groups", [
    (1, 1, 1, 1, 1), (1, 4, 2, 1, 1), (3, 5, 5, 1, 1), (65, 8, 2, 1, 1), (7, 16, 8, 4, 2), (130, 60, 6, 6, 3),
    (33, 64, 6, 8, 4), (40, 96, 4, 3, 1), (17, 129, 8, 1, 1), (21, 256, 8, 8, 4), (9, 210, 8, 30, 7), (5, 512, 16, 64, 5),
    (4, 500, 8, 4, 2), (11, 64, 3, 64, 3), (13, 24, 3, 8, 1), (6, 250, 2, 50, 40)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_matches_64_bits(T, E, k, groups, top_groups, score):
    for i, dtype in enumerate((F32, BF)):
        logits, gen = _logits(T, E, dtype, 100 * T + E + i)
        bias = torch.randn(E, generator=gen) * 0.05 if (T + i) % 2 else None
        _check(logits, k, bias, score, groups, top_groups, best=1 + (T + E + i) % 2, renorm=(E + i) % 3 != 0,
               scale=2.5 if i else 1.0)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties_and_neighbours(score, bias):
    """Equal logits go to the lowest index (of groups too), and logits one step apart
    are told apart, whatever a rounding of their scores would say."""
    T, E, k, G = 24, 64, 6, 8
    logits, gen = _logits(T, E, F32, 5)
    logits[:8] = 0.0                                   # every expert the same
    logits[8:12] = logits[8:12, :1] + torch.zeros(E)   # a row of one value
    base = logits[12:16, :1].abs() + 0.1
    step = torch.randperm(E, generator=gen)
    up = base
    row = torch.empty(4, E)
    for e in step.tolist():
        row[:, e:e + 1] = up
        up = torch.nextafter(up, torch.full_like(up, 9.0))
    logits[12:16] = row
    logits[16:20] = torch.randint(-2, 3, (4, E), generator=gen).float() / 2
    logits[20:] = 40.0 + torch.rand(4, E, generator=gen)  # sigmoid: scores within 2^-58 of 1
    b = None if not bias else torch.randint(0, 2, (E,), generator=gen).float() * 0.25
    if bias and score == "sigmoid":
        logits = logits[:20]  # score + bias of the last rows is the same number for many, by a rounding even in 64 bits
    for groups, tg in ((1, 1), (G, 3)):
        if score == "sigmoid" and groups > 1:
            _check(logits[:20], k, b, score, groups, tg)
        else:
            _check(logits, k, b, score, groups, tg)


def test_route_masked_rows():
    T, E = 12, 32
    logits, gen = _logits(T, E, F32, 6)
    inf = math.inf
    logits[0] = -inf                 # nobody
    logits[1, 3:] = -inf             # fewer than k
    logits[2, :16] = -inf            # half of the groups empty
    logits[3] = torch.finfo(F32).min  # the type's lowest value is a value like another
    logits[4, 7] = torch.finfo(F32).min
    logits[5, 9] = math.nan
    logits[6, 1::2] = -inf           # one live expert in each group of two
    bias = torch.randn(E, generator=gen) * 0.1
    for score in ("softmax", "sigmoid"):
        for b in (None, bias):
            _check(logits, 4, b, score)
            _check(logits, 4, b, score, groups=16, top_groups=5)
            _check(logits, 4, b, score, groups=4, top_groups=1, best=1, renorm=False)
    odd = bias.clone()
    odd[3], odd[4], odd[5] = -inf, math.nan, 3.0  # two experts out, one always in
    _check(logits, 4, odd, "sigmoid", groups=4, top_groups=2)
    get = get_backend("rocm").moe_route(torch.full((2, 8), math.inf, device=DEV), 2)
    assert (get[1] == -1).all() and (get[2] == 0).all()  # softmax of infinities: no score


def test_route_far_logits_and_small_sums():
    """Scores from 2^-100 up, and chosen scores whose sum is below the guard."""
    logits, gen = _logits(50, 48, F32, 7, std=12.0)
    _check(logits, 5, None, "softmax")
    _check(logits, 5, torch.linspace(3, 0, 48), "softmax")   # the bias alone decides
    _check(logits - 40.0, 5, None, "sigmoid", renorm=True)
    _check(logits - 40.0, 5, torch.linspace(3, 0, 48), "sigmoid", groups=6, top_groups=2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_many_tokens(score):
    """Every token of a long call, against sorting in 64 bits."""
    T, E, k = 30011, 64, 6
    logits, gen = _logits(T, E, F32, 8)
    bias = torch.randn(E, generator=gen) * 0.05
    _, topi, topw = get_backend("rocm").moe_route(logits.to(DEV), k, score=score, bias=bias.to(DEV), groups=8,
                                                  top_groups=4, need_prob=False)
    s = ref.scores(logits.double(), score)
    c = s + bias.double()
    g = c.view(T, 8, 8).topk(2, -1)[0].sum(-1).topk(4, -1)[1]
    keep = torch.zeros(T, 8, dtype=torch.bool).scatter(1, g, True).repeat_interleave(8, 1)
    ti = c.masked_fill(~keep, -math.inf).topk(k, -1)[1]
    assert torch.equal(topi.cpu(), ti)
    w = s.gather(1, ti)
    w = w / w.sum(1, keepdim=True)
    assert ((topw.cpu().double() - w).abs() <= 3 * _tol(logits, E) * w).all()


def test_route_strides_streams_and_replay():
    be = get_backend("rocm")
    logits, gen = _logits(40, 96, F32, 9)
    wide = torch.zeros(40, 200)
    wide[:, 5:101] = logits
    bias = torch.randn(96, generator=gen) * 0.05
    want = be.moe_route(logits.to(DEV), 4, score="sigmoid", bias=bias.to(DEV), groups=3, top_groups=2)
    got = be.moe_route(wide.to(DEV)[:, 5:101], 4, score="sigmoid", bias=bias.double().to(DEV), groups=3, top_groups=2)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # unaligned rows: 95 of 96 experts from the second on
    shifted = logits.to(DEV).view(-1)[1:1 + 39 * 95].view(39, 95)
    got = be.moe_route(shifted, 4)
    assert torch.equal(got[1].cpu(), ref.route(shifted.cpu(), 4, "softmax", None, 1, 1, 2, True, 1.0)[1])
    empty = be.moe_route(torch.empty(0, 8, device=DEV), 2)
    assert [tuple(t.shape) for t in empty] == [(0, 8), (0, 2), (0, 2)]
    z, b = logits.to(DEV), bias.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = be.moe_route(z, 4, score="sigmoid", bias=b, groups=3, top_groups=2)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = be.moe_route(z, 4, score="sigmoid", bias=b, groups=3, top_groups=2)
    for i in range(3):
        z.copy_(_logits(40, 96, F32, 20 + i)[0])
        graph.replay()
        eager = be.moe_route(z, 4, score="sigmoid", bias=b, groups=3, top_groups=2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, eager))


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (3, 5, 2), (50, 16, 4), (33, 60, 6), (20, 64, 8), (9, 129, 8), (7, 256, 8),
                                   (5, 512, 16)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_gradient(T, E, k, score, renorm):
    be = get_backend("rocm")
    for i, dtype in enumerate((F32, BF)):
        logits, gen = _logits(T, E, dtype, 300 * T + E + i)
        topi = torch.rand(T, E, generator=gen).topk(k, 1)[1]
        if T > 2:
            topi[1, -1] = -1
            topi[2] = -1
        dtopw = torch.randn(T, k, generator=gen)
        dprob = torch.randn(T, E, generator=gen) * 0.3 if (T + i) % 2 else None
        dt = dtopw.clone()
        dt[topi < 0] = math.nan  # an empty slot's gradient is not read
        scale = 1.0 + 1.5 * i
        got = be.moe_route_backward(dt.to(DEV), logits.to(DEV), topi.to(DEV), score=score, renorm=renorm, scale=scale,
                                    dprob=None if dprob is None else dprob.to(DEV))
        assert got.dtype == dtype and got.shape == logits.shape
        z = logits.double().requires_grad_()
        args = (topi, dtopw.double(), None if dprob is None else dprob.double(), score, renorm, scale)
        want, = torch.autograd.grad(ref.route_loss(z, *args), z)
        # magnitudes of the terms: |ds| and the softmax's mean of them, each through a
        # score and a quotient of sums of E / 16 + 4 roundings
        with torch.no_grad():
            s = ref.scores(z, score)
            w = torch.where(topi >= 0, s.gather(1, topi.clamp_min(0)), torch.zeros((), dtype=torch.float64))
            g = dtopw.double().abs() * scale
            if renorm:
                tot = w.sum(1, keepdim=True).clamp_min(1e-30)
                g = (g + (g * w).sum(1, keepdim=True) / tot) / tot
            g = torch.where(topi >= 0, g, torch.zeros_like(g))
            ds = torch.zeros_like(s).scatter_add(1, topi.clamp_min(0), g) + (0 if dprob is None else dprob.double().abs())
            mag = s * ((ds + (s * ds).sum(1, keepdim=True)) if score == "softmax" else ds * torch.sigmoid(-z))
            tol = 6 * _tol(logits, E) * mag + (2.0 ** -8 if dtype == BF else 0.0) * want.abs() + 1e-37
        assert ((got.cpu().double() - want).abs() <= tol).all()


def test_route_gradient_against_differences():
    """The formula's gradient is that of the forward: central differences of the
    forward's own weights and scores (the choice fixed) in 64 bits."""
    gen = torch.Generator().manual_seed(3)
    z = torch.randn(4, 9, generator=gen, dtype=torch.float64)
    topi = torch.rand(4, 9, generator=gen).topk(3, 1)[1]
    dtopw, dprob = torch.randn(4, 3, generator=gen).double(), torch.randn(4, 9, generator=gen).double()
    for score in ("softmax", "sigmoid"):
        for renorm in (False, True):
            got = get_backend("rocm").moe_route_backward(dtopw.float().to(DEV), z.float().to(DEV), topi.to(DEV),
                                                         score=score, renorm=renorm, scale=2.5,
                                                         dprob=dprob.float().to(DEV)).cpu().double()
            zf = z.float().double()
            for t in range(4):
                for e in range(9):
                    h = torch.zeros_like(zf)
                    h[t, e] = 1e-5
                    args = (topi, dtopw.float().double(), dprob.float().double(), score, renorm, 2.5)
                    diff = (ref.route_loss(zf + h, *args) - ref.route_loss(zf - h, *args)) / 2e-5
                    # terms of at most 40 in magnitude at 6 _tol (see above), _tol here below
                    # 17 * 2^-24; the difference's own error (h^2 / 6 of a third derivative, 1e-16 / h) is less
                    assert abs(float(got[t, e] - diff)) <= 6 * 17 * 2.0 ** -24 * 40


def test_route_gradient_masked_and_guarded():
    be = get_backend("rocm")
    z = torch.tensor([[0.0, -math.inf, 1.0, 2.0], [-40.0, -41.0, 0.0, 0.0]])
    topi = torch.tensor([[3, 1], [0, 1]])
    dt = torch.tensor([[1.0, 2.0], [1.0, -1.0]])
    for score in ("softmax", "sigmoid"):
        got = be.moe_route_backward(dt.to(DEV), z.to(DEV), topi.to(DEV), score=score).cpu()
        assert torch.isfinite(got).all() and float(got[0, 1]) == 0.0
        assert (got[1] == 0).all()  # weights of a sum below the guard are constants
    # the same expert in two slots adds both gradients
    a = be.moe_route_backward(torch.tensor([[1.0, 2.0]], device=DEV), z[:1].to(DEV), torch.tensor([[2, 2]], device=DEV),
                              renorm=False)
    b = be.moe_route_backward(torch.tensor([[3.0]], device=DEV), z[:1].to(DEV), torch.tensor([[2]], device=DEV),
                              renorm=False)
    assert torch.equal(a, b)
    assert be.moe_route_backward(torch.empty(0, 2, device=DEV), torch.empty(0, 4, device=DEV),
                                 torch.empty(0, 2, dtype=torch.int64, device=DEV)).shape == (0, 4)


def test_route_refusals():
    be = get_backend("rocm")
    z = torch.zeros(3, 12, device=DEV)
    for kw, err in ((dict(top_k=0), ValueError), (dict(top_k=13), ValueError), (dict(top_k=2, score="max"), ValueError),
                    (dict(top_k=2, groups=5), ValueError), (dict(top_k=5, groups=4, top_groups=1), ValueError),
                    (dict(top_k=2, groups=4, top_groups=5), ValueError), (dict(top_k=2, group_best=3), ValueError),
                    (dict(top_k=2, bias=torch.zeros(11, device=DEV)), RuntimeError)):
        with pytest.raises(err):
            be.moe_route(z, **kw)
    with pytest.raises(RuntimeError):
        be.moe_route(z.half(), 2)
    with pytest.raises(RuntimeError):
        be.moe_route(z.view(-1), 2)
    with pytest.raises(NotImplementedError):
        be.moe_route(torch.zeros(2, 513, device=DEV), 2)
    with pytest.raises(NotImplementedError):
        be.moe_route(torch.zeros(2, 40, device=DEV), 17)
    topi = torch.zeros(3, 2, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError):
        be.moe_route_backward(torch.zeros(3, 3, device=DEV), z, topi)
    with pytest.raises(RuntimeError):
        be.moe_route_backward(torch.zeros(3, 2, device=DEV), z, topi.int())
    with pytest.raises(RuntimeError):
        be.moe_route_backward(torch.zeros(3, 2, device=DEV), z, topi, dprob=torch.zeros(3, 11, device=DEV))


@pytest.mark.parametrize("E", [7, 8, 60, 100, 256, 512])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_route_gradient_of_rows_without_experts(E, dtype):
    """A row whose logits are all -inf has no gradient, whatever dtopw and dprob hold, nor
    has a masked expert, whatever dprob holds there; the others have theirs."""
    be = get_backend("rocm")
    logits, gen = _logits(9, E, dtype, E)
    empty = torch.tensor([0, 4, 8])
    logits[empty] = -math.inf
    logits[5, 1:] = -math.inf  # one expert left
    rest = torch.tensor([t for t in range(9) if t not in empty.tolist()])
    dtopw, dprob = torch.randn(9, 3, generator=gen), torch.randn(9, E, generator=gen)
    dtopw[4], dprob[8] = math.nan, math.nan
    plain = dprob.clone()
    dprob[5, 2], dprob[5, 3] = math.nan, math.inf
    plain[5, 2:4] = 0.0
    for score in ("softmax", "sigmoid"):
        for renorm in (False, True):
            topi = be.moe_route(logits.to(DEV), 3, score=score, renorm=renorm)[1]
            assert (topi[empty] == -1).all()
            for dp in (None, dprob):
                got = be.moe_route_backward(dtopw.to(DEV), logits.to(DEV), topi, score=score, renorm=renorm,
                                            dprob=None if dp is None else dp.to(DEV)).cpu()
                assert (got[empty] == 0).all()
                alone = be.moe_route_backward(dtopw[rest].to(DEV), logits[rest].to(DEV), topi[rest].contiguous(),
                                              score=score, renorm=renorm,
                                              dprob=None if dp is None else plain[rest].to(DEV))
                assert torch.isfinite(got).all() and torch.equal(got[rest], alone.cpu())
