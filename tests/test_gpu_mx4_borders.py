"""The 4-bit products with infinities and NaN among the activations, values of all of a type's bits, and many rows."""
import math

import pytest
import torch

import _mx4 as ref
from smaulnative_amd.compute import get_backend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def _same_kinds(got, want):
    """Infinities with their signs and NaN where the plain product has them."""
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.where(torch.isinf(got), got, torch.zeros_like(got)),
                       torch.where(torch.isinf(want), want, torch.zeros_like(want)))


def _spoil(x):
    """One value a row is no number; the last payload is in a NaN's lowest bit alone."""
    x[0, 3], x[1, 40], x[2, 70] = math.inf, -math.inf, math.nan
    x[3, 0], x[3, 1] = math.inf, -math.inf
    if x.dtype == F32:
        x[4].view(torch.int32)[5] = 0x7F800001
    return x


@pytest.mark.parametrize("rows", [9, 70, 300])  # the kernel of few rows, and the larger ones
@pytest.mark.parametrize("dtype", [F32, BF])
def test_products_of_infinities(rows, dtype):
    gen = torch.Generator().manual_seed(rows)
    K, N = 96, 80
    x = _spoil(torch.randn(rows, K, generator=gen).to(dtype))
    w, s = ref.weight(N, K, gen)
    got = get_backend("rocm").mx4_forward(x.to(DEV), w.to(DEV), s.to(DEV), K, N)
    want = x.double() @ ref.values(w, s, K).t()
    _same_kinds(got, want)
    clean = torch.isfinite(x).all(-1)
    assert clean.sum() == rows - (5 if dtype == F32 else 4) and torch.isfinite(got.cpu()[clean]).all()

    g = _spoil(torch.randn(rows, N, generator=gen).to(dtype))
    dx = get_backend("rocm").mx4_backward_input(g.to(DEV), w.to(DEV), s.to(DEV), K, N)
    _same_kinds(dx, g.double() @ ref.values(w, s, K))


@pytest.mark.parametrize("T", [9, 150])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_experts_of_nan_rows(T, dtype):
    """A token that is no number takes no other with it."""
    gen = torch.Generator().manual_seed(T)
    E, d, h, k = 4, 64, 96, 2
    x = torch.randn(T, d, generator=gen).to(dtype)
    x[2, 5], x[7, 0] = math.nan, math.inf
    experts = []
    for o, i in ((h, d), (h, d), (d, h)):
        ws = [ref.weight(o, i, gen) for _ in range(E)]
        experts += [torch.stack([w for w, _ in ws]), torch.stack([s for _, s in ws])]
    topi = torch.stack([torch.randperm(E, generator=gen)[:k] for _ in range(T)])
    topw = torch.rand(T, k, generator=gen) + 0.1
    out, _ = get_backend("rocm").mx4_moe_forward(x.to(DEV), topi.to(DEV), topw.to(DEV), [t.to(DEV) for t in experts])
    fine = torch.ones(T, dtype=torch.bool)
    fine[2], fine[7] = False, False
    out = out.cpu()
    assert torch.isfinite(out[fine]).all() and torch.isnan(out[2]).all() and not torch.isfinite(out[7]).any()


@pytest.mark.parametrize("rows", [9, 150])
def test_fp32_activations_keep_all_their_bits(rows):
    """A weight of one code picks single activations: 24 bits come back as they went in."""
    gen = torch.Generator().manual_seed(rows)
    K = 64
    x = torch.randn(rows, K, generator=gen) * torch.pow(2.0, torch.randint(-30, 30, (rows, K), generator=gen).float())
    w, s = ref.quantize(torch.eye(K))
    got = get_backend("rocm").mx4_forward(x.to(DEV), w.to(DEV), s.to(DEV), K, K)
    assert torch.equal(got.cpu(), x)


@pytest.mark.parametrize("rows,K,N", [(4200, 2049, 160), (8230, 4090, 96)])  # both larger tiles of the gradient
def test_large_gradient(rows, K, N):
    gen = torch.Generator().manual_seed(rows)
    w, s = ref.weight(N, K, gen)
    g = torch.randn(rows, N, generator=gen).to(BF)
    got = get_backend("rocm").mx4_backward_input(g.to(DEV), w.to(DEV), s.to(DEV), K, N).cpu()
    some = torch.cat([torch.arange(40), torch.arange(rows - 300, rows)])
    wv = ref.values(w, s, K)
    want = g[some].double() @ wv
    # N products summed in fp32, and half a step of bf16
    tol = N * 2.0 ** -24 * (g[some].double().abs() @ wv.abs()) + 2.0 ** -8 * want.abs()
    assert ((got[some].double() - want).abs() <= tol + 1e-37).all()


@pytest.mark.parametrize("rows,N", [(100, 500), (1100, 900), (1500, 4090), (4100, 4500)])
@pytest.mark.parametrize("act", ["keep", "mx4"])
def test_linear_of_every_tile(rows, N, act):
    """Rows and columns of the products' different tiles, ending inside one."""
    gen = torch.Generator().manual_seed(rows + N)
    K = 200
    w, s = ref.weight(N, K, gen)
    x = torch.randn(rows, K, generator=gen).to(BF)
    got = get_backend("rocm").mx4_forward(x.to(DEV), w.to(DEV), s.to(DEV), K, N, act).cpu()
    some = torch.cat([torch.arange(40), torch.arange(rows - 60, rows)])
    xv = ref.rounded(x[some]) if act == "mx4" else x[some].double()
    wv = ref.values(w, s, K)
    want = xv @ wv.t()
    # K products summed in fp32, and half a step of bf16
    tol = K * 2.0 ** -24 * (xv.abs() @ wv.abs().t()) + 2.0 ** -8 * want.abs()
    assert ((got[some].double() - want).abs() <= tol + 1e-37).all()


@pytest.mark.parametrize("K", [4, 36, 100])
@pytest.mark.parametrize("rows", [1, 9, 64, 65])
def test_infinities_at_the_end_of_a_width_off_eight(rows, K):
    """fp32 rows that end inside a group of 8 values: an infinity among the last four."""
    gen = torch.Generator().manual_seed(rows + K)
    N = 70
    w, s = ref.weight(N, K, gen)
    for at in range(K - 4, K):
        x = torch.randn(rows, K, generator=gen)
        x[rows // 2, at] = -math.inf if at % 2 else math.inf
        got = get_backend("rocm").mx4_forward(x.to(DEV), w.to(DEV), s.to(DEV), K, N)
        want = x.double() @ ref.values(w, s, K).t()
        assert torch.isinf(want).any()
        _same_kinds(got, want)


@pytest.mark.parametrize("T", [9, 150])
def test_infinite_hidden_values_at_the_end_of_a_width_off_eight(T):
    """The same of the experts' hidden rows: the last of 36 overflows fp32."""
    gen = torch.Generator().manual_seed(T)
    d, h = 64, 36
    x = torch.rand(T, d, generator=gen) + 0.5
    gate, up, down = torch.rand(h, d, generator=gen), torch.rand(h, d, generator=gen), torch.randn(d, h, generator=gen)
    gate[-1] *= 2.0 ** 70
    up[-1] *= 2.0 ** 70
    experts = [t[None] for m in (gate, up, down) for t in ref.quantize(m)]
    g, u = (x.double() @ ref.values(experts[i][0], experts[i + 1][0], d).t() for i in (0, 2))
    hid = ref.swiglu(g, u).float()
    assert torch.isinf(hid[:, -1]).all() and torch.isfinite(hid[:, :-1]).all()
    want = hid.double() @ ref.values(experts[4][0], experts[5][0], h).t()
    out, _ = get_backend("rocm").mx4_moe_forward(x.to(DEV), torch.zeros(T, 1, dtype=torch.int64, device=DEV),
                                                 torch.ones(T, 1, device=DEV), [t.to(DEV) for t in experts])
    assert torch.isinf(want).any()
    _same_kinds(out, want)


@pytest.mark.parametrize("rows", [1, 9, 32, 33, 64, 150, 700])  # few rows, and tiles
def test_fp32_gradients_keep_all_their_bits(rows):
    """A weight of one code a row picks single gradients: 24 bits come back as they went in."""
    gen = torch.Generator().manual_seed(rows)
    for K in (64, 100):
        g = torch.randn(rows, K, generator=gen) * torch.pow(2.0, torch.randint(-30, 30, (rows, K), generator=gen).float())
        w, s = ref.quantize(torch.eye(K))
        got = get_backend("rocm").mx4_backward_input(g.to(DEV), w.to(DEV), s.to(DEV), K, K)
        assert torch.equal(got.cpu(), g)


@pytest.mark.parametrize("T", [9, 64, 65, 300])
@pytest.mark.parametrize("d", [64, 104])
def test_fp32_experts_keep_all_their_bits(T, d):
    """Gate, up and down weights of one code a row: an output is silu(x) x of its own x.

    The product's arithmetic alone is left: the argument's rounding (|x| 2^-24 of the
    value), the exponential, sum, reciprocal and two products, a step of 2^-23 each at
    most: |x| + 10 times 2^-24, below 2^-20 for |x| < 6.  A bf16 term dropped from x or from
    the hidden rows is 2^-17 and more on most values."""
    gen = torch.Generator().manual_seed(T + d)
    x = torch.randn(T, d, generator=gen).clamp(-5.5, 5.5)
    w, s = ref.quantize(torch.eye(d))
    out, _ = get_backend("rocm").mx4_moe_forward(x.to(DEV), torch.zeros(T, 1, dtype=torch.int64, device=DEV),
                                                 torch.ones(T, 1, device=DEV), [t[None].to(DEV) for t in (w, s) * 3])
    want = ref.swiglu(x.double(), x.double())
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -20 * want.abs()).all()
