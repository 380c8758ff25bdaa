"""The residual's addition with the norm, its output as rows and as codes, and its
gradients, against plain 64-bit forms."""
import math

import pytest
import torch

import _fp8_block as ref
from smaulnative_amd.compute import get_backend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
EPS = 1e-6


def be():
    return get_backend("rocm")


def inputs(T, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + T * 31 + d)
    x, r = (torch.randn(T, d, generator=g).to(dtype) for _ in range(2))
    return x, r, 1 + 0.3 * torch.randn(d, generator=g), g


SHAPES = [(1, 1), (1, 64), (3, 127), (5, 128), (64, 129), (33, 513), (7, 1000), (130, 2048), (5, 2049), (3, 4099),
          (2, 8192), (2, 9001), (600, 200)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,d", SHAPES)
def test_forward(T, d, dtype):
    x, r, w, _ = inputs(T, d, dtype)
    for residual in (r, None):
        for weight in (w, None):
            s = x if residual is None else (x.float() + residual.float()).to(dtype)
            y, e = ref.norm(s.double(), torch.ones(d).double() if weight is None else weight.double(), EPS)
            dev = [t if t is None else t.to(DEV) for t in (x, residual, weight)]
            got_s, got = be().add_rms_norm(*dev, EPS)
            assert torch.equal(got_s.cpu(), s) and got.dtype == dtype
            ref.check(got, y, e + ref.HALF[dtype] * (y.abs() + e), (T, d, dtype))
            got_s, c, cs = be().add_rms_norm(*dev, EPS, quantize=True)
            assert torch.equal(got_s.cpu(), s)
            n = ref.blocks(d)
            assert c.shape == (T, 128 * n) and cs.shape == (T, (n + 3) // 4 * 4)
            assert not c[:, d:].any() and not cs[:, n:].any()
            ref.check(ref.values(c.cpu(), cs.cpu(), d), ref.rounded(y), ref.moved(y, e), (T, d, dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,d", SHAPES + [(1500, 300), (5000, 64)])
def test_backward(T, d, dtype):
    x, r, w, g = inputs(T, d, dtype, 1)
    dy, ds = (torch.randn(T, d, generator=g).to(dtype) for _ in range(2))
    for extra in (ds, None):
        for weight in (w, None):
            (dx, dxe), (dw, dwe) = ref.norm_grad(dy.double(), x.double(),
                                                 torch.ones(d).double() if weight is None else weight.double(), EPS,
                                                 None if extra is None else extra.double(), dtype)
            dev = [t if t is None else t.to(DEV) for t in (dy, x, weight, extra)]
            got, gw = be().add_rms_norm_backward(*dev[:3], EPS, ds=dev[3])
            assert got.dtype == dtype and gw.dtype == F32
            ref.check(got, dx, dxe, (T, d, dtype))
            ref.check(gw, dw, dwe, (T, d, dtype))
            only, none = be().add_rms_norm_backward(*dev[:3], EPS, ds=dev[3], need_dw=False)
            assert none is None and torch.equal(only, got)


@pytest.mark.parametrize("T,d", [(700, 2049), (1100, 4096), (530, 4097)])
def test_backward_of_more_rows_than_workgroups(T, d):
    """Wide rows in several turns of a workgroup, their shares of the weight's gradient joined."""
    x, _, w, g = inputs(T, d, BF, 5)
    dy = torch.randn(T, d, generator=g).to(BF)
    (dx, dxe), (dw, dwe) = ref.norm_grad(dy.double(), x.double(), w.double(), EPS, None, BF)
    got, gw = be().add_rms_norm_backward(dy.to(DEV), x.to(DEV), w.to(DEV), EPS)
    ref.check(got, dx, dxe, (T, d))
    ref.check(gw, dw, dwe, (T, d))


def test_gradient_against_differences():
    """Central differences of the norm in 64 bits: truncation h^2 times the third derivative
    (of a function of values near 1, order 1) and rounding 2^-53 / h, h = 1e-5; fp32's own
    error is the larger, 1e-5 of the gradient's size."""
    T, d, h = 4, 37, 1e-5
    x, _, w, g = inputs(T, d, F32, 2)
    dy = torch.randn(T, d, generator=g)
    dx, dw = be().add_rms_norm_backward(dy.to(DEV), x.to(DEV), w.to(DEV), EPS)

    def loss(v, u):
        return float((ref.norm(v, u, EPS)[0] * dy.double()).sum())

    for t, got, at in ((0, dx, x), (1, dw, w)):
        flat = at.double().clone().view(-1)
        for i in range(0, flat.numel(), 5):
            step = []
            for sign in (1, -1):
                v = flat.clone()
                v[i] += sign * h
                v = v.view(at.shape)
                step.append(loss(v, w.double()) if t == 0 else loss(x.double(), v))
            assert abs((step[0] - step[1]) / (2 * h) - float(got.view(-1)[i])) <= 1e-5 * (1 + float(got.abs().max()))


def test_zero_infinite_and_nan_rows():
    x, r, w, _ = inputs(40, 300, F32, 3)
    clean = be().add_rms_norm(x.to(DEV), None, w.to(DEV), EPS, quantize=True)
    x[3], x[5, 17], x[9, 250] = 0.0, math.nan, math.inf
    s, c, cs = be().add_rms_norm(x.to(DEV), None, w.to(DEV), EPS, quantize=True)
    v = be().fp8_block_dequantize(c, cs, 300, F32).cpu()
    assert (v[3] == 0).all() and torch.isnan(v[5]).all()
    assert torch.isnan(v[9, 128:256]).all()  # inf / inf; the row's other values are 0
    assert (v[9, :128] == 0).all() and (v[9, 256:] == 0).all()
    others = [i for i in range(40) if i not in (3, 5, 9)]
    assert torch.equal(c.cpu()[others], clean[1].cpu()[others]) and torch.equal(cs.cpu()[others], clean[2].cpu()[others])


def test_layouts_and_empty_calls():
    x, r, w, g = inputs(24, 200, BF, 4)
    dev = [t.to(DEV) for t in (x, r, w)]
    s, y = be().add_rms_norm(*dev, EPS)
    wide = torch.zeros(24, 211, dtype=BF, device=DEV)
    wide[:, 5:205] = dev[0]
    s2, y2 = be().add_rms_norm(wide[:, 5:205], dev[1].t().contiguous().t(), dev[2].double(), EPS)
    assert torch.equal(s, s2) and torch.equal(y, y2)
    s3, y3 = be().add_rms_norm(dev[0].view(2, 3, 4, 200), dev[1].view(2, 3, 4, 200), dev[2], EPS)
    assert torch.equal(s3.view(24, 200), s) and torch.equal(y3.view(24, 200), y)
    s0, c0, cs0 = be().add_rms_norm(dev[0][:0], dev[1][:0], dev[2], EPS, quantize=True)
    assert s0.shape == (0, 200) and c0.shape == (0, 256) and cs0.shape == (0, 4)
    dx, dw = be().add_rms_norm_backward(dev[0][:0], dev[1][:0], dev[2], EPS)
    assert dx.shape == (0, 200) and dw.shape == (200,) and not dw.any()
    same, z = be().add_rms_norm(dev[0])
    assert same is dev[0] and torch.equal(z, be().add_rms_norm(dev[0], None, torch.ones(200, device=DEV), 1e-6)[1])


def test_codes_where_fp32_lands_between_two():
    """Values whose nearest fp32 number is the middle of two codes: rounded twice, to nearest, half of
    them would go to the code on the other side.  y + ye, the value to 2^-47, may lie more than a step
    of fp32 from y (1.5 at most, seldom), and only then the other code is left: less than a quarter."""
    T, d = 4096, 2048
    w = (1 + 0.3 * torch.randn(d, generator=torch.Generator().manual_seed(1))).to(DEV)
    found, other = 0, 0
    for seed in range(8):
        x = torch.randn(T, d, generator=torch.Generator(DEV).manual_seed(seed), device=DEV)
        y = ref.norm(x.double(), w.double(), EPS)[0]
        middle = (y.float().view(torch.int32) & 0xfffff) == 0x80000
        middle &= y.abs() > 1e-2  # no subnormal codes
        rows = middle.any(1).nonzero()[:, 0]
        codes = be().add_rms_norm(x, None, w, EPS, quantize=True)[1][rows].cpu()
        want = ref.quantize(y[rows].cpu())[0]
        at = middle[rows].cpu()
        found += int(at.sum())
        other += int((codes[at] != want[at]).sum())
        assert torch.equal(codes[~at], want[~at])
    assert found >= 20 and other < found / 4, (other, found)


# each width's form; few rows and more than the chip has CUs
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,d", [(20, 64), (300, 300), (20, 900), (300, 1500), (20, 3000), (20, 5000), (20, 9001)])
def test_very_large_and_small_rows(T, d, dtype):
    """Finite rows whose squares, or products with a gradient, fp32 does not hold; and ordinary rows
    with one such value.  The bounds of ordinary rows, and two steps of the type's least value where
    results are that small (a product and its scaling back)."""
    g = torch.Generator().manual_seed(d)
    scales = (2e37, 1e36, 1e34, 1e30, 1e25, 1e20, 3e19, 1e18, 1.0, 1e-18, 1e-20, 1e-25)
    rows = torch.tensor(scales, dtype=torch.float64).repeat(-(-T // 12))[:T, None]
    x, r, dy, ds = ((torch.randn(T, d, generator=g).double() * rows).to(dtype) if i < 2 else
                    torch.randn(T, d, generator=g).to(dtype) for i in range(4))
    x[8, d // 2], x[9, d - 1], x[10, 0] = 1e25, -3e38, 1e20
    dy = (dy.double() * torch.where(rows > 1e15, 1e15, 1.0)).to(dtype)
    w = 1 + 0.3 * torch.randn(d, generator=g)
    wd = w.double()
    s = (x.float() + r.float()).to(dtype)
    least = {BF: 2.0 ** -133, F32: 2.0 ** -149}[dtype]
    assert torch.isfinite(s).all()
    dev = [t.to(DEV) for t in (x, r, w, dy, ds)]
    y, e = ref.norm(s.double(), wd, EPS)
    got_s, got = be().add_rms_norm(*dev[:3], EPS)
    assert torch.equal(got_s.cpu(), s)
    ref.check(got, y, e + ref.HALF[dtype] * (y.abs() + e) + 2 * least, (T, d, dtype))
    _, c, cs = be().add_rms_norm(*dev[:3], EPS, quantize=True)
    ref.check(ref.values(c.cpu(), cs.cpu(), d), ref.rounded(y), ref.moved(y, e + 2.0 ** -148), (T, d, dtype))
    for extra in (ds, None):
        (dx, dxe), (dw, dwe) = ref.norm_grad(dy.double(), s.double(), wd, EPS, None if extra is None else extra.double(), dtype)
        got, gw = be().add_rms_norm_backward(dev[3], got_s, dev[2], EPS, ds=None if extra is None else dev[4])
        ref.check(got, dx, dxe + 2 * least, (T, d, dtype))
        ref.check(gw, dw, dwe, (T, d, dtype))
