"""The 4-bit format: quantisation, products, gradient and routed experts against plain 64-bit forms."""
import math

import pytest
import torch

import _mx4 as ref
from smaulnative_amd.compute import get_backend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def _dev(*ts):
    return [t.to(DEV) for t in ts]


# ---- quantisation ----------------------------------------------------------
def _check_quant(x):
    be = get_backend("rocm")
    codes, scales = be.mx4_quantize(x.to(DEV))
    wc, ws = ref.quantize(x)
    assert torch.equal(scales.cpu(), ws)
    assert torch.equal(codes.cpu(), wc)
    K = x.shape[-1]
    want = ref.values(wc, ws, K)
    for dtype in (F32, BF):
        got = be.mx4_dequantize(codes, scales, K, dtype)
        assert got.dtype == dtype and got.shape == x.shape
        # every value is exact in both types; past their range (codes times 2^126 and up) it is infinite
        assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=7e77), torch.nan_to_num(want.to(dtype).double(), nan=7e77))


@pytest.mark.parametrize("rows,K", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 64), (7, 100), (64, 1024), (33, 1000),
                                    (130, 96), (1, 4097), (300, 8)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_quantize_shapes(rows, K, dtype):
    gen = torch.Generator().manual_seed(rows * 5000 + K)
    x = torch.randn(rows, K, generator=gen) * torch.pow(2.0, torch.randint(-20, 20, (rows, 1), generator=gen).float())
    x[rows // 2] = 0.0
    _check_quant(x.to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_quantize_borders(dtype):
    """Every border between neighbours, its neighbours in the type, and every power of
    two of a block's largest value from the subnormals to the top."""
    vals = torch.tensor([b for b, _ in ref.BORDERS] + [0.0, 0.125, 6.0, 7.0, 7.9, 5.5], dtype=dtype)
    up = torch.nextafter(vals, torch.full_like(vals, 9.0))
    down = torch.nextafter(vals, torch.full_like(vals, -9.0)).abs()
    row = torch.cat([vals, up, down])
    row = torch.cat([row, -row, torch.zeros(96 - 2 * row.numel(), dtype=dtype)]) if 2 * row.numel() <= 96 else row
    blocks = []
    for e in range(-148, 126):
        for part in row.split(31):
            blocks.append(torch.cat([part, torch.full((32 - part.numel(),), 4.0, dtype=dtype)]).double() * 2.0 ** e)
    x = torch.stack(blocks)
    x = torch.where(x.abs() > torch.finfo(dtype).max, torch.zeros_like(x), x).to(dtype)
    _check_quant(x)
    tops = torch.full((1, 32), torch.finfo(dtype).max, dtype=dtype)
    _check_quant(torch.cat([tops, -tops, torch.full((1, 32), torch.finfo(dtype).smallest_normal, dtype=dtype)]))


def test_quantize_not_finite():
    x = torch.ones(4, 96)
    x[0, 5], x[1, 40], x[2, 95] = math.inf, math.nan, -math.inf
    _check_quant(x)
    _check_quant(x[:, :90].bfloat16())
    got = get_backend("rocm").mx4_quantize(x.to(DEV))[1].cpu()
    assert (got == 255).sum() == 3 and (got[3] == 127 - 2).all()


def test_quantize_views_and_empty():
    be = get_backend("rocm")
    x = torch.randn(6, 5, 200, generator=torch.Generator().manual_seed(1))
    _check_quant(x)
    c, s = be.mx4_quantize(x.to(DEV)[:, 1:4, 3:103])
    wc, ws = ref.quantize(x[:, 1:4, 3:103])
    assert torch.equal(c.cpu(), wc) and torch.equal(s.cpu(), ws)
    flat = x.to(DEV).view(-1)[1:1 + 64 * 90].view(90, 64)  # rows that start 4 bytes off
    c, s = be.mx4_quantize(flat)
    wc, ws = ref.quantize(flat.cpu())
    assert torch.equal(c.cpu(), wc) and torch.equal(s.cpu(), ws)
    c, s = be.mx4_quantize(torch.empty(0, 40, device=DEV))
    assert c.shape == (0, 32) and s.shape == (0, 2)
    assert be.mx4_dequantize(c, s, 40).shape == (0, 40)
    # codes and scales that are views
    c, s = be.mx4_quantize(x.to(DEV))
    a, b = be.mx4_dequantize(c[:, 2:4], s[:, 2:4], 200), be.mx4_dequantize(c, s, 200)[:, 2:4]
    assert torch.equal(a, b)


# ---- the product and its input gradient ---------------------------------------
# Tolerances: K 2^-24 of the terms' magnitudes for the fp32 sums, 2^-17 of them for
# fp32 values as two bf16 terms (rounded to the format they are exact), and half a
# step of the output.
def _check_linear(rows, K, N, dtype, act, seed, x=None):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=gen).to(dtype) if x is None else x
    w, s = ref.weight(N, K, gen)
    got = get_backend("rocm").mx4_forward(*_dev(x, w, s), K, N, act=act)
    assert got.dtype == dtype and got.shape == (rows, N)
    xv, wv = ref.rounded(x) if act == "mx4" else x.double(), ref.values(w, s, K)
    want = xv @ wv.t()
    lost = K * 2.0 ** -24 + (2.0 ** -17 if dtype == F32 and act == "keep" else 0.0)
    tol = (xv.abs() @ wv.abs().t()) * lost + (2.0 ** -8 if dtype == BF else 2.0 ** -24) * want.abs() + 1e-37
    bad = (got.cpu().double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


SHAPES = [(1, 1, 1), (1, 32, 16), (1, 1024, 2560), (2, 33, 70), (3, 1000, 129), (16, 96, 64), (17, 512, 48), (31, 160, 257),
          (33, 128, 128), (64, 1024, 320), (65, 256, 200), (100, 1000, 777), (128, 2560, 128), (130, 64, 1), (257, 288, 384),
          (300, 1056, 520), (513, 512, 256), (1, 4000, 31), (48, 8, 8), (1025, 128, 640)]


@pytest.mark.parametrize("rows,K,N", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("act", ["keep", "mx4"])
def test_linear_shapes(rows, K, N, dtype, act):
    _check_linear(rows, K, N, dtype, act, rows + K + N)


@pytest.mark.parametrize("act", ["keep", "mx4"])
def test_linear_special_rows(act):
    """Zero rows stay zero, a NaN stays in its row, and a weight's NaN block in its column."""
    be = get_backend("rocm")
    gen = torch.Generator().manual_seed(2)
    for rows in (4, 200):
        x = torch.randn(rows, 192, generator=gen).bfloat16()
        x[1] = 0.0
        x[2, 100] = math.nan
        w, s = ref.weight(160, 192, gen)
        s[7, 3] = 255
        got = be.mx4_forward(*_dev(x, w, s), 192, 160, act=act).cpu().float()
        fine = torch.ones_like(got, dtype=torch.bool)
        fine[2], fine[:, 7] = False, False
        assert torch.isnan(got[2]).all() and torch.isnan(got[:, 7]).all() and torch.isfinite(got[fine]).all()
        assert (got[1][torch.arange(160) != 7] == 0).all()


@pytest.mark.parametrize("K", [32, 128, 160, 384])
@pytest.mark.parametrize("act", ["keep", "mx4"])
def test_linear_nan_scales_stay_in_their_row(K, act):
    """Widths that the products pad: the padding of a row takes nothing from the next one."""
    gen = torch.Generator().manual_seed(K)
    x = torch.randn(100, K, generator=gen).bfloat16()
    w, s = ref.weight(48, K, gen)
    s[1::2] = 255
    got = get_backend("rocm").mx4_forward(*_dev(x, w, s), K, 48, act=act).cpu()
    assert torch.isnan(got[:, 1::2]).all() and torch.isfinite(got[:, 0::2]).all()
    dx = get_backend("rocm").mx4_backward_input(*_dev(got[:, :48].nan_to_num(), w, torch.where(s == 255, 120, s)), K, 48)
    assert torch.isfinite(dx).all()


def test_linear_wide_range():
    """Scales from one end to the other: the products keep their powers of two."""
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(70, 96, generator=gen) * torch.pow(2.0, torch.randint(-60, 60, (70, 1), generator=gen).float())
    w, s = ref.quantize(torch.randn(40, 96, generator=gen) * torch.pow(2.0, torch.randint(-60, 60, (40, 1), generator=gen).float()))
    for act in ("keep", "mx4"):
        for dtype in (F32, BF):
            xd = x.to(dtype)
            got = get_backend("rocm").mx4_forward(*_dev(xd, w, s), 96, 40, act=act).cpu().double()
            xv, wv = ref.rounded(xd) if act == "mx4" else xd.double(), ref.values(w, s, 96)
            want = xv @ wv.t()
            lost = 96 * 2.0 ** -24 + (2.0 ** -17 if dtype == F32 and act == "keep" else 0.0)
            tol = (xv.abs() @ wv.abs().t()) * lost + (2.0 ** -8 if dtype == BF else 2.0 ** -24) * want.abs()
            assert ((got - want).abs() <= tol + 1e-37).all()


def test_linear_views():
    be = get_backend("rocm")
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(70, 300, generator=gen)
    w, s = ref.weight(96, 128, gen)
    xd, wd, sd = _dev(x, w, s)
    want = be.mx4_forward(xd[:, 7:135].contiguous(), wd, sd, 128, 96)
    assert torch.equal(want, be.mx4_forward(xd[:, 7:135], wd, sd, 128, 96))
    off = xd.view(-1)[3:3 + 128 * 70].view(70, 128)  # rows 12 bytes off 16
    assert torch.equal(be.mx4_forward(off, wd, sd, 128, 96), be.mx4_forward(off.clone(), wd, sd, 128, 96))
    ww = torch.zeros(96, 80, dtype=torch.uint8, device=DEV)
    ww[:, 5:69] = wd
    assert torch.equal(want, be.mx4_forward(xd[:, 7:135], ww[:, 5:69], sd, 128, 96))
    assert be.mx4_forward(xd[:0, :128], wd, sd, 128, 96).shape == (0, 96)


@pytest.mark.parametrize("rows,K,N", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF])
def test_input_gradient(rows, K, N, dtype):
    gen = torch.Generator().manual_seed(7 * rows + K + N)
    g = torch.randn(rows, N, generator=gen).to(dtype)
    w, s = ref.weight(N, K, gen)
    got = get_backend("rocm").mx4_backward_input(*_dev(g, w, s), K, N)
    assert got.dtype == dtype and got.shape == (rows, K)
    wv = ref.values(w, s, K)
    want = g.double() @ wv
    lost = N * 2.0 ** -24 + (2.0 ** -17 if dtype == F32 else 0.0)
    tol = (g.double().abs() @ wv.abs()) * lost + (2.0 ** -8 if dtype == BF else 2.0 ** -24) * want.abs() + 1e-37
    assert ((got.cpu().double() - want).abs() <= tol).all()


def test_input_gradient_against_differences():
    """<dx, v> is the change of <g, forward(x)> along v: the forward is linear, so the
    difference of two calls is the derivative up to their fp32 sums."""
    be = get_backend("rocm")
    gen = torch.Generator().manual_seed(8)
    x, v, g = (torch.randn(20, n, generator=gen) for n in (90, 90, 70))
    w, s = ref.weight(70, 90, gen)
    xd, vd, gd, wd, sd = _dev(x, v, g, w, s)
    dx = be.mx4_backward_input(gd, wd, sd, 90, 70).cpu().double()
    diff = (be.mx4_forward(xd + vd, wd, sd, 90, 70) - be.mx4_forward(xd - vd, wd, sd, 90, 70)).cpu().double() / 2
    left, right = (dx * v.double()).sum(), (diff * g.double()).sum()
    wv = ref.values(w, s, 90).abs()
    mag = ((x.abs().double() + v.abs().double()) @ wv.t() * g.abs().double()).sum() * 2
    assert abs(float(left - right)) <= float(mag) * (2.0 ** -16 + 200 * 2.0 ** -24)


# ---- the routed experts -------------------------------------------------------
def _experts(E, d, h, gen):
    out = []
    for n, m in ((h, d), (h, d), (d, h)):
        c, s = zip(*(ref.weight(n, m, gen, std=0.05) for _ in range(E)))
        out += [torch.stack(c), torch.stack(s)]
    return out


def _routing(T, E, k, gen):
    topw, topi = torch.rand(T, E, generator=gen).topk(k, 1)
    return topi, topw / topw.sum(1, keepdim=True)


def _check_moe(x, topi, topw, experts, act):
    out, counts = get_backend("rocm").mx4_moe_forward(*_dev(x, topi, topw), tuple(_dev(*experts)), act=act)
    d, h = x.shape[-1], experts[0].shape[1]
    flat = x.reshape(-1, d)
    k = topi.shape[-1]
    want, bound, wc = ref.moe(flat, topi.reshape(-1, k), topw.reshape(-1, k), experts, act)
    assert out.dtype == x.dtype and out.shape == x.shape
    assert torch.equal(counts.cpu(), wc)
    off = (out.cpu().double().reshape(-1, d) - want).abs()
    assert (off <= bound).all(), float((off / bound).max())
    return out


@pytest.mark.parametrize("T,d,h,E,k", [(1, 64, 128, 4, 2), (5, 128, 64, 8, 8), (64, 256, 320, 8, 2), (64, 1024, 2560, 8, 2),
                                       (65, 128, 192, 3, 1), (130, 200, 104, 5, 2), (300, 256, 640, 8, 2), (77, 40, 24, 64, 3),
                                       (1000, 128, 256, 4, 2), (33, 136, 1000, 16, 4), (2, 8, 8, 1, 1), (700, 512, 96, 2, 2)])
@pytest.mark.parametrize("dtype,act", [(BF, "keep"), (F32, "keep"), (BF, "mx4")])
def test_moe_shapes(T, d, h, E, k, dtype, act):
    gen = torch.Generator().manual_seed(T + d + h + E)
    x = torch.randn(T, d, generator=gen).to(dtype)
    topi, topw = _routing(T, E, k, gen)
    _check_moe(x, topi, topw, _experts(E, d, h, gen), act)


@pytest.mark.parametrize("T", [9, 150])
@pytest.mark.parametrize("dtype,act", [(BF, "keep"), (F32, "keep"), (BF, "mx4")])
def test_moe_uneven_and_dropped(T, dtype, act):
    gen = torch.Generator().manual_seed(T)
    d, h, E = 96, 160, 6
    ex = _experts(E, d, h, gen)
    x = torch.randn(T, d, generator=gen).to(dtype)
    topi, topw = _routing(T, E, 2, gen)
    one = torch.full_like(topi[:, :1], 3)
    _check_moe(x, one, torch.ones(T, 1), ex, act)              # everyone at one expert
    topi[::2, 1], topw[::2, 1] = -1, 0.0                        # empty slots
    topw[1, 0] = 0.0                                            # a weight of nothing
    topw[3] = math.nan                                          # a token whose routing failed
    topi[5] = -1                                                # a padding row
    w0 = torch.nan_to_num(topw)
    w0[5] = 0.0
    out = _check_moe(x, topi, w0, ex, act)
    be = get_backend("rocm")
    again, _ = be.mx4_moe_forward(*_dev(x, topi, torch.where(topi < 0, torch.full_like(topw, 0.7), topw)),
                                  tuple(_dev(*ex)), act=act)
    assert torch.equal(out, again)                              # a dropped slot's weight is not read
    assert (out[5] == 0).all() and (out[3] == 0).all()
    nobody, counts = be.mx4_moe_forward(*_dev(x, torch.full_like(topi, -1), torch.zeros_like(topw)), tuple(_dev(*ex)),
                                        act=act)
    assert (nobody == 0).all() and (counts == 0).all()
    empty, counts = be.mx4_moe_forward(*_dev(x[:0], topi[:0], topw[:0]), tuple(_dev(*ex)), act=act)
    assert empty.shape == (0, d) and (counts == 0).all()


@pytest.mark.parametrize("act", ["keep", "mx4"])
def test_routed_layer_together(act):
    """Logits to outputs, as a layer runs it: leading dimensions, another stream, and a
    captured graph replayed over changing inputs beside eager calls."""
    be = get_backend("rocm")
    gen = torch.Generator().manual_seed(11)
    B, S, d, h, E, k = 3, 7, 256, 192, 16, 4
    ex = _experts(E, d, h, gen)
    exd = tuple(_dev(*ex))
    x = torch.randn(B, S, d, generator=gen).bfloat16()
    gate = torch.randn(E, d, generator=gen) * 0.05
    bias = torch.randn(E, generator=gen) * 0.02
    xd, gd, bd = _dev(x, gate, bias)

    def layer(x):
        logits = x.reshape(-1, d).float() @ gd.t()
        _, ti, tw = be.moe_route(logits, k, score="sigmoid", bias=bd, groups=4, top_groups=2, scale=2.5, need_prob=False)
        out, counts = be.mx4_moe_forward(x, ti.view(B, S, k), tw.view(B, S, k), exd, act=act)
        return out, counts, ti, tw

    out, counts, ti, tw = layer(xd)
    logits = (xd.reshape(-1, d).float() @ gd.t()).cpu()
    assert torch.equal(ti.cpu(), ref.route(logits, k, "sigmoid", bias, 4, 2, 2, True, 2.5)[1])
    _check_moe(x, ti.cpu().view(B, S, k), tw.cpu().view(B, S, k), ex, act)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = layer(xd)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip((out, counts, ti, tw), other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(xd)
    for i in range(3):
        xd.copy_(torch.randn(B, S, d, generator=gen))
        graph.replay()
        want = layer(xd)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_linear_streams_and_replay():
    be = get_backend("rocm")
    gen = torch.Generator().manual_seed(12)
    w, s = ref.weight(256, 256, gen)
    wd, sd = _dev(w, s)
    for rows in (1, 200):
        x = torch.randn(rows, 256, generator=gen).bfloat16().to(DEV)
        for act in ("keep", "mx4"):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = be.mx4_forward(x, wd, sd, 256, 256, act=act)
                dx = be.mx4_backward_input(y, wd, sd, 256, 256)
            for i in range(3):
                x.copy_(torch.randn(rows, 256, generator=gen))
                graph.replay()
                y2 = be.mx4_forward(x, wd, sd, 256, 256, act=act)
                dx2 = be.mx4_backward_input(y2, wd, sd, 256, 256)
                torch.cuda.synchronize()
                assert torch.equal(y, y2) and torch.equal(dx, dx2)


def test_refusals():
    be = get_backend("rocm")
    x = torch.zeros(4, 64, device=DEV)
    w, s = be.mx4_quantize(torch.zeros(96, 64, device=DEV))
    with pytest.raises(RuntimeError):
        be.mx4_quantize(x.half())
    with pytest.raises(RuntimeError):
        be.mx4_quantize(torch.zeros(4, 0, device=DEV))
    with pytest.raises(RuntimeError):
        be.mx4_dequantize(w, s, 65)
    with pytest.raises(RuntimeError):
        be.mx4_dequantize(w, s, 64, torch.float16)
    with pytest.raises(ValueError):
        be.mx4_forward(x, w, s, 64, 96, act="fp8")
    with pytest.raises(RuntimeError):
        be.mx4_forward(x, w, s, 32, 96)
    with pytest.raises(RuntimeError):
        be.mx4_forward(x, w, s, 64, 95)
    with pytest.raises(RuntimeError):
        be.mx4_forward(x.double(), w, s, 64, 96)
    with pytest.raises(RuntimeError):
        be.mx4_forward(x, w.char(), s, 64, 96)
    with pytest.raises(RuntimeError):
        be.mx4_backward_input(x, w, s, 64, 96)
    gen = torch.Generator().manual_seed(1)
    ex = tuple(_dev(*_experts(4, 64, 32, gen)))
    ti, tw = torch.zeros(4, 2, dtype=torch.int64, device=DEV), torch.ones(4, 2, device=DEV)
    with pytest.raises(NotImplementedError):
        be.mx4_moe_forward(x, ti, tw, ex, act="mx4")  # fp32 rows
    with pytest.raises(RuntimeError):
        be.mx4_moe_forward(x, ti[:3], tw[:3], ex)
    with pytest.raises(RuntimeError):
        be.mx4_moe_forward(x, ti.int(), tw, ex)
    with pytest.raises(RuntimeError):
        be.mx4_moe_forward(x, ti, tw, ex[:4] + ex[:2])
    with pytest.raises(ValueError):
        be.mx4_moe_forward(x, torch.zeros(4, 5, dtype=torch.int64, device=DEV), torch.ones(4, 5, device=DEV), ex)
    bad = tuple(_dev(*_experts(2, 60, 32, gen)))
    with pytest.raises(NotImplementedError):
        be.mx4_moe_forward(torch.zeros(3, 60, device=DEV), ti[:3], tw[:3], bad)  # d off 8
