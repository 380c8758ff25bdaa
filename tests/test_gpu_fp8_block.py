"""Rows in blocks of 128 8-bit codes on the device: quantisation, products and input
gradients against plain 64-bit forms."""
import math

import pytest
import torch

import _fp8_block as ref
from smaulnative_amd.compute import get_backend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def be():
    return get_backend("rocm")


def gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("K", [1, 7, 127, 128, 129, 500, 512, 513, 1000, 1536])
def test_quantize_is_the_definition(K, dtype):
    x = (torch.randn(37, K, generator=gen(K)) * torch.exp(4 * torch.randn(37, 1, generator=gen(K + 1)))).to(dtype)
    codes, scales = be().fp8_block_quantize(x.to(DEV))
    want = ref.quantize(x)
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])
    for out in (F32, BF):
        y = be().fp8_block_dequantize(codes, scales, K, out)
        assert y.dtype == out and torch.equal(y.cpu().double(), ref.values(*want, K))


def test_quantize_at_the_borders():
    """Ties, the largest code and the next scale, subnormals, zeros of both signs, the ends of
    fp32, infinities and NaN."""
    grid = ref.GRID
    mids = (grid[1:] + grid[:-1]) / 2
    rows = []
    for e in (0, -20, 100, -118, -119, -126):
        v = torch.cat([mids, mids * (1 + 2.0 ** -12), mids * (1 - 2.0 ** -12)]).float() * 2.0 ** e
        v = torch.cat([v, -v])
        v = torch.nn.functional.pad(v, (0, -v.numel() % 127)).view(-1, 127)
        rows.append(torch.cat([v, torch.full((v.shape[0], 1), 448.0 * 2.0 ** e)], 1))
    for top in (448.0, 449.0, 447.0, 256.0, 255.0, 480.0, 511.9, 512.0):
        rows.append(torch.cat([torch.linspace(-top, top, 127), torch.tensor([top])])[None])
    x = torch.cat(rows)
    tiny = torch.zeros(9, 128)
    tiny[0, 5], tiny[1, 0], tiny[1, 1] = 2.0 ** -149, 2.0 ** -126, -(2.0 ** -130)
    tiny[2, 3], tiny[2, 4] = 2.0 ** -118, 2.0 ** -140
    tiny[3] = -0.0
    tiny[4, 7], tiny[4, 8] = torch.finfo(F32).max, 2.0 ** 118
    tiny[5, 2], tiny[5, 9] = math.inf, 1.0
    tiny[6, 2], tiny[6, 9] = math.nan, 1.0
    tiny[7, 127] = -math.inf
    x = torch.cat([x, tiny])
    for t in (x, x.to(BF)):
        codes, scales = be().fp8_block_quantize(t.to(DEV))
        want = ref.quantize(t)
        assert torch.equal(scales.cpu(), want[1])
        assert torch.equal(codes.cpu(), want[0])
        y = be().fp8_block_dequantize(codes, scales, 128, F32).cpu().double()
        v = ref.values(*want, 128).float().double()  # fp32's largest value rounds up to 2^128, which is not one
        assert torch.equal(torch.isnan(y), torch.isnan(v)) and torch.equal(y[~torch.isnan(v)], v[~torch.isnan(v)])


def test_quantize_other_layouts():
    x = torch.randn(6, 5, 200, generator=gen(0)).to(DEV)
    want = ref.quantize(x.cpu())
    for t in (x, x.transpose(0, 1).contiguous().transpose(0, 1), torch.randn(6, 5, 203, device=DEV)[..., 1:201].copy_(x)):
        codes, scales = be().fp8_block_quantize(t)
        assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])
    codes, scales = be().fp8_block_quantize(x[:0])
    assert codes.shape == (0, 5, 256) and scales.shape == (0, 5, 4)
    assert be().fp8_block_dequantize(codes, scales, 200).shape == (0, 5, 200)


ROWS = [1, 2, 31, 33, 64, 65, 200, 515]


@pytest.mark.parametrize("K,N", [(1, 1), (64, 31), (128, 128), (129, 130), (640, 513), (1000, 777), (2048, 260)])
@pytest.mark.parametrize("rows", ROWS)
def test_forward(rows, K, N):
    g = gen(rows * K + N)
    w, s = ref.weight(N, K, g)
    wv = ref.values(w, s, K)
    x = torch.randn(rows, K, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))
    wd, sd = w.to(DEV), s.to(DEV)
    for dtype in (BF, F32):
        t = x.to(dtype)
        y = be().fp8_block_forward(t.to(DEV), wd, sd, K, N)
        assert y.dtype == dtype
        ref.check(y, *ref.product(ref.rounded(t), wv, dtype, codes=True), (rows, K, N, dtype))
        c, cs = ref.quantize(t)
        again = be().fp8_block_forward(c.to(DEV), wd, sd, K, N, xs=cs.to(DEV), dtype=dtype)
        assert torch.equal(y, again)
    assert be().fp8_block_forward(c.to(DEV), wd, sd, K, N, xs=cs.to(DEV)).dtype == BF


# a size for each tile of products with fp32 results, ragged in rows, columns and K
@pytest.mark.parametrize("rows,K,N", [(600, 130, 1000), (3001, 300, 2602), (1473, 233, 4821), (7108, 290, 1843)])
def test_forward_of_many_rows_in_fp32(rows, K, N):
    g = gen(rows)
    w, s = ref.weight(N, K, g)
    x = torch.randn(rows, K, generator=g)
    y = be().fp8_block_forward(x.to(DEV), w.to(DEV), s.to(DEV), K, N).cpu()
    at = torch.cat([torch.tensor([0, 63, 64, 255, 256, rows - 1]), torch.randperm(rows, generator=g)[:300]])
    ref.check(y[at], *ref.product(ref.rounded(x[at]), ref.values(w, s, K), F32), (rows, K, N))
    few = be().fp8_block_forward(x[:50].to(DEV), w.to(DEV), s.to(DEV), K, N).cpu()
    bound = 2 * ref.product(ref.rounded(x[:50]), ref.values(w, s, K), F32)[1]
    assert bool(((y[:50].double() - few.double()).abs() <= bound).all())


@pytest.mark.parametrize("rows,K", [(1, 300), (8, 300), (16, 1000), (17, 300), (32, 2000)])
def test_products_of_few_rows_are_exact(rows, K):
    """Two large products that cancel, each among seven of 2^-15 of it: the sum of the small ones is
    left, whatever the result's type (their sum is short enough for fp32 and bf16)."""
    x = torch.zeros(rows, K)
    x[:, :16] = 2.0 ** -7
    x[:, 0], x[:, 8] = 256.0, -256.0
    x *= (2.0 ** torch.arange(rows).remainder(5))[:, None]
    want = x[:, :16].double().sum(-1, keepdim=True).expand(-1, 40)
    w = torch.zeros(40, K)
    w[:, :16] = 1.0
    w, s = ref.quantize(w)
    for dtype in (BF, F32):
        y = be().fp8_block_forward(x.to(dtype).to(DEV), w.to(DEV), s.to(DEV), K, 40)
        assert torch.equal(y.cpu().double(), want)


def test_forward_layouts_and_leading_dimensions():
    K, N = 200, 96
    g = gen(1)
    w, s = (t.to(DEV) for t in ref.weight(N, K, g))
    x = torch.randn(4, 25, K, generator=g).to(BF).to(DEV)
    want = be().fp8_block_forward(x.view(100, K), w, s, K, N)
    assert torch.equal(be().fp8_block_forward(x, w, s, K, N), want.view(4, 25, N))
    wide = torch.zeros(100, K + 3, dtype=BF, device=DEV)
    wide[:, 1:K + 1] = x.view(100, K)
    assert torch.equal(be().fp8_block_forward(wide[:, 1:K + 1], w, s, K, N), want)
    off = torch.zeros(w.numel() + 3, dtype=torch.uint8, device=DEV)
    off[3:] = w.view(-1)
    soff = torch.zeros(s.numel() + 1, dtype=torch.uint8, device=DEV)
    soff[1:] = s.view(-1)
    assert torch.equal(be().fp8_block_forward(x.view(100, K), off[3:].view(N, -1), soff[1:].view(N, -1), K, N), want)
    assert be().fp8_block_forward(x[:0], w, s, K, N).shape == (0, 25, N)


@pytest.mark.parametrize("rows", [3, 64, 300])
def test_forward_with_infinities_and_nan(rows):
    """A block that holds one is all NaN: its row's outputs are, and no other's."""
    K, N = 300, 140
    g = gen(rows)
    w, s = ref.weight(N, K, g)
    x = torch.randn(rows, K, generator=g)
    clean = be().fp8_block_forward(x.to(DEV), w.to(DEV), s.to(DEV), K, N).cpu()
    x[1, 7], x[rows - 1, 299] = math.inf, math.nan
    y = be().fp8_block_forward(x.to(DEV), w.to(DEV), s.to(DEV), K, N).cpu()
    bad = torch.zeros(rows, dtype=torch.bool)
    bad[1] = bad[rows - 1] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])
    s[5, 1] = 255
    y = be().fp8_block_forward(x.to(DEV), w.to(DEV), s.to(DEV), K, N).cpu()
    assert torch.isnan(y[:, 5]).all()
    keep = [n for n in range(N) if n != 5]
    assert torch.equal(y[~bad][:, keep], clean[~bad][:, keep])


@pytest.mark.parametrize("K,N", [(1, 1), (64, 31), (128, 128), (129, 130), (513, 640), (777, 1000), (260, 2048)])
@pytest.mark.parametrize("rows", ROWS)
def test_backward_input(rows, K, N):
    g = gen(rows * K + N)
    w, s = ref.weight(N, K, g)
    wv = ref.values(w, s, K)
    dy = torch.randn(rows, N, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))
    for dtype in (BF, F32):
        t = dy.to(dtype)
        dx = be().fp8_block_backward_input(t.to(DEV), w.to(DEV), s.to(DEV), K, N)
        assert dx.dtype == dtype
        ref.check(dx, *ref.product(t.double(), wv.t().contiguous(), dtype), (rows, K, N, dtype))
    assert be().fp8_block_backward_input(t[:0].to(DEV), w.to(DEV), s.to(DEV), K, N).shape == (0, K)


@pytest.mark.parametrize("rows,K,N", [(70, 8192, 140), (130, 6000, 300), (65, 5001, 70), (200, 16384, 96)])
def test_few_tiles_of_a_long_axis(rows, K, N):
    """K in slices that are joined: forward, and the input gradient over as many outputs."""
    g = gen(rows)
    w, s = ref.weight(N, K, g)
    wv = ref.values(w, s, K)
    x = torch.randn(rows, K, generator=g)
    for dtype in (BF, F32):
        y = be().fp8_block_forward(x.to(dtype).to(DEV), w.to(DEV), s.to(DEV), K, N)
        ref.check(y, *ref.product(ref.rounded(x.to(dtype)), wv, dtype, codes=True), (rows, K, N, dtype))
    w, s = ref.weight(K, N, g)
    wv = ref.values(w, s, N)
    for dtype in (BF, F32):
        dx = be().fp8_block_backward_input(x.to(dtype).to(DEV), w.to(DEV), s.to(DEV), N, K)
        ref.check(dx, *ref.product(x.to(dtype).double(), wv.t().contiguous(), dtype), (rows, K, N, dtype))


# a wave's steps and the rounds of workgroups on either side of what one launch has
@pytest.mark.parametrize("rows,K,N", [(65, 513, 1024), (65, 513, 1025), (300, 131, 1101), (257, 64, 777), (1001, 1000, 777),
                                      (520, 1000, 1000), (2100, 250, 500), (2100, 260, 520), (900, 1090, 520), (1024, 1025, 512)])
def test_backward_input_by_either_way(rows, K, N):
    g = gen(rows * K + N)
    w, s = ref.weight(N, K, g)
    wv = ref.values(w, s, K).t().contiguous()
    dy = torch.randn(rows, N, generator=g)
    for dtype in (BF, F32):
        t = dy.to(dtype)
        dx = be().fp8_block_backward_input(t.to(DEV), w.to(DEV), s.to(DEV), K, N)
        ref.check(dx, *ref.product(t.double(), wv, dtype), (rows, K, N, dtype))
        t[1, N - 1], t[rows - 1, 0], t[rows // 2, 5] = float("nan"), float("inf"), float("-inf")
        bad = dx.clone()
        bad[[1, rows - 1, rows // 2]] = 0
        dx = be().fp8_block_backward_input(t.to(DEV), w.to(DEV), s.to(DEV), K, N)
        assert not torch.isfinite(dx[[1, rows - 1, rows // 2]]).any()
        dx[[1, rows - 1, rows // 2]] = 0
        assert torch.equal(dx, bad)


# one workgroup a CU and one more, of 32 and of 64 columns (256 CUs), and two rounds of them
@pytest.mark.parametrize("rows,K,N", [(1024, 510, 300), (1024, 520, 300), (1000, 1024, 600), (1030, 1010, 600), (2200, 140, 470),
                                      (1790, 70, 880), (3800, 380, 150), (70, 8192, 65), (200, 4090, 1024)])
def test_backward_input_about_one_round(rows, K, N):
    g = gen(rows)
    w, s = ref.weight(N, K, g)
    wv = ref.values(w, s, K).t().contiguous()
    dy = torch.randn(rows, N, generator=g)
    for dtype in (BF, F32):
        t = dy.to(dtype)
        dx = be().fp8_block_backward_input(t.to(DEV), w.to(DEV), s.to(DEV), K, N)
        ref.check(dx, *ref.product(t.double(), wv, dtype), (rows, K, N, dtype))


def room(bytes_):
    free = torch.cuda.mem_get_info()[0]
    if free < bytes_:
        pytest.skip(f"needs {bytes_ >> 30} GiB of device memory, {free >> 30} are free")


def repeats(y, y0):
    """Whether y's columns are y0's, over and over."""
    P = y0.shape[1]
    return all(torch.equal(y[:, k:k + P], y0[:, :y.shape[1] - k]) for k in range(0, y.shape[1], P))


# 31 rows of the result pass 32 bits of bytes, whole vectors a row
@pytest.mark.parametrize("dtype,N", [(F32, 44739248), (BF, 89478488)])
def test_forward_of_very_wide_results(dtype, N):
    """Columns repeat with a period that no tile has, and are the narrow product's."""
    room(40 << 30)
    K, P, rows = 100, 60011, 70
    w0, s0 = ref.weight(P, K, gen(3))
    w0, s0 = w0.to(DEV), s0.to(DEV)
    x = torch.randn(rows, K, generator=gen(4)).to(dtype).to(DEV)
    y0 = be().fp8_block_forward(x, w0, s0, K, P)
    at = torch.randint(0, P, (50,), generator=gen(5))
    wv = ref.values(w0[at.to(DEV)].cpu(), s0[at.to(DEV)].cpu(), K)
    ref.check(y0[:, at.to(DEV)], *ref.product(ref.rounded(x.cpu()), wv, dtype, codes=True), (dtype, N))
    w, s = (t.repeat(-(-N // P), 1)[:N] for t in (w0, s0))
    assert repeats(be().fp8_block_forward(x, w, s, K, N), y0)


@pytest.mark.parametrize("dtype,K", [(F32, 44739248), (BF, 89478488)])
def test_backward_input_of_very_wide_results(dtype, K):
    room(80 << 30)
    N, P, rows = 20, 60416, 70  # the scales repeat with the codes: a period of whole words of them
    w0, s0 = ref.weight(N, P, gen(6))
    w, s = w0.to(DEV).repeat(1, -(-K // P)), s0.to(DEV).repeat(1, -(-K // P))
    n = ref.blocks(K)
    w, s = w[:, :128 * n].contiguous(), s[:, :(n + 3) // 4 * 4].contiguous()
    w[:, K:], s[:, n:] = 0, 0
    g = torch.randn(rows, N, generator=gen(7)).to(dtype)
    dx0 = be().fp8_block_backward_input(g.to(DEV), w0.to(DEV), s0.to(DEV), P, N)
    wv = ref.values(w0, s0, P)[:, :1000].t().contiguous()
    ref.check(dx0[:, :1000], *ref.product(g.double(), wv, dtype), (dtype, K))
    assert repeats(be().fp8_block_backward_input(g.to(DEV), w, s, K, N), dx0)
