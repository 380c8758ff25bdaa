"""The 8-bit feed-forward path as a program uses it: layers in a row, other streams,
captured graphs, long tensors, other layouts, rows that are not finite."""
import gc

import pytest
import torch

import _fp8_block as ref
from smaulnative_amd import AddRMSNorm, FP8BlockFFN, FP8BlockLinear, FP8BlockNormFFN
from smaulnative_amd.compute import get_backend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def be():
    return get_backend("rocm")


def block(d, h, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [t.to(DEV) for n, k in ((h, d), (h, d), (d, h)) for t in ref.weight(n, k, g, 1.5 / k ** 0.5)]


def ask(T, d, h, seed, dtype=BF):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(T, d, generator=g).to(dtype).to(DEV) for _ in range(2)]


def run(x, r, dy, w, norm, lin, d, h):
    """Every operator once, as a layer runs them: outputs and gradients."""
    b = be()
    s, codes, scales = b.add_rms_norm(x, r, norm, 1e-6, quantize=True)
    y, saved = b.fp8_block_ffn_forward(codes, w, d, h, xs=scales, save=True)
    q, qs = b.fp8_block_quantize(y)
    out = b.fp8_block_forward(q, *lin, d, h, xs=qs)
    grad = b.fp8_block_backward_input(out, *lin, d, h) + dy
    dx, *dw = b.fp8_block_ffn_backward(grad, w, saved, d, h)
    dx, dn = b.add_rms_norm_backward(dx, s, norm, 1e-6, grad)
    return (s, y, b.fp8_block_dequantize(q, qs, d, BF), out, dx, dn, *dw)


# few rows; few tiles in slices of a long K; many tiles
@pytest.mark.parametrize("T,d,h", [(1, 128, 200), (20, 200, 333), (70, 256, 4200), (700, 320, 1100)])
def test_together_streams_and_replays(T, d, h):
    w, lin = block(d, h), block(d, h, 1)[:2]
    norm = torch.rand(d, device=DEV) + 0.5
    x, r = ask(T, d, h, 2)
    dy = ask(T, d, h, 3)[0]
    args = (x, r, dy, w, norm, lin, d, h)
    want = run(*args)
    assert all(torch.equal(a, b) for a, b in zip(run(*args), want))
    # two calls at once, on streams of their own
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in sides:
        with torch.cuda.stream(s):
            got.append([run(*args) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for side in got for o in side for a, b in zip(o, want))
    # two graphs of one program, replayed at once beside eager calls over changing inputs
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(*args)
        graphs.append((g, out))
    for i in range(3):
        for t in (x, r, dy):
            t.copy_(torch.randn(T, d, generator=torch.Generator().manual_seed(10 * i)))
        torch.cuda.synchronize()
        for s, (g, _) in zip(sides, graphs):
            with torch.cuda.stream(s):
                g.replay()
        want = run(*args)
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("trainable", [False, True])
@pytest.mark.parametrize("T", [5, 300])
def test_layers_in_a_captured_step(T, trainable):
    """Two layers and a product, their loss and gradients, in a graph; a capture is refused as
    long as an eager pass holds the parameters."""
    torch.manual_seed(0)
    d, h = 136, 264
    a, b = (FP8BlockNormFFN(d, h, trainable).to(DEV) for _ in range(2))
    c, n, f = FP8BlockLinear(d, 100, bias=True).to(DEV), AddRMSNorm(d).to(DEV), FP8BlockFFN(d, h, trainable).to(DEV)
    params = [p for m in (a, b, c, n, f) for p in m.parameters()]
    x = torch.randn(T, d, device=DEV)

    def step():
        y, s = a(x)
        y, s = b(y, s)
        y, s = n(y, s)
        y = c(f(y) + s)
        for p in params:
            p.grad = None
        (y * y).mean().backward()
        return y.detach(), [p.grad for p in params]

    eager = a(x)
    held = n(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="outside of this capture"):
            a(x)
        with pytest.raises(RuntimeError, match="outside of this capture"):
            n(x)
        with torch.no_grad():
            a(x)
    assert eager[0].requires_grad and held[0].requires_grad
    del eager, held
    gc.collect()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, grads = step()
    for i in range(3):
        x.copy_(torch.randn(T, d, generator=torch.Generator().manual_seed(i)))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, *grads)]
        y2, grads2 = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, (y2, *grads2)))
        del y2, grads2


@pytest.mark.parametrize("T,h", [(10, 300), (200, 300), (1100, 2200)])
def test_rows_that_are_not_finite(T, h):
    """They spoil their own rows, and sums over rows; the other rows are as without them."""
    d = 200
    w = block(d, h)
    x, dy = ask(T, d, h, 5)
    bad = [0, T // 2, T - 1]
    ok = torch.ones(T, dtype=torch.bool, device=DEV)
    ok[bad] = False
    y, saved = be().fp8_block_ffn_forward(x, w, d, h, save=True)
    dx = be().fp8_block_ffn_backward(dy, w, saved, d, h)[0]
    for row, v in zip(bad, (float("nan"), float("inf"), float("-inf"))):
        x[row, 7] = v
    y2, saved = be().fp8_block_ffn_forward(x, w, d, h, save=True)
    dx2, *dw = be().fp8_block_ffn_backward(dy, w, saved, d, h)
    assert torch.equal(y[ok], y2[ok]) and torch.equal(dx[ok], dx2[ok])
    assert bool(y2[~ok].isnan().all()) and bool(dx2[~ok].isnan().all())
    assert all(bool(t.isnan().all()) for t in dw)
    # a gradient that is not finite
    x, dy = ask(T, d, h, 5)
    y, saved = be().fp8_block_ffn_forward(x, w, d, h, save=True)
    dy[bad[1], 3] = float("nan")
    dx2 = be().fp8_block_ffn_backward(dy, w, saved, d, h, need_dw=False)[0]
    ok[:] = True
    ok[bad[1]] = False
    assert torch.equal(dx[ok], dx2[ok]) and bool(dx2[~ok].isnan().all())


@pytest.mark.parametrize("T", [3, 130])
def test_other_layouts(T):
    """Strided rows, codes at odd addresses, leading dimensions, one tensor twice."""
    d, h = 136, 300
    w = block(d, h)
    x, dy = ask(T, d, h, 8)
    y, saved = be().fp8_block_ffn_forward(x, w, d, h, save=True)
    grads = be().fp8_block_ffn_backward(dy, w, saved, d, h)

    def odd(t):
        b = torch.empty(t.numel() + 3, dtype=t.dtype, device=DEV)
        v = b[3:].view(t.shape)
        return v.copy_(t)

    wide = torch.randn(T, d + 5, device=DEV).to(BF)
    for form in (odd, lambda t: t.t().contiguous().t(), lambda t: t.unsqueeze(0).expand(2, *t.shape)[1]):
        w2 = [form(t) for t in w]
        y2, saved2 = be().fp8_block_ffn_forward(form(x), w2, d, h, save=True)
        got = be().fp8_block_ffn_backward(form(dy), w2, saved2, d, h)
        assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(grads, got))
    wide[:, 2:2 + d] = x
    assert torch.equal(be().fp8_block_ffn_forward(wide[:, 2:2 + d], w, d, h), y)
    s, n = be().add_rms_norm(x, x, None, 1e-6)
    assert torch.equal(s, (2 * x.float()).to(BF))
    dx, _ = be().add_rms_norm_backward(n, s, None, 1e-6, n, need_dw=False)
    assert torch.isfinite(dx).all()
    one = be().fp8_block_ffn_forward(x[:, None], w, d, h)
    assert one.shape == (T, 1, d) and torch.equal(one[:, 0], y)
    # gate and up may be one matrix
    w3 = [*w[:2], *w[:2], *w[4:]]
    ref_y, bound = ref.ffn(ref.rounded(x.cpu()), *[ref.values(w3[i].cpu(), w3[i + 1].cpu(), k)
                                                   for i, k in ((0, d), (2, d), (4, h))])[:2]
    ref.check(be().fp8_block_ffn_forward(x, w3, d, h), ref_y, bound)


def room(bytes_):
    free = torch.cuda.mem_get_info()[0]
    if free < bytes_:
        pytest.skip(f"needs {bytes_ >> 30} GiB of device memory, {free >> 30} are free")


def periods(T, t):
    """Rows 0 to T - 1 of a tensor that repeats t's."""
    return t.repeat(-(-T // t.shape[0]), 1)[:T]


def test_more_than_32_bits_of_rows():
    """Rows repeat with a period that no tile has: each period as the first, whose rows are
    checked against the same rows alone."""
    room(90 << 30)
    T, P, K, N = (1 << 25) + 1000, 20011, 256, 136  # 8.6 G codes
    g = torch.Generator().manual_seed(4)
    lin = [t.to(DEV) for t in ref.weight(N, K, g)]
    base = torch.randn(P, K, generator=g).to(BF).to(DEV)
    x = periods(T, base)
    q, s = be().fp8_block_quantize(x)
    del x
    q0, s0 = be().fp8_block_quantize(base)
    last = T // P * P
    for a, b in ((q, q0), (s, s0)):
        assert torch.equal(a[:P], b) and torch.equal(a[last - P:last], b) and torch.equal(a[last:], b[:T - last])
    y = be().fp8_block_forward(q, *lin, K, N, xs=s)
    y0 = be().fp8_block_forward(q0, *lin, K, N, xs=s0)
    for k in range(0, last, P):
        assert torch.equal(y[k:k + P], y0), k
    assert torch.equal(y[last:], y0[:T - last])
    v = be().fp8_block_dequantize(q, s, K, BF)
    assert torch.equal(v[last - P:last], be().fp8_block_dequantize(q0, s0, K, BF))
    del q, s
    dx = be().fp8_block_backward_input(y, *lin, K, N)
    dx0 = be().fp8_block_backward_input(y0, *lin, K, N)
    assert torch.equal(dx[:P], dx0) and torch.equal(dx[last - P:last], dx0)
    sums, n = be().add_rms_norm(v, dx, None, 1e-6)
    assert torch.equal(n[last - P:last], be().add_rms_norm(v[:P], dx0, None, 1e-6)[1])
    del dx, v
    d2 = be().add_rms_norm_backward(n, sums, None, 1e-6, None, need_dw=False)[0]
    assert torch.equal(d2[last - P:last], be().add_rms_norm_backward(n[:P], sums[:P], None, 1e-6, None, False)[0])


def test_more_than_32_bits_of_hidden_rows():
    room(120 << 30)
    T, P, d, h = 7_000_000, 20011, 128, 640  # 4.5 G hidden codes
    w = block(d, h)
    x0, dy0 = ask(P, d, h, 9)
    x, dy = periods(T, x0), periods(T, dy0)
    last = T // P * P
    y, saved = be().fp8_block_ffn_forward(x, w, d, h, save=True)
    y0, saved0 = be().fp8_block_ffn_forward(x0, w, d, h, save=True)
    for k in range(0, last, P):
        assert torch.equal(y[k:k + P], y0), k
    assert torch.equal(y[last:], y0[:T - last])
    dx, *dw = be().fp8_block_ffn_backward(dy, w, saved, d, h)
    dx0, *dw0 = be().fp8_block_ffn_backward(dy0, w, saved0, d, h)
    for k in range(0, last, P):
        assert torch.equal(dx[k:k + P], dx0), k
    # T / P periods, the last one in part (0.002 for it): fp32 sums over T rows 16 an instruction, half
    # a step each, and two roundings to bf16
    for a, b in zip(dw, dw0):
        scale = float(b.double().abs().max()) * T / P
        off = (a.double() - b.double() * (T / P)).abs().max()
        assert float(off) <= scale * (T / 16 * 2.0 ** -24 + 2 * 2.0 ** -8 + 0.002), float(off) / scale
