"""The gated feed-forward block in 8 bits and its gradients, and the layers over it,
against plain 64-bit forms."""
import pytest
import torch
import torch.nn as nn

import _fp8_block as ref
from smaulnative_amd import AddRMSNorm, FP8BlockFFN, FP8BlockLinear, FP8BlockNormFFN, FP8Linear, SwiFFN, MoEConfig
from smaulnative_amd import _lib, fp8_block
from smaulnative_amd.compute import get_backend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
KEPT = 2.0 ** -16  # what the forward pass keeps for the gradients has 16 significant bits or more


def be():
    return get_backend("rocm")


def block(T, d, h, seed=0):
    g = torch.Generator().manual_seed(seed * 104729 + T * 31 + d * 7 + h)
    x, dy = (torch.randn(T, d, generator=g).to(BF) for _ in range(2))
    weights = [t for n, k in ((h, d), (h, d), (d, h)) for t in ref.weight(n, k, g, 1.5 / k ** 0.5)]
    plain = [ref.values(weights[i], weights[i + 1], k) for i, k in ((0, d), (2, d), (4, h))]
    return x, dy, [t.to(DEV) for t in weights], plain


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 64, 200), (3, 300, 129), (33, 128, 384), (64, 200, 640), (65, 130, 257),
          (130, 256, 512), (300, 500, 1251), (257, 129, 130), (70, 130, 4200)]


@pytest.mark.parametrize("T,d,h", SHAPES)
def test_forward(T, d, h):
    x, _, w, plain = block(T, d, h)
    y, bound = ref.ffn(ref.rounded(x), *plain, exact=True)[:2]
    got = be().fp8_block_ffn_forward(x.to(DEV), w, d, h)
    assert got.dtype == BF
    ref.check(got, y, bound, (T, d, h))
    c, cs = ref.quantize(x)
    assert torch.equal(be().fp8_block_ffn_forward(c.to(DEV), w, d, h, xs=cs.to(DEV)), got)


@pytest.mark.parametrize("given", ["rows", "codes"])
@pytest.mark.parametrize("T,d,h", SHAPES)
def test_backward(T, d, h, given):
    x, dy, w, plain = block(T, d, h, 1)
    want = ref.ffn_grad(ref.rounded(x), dy.double(), *plain, KEPT, exact=True)
    c, cs = (t.to(DEV) for t in ref.quantize(x))
    arg = (x.to(DEV), None) if given == "rows" else (c, cs)
    y, saved = be().fp8_block_ffn_forward(arg[0], w, d, h, xs=arg[1], save=True)
    assert torch.equal(y, be().fp8_block_ffn_forward(arg[0], w, d, h, xs=arg[1]))
    grads = be().fp8_block_ffn_backward(dy.to(DEV), w, saved, d, h)
    for name, got in zip(("y", "dx", "dgate", "dup", "ddown"), (y, *grads)):
        assert got.dtype == BF
        ref.check(got, *want[name], (name, T, d, h))
    dx = be().fp8_block_ffn_backward(dy.to(DEV), w, saved, d, h, need_dw=False)
    assert torch.equal(dx[0], grads[0]) and dx[1:] == (None, None, None)
    dw = be().fp8_block_ffn_backward(dy.to(DEV), w, saved, d, h, need_dx=False)
    assert dw[0] is None and all(torch.equal(a, b) for a, b in zip(dw[1:], grads[1:]))


# more tiles of 64 rows by a block than the chip has CUs: each of the larger tiles
@pytest.mark.parametrize("T,d,h", [(1100, 130, 2200), (129, 64, 32896), (2040, 150, 4090)])
def test_many_tiles(T, d, h):
    x, dy, w, plain = block(T, d, h, 6)
    assert -(-T // 64) * ref.blocks(h) > torch.cuda.get_device_properties(0).multi_processor_count
    y, saved = be().fp8_block_ffn_forward(x.to(DEV), w, d, h, save=True)
    assert torch.equal(y, be().fp8_block_ffn_forward(x.to(DEV), w, d, h))
    dx = be().fp8_block_ffn_backward(dy.to(DEV), w, saved, d, h, need_dw=False)[0]
    at = torch.cat([torch.tensor([0, 63, 64, 127, 128, T - 1]), torch.randperm(T, generator=torch.Generator().manual_seed(1))[:20]])
    want = ref.ffn_grad(ref.rounded(x[at]), dy[at].double(), *plain, KEPT)
    ref.check(y[at.to(DEV)], *want["y"], (T, d, h))
    ref.check(dx[at.to(DEV)], *want["dx"], (T, d, h))


@pytest.mark.parametrize("T", [20, 300])
def test_few_hidden_rows_are_exact(T):
    """Most of y is 64 bits' y rounded once.  Sums in fp32 are off by 2e-6 in the mean (16 roundings
    of partial sums), a code's step is 2^-4 of it and more: 6e-5 of the codes move, a code in one
    row of 20, and it moves less than half of the row's outputs by a step of bf16 (a hidden value is
    768^-0.5 of an output, its step 2^-4 of that, bf16's 2^-8): less than 5 % in all."""
    d, h = 256, 768
    x, _, w, plain = block(T, d, h, 7)
    y = ref.ffn(ref.rounded(x), *plain)[0]
    got = be().fp8_block_ffn_forward(x.to(DEV), w, d, h).cpu()
    assert float((got == y.to(BF)).double().mean()) >= 0.95


def test_empty_batch():
    d, h = 130, 200
    _, _, w, _ = block(1, d, h)
    x = torch.zeros(0, d, dtype=BF, device=DEV)
    y, saved = be().fp8_block_ffn_forward(x, w, d, h, save=True)
    assert y.shape == (0, d)
    dx, *dw = be().fp8_block_ffn_backward(x, w, saved, d, h)
    assert dx.shape == (0, d) and all(not t.any() for t in dw)


def test_gradients_against_differences():
    """Central differences in 64 bits of the block with its rounding held: h moves the rounded
    hidden rows as much as the unrounded ones.  The bounds of the gradients, and 1e-6 for the
    differences (step 1e-4, third derivatives of order 1)."""
    T, d, h = 5, 40, 24
    x, dy, w, plain = block(T, d, h, 2)
    xv = ref.rounded(x)
    want = ref.ffn_grad(xv, dy.double(), *plain, KEPT)
    y, saved = be().fp8_block_ffn_forward(x.to(DEV), w, d, h, save=True)
    grads = dict(zip(("dx", "dgate", "dup", "ddown"), be().fp8_block_ffn_backward(dy.to(DEV), w, saved, d, h)))
    v = ref.silu(xv @ plain[0].t()) * (xv @ plain[1].t())
    held = ref.rounded(v) - v

    def loss(p):
        hid = ref.silu(p[0] @ p[1].t()) * (p[0] @ p[2].t()) + held
        return float((hid @ p[3].t() * dy.double()).sum())

    at = [xv, *plain]
    for i, name in enumerate(("dx", "dgate", "dup", "ddown")):
        for j in range(0, at[i].numel(), 17):
            side = []
            for step in (1e-4, -1e-4):
                p = [t.clone() for t in at]
                p[i].view(-1)[j] += step
                side.append(loss(p))
            slope = (side[0] - side[1]) / 2e-4
            off = abs(slope - float(grads[name].reshape(-1)[j]))
            assert off <= float(want[name][1].reshape(-1)[j]) + 1e-6 * (1 + abs(slope)), (name, j, off)


def test_linear_layer():
    torch.manual_seed(0)
    K, N = 200, 150
    lin = nn.Linear(K, N).to(DEV)
    m = FP8BlockLinear.from_float(lin)
    w = ref.rounded(lin.weight.detach().cpu())
    assert torch.equal(fp8_block.decode(m.w8, m.ws, K).cpu().double(), w)
    for dtype in (F32, BF, torch.float16):
        x = torch.randn(3, 70, K).to(dtype).to(DEV).requires_grad_()
        y = m(x)
        assert y.shape == (3, 70, N)
        xv = ref.rounded(x.detach().cpu().float().view(-1, K))
        want, bound = ref.product(xv, w, F32)
        if dtype == BF:
            bound = bound + ref.aligned(xv, w)
        half = {F32: ref.U, BF: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
        bound = bound + half * (want.abs() + bound)  # the product is rounded to x's type, then the bias added in fp32
        want = want + lin.bias.detach().cpu().double()
        ref.check(y.view(-1, N), want, bound + ref.U * (want.abs() + bound))
        dy = torch.randn(3, 70, N).to(y.dtype).to(DEV)
        y.backward(dy)
        dx, bound = ref.product(dy.cpu().double().view(-1, N).to(dtype).double(), w.t().contiguous(), F32)
        assert x.grad.dtype == dtype
        # the bias is fp32: a gradient comes back through a cast to y's own type
        ref.check(x.grad.view(-1, K), dx, bound + 3 * half * (dy.cpu().double().view(-1, N).abs() @ w.abs() + bound))
    fp8 = FP8Linear(K, N).to(DEV)
    m = FP8BlockLinear.from_fp8(fp8)
    assert m(torch.randn(5, K, device=DEV)).shape == (5, N)


def test_host_quantizer_is_the_device_one():
    x = torch.randn(20, 300) * torch.exp(3 * torch.randn(20, 1))
    x[3, 5], x[4, 250], x[6] = float("inf"), float("nan"), 0.0
    for t in (x, x.to(BF)):
        host, dev = fp8_block.quantize(t), fp8_block.quantize(t.to(DEV))
        assert all(torch.equal(a, b.cpu()) for a, b in zip(host, dev))
        a, b = fp8_block.decode(*host, 300), fp8_block.decode(*dev, 300).cpu()
        assert torch.equal(torch.nan_to_num(a, nan=7.0), torch.nan_to_num(b, nan=7.0))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("residual", [True, False])
def test_norm_layer(dtype, residual):
    torch.manual_seed(1)
    T, d = 50, 300
    m = AddRMSNorm(d, 1e-5).to(DEV)
    with torch.no_grad():
        m.weight.add_(0.2 * torch.randn(d, device=DEV))
    x, r = (torch.randn(2, T // 2, d).to(dtype).to(DEV).requires_grad_() for _ in range(2))
    y, s = m(x, r if residual else None)
    dy, ds = (torch.randn(2, T // 2, d).to(dtype).to(DEV) for _ in range(2))
    torch.autograd.backward([y, s], [dy, ds])
    sv = s.detach().cpu().double().view(T, d)
    w = m.weight.detach().cpu().double()
    want, e = ref.norm(sv, w, 1e-5)
    ref.check(y.view(T, d), want, e + ref.HALF[dtype] * (want.abs() + e))
    (dx, dxe), (dw, dwe) = ref.norm_grad(dy.cpu().double().view(T, d), sv, w, 1e-5, ds.cpu().double().view(T, d), dtype)
    ref.check(x.grad.view(T, d), dx, dxe)
    ref.check(m.weight.grad, dw, dwe)
    if residual:
        assert torch.equal(r.grad, x.grad)


F16 = torch.float16
STEP = {F32: (ref.U, 2.0 ** -149), BF: (2.0 ** -8, 2.0 ** -133), F16: (2.0 ** -11, 2.0 ** -25), torch.float64: (0.0, 0.0)}
# x's type, the residual's, the sum's
TYPES = [(F16, None, F16), (F16, F16, F16), (BF, F32, F32), (F32, BF, F32), (F16, BF, F32), (BF, F16, F32),
         (torch.float64, torch.float64, torch.float64)]


def typed(T, d, xt, rt, seed):
    """x, the residual (or None) as leaves, and gradients of the outputs, which the sum's type holds."""
    torch.manual_seed(seed)
    x = torch.randn(T, d).to(xt).to(DEV).requires_grad_()
    r = None if rt is None else torch.randn(T, d).to(rt).to(DEV).requires_grad_()
    return x, r, torch.randn(T, d).to(xt).to(DEV), torch.randn(T, d).to(BF).to(DEV)


@pytest.mark.parametrize("xt,rt,total", TYPES)
def test_norm_layer_of_other_types(xt, rt, total):
    """Computed in fp32 on fp32 addends, each output and gradient rounded to its own type once more."""
    T, d = 50, 300
    m = AddRMSNorm(d, 1e-5).to(DEV)
    x, r, dy, ds = typed(T, d, xt, rt, 4)
    y, s = m(x, r)
    assert y.dtype == xt and s.dtype == total
    torch.autograd.backward([y, s], [dy, ds.to(total)])
    sv = x.detach().cpu().float()
    if r is not None:
        sv = sv + r.detach().cpu().float()
    assert torch.equal(s.detach().cpu(), sv.to(total))

    def again(v, e, dtype):  # rounded to fp32, then to dtype
        half, least = STEP[dtype]
        e = e + ref.U * (v.abs() + e)
        return v, e + half * (v.abs() + e) + least

    w = torch.ones(d).double()
    ref.check(y, *again(*ref.norm(sv.double(), w, 1e-5), xt))
    (dx, dxe), (dw, dwe) = ref.norm_grad(dy.cpu().double(), sv.double(), w, 1e-5, ds.cpu().double(), F32)
    ref.check(m.weight.grad, dw, dwe)
    for leaf, dtype in ((x, xt), (r, rt)):
        if leaf is not None:
            assert leaf.grad.dtype == dtype
            ref.check(leaf.grad, *again(dx, dxe, dtype))


@pytest.mark.parametrize("xt,rt,total", TYPES)
@pytest.mark.parametrize("T", [7, 130])
def test_norm_block_layer_of_other_types(T, xt, rt, total):
    """As the layer on fp32 addends."""
    torch.manual_seed(T)
    d, h = 136, 300
    m = FP8BlockNormFFN(d, h, True).to(DEV)
    x, r, dy, ds = typed(T, d, xt, rt, T)
    y, s = m(x, r)
    assert y.dtype == xt and s.dtype == total
    torch.autograd.backward([y, s], [dy, ds.to(total)])
    grads = [p.grad for p in m.parameters()]
    m.zero_grad(set_to_none=True)
    x2, r2 = (t if t is None else t.detach().float().requires_grad_() for t in (x, r))
    y2, s2 = m(x2, r2)
    torch.autograd.backward([y2, s2], [dy.float(), ds.float()])
    assert torch.equal(y, y2.to(xt)) and torch.equal(s, s2.to(total))
    assert all(torch.equal(a, p.grad) for a, p in zip(grads, m.parameters()))
    for a, b in ((x, x2), (r, r2)):
        assert a is None or (a.grad.dtype == a.dtype and torch.equal(a.grad, b.grad.to(a.dtype)))


def _module_weights(m):
    if m.trainable:
        return [ref.rounded(t.detach().cpu().float()) for t in (m.gate, m.up, m.down)]
    return [fp8_block.decode(getattr(m, n + "_w").cpu(), getattr(m, n + "_s").cpu(), k).double()
            for n, k in (("gate", m.d), ("up", m.d), ("down", m.h))]


@pytest.mark.parametrize("trainable", [True, False])
@pytest.mark.parametrize("T", [5, 64, 200])
def test_block_layer(T, trainable):
    torch.manual_seed(T)
    d, h = 136, 300
    m = FP8BlockFFN(d, h, trainable).to(DEV)
    x = torch.randn(T, d).to(BF).to(DEV).requires_grad_()
    y = m(x)
    dy = torch.randn(T, d).to(BF).to(DEV)
    y.backward(dy)
    want = ref.ffn_grad(ref.rounded(x.detach().cpu()), dy.cpu().double(), *_module_weights(m), KEPT)
    ref.check(y, *want["y"])
    ref.check(x.grad, *want["dx"])
    if trainable:
        for name in ("gate", "up", "down"):
            g = getattr(m, name).grad
            assert g.dtype == F32
            ref.check(g, *want["d" + name])
    with torch.no_grad():
        assert torch.equal(m(x), y)


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("layer", [lambda: AddRMSNorm(136), lambda: FP8BlockNormFFN(136, 200, True), lambda: FP8BlockNormFFN(136, 200)])
def test_an_output_that_nothing_uses(layer, residual, monkeypatch):
    """Its gradient is zeros, which for the sum are neither filled in nor read."""
    torch.manual_seed(0)
    m = layer().to(DEV)
    x, r = (torch.randn(20, 136, device=DEV).to(BF).requires_grad_() for _ in range(2))
    inputs = [x, *([r] if residual else []), *m.parameters()]
    dy, ds = (torch.randn(20, 136, device=DEV).to(BF) for _ in range(2))
    seen, entry = [], type(be()).add_rms_norm_backward

    def look(self, dy, s, weight=None, eps=1e-6, ds=None, need_dw=True):
        seen.append(ds)
        return entry(self, dy, s, weight, eps, ds, need_dw)

    monkeypatch.setattr(type(be()), "add_rms_norm_backward", look)
    y, s = m(x, r if residual else None)
    got = torch.autograd.grad(y, inputs, dy)
    assert seen == [None]
    y, s = m(x, r if residual else None)
    want = torch.autograd.grad([y, s], inputs, [dy, torch.zeros_like(s)])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    y, s = m(x, r if residual else None)
    got = torch.autograd.grad(s, inputs, ds)
    assert torch.equal(got[0], ds) and not any(t.any() for t in got[1 + residual:])


def test_memory_of_a_frozen_block():
    """Its pass keeps the factors (6 bytes a hidden value) beside its input and output, and its
    gradient makes room for dx alone."""
    T, d, h, slack = 2048, 256, 2048, 1 << 21
    m = FP8BlockFFN(d, h).to(DEV)
    x = torch.randn(T, d, device=DEV).to(BF).requires_grad_()
    dy = torch.randn(T, d, device=DEV).to(BF)
    want = torch.autograd.grad(m(x), x, dy)[0]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = m(x)
    held = torch.cuda.memory_allocated() - before
    assert 6 * T * h <= held <= 6 * T * h + 2 * T * d + slack
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)
    # dg and du, the three weights turned round, dx in slices and itself
    need = _lib.load().smaul_fp8_block_ffn_backward_part_workspace_size(T, d, h, 1, 0)
    assert torch.cuda.max_memory_allocated() - before <= need + 2 * T * d + slack
    # and the codes are asked for where weights' gradients are
    w = [getattr(m, n) for n in m._NAMES]
    _, saved = be().fp8_block_ffn_forward(x.detach(), w, d, h, save=True)
    bare = (None, None, None, None, saved[4])
    assert torch.equal(be().fp8_block_ffn_backward(dy, w, bare, d, h, need_dw=False)[0], want)
    with pytest.raises(RuntimeError, match="need the codes"):
        be().fp8_block_ffn_backward(dy, w, bare, d, h)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("T", [7, 130])
def test_norm_block_layer(T, residual, dtype):
    """The norm's codes go straight to the block: as its entry points one after the other."""
    torch.manual_seed(T)
    d, h = 136, 300
    m = FP8BlockNormFFN(d, h, True).to(DEV)
    with torch.no_grad():
        m.norm.add_(0.2 * torch.randn(d, device=DEV))
    x, r = (torch.randn(T, d).to(dtype).to(DEV).requires_grad_() for _ in range(2))
    y, s = m(x, r if residual else None)
    dy, ds = (torch.randn(T, d).to(dtype).to(DEV) for _ in range(2))
    torch.autograd.backward([y, s], [dy, ds])
    b = be()
    w = [t for p in (m.gate, m.up, m.down) for t in b.fp8_block_quantize(p.detach())]
    with torch.no_grad():
        s1, c, cs = b.add_rms_norm(x, r if residual else None, m.norm, m.eps, quantize=True)
        y1, saved = b.fp8_block_ffn_forward(c, w, d, h, xs=cs, save=True)
        dn, *dw = b.fp8_block_ffn_backward(dy.to(BF), w, saved, d, h)
        dx, dnorm = b.add_rms_norm_backward(dn.to(dtype), s1, m.norm, m.eps, ds)
    assert torch.equal(y, y1.to(dtype)) and torch.equal(s, s1)
    assert torch.equal(x.grad, dx) and torch.equal(m.norm.grad, dnorm)
    assert all(torch.equal(p.grad, g.float()) for p, g in zip((m.gate, m.up, m.down), dw))
    if residual:
        assert torch.equal(r.grad, dx)


def test_block_of_a_tiled_layer():
    torch.manual_seed(3)
    ffn = SwiFFN(MoEConfig(d_model=128)).to(DEV)
    x = torch.randn(60, 128).to(BF).to(DEV)
    with torch.no_grad():
        want = ffn(x).double()
        got = FP8BlockFFN.from_swiffn(ffn)(x).double()
        same = FP8BlockFFN.from_swiffn(ffn, trainable=True)(x).double()
    # rounded activations, weights and hidden rows: each value off by 2^-4 at most, by 2^-5.5 in the mean
    assert float((got - want).norm() / want.norm()) < 3 * 2.0 ** -4 and torch.equal(got, same)
