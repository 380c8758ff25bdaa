"""CPU checks of the 8-bit feed-forward path: what its entry points refuse before anything
reaches a device, and the host quantizer."""
import pytest
import torch

import _fp8_block as ref
from smaulnative_amd import AddRMSNorm, FP8BlockFFN, FP8BlockLinear, FP8BlockNormFFN, _lib, fp8_block
from smaulnative_amd.compute import get_backend

P = 4096  # a pointer that is only looked at
OK, BAD, NO = _lib.SMAUL_OK, _lib.SMAUL_ERR_INVALID, _lib.SMAUL_ERR_UNSUPPORTED


def test_host_tensors_are_refused():
    be = get_backend("rocm")
    x, b = torch.zeros(3, 8), torch.zeros(3, 8, dtype=torch.bfloat16)
    w, s = torch.zeros(8, 128, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8)
    saved = (w[:3], s[:3], w[:3], s[:3], torch.zeros(3 * 8 * 8, dtype=torch.uint8))
    calls = (lambda: be.fp8_block_quantize(x), lambda: be.fp8_block_dequantize(w, s, 8),
             lambda: be.fp8_block_forward(x, w, s, 8, 8), lambda: be.fp8_block_backward_input(x, w, s, 8, 8),
             lambda: be.fp8_block_ffn_forward(b, (w, s) * 3, 8, 8),
             lambda: be.fp8_block_ffn_backward(b, (w, s) * 3, saved, 8, 8), lambda: be.add_rms_norm(x, x),
             lambda: be.add_rms_norm_backward(x, x))
    for call in calls:
        with pytest.raises(RuntimeError, match="HIP device tensors"):
            call()


def test_quantize_arguments():
    lib = _lib.load()
    assert lib.smaul_fp8_block_quantize(None, 0, None, None, 4, 32, None) == BAD
    assert lib.smaul_fp8_block_quantize(P, 2, P, P, 4, 32, None) == BAD
    assert lib.smaul_fp8_block_quantize(P, 0, P, P, 4, 0, None) == BAD
    assert lib.smaul_fp8_block_quantize(P, 0, P, P, -1, 32, None) == BAD
    assert lib.smaul_fp8_block_quantize(P, 0, P + 4, P, 4, 32, None) == BAD
    assert lib.smaul_fp8_block_quantize(P, 0, P, P, 0, 32, None) == OK
    assert lib.smaul_fp8_block_quantize(P, 0, P, P, 1 << 40, 128, None) == NO
    assert lib.smaul_fp8_block_dequantize(P, P, None, 0, 4, 32, None) == BAD
    assert lib.smaul_fp8_block_dequantize(P + 1, P, P, 0, 4, 32, None) == BAD
    assert lib.smaul_fp8_block_dequantize(P, P, P, 1, 1 << 40, 128, None) == NO


def test_product_arguments():
    lib = _lib.load()
    size = lib.smaul_fp8_block_linear_workspace_size
    for xt in (0, 1, 2):
        need = size(100, 64, 32, xt)
        assert need >= (0 if xt == 2 else 100 * 132)

        def call(x=P, xs=P, w=P, s=P, y=P, yt=1, rows=100, K=64, N=32, ws=P, nb=need, xt=xt):
            return lib.smaul_fp8_block_linear(x, xt, xs, w, s, y, yt, rows, K, N, ws, nb, None)

        assert call(rows=0) == OK and call(K=0) == BAD and call(N=-1) == BAD and call(yt=2) == BAD and call(xt=3) == BAD
        assert call(x=None) == BAD and call(w=None) == BAD and call(s=None) == BAD and call(y=None) == BAD
        assert call(x=P + 8) == BAD and call(w=P + 8) == BAD and call(y=P + 2) == BAD and call(s=P + 1) == BAD
        if xt == 2:
            assert call(xs=None) == BAD and call(xs=P + 2) == BAD
        if need:
            assert call(nb=need - 1) == BAD and call(ws=P + 16) == BAD and call(ws=None) == BAD
        big = size(1 << 40, 64, 32, xt)
        assert call(rows=1 << 40, nb=big) == NO
    assert size(-1, 64, 32, 0) == -1 and size(4, 64, 32, 5) == -1
    dsize = lib.smaul_fp8_block_backward_input_workspace_size
    assert dsize(4, 0, 32, 0) == -1 and dsize(4, 64, 32, 2) == -1
    for rows in (4, 100):
        need = dsize(rows, 64, 32, 1)

        def dx(g=P, t=1, w=P, s=P, o=P, rows=rows, K=64, N=32, ws=P, nb=need):
            return lib.smaul_fp8_block_backward_input(g, t, w, s, o, rows, K, N, ws, nb, None)

        assert dx(rows=0) == OK and dx(t=2) == BAD and dx(K=0) == BAD and dx(N=0) == BAD
        assert dx(g=None) == BAD and dx(o=None) == BAD and dx(g=P + 4) == BAD and dx(w=P + 4) == BAD
        if need:
            assert dx(nb=need - 1) == BAD and dx(ws=P + 8) == BAD


def test_block_arguments():
    lib = _lib.load()
    need = [lib.smaul_fp8_block_ffn_workspace_size(70, 64, 96, 1, save) for save in (0, 1)]

    def fwd(x=P, xt=1, xs=P, gw=P, gs=P, y=P, kept=P, saved=None, T=70, d=64, h=96, ws=P, nb=need[0]):
        return lib.smaul_fp8_block_ffn_forward(x, xt, xs, gw, gs, P, P, P, P, y, kept, kept, kept, kept, saved, T, d, h,
                                               ws, nb, None)

    assert fwd(T=0) == OK and fwd(d=0) == BAD and fwd(h=0) == BAD and fwd(xt=0) == BAD and fwd(T=-1) == BAD
    assert fwd(x=None) == BAD and fwd(gw=None) == BAD and fwd(y=None) == BAD and fwd(xt=2, xs=None) == BAD
    assert fwd(x=P + 8) == BAD and fwd(gw=P + 8) == BAD and fwd(gs=P + 2) == BAD
    assert fwd(nb=need[0] - 1) == BAD and fwd(ws=P + 16) == BAD
    assert fwd(saved=P, kept=None, nb=need[1]) == BAD and fwd(saved=P + 8, nb=need[1]) == BAD
    assert lib.smaul_fp8_block_ffn_workspace_size(4, 64, 96, 0, 0) == -1
    assert lib.smaul_fp8_block_ffn_saved_size(4, 0) == -1 and lib.smaul_fp8_block_ffn_saved_size(4, 96) > 0
    assert lib.smaul_fp8_block_ffn_backward_workspace_size(-1, 64, 96) == -1
    need = lib.smaul_fp8_block_ffn_backward_workspace_size(70, 64, 96)

    def bwd(dy=P, gw=P, kept=P, dx=P, dg=P, du=P, dd=P, T=70, d=64, h=96, ws=P, nb=need):
        return lib.smaul_fp8_block_ffn_backward(dy, gw, P, P, P, P, P, P, P, P, P, kept, dx, dg, du, dd, T, d, h, ws, nb,
                                                None)

    assert bwd(dg=None) == BAD and bwd(dd=None) == BAD and bwd(d=0) == BAD
    assert bwd(dx=None, dg=None, du=None, dd=None) == OK and bwd(T=0, dg=None, du=None, dd=None) == OK
    assert bwd(dy=None) == BAD and bwd(kept=None) == BAD and bwd(dx=P + 2) == BAD and bwd(gw=P + 4) == BAD
    assert bwd(nb=need - 1) == BAD and bwd(ws=P + 64) == BAD


def test_block_backward_workspace_of_what_is_asked_for():
    lib = _lib.load()
    size = lib.smaul_fp8_block_ffn_backward_part_workspace_size
    assert size(-1, 64, 96, 1, 1) == size(70, 0, 96, 1, 1) == size(70, 64, 0, 1, 1) == -1
    for T, d, h in ((70, 64, 96), (300, 130, 1000)):
        every = lib.smaul_fp8_block_ffn_backward_workspace_size(T, d, h)
        need = {(dx, dw): size(T, d, h, dx, dw) for dx in (0, 1) for dw in (0, 1)}
        assert need[1, 1] == every and need[1, 0] < every and need[0, 1] < every
        # dx alone: no copy of x's, dy's, h's rows, dg or du turned round
        assert need[1, 0] <= every - 2 * T * (2 * d + 3 * h)
        for dx, dw in ((1, 0), (0, 1), (1, 1)):
            w = P if dw else None
            assert lib.smaul_fp8_block_ffn_backward(P, P, P, P, P, P, P, *[w] * 4, P, P if dx else None, w, w, w, T, d, h, P,
                                                    need[dx, dw] - 1, None) == BAD


def test_norm_arguments():
    lib = _lib.load()

    def fwd(x=P, r=P, t=1, eps=1e-6, s=P, o=P, sc=P, T=4, d=64):
        return lib.smaul_add_rms_norm(x, r, t, P, eps, s, o, sc, T, d, None)

    assert fwd(T=0) == OK and fwd(t=2) == BAD and fwd(d=0) == BAD and fwd(T=-1) == BAD
    assert fwd(eps=0.0) == BAD and fwd(eps=float("inf")) == BAD and fwd(eps=float("nan")) == BAD
    assert fwd(x=None) == BAD and fwd(s=None) == BAD and fwd(o=None) == BAD and fwd(o=P + 4) == BAD
    assert fwd(T=1 << 40) == NO
    assert lib.smaul_add_rms_norm_backward_workspace_size(4, 0) == -1
    need = lib.smaul_add_rms_norm_backward_workspace_size(40, 64)

    def bwd(dy=P, s=P, t=1, eps=1e-6, dx=P, dw=P, T=40, d=64, ws=P, nb=need):
        return lib.smaul_add_rms_norm_backward(dy, s, None, t, P, eps, dx, dw, T, d, ws, nb, None)

    assert bwd(t=2) == BAD and bwd(d=0) == BAD and bwd(eps=-1.0) == BAD and bwd(dy=None) == BAD and bwd(dx=None) == BAD
    assert bwd(nb=need - 1) == BAD and bwd(ws=P + 4) == BAD and bwd(T=0, dw=None) == OK


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [1, 127, 128, 129, 513, 700])
def test_host_quantizer_is_the_definition(K, dtype):
    g = torch.Generator().manual_seed(K)
    x = (torch.randn(9, K, generator=g) * torch.exp(4 * torch.randn(9, 1, generator=g))).to(dtype)
    x[1] = 0
    codes, scales = fp8_block.quantize(x)
    want = ref.quantize(x)
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    assert torch.equal(fp8_block.decode(codes, scales, K).double(), ref.values(*want, K))
    x[0, K // 2], x[2, 0] = float("nan"), float("-inf")
    codes, scales = fp8_block.quantize(x)
    want = ref.quantize(x)
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])


def test_layers_refuse_and_hold():
    for bad in (lambda: FP8BlockLinear(0, 4), lambda: FP8BlockFFN(4, 0), lambda: AddRMSNorm(0),
                lambda: AddRMSNorm(4, 0.0), lambda: FP8BlockNormFFN(4, 4, eps=float("nan")),
                lambda: fp8_block.quantize(torch.zeros(3, 0)), lambda: fp8_block.quantize(torch.zeros(3, 4).long())):
        with pytest.raises(ValueError):
            bad()
    m = FP8BlockFFN(130, 200)
    assert not list(m.parameters()) and m.gate_w.shape == (200, 256) and m.down_s.shape == (130, 4)
    t = FP8BlockNormFFN(130, 200, trainable=True)
    assert {n for n, _ in t.named_parameters()} == {"gate", "up", "down", "norm"}
    assert FP8BlockLinear(5, 7, bias=True).state_dict().keys() == {"w8", "ws", "bias"}


def test_gradient_formulas_against_autograd():
    """The plain forms that the device is held to, against autograd in 64 bits with the roundings
    held (up to what 64 bits lose, 1e-12 of the largest)."""
    g = torch.Generator().manual_seed(0)
    T, d, h = 6, 40, 24
    x, dy = (torch.randn(T, d, generator=g, dtype=torch.float64) for _ in range(2))
    ws = [ref.rounded(torch.randn(n, k, generator=g)) for n, k in ((h, d), (h, d), (d, h))]
    want = ref.ffn_grad(x, dy, *ws, 0.0)
    leaves = [t.clone().requires_grad_() for t in (x, *ws)]
    v = ref.silu(leaves[0] @ leaves[1].t()) * (leaves[0] @ leaves[2].t())
    hid = v + (ref.rounded(v.detach()) - v.detach())
    grads = torch.autograd.grad((hid @ leaves[3].t() * dy).sum(), leaves)
    for name, got in zip(("dx", "dgate", "dup", "ddown"), grads):
        assert float((want[name][0] - got).abs().max()) <= 1e-12 * float(got.abs().max())
    s, w = (torch.randn(*n, generator=g, dtype=torch.float64).requires_grad_() for n in ((T, d), (d,)))
    ds = torch.randn(T, d, generator=g, dtype=torch.float64)
    grads = torch.autograd.grad((ref.norm(s, w, 1e-6)[0] * dy).sum() + (s * ds).sum(), (s, w))
    got = ref.norm_grad(dy, s.detach(), w.detach(), 1e-6, ds, torch.float32)
    for (v, _), want in zip(got, grads):
        assert float((v - want).abs().max()) <= 1e-12 * float(want.abs().max())
