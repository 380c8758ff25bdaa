"""CPU checks of the routing's and the 4-bit products' entry points: what they refuse,
before anything reaches a device."""
import pytest
import torch

from smaulnative_amd import _lib
from smaulnative_amd.compute import get_backend

P = 4096  # a pointer that is only looked at


def test_host_tensors_are_refused():
    be = get_backend("rocm")
    z = torch.zeros(3, 8)
    topi, topw = torch.zeros(3, 2, dtype=torch.int64), torch.ones(3, 2)
    w, s = torch.zeros(8, 16, dtype=torch.uint8), torch.zeros(8, 1, dtype=torch.uint8)
    calls = (lambda: be.moe_route(z, 2), lambda: be.moe_route_backward(topw, z, topi), lambda: be.mx4_quantize(z),
             lambda: be.mx4_dequantize(w, s, 8), lambda: be.mx4_forward(z, w, s, 8, 8),
             lambda: be.mx4_backward_input(z, w, s, 8, 8),
             lambda: be.mx4_moe_forward(z, topi, topw, (w[None], s[None]) * 3))
    for call in calls:
        with pytest.raises(RuntimeError, match="HIP device tensors"):
            call()


@pytest.mark.parametrize("T,E,k,score,groups,top,best,rc", [
    (4, 0, 1, 0, 1, 1, 2, _lib.SMAUL_ERR_INVALID), (4, 8, 9, 0, 1, 1, 2, _lib.SMAUL_ERR_INVALID),
    (-1, 8, 2, 0, 1, 1, 2, _lib.SMAUL_ERR_INVALID), (4, 8, 2, 2, 1, 1, 2, _lib.SMAUL_ERR_INVALID),
    (4, 8, 2, 0, 3, 1, 2, _lib.SMAUL_ERR_INVALID), (4, 8, 3, 0, 4, 1, 2, _lib.SMAUL_ERR_INVALID),
    (4, 8, 2, 0, 4, 5, 2, _lib.SMAUL_ERR_INVALID), (4, 8, 2, 0, 4, 2, 0, _lib.SMAUL_ERR_INVALID),
    (4, 1024, 2, 0, 1, 1, 2, _lib.SMAUL_ERR_UNSUPPORTED), (4, 64, 17, 0, 1, 1, 2, _lib.SMAUL_ERR_UNSUPPORTED),
    (4, 256, 2, 0, 128, 8, 2, _lib.SMAUL_ERR_UNSUPPORTED), ((1 << 31) + 1, 8, 2, 0, 1, 1, 2, _lib.SMAUL_ERR_UNSUPPORTED),
    (0, 8, 2, 0, 1, 1, 2, _lib.SMAUL_OK), (4, 8, 2, 0, 1, 1, 2, _lib.SMAUL_ERR_INVALID)])
def test_route_arguments(T, E, k, score, groups, top, best, rc):
    lib = _lib.load()
    assert lib.smaul_moe_route(None, 0, None, None, None, None, T, E, k, score, groups, top, best, 1, 1.0, None) == rc
    if groups == 1:
        assert lib.smaul_moe_route_backward(None, None, 0, None, None, None, T, E, k, score, 1, 1.0, None) == rc
    assert lib.smaul_moe_route(P, 5, None, None, P, P, 4, 8, 2, 0, 1, 1, 2, 1, 1.0, None) == _lib.SMAUL_ERR_INVALID


def test_mx4_arguments():
    lib = _lib.load()
    bad, no = _lib.SMAUL_ERR_INVALID, _lib.SMAUL_ERR_UNSUPPORTED
    assert lib.smaul_mx4_quantize(None, 0, None, None, 4, 32, None) == bad
    assert lib.smaul_mx4_quantize(P, 3, P, P, 4, 32, None) == bad
    assert lib.smaul_mx4_quantize(P, 0, P, P, 4, 0, None) == bad
    assert lib.smaul_mx4_quantize(P, 0, P + 2, P, 4, 32, None) == bad
    assert lib.smaul_mx4_quantize(P, 0, P, P, 0, 32, None) == _lib.SMAUL_OK
    assert lib.smaul_mx4_dequantize(P, P, None, 0, 4, 32, None) == bad
    assert lib.smaul_mx4_dequantize(P + 1, P, P, 0, 4, 32, None) == bad
    for act in (0, 1):
        need = lib.smaul_mx4_linear_workspace_size(100, 64, 32, 1, act)
        assert need >= (100 * 2 * 17 if act else 0)
        assert lib.smaul_mx4_linear(P, 1, P, P, P, 100, 64, 32, act, None, max(need, 1) - 1, None) == bad or need == 0
        assert lib.smaul_mx4_linear(P, 1, P + 4, P, P, 100, 64, 32, act, P, need, None) == bad
        assert lib.smaul_mx4_linear(P, 1, P, P, P, 0, 64, 32, act, None, 0, None) == _lib.SMAUL_OK
    assert lib.smaul_mx4_linear(P, 1, P, P, P, 100, 64, 32, 2, P, 1 << 20, None) == bad
    assert lib.smaul_mx4_linear(P, 1, P, P, P, 100, 0, 32, 0, None, 0, None) == bad
    assert lib.smaul_mx4_linear_workspace_size(-1, 64, 32, 1, 1) == -1
    assert lib.smaul_mx4_backward_input(P, 0, P, P, None, 4, 64, 32, P, 1 << 20, None) == bad
    assert lib.smaul_mx4_backward_input(P, 0, P + 8, P, P, 4, 64, 32, P, 1 << 20, None) == bad
    assert lib.smaul_mx4_backward_input(P + 4, 0, P, P, P, 4, 64, 32, P, 1 << 20, None) == bad
    need = lib.smaul_mx4_backward_input_workspace_size(100, 64, 32, 0)
    assert need > 0 and lib.smaul_mx4_backward_input_workspace_size(100, 0, 32, 0) == -1
    assert lib.smaul_mx4_backward_input(P, 0, P, P, P, 100, 64, 32, P, need - 1, None) == bad
    assert lib.smaul_mx4_backward_input(P, 0, P, P, P, 100, 64, 32, P + 16, need, None) == bad
    assert lib.smaul_mx4_linear(P + 4, 1, P, P, P, 10, 64, 32, 0, None, 0, None) == bad
    size = lib.smaul_mx4_moe_workspace_size(64, 128, 256, 8, 2, 1, 1)
    assert size > 0 and lib.smaul_mx4_moe_workspace_size(64, 128, 0, 8, 2, 1, 1) == -1

    def moe(dtype=1, T=64, d=128, h=256, E=8, k=2, act=1, ws=P, bytes_=size, gate=P):
        return lib.smaul_mx4_moe_forward(P, dtype, P, P, gate, P, P, P, P, P, P, P, T, d, h, E, k, act, ws, bytes_, None)

    assert moe(E=65) == bad and moe(k=9) == bad and moe(k=0) == bad and moe(act=3) == bad
    assert moe(d=124) == no and moe(dtype=0) == no and moe(T=1 << 40) == no
    assert moe(bytes_=size - 1) == bad and moe(ws=None) == bad and moe(ws=P + 16) == bad and moe(gate=P + 2) == bad
    assert moe(T=0) == _lib.SMAUL_OK


def test_calls_past_a_launch_are_refused():
    """A launch counts its work-items in 32 bits, and runs what is left of a division by
    2^32 of a larger grid without a word: refused before anything is launched."""
    lib = _lib.load()
    bad, no = _lib.SMAUL_ERR_INVALID, _lib.SMAUL_ERR_UNSUPPORTED
    for T, rc in (((1 << 28) - 16, bad), (1 << 28, no), (1 << 30, no)):  # bad: null pointers are looked at next
        assert lib.smaul_moe_route(None, 0, None, None, None, None, T, 4, 2, 0, 1, 1, 2, 1, 1.0, None) == rc
        assert lib.smaul_moe_route_backward(None, None, 0, None, None, None, T, 4, 2, 0, 1, 1.0, None) == rc
    assert lib.smaul_mx4_quantize(P, 1, P, P, 1 << 32, 32, None) == no
    assert lib.smaul_mx4_dequantize(P, P, P, 1, 1 << 32, 32, None) == no
    for rows, K, N in ((1 << 27, 1, 1), (1 << 30, 1, 1), (1 << 22, 8200, 8), (100, 1 << 20, 1 << 20)):
        for act in (0, 1):
            need = lib.smaul_mx4_linear_workspace_size(rows, K, N, 1, act)
            assert lib.smaul_mx4_linear(P, 1, P, P, P, rows, K, N, act, P, need, None) == no
    for rows, K, N in ((100, 1 << 19, 1 << 17), (1 << 27, 1, 3)):
        need = lib.smaul_mx4_backward_input_workspace_size(rows, K, N, 1)
        assert lib.smaul_mx4_backward_input(P, 1, P, P, P, rows, K, N, P, need, None) == no
    assert lib.smaul_mx4_backward_input(P, 1, P, P, P, 4, 1 << 29, 8, P, 0, None) == no
    assert lib.smaul_mx4_linear(P, 1, P, P, P, 4, 8, 1 << 29, 0, None, 0, None) == no
