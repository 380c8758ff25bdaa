"""Routing among experts that tie, or nearly: padding, equal logits beside others a bit away."""
import pytest
import torch

import _mx4 as ref
from smaulnative_amd.compute import get_backend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF = torch.float32, torch.bfloat16


def _check(z, k, score, bias, groups, top_groups, best):
    _, topi, topw = get_backend("rocm").moe_route(z.to(DEV), k, score=score, groups=groups, top_groups=top_groups,
                                                  group_best=best, bias=None if bias is None else bias.to(DEV))
    _, ti, tw = ref.route(z, k, score, bias, groups, top_groups, best, True, 1.0)
    assert torch.equal(topi.cpu(), ti)
    # a score is off by the roundings of a sum of E / 16 + 4 and 12 more, a weight by three of those
    assert ((topw.cpu().double() - tw).abs() <= 3 * (z.shape[1] / 16 + 16) * 2.0 ** -24 * tw + 1e-37).all()


@pytest.mark.parametrize("E,k,groups,top_groups", [(12, 3, 1, 1), (64, 8, 1, 1), (64, 6, 8, 4), (120, 16, 1, 1),
                                                   (256, 8, 8, 3), (60, 4, 5, 2), (320, 8, 1, 1), (512, 10, 64, 9)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [None, "zero", "own"])
def test_padding_among_tokens(E, k, groups, top_groups, score, biased):
    gen = torch.Generator().manual_seed(E + k)
    bias = None if biased is None else torch.zeros(E) if biased == "zero" else torch.randn(E, generator=gen) * 0.05
    for dtype in (F32, BF):
        z = (torch.randn(41, E, generator=gen) * 0.64).to(dtype)
        z[5:9], z[17], z[39:] = 0.0, 1.25, -0.0
        _check(z, k, score, bias, groups, top_groups, 1 + E % 2)


@pytest.mark.parametrize("E,k", [(48, 4), (128, 8), (256, 16)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_equal_experts_beside_near_ones(E, k, score, biased):
    """More than k of one logit, among them some a step or a few above and below it."""
    gen = torch.Generator().manual_seed(E * k)
    z = torch.randn(48, E, generator=gen) * 0.3 - 2.0
    for t in range(z.shape[0]):
        n = int(torch.randint(2, 2 * k + 2, (1,), generator=gen))
        at = torch.randperm(E, generator=gen)[:n]
        z[t, at] = 1.0 + t / 16
        for e in at[:n // 3].tolist():
            steps = int(torch.randint(-4, 5, (1,), generator=gen))
            z[t, e] = (z[t, e].view(torch.int32) + steps).view(torch.float32)
    _check(z, k, score, torch.zeros(E) if biased else None, 1, 1, 2)
