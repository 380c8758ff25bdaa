"""Plain 64-bit forms of the routing and of the 4-bit format, for the tests (host tensors)."""
import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
# the borders between neighbours; a value on one goes to the even code
BORDERS = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))


def blocks(K):
    return -(-K // 32)


def quantize(x):
    """(codes [..., 16 n], scales [..., n]) of x [..., K], by the definition."""
    K, n = x.shape[-1], blocks(x.shape[-1])
    b = torch.zeros(*x.shape[:-1], n * 32, dtype=torch.float64)
    b[..., :K] = x.double()
    b = b.view(*x.shape[:-1], n, 32)
    amax = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    safe = torch.where(bad | (amax == 0), torch.ones_like(amax), amax)
    e = torch.frexp(safe).exponent - 1 - 2
    e = torch.where(amax == 0, torch.full_like(e, -127), e).clamp(-127, 125)
    a = b.abs() * torch.pow(2.0, -e.double()).unsqueeze(-1)
    code = torch.zeros(b.shape, dtype=torch.int64)
    for border, up in BORDERS:
        code += ((a >= border) if up else (a > border)).long()
    code += 8 * torch.signbit(b).long()
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).view(*x.shape[:-1], n * 16, 2)
    scale = torch.where(bad, torch.full_like(e, 255), e + 127)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), scale.to(torch.uint8)


def values(codes, scales, K):
    """What codes stand for, float64 [..., K]."""
    nib = torch.stack([codes & 15, codes >> 4], -1).long().view(*scales.shape, 32)
    v = GRID[nib & 7] * torch.where(nib >= 8, -1.0, 1.0).double()
    unit = torch.where(scales == 255, torch.full(scales.shape, math.nan, dtype=torch.float64),
                       torch.pow(2.0, scales.double() - 127))
    return (v * unit.unsqueeze(-1)).reshape(*scales.shape[:-1], -1)[..., :K]


def rounded(x):
    return values(*quantize(x), x.shape[-1])


def weight(out_f, in_f, gen, std=0.02):
    return quantize(torch.randn(out_f, in_f, generator=gen) * std)


def scores(z, score):
    return torch.softmax(z, -1) if score == "softmax" else torch.sigmoid(z)


def route(logits, k, score, bias, groups, top_groups, group_best, renorm, scale):
    """(prob, topi, topw) float64 / int64, a token at a time."""
    z = logits.double()
    s = scores(z, score)
    T, E = z.shape
    per = E // groups
    topi = torch.full((T, k), -1, dtype=torch.int64)
    topw = torch.zeros(T, k, dtype=torch.float64)
    for t in range(T):
        c = [float(s[t, e]) + (float(bias[e]) if bias is not None else 0.0) for e in range(E)]
        live = [e for e in range(E) if float(z[t, e]) > -math.inf and c[e] > -math.inf]
        if top_groups < groups:
            rank = []
            for g in range(groups):
                best = sorted((c[e] for e in live if e // per == g), reverse=True)[:group_best]
                rank.append((-sum(best) if best else math.inf, g))
            kept = {g for _, g in sorted(rank)[:top_groups]}
            live = [e for e in live if e // per in kept]
        key = (lambda e: (-float(z[t, e]), e)) if bias is None else (lambda e: (-c[e], e))
        chosen = sorted(live, key=key)[:k]
        w = [float(s[t, e]) for e in chosen]
        if renorm and chosen:
            w = [1.0 / len(w)] * len(w) if sum(w) < 1e-6 else [v / sum(w) for v in w]
        for j, e in enumerate(chosen):
            topi[t, j], topw[t, j] = e, w[j] * scale
    return s, topi, topw


def route_loss(logits, topi, dtopw, dprob, score, renorm, scale):
    """sum(topw * dtopw) + sum(prob * dprob) as a function of the logits (float64, differentiable)."""
    s = scores(logits, score)
    has = topi >= 0
    w = torch.where(has, s.gather(1, topi.clamp_min(0)), torch.zeros((), dtype=s.dtype))
    if renorm:
        total = w.sum(1, keepdim=True)
        even = has.double() / has.sum(1, keepdim=True).clamp_min(1)
        w = torch.where(total < 1e-6, even, w / total.clamp_min(1e-9))
    loss = torch.where(has, w * scale * dtopw, torch.zeros_like(w)).sum()
    return loss if dprob is None else loss + (s * dprob).sum()


def swiglu(g, u):
    return g * torch.sigmoid(g) * u


def moe(x, topi, topw, experts, act):
    """(out, bound): the routed experts in float64 and how far an element may be off.

    The bound adds up, per slot and with absolute values through the products:
    - keep: the rounding of the hidden rows to x's type (half a step each; fp32 rows
      go on as two bf16 terms, 2^-17), of x likewise in fp32, and 2^-19 of the
      SwiGLU product's own arithmetic;
    - mx4: where the error of the fp32 hidden values changes a code, the whole step;
    - the fp32 sums, K 2^-24 of the terms' magnitudes (K of the products' lengths);
    - the rounding of the slot's output to x's type, and of the sum.
    """
    d = x.shape[-1]
    E, h = experts[0].shape[:2]
    bf16 = x.dtype == torch.bfloat16
    half = 2.0 ** -8 if bf16 else 2.0 ** -24
    xv = rounded(x) if act == "mx4" else x.double()
    xe = 0.0 if bf16 else 2.0 ** -17
    out = torch.zeros(x.shape, dtype=torch.float64)
    bound = torch.zeros(x.shape, dtype=torch.float64)
    counts = torch.zeros(E, dtype=torch.int32)
    for e in range(E):
        tok, slot = ((topi == e) & (topw > 0)).nonzero(as_tuple=True)
        counts[e] = tok.numel()
        if not tok.numel():
            continue
        wg, wu, wd = (values(experts[i][e], experts[i + 1][e], n) for i, n in ((0, d), (2, d), (4, h)))
        xt = xv[tok]
        g, u = xt @ wg.t(), xt @ wu.t()
        rel = xe + d * 2.0 ** -24
        ge, ue = xt.abs() @ wg.abs().t() * rel, xt.abs() @ wu.abs().t() * rel
        hid = swiglu(g, u)
        # |d silu| <= 1.1, |silu(g)| <= |g|
        he = 1.1 * ge * (u.abs() + ue) + g.abs() * ue + 2.0 ** -19 * hid.abs()
        if act == "mx4":
            # every value up or down by its error, and in or out (a block's largest value)
            mid, out_ = rounded(hid), torch.sign(hid) * he
            moved = [rounded(v) for v in (hid - he, hid + he, hid - out_, hid + out_)]
            he = torch.stack([(v - mid).abs() for v in moved]).amax(0)
            hid = mid
        else:
            he = he + hid.abs() * (half if bf16 else 2.0 ** -17)
        y = hid @ wd.t()
        ye = he @ wd.abs().t() + h * 2.0 ** -24 * (hid.abs() @ wd.abs().t())
        ye = ye + half * (y.abs() + ye)
        w = topw[tok, slot].double().unsqueeze(1)
        out[tok] += y * w
        bound[tok] += ye * w + 2.0 ** -23 * (y * w).abs()
    return out, bound + half * (out.abs() + bound) + 1e-30, counts
