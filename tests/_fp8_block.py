"""Plain 64-bit forms of the 8-bit feed-forward path, for the tests (host tensors)."""
import math

import torch

U = 2.0 ** -24  # half a step of fp32, relative
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
# what the codes 0 to 126 stand for, ascending; 127 is NaN
GRID = torch.tensor([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127],
                    dtype=torch.float64)


def blocks(K):
    return -(-K // 128)


def quantize(x):
    """(codes [..., 128 n], scales [..., 4 ceil(n / 4)]) of x [..., K], by the definition."""
    K, n = x.shape[-1], blocks(x.shape[-1])
    b = torch.zeros(*x.shape[:-1], n * 128, dtype=torch.float64)
    b[..., :K] = x.double()
    b = b.view(*x.shape[:-1], n, 128)
    bad = ~torch.isfinite(b).all(-1)
    amax = torch.where(bad, torch.ones((), dtype=torch.float64), b.abs().amax(-1))
    scale = torch.zeros(amax.shape, dtype=torch.int64)
    for byte in range(254):  # the least that does not pass 448
        scale = torch.where((scale == byte) & (amax > 448 * 2.0 ** (byte - 127)), byte + 1, scale)
    a = b.abs() * torch.pow(2.0, 127 - scale.double()).unsqueeze(-1)
    a = torch.where(bad.unsqueeze(-1), torch.zeros_like(a), a)
    up = torch.searchsorted(GRID, a.contiguous()).clamp(max=126)  # the first code at or above
    lo = (up - 1).clamp_min(0)
    dlo, dup = a - GRID[lo], GRID[up] - a
    code = torch.where((dlo < dup) | ((dlo == dup) & (lo % 2 == 0)), lo, up)
    code = code + 128 * torch.signbit(b).long()
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code)
    scale = torch.where(bad, torch.full_like(scale, 255), scale)
    return (code.view(*x.shape[:-1], n * 128).to(torch.uint8),
            torch.nn.functional.pad(scale, (0, -n % 4)).to(torch.uint8))


def values(codes, scales, K):
    """What codes stand for, float64 [..., K]."""
    n = codes.shape[-1] // 128
    c = codes.long().view(*codes.shape[:-1], n, 128)
    v = torch.cat([GRID, torch.tensor([math.nan], dtype=torch.float64)])[c & 127]
    v = torch.where(c >= 128, -v, v)
    s = scales[..., :n].double()
    unit = torch.where(s == 255, torch.full_like(s, math.nan), torch.pow(2.0, s - 127))
    return (v * unit.unsqueeze(-1)).reshape(codes.shape)[..., :K]


def rounded(x):
    return values(*quantize(x), x.shape[-1])


def moved(v, err):
    """How far codes of values within err of v may stand from v's: each value up or down by
    its error, and in or out (a block's largest value may take another scale)."""
    mid, out = rounded(v), torch.sign(v) * err
    return torch.stack([(rounded(w) - mid).abs() for w in (v - err, v + err, v - out, v + out)]).amax(0)


def weight(out_f, in_f, gen, std=0.05):
    return quantize(torch.randn(out_f, in_f, generator=gen) * std)


def _tops(x):
    """The largest magnitude of each 8 neighbouring values of a row, [..., K / 8]."""
    x = torch.nn.functional.pad(x.abs(), (0, -x.shape[-1] % 8))
    return x.view(*x.shape[:-1], -1, 8).amax(-1)


def aligned(x, w):
    """What an 8-bit matrix instruction may lose of x w^T: 8 neighbouring products are summed
    with the last bit 2^-13 of the largest's power of two (measured on the device: a product
    2^-13 of its neighbour counts, one of 2^-14 does not), so up to 7 of them lose less than
    2^-13 of the largest each."""
    return 7 * 2.0 ** -13 * (_tops(x) @ _tops(w).t())


def product(x, w, dtype, codes=False):
    """(y, bound) of x w^T: products exact, sums fp32 over whole blocks, y rounded once;
    ``codes``: bf16 results of the 8-bit instructions."""
    y = x @ w.t()
    err = 128 * blocks(x.shape[-1]) * U * (x.abs() @ w.abs().t())
    if codes and dtype == torch.bfloat16:
        err = err + aligned(x, w)
    return y, err + HALF[dtype] * (y.abs() + err) + 1e-44


def norm(s, weight, eps):
    """(y, bound) before y's own rounding: a sum of d squares, a root, a division and two products in fp32."""
    d = s.shape[-1]
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps) * weight
    return y, (d / 2 + 8) * U * y.abs()


def norm_grad(dy, s, weight, eps, ds, dtype):
    """((dx, bound), (dw, bound)): dx from two sums of d terms, dw one of T."""
    T, d = s.shape
    r = 1 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    wg = weight * dy
    dot = (wg * s).mean(-1, keepdim=True) * r * r
    dx = (wg - s * dot) * r
    dot_abs = (wg * s).abs().mean(-1, keepdim=True) * r * r
    err = r * (wg.abs() * (d / 2 + 8) + s.abs() * dot_abs * (2 * d + 16) + (s * dot).abs() * (d / 2 + 8)) * U
    if ds is not None:
        dx = dx + ds
        err = err + dx.abs() * U
    terms = dy * s * r
    return (dx, err + HALF[dtype] * (dx.abs() + err) + 1e-44), \
        (terms.sum(0), terms.abs().sum(0) * (T + d / 2 + 8) * U + 1e-44)


def silu(g):
    return g * torch.sigmoid(g)


def ffn(x, gate, up, down, exact=False):
    """(y, bound, g, u, h, bound of h's values): hidden rows rounded from fp32, y to bf16.
    ``exact``: hidden rows of exact products (few of them), else of the 8-bit instructions."""
    g, u = x @ gate.t(), x @ up.t()
    rel = 128 * blocks(x.shape[-1]) * U
    ge, ue = (x.abs() @ w.abs().t() * rel + (0 if exact else aligned(x, w)) for w in (gate, up))
    v = silu(g) * u
    # |silu'| <= 1.1, |silu(g)| <= |g|; 2^-19 for the product's own arithmetic
    ve = 1.1 * ge * (u.abs() + ue) + g.abs() * ue + 2.0 ** -19 * v.abs()
    h, he = rounded(v), moved(v, ve)
    y = h @ down.t()
    ye = he @ down.abs().t() + 128 * blocks(h.shape[-1]) * U * ((h.abs() + he) @ down.abs().t()) + aligned(h.abs() + he, down)
    return y, ye + HALF[torch.bfloat16] * (y.abs() + ye), g, u, h, he, ge, ue


def ffn_grad(x, dy, gate, up, down, kept, exact=False):
    """{name: (gradient, bound)} of the block; ``kept``: how far what the forward pass keeps of
    u silu'(g) and silu(g) is rounded, relative.  dg and du are rounded to bf16."""
    y, ye, g, u, h, he, ge, ue = ffn(x, gate, up, down, exact)
    d, n, T = x.shape[-1], gate.shape[0], x.shape[0]
    half = HALF[torch.bfloat16]
    sig = torch.sigmoid(g)
    a, b = u * sig * (1 + g * (1 - sig)), g * sig
    # |silu''| <= 0.5
    ae = ue * 1.1 + (u.abs() + ue) * 0.5 * ge + (2.0 ** -19 + kept) * (u.abs() * 1.1)
    be = 1.1 * ge + (2.0 ** -19 + kept) * b.abs()
    dh = dy @ down
    dhe = (d + 128) * U * (dy.abs() @ down.abs())
    dg, du = dh * a, dh * b
    dge = dhe * (a.abs() + ae) + dh.abs() * ae
    due = dhe * (b.abs() + be) + dh.abs() * be
    dge, due = dge + half * (dg.abs() + dge), due + half * (du.abs() + due)

    def out(v, e):
        return v, e + half * (v.abs() + e) + 1e-44

    sums = 2 * (n + 128) * U
    dx = out(dg @ gate + du @ up, dge @ gate.abs() + due @ up.abs() +
             sums * ((dg.abs() + dge) @ gate.abs() + (du.abs() + due) @ up.abs()))
    sums = (T + 128) * U
    return {"y": (y, ye), "dx": dx,
            "dgate": out(dg.t() @ x, dge.t() @ x.abs() + sums * ((dg.abs() + dge).t() @ x.abs())),
            "dup": out(du.t() @ x, due.t() @ x.abs() + sums * ((du.abs() + due).t() @ x.abs())),
            "ddown": out(dy.t() @ h, dy.abs().t() @ he + sums * (dy.abs().t() @ (h.abs() + he)))}


def check(got, want, bound, what=""):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    assert bool((off <= bound).all()), (what, float((off - bound).max()), float((off / bound).max()))
