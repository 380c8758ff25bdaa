"""The routing and the 4-bit products of a mixture-of-experts layer, as measurable cases.

Each case is one pass through an operator.  With ``own`` false ``run`` computes
it in elementary tensor operations, otherwise through ``RocmBackend``:

- ``route``: scores of every expert (softmax or sigmoid), a balance bias, groups,
  top-k and renormalised weights (``moe_route``);
- ``route_grad``: the logits' gradient from those of the weights and the scores
  (``moe_route_backward``);
- ``quant``: rows rounded to blocks of 32 4-bit floating point values with a
  shared power of two, and the values they stand for (``mx4_quantize``,
  ``mx4_dequantize``);
- ``linear``: the product with such a weight, the activations as they are or
  rounded to the format too (``mx4_forward``);
- ``dx``: the input gradient of that product (``mx4_backward_input``);
- ``moe``: the routed SwiGLU experts in the format (``mx4_moe_forward``).
"""
import math

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # what the codes 0 to 7 stand for; +8 is the sign


def listed():
    return [
        # a decode step of 64 sequences, routed the balanced way: 64 experts in 8 groups, 4 of them, 6 experts
        dict(name="route_step_64", kind="route", T=64, E=64, k=6, score="sigmoid", groups=8, top_groups=4, best=2,
             bias=True, renorm=True, scale=2.5, dtype="f32", prob=False),
        # a prefill of 65536 tokens over 256 experts in 8 groups, the scores kept for the usage reports
        dict(name="route_prefill_64k", kind="route", T=65536, E=256, k=8, score="sigmoid", groups=8, top_groups=4,
             best=2, bias=True, renorm=True, scale=2.5, dtype="f32", prob=True),
        # training: 16384 tokens, 64 experts, softmax top-8 renormalised, with the balance loss's gradient of the scores
        dict(name="route_grad_softmax_16k", kind="route_grad", T=16384, E=64, k=8, score="softmax", renorm=True,
             scale=1.0, dtype="f32", prob=True),
        # training a short ragged batch with sigmoid scores over 60 experts
        dict(name="route_grad_sigmoid_odd", kind="route_grad", T=4099, E=60, k=6, score="sigmoid", renorm=True,
             scale=2.5, dtype="f32", prob=False),
        # the hidden rows of a long prefill (65536 tokens, d = 2048) rounded to the format
        dict(name="quant_rows_64k_bf16", kind="quant", rows=65536, K=2048, dtype="bf16"),
        # one weight of an odd width, from fp32
        dict(name="quant_weight_odd_f32", kind="quant", rows=2560, K=1000, dtype="f32"),
        # one token through a projection, bf16 activations as they are: the weight's bytes and the launch
        dict(name="linear_token_bf16", kind="linear", rows=1, K=1024, N=2560, act="keep", dtype="bf16"),
        # a prefill through the same projection, activations rounded to the format
        dict(name="linear_prefill_mx4", kind="linear", rows=16384, K=1024, N=2560, act="mx4", dtype="bf16"),
        # training through a frozen projection: 4096 rows
        dict(name="dx_4096_bf16", kind="dx", rows=4096, K=1024, N=2560, dtype="bf16"),
        # the same with fp32 gradients, ragged rows and widths
        dict(name="dx_odd_f32", kind="dx", rows=1001, K=1000, N=777, dtype="f32"),
        # a decode step of 64 sequences through eight experts, top-2
        dict(name="moe_decode_64_bf16", kind="moe", T=64, d=1024, h=2560, E=8, k=2, act="keep", dtype="bf16"),
        # a prefill of 16384 tokens through the same layer, activations and hidden rows rounded to the format
        dict(name="moe_prefill_16k_mx4", kind="moe", T=16384, d=1024, h=2560, E=8, k=2, act="mx4", dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "route_grad", "quant", "linear", "dx", "moe"])
    dtype = rng.choice(["f32", "bf16"])
    if kind in ("route", "route_grad"):
        groups = rng.choice([1, 1, 2, 4, 8])
        per = _spread(rng, 4, 256 // groups)
        E = groups * per
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(8, per * top_groups))
        T = min(_spread(rng, 1, 65536), (65536 * 256) // E)
        c = dict(kind=kind, T=T, E=E, k=k, score=rng.choice(["softmax", "sigmoid"]),
                 renorm=rng.random() < 0.7 if kind == "route" else k > 1, scale=rng.choice([1.0, 2.5]), dtype=dtype,
                 prob=rng.random() < 0.5)
        if kind == "route":
            c.update(groups=groups, top_groups=top_groups, best=rng.randint(1, 2), bias=rng.random() < 0.6)
        return c
    if kind == "quant":
        K = _spread(rng, 32, 8192)
        return dict(kind=kind, rows=min(_spread(rng, 1, 65536), 65536 * 2048 // K), K=K, dtype=dtype)
    if kind in ("linear", "dx"):
        K, N = _spread(rng, 64, 4096), _spread(rng, 64, 4096)
        rows = min(_spread(rng, 1, 16384 if kind == "linear" else 8192), 16384 * 1024 * 2560 // (K * N))
        c = dict(kind=kind, rows=rows, K=K, N=N, dtype=dtype)
        if kind == "linear":
            c["act"] = rng.choice(["keep", "mx4"])
        return c
    E = rng.randint(2, 16)
    k = rng.randint(1, min(4, E))
    d, h = 8 * _spread(rng, 16, 192), 8 * _spread(rng, 16, 384)
    T = min(_spread(rng, 1, 16384), 16384 * 2 * 1024 * 2560 // (k * d * h))
    act = rng.choice(["keep", "mx4"])
    # rows rounded to 4 bits between two products: a bf16 layer's case
    return dict(kind=kind, T=T, d=d, h=h, E=E, k=k, act=act, dtype="bf16" if act == "mx4" else dtype)


# ---- the plain forms ------------------------------------------------------
def _tensor(values, like):
    return torch.tensor(values, device=like.device)


def _codes(x):
    """(codes [..., 16 n], scale bytes [..., n]) of x [..., K], n = ceil(K / 32)."""
    K = x.shape[-1]
    n = -(-K // 32)
    b = F.pad(x.float(), (0, n * 32 - K)).view(*x.shape[:-1], n, 32)
    amax = b.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, torch.full_like(amax, -127, dtype=torch.int32))
    e = e.clamp(-127, 125)
    a = b.abs() * torch.exp2(-e.float()).unsqueeze(-1)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    half = (torch.round(a / step) * step).clamp_max(6.0) * 2  # 0 to 12, round ties to even
    code = _tensor([0, 1, 2, 3, 4, 4, 5, 5, 6, 6, 6, 6, 7], x)[half.long()] + 8 * torch.signbit(b)
    code = code.view(*x.shape[:-1], n * 16, 2)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), (e + 127).to(torch.uint8)


def _values(codes, scales, K):
    """What codes stand for, fp32 [..., K]."""
    lut = _tensor(GRID + tuple(-v for v in GRID), codes)
    pair = torch.stack([codes & 15, codes >> 4], -1).long()
    v = lut[pair].view(*scales.shape, 32) * torch.exp2(scales.float() - 127.0).unsqueeze(-1)
    return v.reshape(*scales.shape[:-1], -1)[..., :K]


def _rounded(x):
    return _values(*_codes(x), x.shape[-1])


def _scores(z, score):
    return torch.softmax(z, -1) if score == "softmax" else 1 / (1 + torch.exp(-z))


def _weights(s, topi, renorm, scale):
    """The chosen slots' weights before the scale, and their sum."""
    has = topi >= 0
    w = torch.where(has, s.gather(1, topi.clamp_min(0)), torch.zeros((), dtype=s.dtype, device=s.device))
    total = w.sum(1, keepdim=True)
    if renorm:
        even = has.to(s.dtype) / has.sum(1, keepdim=True).clamp_min(1)
        w = torch.where(total < 1e-6, even, w / total.clamp_min(1e-9))
    return w, total


def _route(c, logits, bias):
    # 64 bits: the choice between two experts next to each other must not depend on a rounding
    z = logits.double()
    s = _scores(z, c["score"])
    T, E = z.shape
    G, low = c["groups"], -math.inf
    live = (z > low) & ~torch.isnan(s)
    sel = s if bias is None else s + bias.double()
    key = torch.where(live, z if bias is None else sel, torch.full_like(z, low))
    if c["top_groups"] < G:
        sel = torch.where(live, sel, torch.full_like(z, low)).view(T, G, E // G)
        best = sel.sort(-1, descending=True)[0][..., :c["best"]]
        first = best[..., 0]
        score = torch.where(best > low, best, torch.zeros_like(best)).sum(-1)
        score = torch.where(first > low, score, first)
        order = score.sort(dim=-1, descending=True, stable=True)[1][:, :c["top_groups"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=z.device).scatter(1, order, True)
        key = torch.where(keep.unsqueeze(-1), key.view(T, G, E // G), torch.full_like(sel, low)).view(T, E)
    best, topi = key.sort(dim=-1, descending=True, stable=True)
    topi = torch.where(best[:, :c["k"]] > low, topi[:, :c["k"]], torch.full_like(topi[:, :c["k"]], -1))
    w, _ = _weights(s, topi, c["renorm"], c["scale"])
    return s.float() if c["prob"] else None, topi, (w * c["scale"]).float()


def _route_grad(c, dtopw, logits, topi, dprob):
    z = logits.float()
    s = _scores(z, c["score"])
    has = topi >= 0
    g = torch.where(has, dtopw, torch.zeros_like(dtopw)) * c["scale"]
    if c["renorm"]:
        w, total = _weights(s, topi, True, 1.0)
        g = (g - (g * w).sum(1, keepdim=True)) / total.clamp_min(1e-9)
        g = torch.where(has & (total >= 1e-6), g, torch.zeros_like(g))
    ds = torch.zeros_like(z) if dprob is None else dprob
    ds = ds.scatter_add(1, topi.clamp_min(0), g)
    if c["score"] == "softmax":
        dz = s * (ds - (ds * s).sum(1, keepdim=True))
    else:
        dz = ds * s * (1 / (1 + torch.exp(z)))
    return dz.to(logits.dtype)


def _moe(c, x, topi, topw, experts):
    gate, up, down = (_values(experts[i], experts[i + 1], n) for i, n in ((0, c["d"]), (2, c["d"]), (4, c["h"])))
    T, k = topi.shape
    slot_expert, order = topi.reshape(-1).sort(stable=True)
    counts = torch.bincount(slot_expert, minlength=c["E"])
    place = torch.arange(T * k, device=x.device) - (counts.cumsum(0) - counts)[slot_expert]
    rows = torch.zeros(c["E"], int(counts.max()), c["d"], device=x.device)  # every expert's rows, padded to the most
    xv = _rounded(x) if c["act"] == "mx4" else x.float()
    rows[slot_expert, place] = xv[order // k]
    g = torch.bmm(rows, gate.transpose(1, 2).contiguous())
    hidden = g / (1 + torch.exp(-g)) * torch.bmm(rows, up.transpose(1, 2).contiguous())
    if c["act"] == "mx4":
        hidden = _rounded(hidden)
    y = torch.bmm(hidden, down.transpose(1, 2).contiguous())
    slots = torch.empty(T * k, c["d"], device=x.device)
    slots[order] = y[slot_expert, place]
    out = (slots.view(T, k, c["d"]) * topw.unsqueeze(-1)).sum(1)
    return out.to(x.dtype), counts.to(torch.int32)


# ---- what a program has in hand ---------------------------------------------
def _logits(gen, T, E, dtype):
    z = torch.randn(T, E, generator=gen, device=DEV) * 0.64  # hidden states N(0, 1), router N(0, 0.02), d = 1024
    z[T - T // 32:] = 0.0  # the padding at the end of a batch: every expert the same
    return z.to(DTYPES[dtype])


def prepare(case, seed):
    c = case
    gen = torch.Generator(DEV).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device=DEV) * std

    if c["kind"] == "route":
        bias = normal(c["E"], std=0.05) if c["bias"] else None
        return c, _logits(gen, c["T"], c["E"], c["dtype"]), bias
    if c["kind"] == "route_grad":
        z = _logits(gen, c["T"], c["E"], c["dtype"])
        topi = z.sort(dim=-1, descending=True, stable=True)[1][:, :c["k"]].contiguous()
        return c, normal(c["T"], c["k"]), z, topi, normal(c["T"], c["E"], std=0.1) if c["prob"] else None
    if c["kind"] == "quant":
        return c, normal(c["rows"], c["K"]).to(DTYPES[c["dtype"]])
    if c["kind"] in ("linear", "dx"):
        w, s = _codes(normal(c["N"], c["K"], std=0.02))
        return c, normal(c["rows"], c["K"] if c["kind"] == "linear" else c["N"]).to(DTYPES[c["dtype"]]), w, s
    x = normal(c["T"], c["d"]).to(DTYPES[c["dtype"]])
    prob = torch.softmax(normal(c["T"], c["E"], std=0.64), -1)
    topw, topi = prob.sort(dim=-1, descending=True, stable=True)
    topw, topi = topw[:, :c["k"]], topi[:, :c["k"]].contiguous()
    experts = []
    for n, m in ((c["h"], c["d"]), (c["h"], c["d"]), (c["d"], c["h"])):
        experts += _codes(normal(c["E"], n, m, std=0.02))
    return c, x, topi, (topw / topw.sum(1, keepdim=True)).contiguous(), tuple(experts)


def run(state):
    c = state[0]
    if own:
        return _run_own(*state)
    if c["kind"] == "route":
        return _route(*state)
    if c["kind"] == "route_grad":
        return _route_grad(*state)
    if c["kind"] == "quant":
        codes, scales = _codes(state[1])
        return _values(codes, scales, c["K"]).to(state[1].dtype)
    if c["kind"] == "linear":
        x = _rounded(state[1]) if c["act"] == "mx4" else state[1].float()
        return (x @ _values(state[2], state[3], c["K"]).t()).to(state[1].dtype)
    if c["kind"] == "dx":
        return (state[1].float() @ _values(state[2], state[3], c["K"])).to(state[1].dtype)
    return _moe(*state)


def _run_own(c, *t):
    from smaulnative_amd.compute import get_backend
    be = get_backend("rocm")
    if c["kind"] == "route":
        return be.moe_route(t[0], c["k"], score=c["score"], bias=t[1], groups=c["groups"], top_groups=c["top_groups"],
                            group_best=c["best"], renorm=c["renorm"], scale=c["scale"], need_prob=c["prob"])
    if c["kind"] == "route_grad":
        return be.moe_route_backward(t[0], t[1], t[2], score=c["score"], renorm=c["renorm"], scale=c["scale"],
                                     dprob=t[3])
    if c["kind"] == "quant":
        codes, scales = be.mx4_quantize(t[0])
        return be.mx4_dequantize(codes, scales, c["K"], t[0].dtype)
    if c["kind"] == "linear":
        return be.mx4_forward(t[0], t[1], t[2], c["K"], c["N"], act=c["act"])
    if c["kind"] == "dx":
        return be.mx4_backward_input(t[0], t[1], t[2], c["K"], c["N"])
    return be.mx4_moe_forward(*t, act=c["act"])


# ---- what the work is, and its outputs in 64 bits ----------------------------
def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    packed = 0.5 + 1 / 32  # bytes of a 4-bit value with its share of a scale
    if c["kind"] == "route":
        n = c["T"] * c["E"]
        return {"bytes": n * size + (n * 4 if c["prob"] else 0) + c["T"] * c["k"] * 12, "flops": 4 * n}
    if c["kind"] == "route_grad":
        n = c["T"] * c["E"]
        return {"bytes": 2 * n * size + (n * 4 if c["prob"] else 0) + c["T"] * c["k"] * 12, "flops": 8 * n}
    if c["kind"] == "quant":  # there and back
        n = c["rows"] * c["K"]
        return {"bytes": 2 * n * size + 2 * n * packed, "flops": 4 * n}
    if c["kind"] in ("linear", "dx"):
        m, n = c["rows"], c["K"] * c["N"]
        return {"bytes": m * (c["K"] + c["N"]) * size + n * packed, "flops": 2 * m * n}
    rows = c["T"] * c["k"]
    used = min(c["E"], rows)
    return {"bytes": 2 * c["T"] * c["d"] * size + rows * 12 + 3 * used * c["d"] * c["h"] * packed,
            "flops": 6 * rows * c["d"] * c["h"]}


def _exact_rounded(x):
    """x in 64 bits, each block of 32 rounded: by comparisons with the borders between neighbours."""
    K = x.shape[-1]
    n = -(-K // 32)
    out = torch.zeros(*x.shape[:-1], n * 32, dtype=torch.float64, device=x.device)
    out[..., :K] = x
    out = out.view(*x.shape[:-1], n, 32)
    top = out.abs().max(-1, keepdim=True)[0]
    unit = 2.0 ** (torch.floor(torch.log2(top.clamp_min(2.0 ** -140))) - 2).clamp(-127, 125)
    unit = torch.where(top >= unit * 8, unit * 2, torch.where(top < unit * 4, unit / 2, unit))  # a log2 next to a whole number
    unit = unit.clamp_min(2.0 ** -127)
    a = out.abs() / unit
    q = torch.zeros_like(a)
    for border, up, low, high in ((0.25, False, 0.0, 0.5), (0.75, True, 0.5, 1.0), (1.25, False, 1.0, 1.5),
                                  (1.75, True, 1.5, 2.0), (2.5, False, 2.0, 3.0), (3.5, True, 3.0, 4.0),
                                  (5.0, False, 4.0, 6.0)):
        q += ((a >= border) if up else (a > border)) * (high - low)
    return (torch.sign(out) * q * unit).view(*x.shape[:-1], n * 32)[..., :K]


def _exact_values(codes, scales, K):
    nibble = torch.stack([codes % 16, codes // 16], -1).view(*codes.shape[:-1], -1)[..., :K]
    mag = torch.tensor(GRID, dtype=torch.float64, device=codes.device)[(nibble % 8).long()]
    unit = 2.0 ** (scales.double() - 127)
    return torch.where(nibble >= 8, -mag, mag) * unit.repeat_interleave(32, -1)[..., :K]


def exact(case, seed):
    c = case
    t = prepare(case, seed)[1:]
    if c["kind"] == "quant":
        return _exact_rounded(t[0].double())
    if c["kind"] == "linear":
        x = _exact_rounded(t[0].double()) if c["act"] == "mx4" else t[0].double()
        return x @ _exact_values(t[1], t[2], c["K"]).t()
    if c["kind"] == "dx":
        return t[0].double() @ _exact_values(t[1], t[2], c["K"])
    if c["kind"] == "route":
        return _exact_route(c, *t)
    if c["kind"] == "route_grad":
        return _exact_route_grad(c, *t)
    x, topi, topw, ex = t
    xv = _exact_rounded(x.double()) if c["act"] == "mx4" else x.double()
    out = torch.zeros(c["T"], c["d"], dtype=torch.float64, device=x.device)
    counts = []
    for e in range(c["E"]):
        tok, slot = (topi == e).nonzero(as_tuple=True)
        counts.append(tok.numel())
        a = xv[tok] @ _exact_values(ex[0][e], ex[1][e], c["d"]).t()
        b = xv[tok] @ _exact_values(ex[2][e], ex[3][e], c["d"]).t()
        hid = a * torch.sigmoid(a) * b
        if c["act"] == "mx4":
            hid = _exact_rounded(hid)
        y = hid @ _exact_values(ex[4][e], ex[5][e], c["h"]).t()
        out[tok] += y * topw[tok, slot].double().unsqueeze(1)
    return out, torch.tensor(counts, dtype=torch.int32)


def _exact_scores(z, score):
    if score == "sigmoid":
        return torch.sigmoid(z)
    e = torch.exp(z - z.max(1, keepdim=True)[0])
    return e / e.sum(1, keepdim=True)


def _exact_route(c, logits, bias):
    z = logits.double()
    s = _exact_scores(z, c["score"])
    choice = s if bias is None else s + bias.double()
    T, E = z.shape
    per = E // c["groups"]
    mine = torch.arange(E, device=z.device)
    alive = torch.ones_like(z, dtype=torch.bool)
    if c["top_groups"] < c["groups"]:
        # a group is in where fewer than top_groups others are ahead of it
        best = choice.view(T, c["groups"], per).topk(min(c["best"], per), -1)[0].sum(-1)
        g = torch.arange(c["groups"], device=z.device)
        a, b = best.unsqueeze(2), best.unsqueeze(1)
        ahead = ((b > a) | ((b == a) & (g.view(1, 1, -1) < g.view(1, -1, 1)))).sum(2)
        alive = (ahead < c["top_groups"]).repeat_interleave(per, 1)
    key = z if bias is None else choice
    topi = torch.empty(T, c["k"], dtype=torch.int64, device=z.device)
    for j in range(c["k"]):  # the highest left, the lowest index among equals
        left = torch.where(alive, key, torch.full_like(key, -math.inf))
        first = torch.where(alive & (left == left.max(1, keepdim=True)[0]), mine, E).min(1)[0]
        topi[:, j] = first
        alive = alive & (mine != first.unsqueeze(1))
    w = s.gather(1, topi)
    if c["renorm"]:
        w = torch.where(w.sum(1, keepdim=True) < 1e-6, torch.full_like(w, 1 / c["k"]), w / w.sum(1, keepdim=True))
    return s if c["prob"] else None, topi, w * c["scale"]


def _exact_route_grad(c, dtopw, logits, topi, dprob):
    with torch.enable_grad():
        z = logits.double().requires_grad_()
        s = _exact_scores(z, c["score"])
        w = s.gather(1, topi)
        if c["renorm"]:
            w = w / w.sum(1, keepdim=True)
        loss = (w * c["scale"] * dtopw.double()).sum()
        if dprob is not None:
            loss = loss + (s * dprob.double()).sum()
        return torch.autograd.grad(loss, z)[0]
