"""The 8-bit feed-forward path, as measurable cases: rows in blocks of 128 E4M3
codes with a shared power of two.

Each case is one pass through an operator.  With ``own`` false ``run`` computes
it in elementary tensor operations, otherwise through ``RocmBackend``:

- ``norm``: the residual's addition, the root-mean-square norm and its output in
  blocks, read back as values (``add_rms_norm``, ``fp8_block_dequantize``);
- ``norm_grad``: the gradients of that norm's input and weight
  (``add_rms_norm_backward``);
- ``linear``: the product of rows in the format with a weight in the format, the
  rows given so or rounded in the call (``fp8_block_forward``);
- ``dx``: the input gradient of that product (``fp8_block_backward_input``);
- ``ffn``: the gated feed-forward block, its hidden rows in the format
  (``fp8_block_ffn_forward``);
- ``ffn_grad``: a training step of that block: the float weights rounded, the
  forward pass, and the gradients of the input and of the three weights
  (``fp8_block_quantize``, ``fp8_block_ffn_forward``, ``fp8_block_ffn_backward``).
"""
import math

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6
BLOCK = 128
TOP = 448.0  # the largest code's value


def listed():
    return [
        # a decode step of 64 sequences: the residual's addition, the norm and its codes between two layers
        dict(name="norm_step_64", kind="norm", T=64, d=1024, dtype="bf16", residual=True),
        # a long prefill: 32768 hidden rows of a wider model
        dict(name="norm_prefill_32k", kind="norm", T=32768, d=2048, dtype="bf16", residual=True),
        # training: the norm's gradients, added to what comes along the residual path
        dict(name="norm_grad_16k", kind="norm_grad", T=16384, d=2048, dtype="bf16", residual=True),
        # a short ragged batch in fp32, an odd width, nothing along the residual path
        dict(name="norm_grad_odd_f32", kind="norm_grad", T=4099, d=1001, dtype="f32", residual=False),
        # one token through a projection: the weight's bytes and the launches
        dict(name="linear_token", kind="linear", T=1, K=1024, N=2560, dtype="bf16", given="rows"),
        # a prefill through a projection, on the codes that a norm left
        dict(name="linear_prefill_codes", kind="linear", T=16384, K=2048, N=5120, dtype="bf16", given="codes"),
        # training through a frozen projection: 4096 rows
        dict(name="dx_4096", kind="dx", T=4096, K=1024, N=2560, dtype="bf16"),
        # the same with fp32 gradients, ragged rows and widths
        dict(name="dx_odd_f32", kind="dx", T=1001, K=1000, N=777, dtype="f32"),
        # a decode step of 64 sequences through the block, on a norm's codes
        dict(name="ffn_step_64", kind="ffn", T=64, d=1024, h=2560, given="codes"),
        # a prefill of 16384 tokens through a wider one
        dict(name="ffn_prefill_16k", kind="ffn", T=16384, d=2048, h=5120, given="codes"),
        # training: a step of 8192 tokens, bf16 weights
        dict(name="ffn_grad_8k", kind="ffn_grad", T=8192, d=1024, h=2560, dtype="bf16"),
        # the small model's block on a ragged batch of byte tokens, odd widths, fp32 weights
        dict(name="ffn_grad_odd", kind="ffn_grad", T=509, d=500, h=1251, dtype="f32"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "linear", "dx", "ffn", "ffn_grad"])
    dtype = rng.choice(["f32", "bf16"])
    if kind in ("norm", "norm_grad"):
        d = _spread(rng, 64, 8192)
        T = min(_spread(rng, 1, 32768), 32768 * 2048 // d)
        return dict(kind=kind, T=T, d=d, dtype=dtype, residual=rng.random() < 0.7)
    if kind in ("linear", "dx"):
        K, N = _spread(rng, 64, 8192), _spread(rng, 64, 8192)
        T = min(_spread(rng, 1, 16384 if kind == "linear" else 8192), 16384 * 2048 * 5120 // (K * N))
        c = dict(kind=kind, T=T, K=K, N=N, dtype=dtype)
        if kind == "linear":
            c["given"] = rng.choice(["rows", "codes"])
        return c
    d, h = _spread(rng, 64, 4096), _spread(rng, 64, 8192)
    if kind == "ffn":
        T = min(_spread(rng, 1, 16384), 16384 * 2048 * 5120 // (d * h))
        return dict(kind=kind, T=T, d=d, h=h, given=rng.choice(["rows", "codes"]))
    T = min(_spread(rng, 1, 8192), 8192 * 2048 * 2560 // (d * h))
    return dict(kind=kind, T=T, d=d, h=h, dtype=dtype)


# ---- the plain forms ------------------------------------------------------
def _encode(x):
    """(codes uint8 [..., 128 n], scales uint8 [..., 4 ceil(n / 4)]) of rows x [..., K], n = ceil(K / 128).

    A block's scale is the least power of two 2^(byte - 127), byte >= 0, that its largest magnitude divided by
    does not pass 448 with; a code is the nearest value, ties to the even one."""
    K = x.shape[-1]
    n = -(-K // BLOCK)
    b = F.pad(x.float(), (0, n * BLOCK - K)).view(*x.shape[:-1], n, BLOCK)
    mantissa, exponent = torch.frexp(b.abs().amax(-1))  # mantissa in [0.5, 1)
    e = torch.where(mantissa > 0, exponent - 9 + (mantissa > TOP / 512).int(), torch.full_like(exponent, -127))
    e = e.clamp_min(-127)
    codes = torch.ldexp(b, -e.unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8)
    scales = F.pad(e + 127, (0, -n % 4)).to(torch.uint8)
    return codes.view(*x.shape[:-1], n * BLOCK), scales


def _values(codes, scales, K):
    """What codes and scales stand for, fp32 [..., K]."""
    n = codes.shape[-1] // BLOCK
    v = codes.view(torch.float8_e4m3fn).float().view(*codes.shape[:-1], n, BLOCK)
    v = torch.ldexp(v, scales[..., :n].int().unsqueeze(-1) - 127)
    return v.view(codes.shape)[..., :K]


def _rounded(x):
    return _values(*_encode(x), x.shape[-1])


def _norm(c, x, residual, weight):
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v = s.float()
    y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * weight
    return {"s": s, "y": _rounded(y).to(torch.bfloat16)}


def _norm_grad(c, dy, s, weight, ds):
    v, g = s.float(), dy.float()
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    u = v * r
    dx = r * (g * weight - u * (g * weight * u).mean(-1, keepdim=True))
    if ds is not None:
        dx = dx + ds.float()
    return {"dx": dx.to(s.dtype), "dw": (g * u).sum(0)}


def _ffn(x, gate, up, down):
    g, u = x @ gate.t(), x @ up.t()
    h = _rounded(g / (1 + torch.exp(-g)) * u)
    return (h @ down.t()).to(torch.bfloat16), g, u, h


def _ffn_grad(c, x, dy, *weights):
    xq = _rounded(x)
    gate, up, down = (_rounded(w) for w in weights)
    y, g, u, h = _ffn(xq, gate, up, down)
    dout = dy.float()
    sig = 1 / (1 + torch.exp(-g))
    dh = dout @ down
    dg, du = dh * u * sig * (1 + g * (1 - sig)), dh * g * sig
    out = {"y": y, "dx": dg @ gate + du @ up, "dgate": dg.t() @ xq, "dup": du.t() @ xq, "ddown": dout.t() @ h}
    return {k: v.to(torch.bfloat16) for k, v in out.items()}


# ---- the cases ------------------------------------------------------------
def _rows(gen, T, d, dtype, scale=1.0):
    """Hidden rows: N(0, 1) with a few wide channels, as a model's residual stream has them."""
    wide = 1 + 7 * (torch.rand(d, generator=gen, device=DEV) < 0.02)
    return (scale * wide * torch.randn(T, d, generator=gen, device=DEV)).to(dtype)


def _weight(gen, N, K, dtype=torch.float32):
    return (torch.randn(N, K, generator=gen, device=DEV) / math.sqrt(K)).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    c, kind = case, case["kind"]
    if kind in ("norm", "norm_grad"):
        dtype = DTYPES[c["dtype"]]
        a, b = (_rows(gen, c["T"], c["d"], dtype) for _ in range(2))
        weight = 1 + 0.2 * torch.randn(c["d"], generator=gen, device=DEV)
        third = (torch.randn(c["T"], c["d"], generator=gen, device=DEV) * 0.1).to(dtype)
        if kind == "norm":
            return c, a, b if c["residual"] else None, weight
        return c, third, a, weight, b if c["residual"] else None
    if kind == "linear":
        x = _rows(gen, c["T"], c["K"], DTYPES[c["dtype"]])
        w, s = _encode(_weight(gen, c["N"], c["K"]))
        return (c, *(_encode(x) if c["given"] == "codes" else (x, None)), w, s)
    if kind == "dx":
        g = torch.randn(c["T"], c["N"], generator=gen, device=DEV).to(DTYPES[c["dtype"]])
        return (c, g, *_encode(_weight(gen, c["N"], c["K"])))
    x = _rows(gen, c["T"], c["d"], torch.bfloat16)
    shapes = ((c["h"], c["d"]), (c["h"], c["d"]), (c["d"], c["h"]))
    if kind == "ffn":
        weights = [t for n, k in shapes for t in _encode(_weight(gen, n, k))]
        return (c, *(_encode(x) if c["given"] == "codes" else (x, None)), *weights)
    dy = torch.randn(c["T"], c["d"], generator=gen, device=DEV).to(torch.bfloat16)
    return (c, x, dy, *(_weight(gen, n, k, DTYPES[c["dtype"]]) for n, k in shapes))


def run(state):
    c, *t = state
    if own:
        return _run_own(c, *t)
    kind = c["kind"]
    if kind == "norm":
        return _norm(c, *t)
    if kind == "norm_grad":
        return _norm_grad(c, *t)
    if kind == "linear":
        x, xs, w, s = t
        v = _rounded(x) if xs is None else _values(x, xs, c["K"])
        return (v @ _values(w, s, c["K"]).t()).to(DTYPES[c["dtype"]])
    if kind == "dx":
        g, w, s = t
        return (g.float() @ _values(w, s, c["K"])).to(g.dtype)
    if kind == "ffn":
        x, xs, *w = t
        v = _rounded(x) if xs is None else _values(x, xs, c["d"])
        gate, up, down = (_values(w[i], w[i + 1], k) for i, k in ((0, c["d"]), (2, c["d"]), (4, c["h"])))
        return _ffn(v, gate, up, down)[0]
    return _ffn_grad(c, *t)


def _run_own(c, *t):
    from smaulnative_amd.compute import get_backend
    be = get_backend("rocm")
    kind = c["kind"]
    if kind == "norm":
        x, residual, weight = t
        s, codes, scales = be.add_rms_norm(x, residual, weight, EPS, quantize=True)
        return {"s": s, "y": be.fp8_block_dequantize(codes, scales, c["d"], torch.bfloat16)}
    if kind == "norm_grad":
        dy, s, weight, ds = t
        dx, dw = be.add_rms_norm_backward(dy, s, weight, EPS, ds=ds)
        return {"dx": dx, "dw": dw}
    if kind == "linear":
        x, xs, w, s = t
        return be.fp8_block_forward(x, w, s, c["K"], c["N"], xs=xs, dtype=DTYPES[c["dtype"]])
    if kind == "dx":
        g, w, s = t
        return be.fp8_block_backward_input(g, w, s, c["K"], c["N"])
    if kind == "ffn":
        x, xs, *w = t
        return be.fp8_block_ffn_forward(x, w, c["d"], c["h"], xs=xs)
    x, dy, *weights = t
    w = [q for m in weights for q in be.fp8_block_quantize(m)]
    y, saved = be.fp8_block_ffn_forward(x, w, c["d"], c["h"], save=True)
    dx, dgate, dup, ddown = be.fp8_block_ffn_backward(dy, w, saved, c["d"], c["h"])
    return {"y": y, "dx": dx, "dgate": dgate, "dup": dup, "ddown": ddown}


def work(case):
    c, kind = case, case["kind"]
    size = 4 if c.get("dtype") == "f32" else 2
    if kind == "norm":  # the sum (written where there is one), the codes and the values read back from them
        n = c["T"] * c["d"]
        return {"bytes": n * (size * (3 if c["residual"] else 1) + 1 + 1 + 2) + 4 * c["d"], "flops": 6 * n}
    if kind == "norm_grad":
        n = c["T"] * c["d"]
        return {"bytes": n * size * (4 if c["residual"] else 3) + 8 * c["d"], "flops": 12 * n}
    if kind in ("linear", "dx"):
        T, K, N = c["T"], c["K"], c["N"]
        given = K if c.get("given") == "codes" else K * size
        return {"bytes": T * (given + N * size) + N * K, "flops": 2 * T * K * N}
    T, d, h = c["T"], c["d"], c["h"]
    if kind == "ffn":
        return {"bytes": T * d * (3 if c["given"] == "codes" else 4) + 3 * d * h, "flops": 6 * T * d * h}
    # in: x, dy and the weights; out: y, dx and the weights' gradients
    return {"bytes": 8 * T * d + 3 * d * h * (size + 2), "flops": 18 * T * d * h}


# ---- in 64 bits -----------------------------------------------------------
def _exact_rounded(x):
    """Rows rounded to blocks, by arithmetic on doubles."""
    x = x.double()
    K = x.shape[-1]
    pad = -K % BLOCK
    b = torch.cat([x, x.new_zeros(*x.shape[:-1], pad)], -1).unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp_min(2.0 ** -200) / TOP))
    e = torch.where(torch.exp2(e - 1) * TOP >= top, e - 1, e)  # the logarithm's last bit
    e = torch.where(torch.exp2(e) * TOP < top, e + 1, e).clamp_min(-127)
    unit = torch.exp2(e)
    a = b / unit
    step = torch.exp2(torch.floor(torch.log2(a.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(a / step) * step * unit).flatten(-2)[..., :K]


def _exact_decoded(codes, scales, K):
    c = codes.long()
    e, m = c >> 3 & 15, c & 7
    v = torch.where(e > 0, (8 + m) * torch.exp2(e.double() - 10), m * 2.0 ** -9)
    v = torch.where(c >= 128, -v, v).unflatten(-1, (-1, BLOCK))
    unit = torch.exp2(scales[..., :v.shape[-2]].double() - 127)
    return (v * unit.unsqueeze(-1)).flatten(-2)[..., :K]


def _exact_block(x, gate, up, down):
    """The block's output and the pieces that its gradients need."""
    g, u = x.matmul(gate.T), x.matmul(up.T)
    sig = torch.sigmoid(g)
    h = _exact_rounded(g * sig * u)
    return h.matmul(down.T), h, u * (sig + g * sig * (1 - sig)), g * sig


def exact(case, seed):
    c, *t = prepare(case, seed)
    kind = c["kind"]
    if kind == "norm":
        x, residual, weight = t
        s = x.double() if residual is None else x.double() + residual.double()
        v = s.to(x.dtype).double()  # the norm is of the rounded sum
        rms = torch.sqrt(v.square().mean(1, keepdim=True) + EPS)
        return {"s": s, "y": _exact_rounded(v / rms * weight.double())}
    if kind == "norm_grad":
        dy, s, weight, ds = t
        v, g = s.double(), dy.double()
        rms = torch.sqrt(v.square().mean(1, keepdim=True) + EPS)
        wg = weight.double() * g
        dx = wg / rms - v * (wg * v).mean(1, keepdim=True) / rms ** 3
        return {"dx": dx if ds is None else dx + ds.double(), "dw": (g * v / rms).sum(0)}
    if kind == "linear":
        x, xs, w, s = t
        v = _exact_rounded(x) if xs is None else _exact_decoded(x, xs, c["K"])
        return v.matmul(_exact_decoded(w, s, c["K"]).T)
    if kind == "dx":
        g, w, s = t
        return g.double().matmul(_exact_decoded(w, s, c["K"]))
    if kind == "ffn":
        x, xs, *w = t
        v = _exact_rounded(x) if xs is None else _exact_decoded(x, xs, c["d"])
        return _exact_block(v, *(_exact_decoded(w[i], w[i + 1], k) for i, k in ((0, c["d"]), (2, c["d"]), (4, c["h"]))))[0]
    x, dy, *w = t
    x, gate, up, down = (_exact_rounded(m) for m in (x, *w))
    y, h, da, db = _exact_block(x, gate, up, down)
    dout = dy.double()
    dh = dout.matmul(down)
    dg, du = dh * da, dh * db
    return {"y": y, "dx": dg.matmul(gate) + du.matmul(up), "dgate": dg.T.matmul(x), "dup": du.T.matmul(x),
            "ddown": dout.T.matmul(h)}
