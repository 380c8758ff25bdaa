"""Weights in microscaled 4-bit floating point: ``MX4Linear`` and ``MX4Experts``.

The format (beside ``FP8Linear``'s tiled E4M3; no counterpart in the reference): a
row of in_f weights is ceil(in_f / 32) blocks of 32 E2M1 codes (16 bytes) with one
E8M0 scale, a power of two: 4.25 bits a weight.  The products run through the
backend's ``mx4_forward`` / ``mx4_moe_forward``, ``act="keep"`` with the activations
as they are, ``act="mx4"`` with their rows rounded to the format too (for prefills:
the matrix cores multiply the codes of both as they are).

Weights are frozen buffers.  Gradients reach the input through ``mx4_backward_input``
(with ``act="mx4"`` the rounding of the activations is taken as the identity), so
what stands before them, the router included, can be trained; a weight gradient is
not formed.  With gradients a layer runs expert by expert, each product's outputs of
its input's type: of bf16 rows that rounds gate's and up's products and each expert's
output too, and with ``act="mx4"`` the hidden rows before they become codes, so that
some are the neighbouring code (outputs 3 % off what the layer gives without
gradients; of fp32 rows it is the same).
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from smaulnative_amd import _lib
from smaulnative_amd.compute import get_backend
from smaulnative_amd.fp8_tile import decode_block

BLOCK = 32
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def check_act(act):
    if act not in _lib.ACTS:
        raise ValueError(f"act must be one of {sorted(_lib.ACTS)}, got {act!r}")
    return act


def _quantize_torch(w):
    """The backend's ``mx4_quantize`` in torch ops, for host tensors."""
    n = -(-w.shape[-1] // BLOCK)
    b = torch.nn.functional.pad(w.float(), (0, n * BLOCK - w.shape[-1])).view(*w.shape[:-1], n, BLOCK)
    finite = torch.isfinite(b).all(-1)
    amax = torch.where(finite, b.abs().amax(-1), torch.ones((), device=w.device))
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, torch.tensor(-127, dtype=torch.int32, device=w.device))
    e = e.clamp_min(-127)
    # powers of two are exact, and 2^127 and less are numbers of fp32
    a = b.abs() * torch.ldexp(torch.ones((), device=w.device), -e).unsqueeze(-1)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp_max(6.0)  # to nearest, ties to even
    code = torch.bucketize(q, torch.tensor(_VALUES, device=w.device)) + 8 * torch.signbit(b)
    code = torch.where(finite.unsqueeze(-1), code, torch.zeros_like(code)).view(*w.shape[:-1], n * BLOCK // 2, 2)
    scale = torch.where(finite, e + 127, torch.full_like(e, 255))
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), scale.to(torch.uint8)


def quantize(w):
    """(codes uint8 [..., 16 n], scales uint8 [..., n]) of w [..., in_f], n = ceil(in_f / 32)."""
    if w.dim() < 1 or w.shape[-1] < 1 or not w.is_floating_point():
        raise ValueError(f"quantize: floating point rows expected, got {w.dtype} {tuple(w.shape)}")
    with torch.no_grad():
        w = w.detach()
        if w.dtype not in (torch.float32, torch.bfloat16):
            w = w.float()
        return get_backend().mx4_quantize(w) if w.is_cuda else _quantize_torch(w)


def decode(codes, scales, in_f, dtype=torch.float32):
    """The values [..., in_f] that codes and scales stand for."""
    if codes.is_cuda:
        return get_backend().mx4_dequantize(codes, scales, in_f, dtype)
    lut = torch.tensor(_VALUES + tuple(-v for v in _VALUES))
    v = lut[torch.stack([codes & 15, codes >> 4], -1).long()].view(*scales.shape, BLOCK)
    # in 64 bits: the smallest scale is a subnormal of fp32
    unit = torch.where(scales == 255, math.nan, torch.pow(2.0, scales.double() - 127.0))
    return (v * unit.unsqueeze(-1)).reshape(*scales.shape[:-1], -1)[..., :in_f].to(dtype)


class _MX4Matmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, codes, scales, in_f, out_f, act):
        ctx.save_for_backward(codes, scales)
        ctx.dims = (in_f, out_f, x.shape, x.dtype)
        rows = x.reshape(-1, in_f)
        if rows.dtype not in (torch.float32, torch.bfloat16):
            rows = rows.float()
        y = get_backend().mx4_forward(rows, codes, scales, in_f, out_f, act)
        return y.reshape(*x.shape[:-1], out_f).to(x.dtype if x.is_floating_point() else torch.float32)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        if not ctx.needs_input_grad[0]:
            return None, None, None, None, None, None
        codes, scales = ctx.saved_tensors
        in_f, out_f, shape, dtype = ctx.dims
        g = grad.reshape(-1, out_f)
        if g.dtype not in (torch.float32, torch.bfloat16):
            g = g.float()
        dx = get_backend().mx4_backward_input(g, codes, scales, in_f, out_f)
        return dx.reshape(shape).to(dtype), None, None, None, None, None


def matmul(x, codes, scales, in_f, out_f, act="keep"):
    """x [..., in_f] . W^T in x's type, differentiable in x."""
    return _MX4Matmul.apply(x, codes, scales, in_f, out_f, act)


class MX4Linear(nn.Module):
    """Linear layer over 4-bit weights: buffers ``w4`` / ``ws``, optional fp32 ``bias``."""

    def __init__(self, in_f, out_f, act="keep", bias=False):
        super().__init__()
        if in_f <= 0 or out_f <= 0:
            raise ValueError(f"in_f/out_f must be positive, got {in_f}/{out_f}")
        self.in_f, self.out_f, self.act = in_f, out_f, check_act(act)
        bound = 1.0 / math.sqrt(in_f)  # nn.Linear's default distribution
        w4, ws = quantize(torch.empty(out_f, in_f).uniform_(-bound, bound))
        self.register_buffer("w4", w4)
        self.register_buffer("ws", ws)
        self.bias = nn.Parameter(torch.zeros(out_f)) if bias else None

    @classmethod
    def from_float(cls, lin, act="keep"):
        """An MX4Linear holding ``lin``'s weight (and bias) quantized."""
        m = cls(lin.in_features, lin.out_features, act, lin.bias is not None).to(lin.weight.device)
        m._set(lin.weight, lin.bias)
        return m

    @classmethod
    def from_fp8(cls, lin, act="keep"):
        """An MX4Linear holding an ``FP8Linear``'s decoded weight (and bias) quantized."""
        m = cls(lin.in_f, lin.out_f, act, lin.bias is not None).to(lin.w8.device)
        m._set(decode_block(lin.w8, lin.sc.float(), 0, lin.out_f, lin.in_f, lin.tile), lin.bias)
        return m

    @torch.no_grad()
    def _set(self, weight, bias):
        w4, ws = quantize(weight)
        self.w4.copy_(w4)
        self.ws.copy_(ws)
        if bias is not None:
            self.bias.copy_(bias.detach())

    def forward(self, x):
        y = matmul(x, self.w4, self.ws, self.in_f, self.out_f, self.act)
        return y if self.bias is None else y + self.bias

    def extra_repr(self):
        return f"in_f={self.in_f}, out_f={self.out_f}, act={self.act!r}, bias={self.bias is not None}"


class _Expert:
    """One expert of an ``MX4Experts``, called as a SwiFFN is."""

    def __init__(self, owner, index):
        self.owner, self.index = owner, index

    def __call__(self, x):
        from smaulnative_amd.moe import _swiglu
        o, i = self.owner, self.index
        dtype = x.dtype if x.is_floating_point() else torch.float32
        gate = matmul(x, o.gate_w[i], o.gate_s[i], o.d, o.h, o.act)
        up = matmul(x, o.up_w[i], o.up_s[i], o.d, o.h, o.act)
        return matmul(_swiglu(gate, up, dtype), o.down_w[i], o.down_s[i], o.h, o.d, o.act)


class MX4Experts(nn.Module):
    """The SwiGLU experts of a MoE layer in the 4-bit format, each projection's weights in
    one buffer: ``gate_w`` / ``up_w`` [E, h, 16 n] and ``down_w`` [E, d, 16 n] codes with
    their scales.  Indexing and iterating give callable experts."""

    _NAMES = ("gate_w", "gate_s", "up_w", "up_s", "down_w", "down_s")

    def __init__(self, num_experts, d, h, act="keep"):
        super().__init__()
        if num_experts <= 0 or d <= 0 or h <= 0:
            raise ValueError(f"num_experts, d and h must be positive, got {num_experts}, {d}, {h}")
        self.num_experts, self.d, self.h, self.act = num_experts, d, h, check_act(act)
        for name, n, m in (("gate", h, d), ("up", h, d), ("down", d, h)):
            bound = 1.0 / math.sqrt(m)
            w, s = quantize(torch.empty(num_experts, n, m).uniform_(-bound, bound))
            self.register_buffer(name + "_w", w)
            self.register_buffer(name + "_s", s)

    @classmethod
    def from_experts(cls, experts, act="keep"):
        """The experts of a layer of ``SwiFFN`` (tiled FP8), decoded and quantized."""
        first = experts[0].gate
        m = cls(len(experts), first.in_f, first.out_f, act).to(first.w8.device)
        with torch.no_grad():
            for i, ex in enumerate(experts):
                for name in ("gate", "up", "down"):
                    lin = getattr(ex, name)
                    w, s = quantize(decode_block(lin.w8, lin.sc.float(), 0, lin.out_f, lin.in_f, lin.tile))
                    getattr(m, name + "_w")[i].copy_(w)
                    getattr(m, name + "_s")[i].copy_(s)
        return m

    def buffers6(self):
        """(gate_w, gate_s, up_w, up_s, down_w, down_s), as the backend takes them."""
        b = self._buffers
        return tuple(b[n] for n in self._NAMES)

    def __len__(self):
        return self.num_experts

    def __getitem__(self, index):
        if not -self.num_experts <= index < self.num_experts:
            raise IndexError(f"expert {index} of {self.num_experts}")
        return _Expert(self, index % self.num_experts)

    def __iter__(self):
        return (self[i] for i in range(self.num_experts))

    def extra_repr(self):
        return f"num_experts={self.num_experts}, d={self.d}, h={self.h}, act={self.act!r}"
