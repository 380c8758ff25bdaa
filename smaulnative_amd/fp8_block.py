"""8-bit feed-forward layers: ``FP8BlockLinear``, ``FP8BlockFFN``, ``AddRMSNorm`` and
``FP8BlockNormFFN``.

The format (beside ``FP8Linear``'s tiled E4M3, whose activations stay as they are; no
counterpart in the reference): rows in blocks of 128 E4M3 codes with a shared power of
two.  Both sides of a product are in it, so it runs on the matrix cores' 8-bit
instructions, and the codes that a norm writes are what the next product reads.

Weights are frozen codes, or with ``trainable`` float parameters that every forward pass
rounds.  Gradients go straight through the roundings: to the input, the norm's weight
and the float weights, whose gradients are formed in bf16.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from smaulnative_amd.compute import get_backend
from smaulnative_amd.fp8_tile import decode_block

BLOCK = 128
TOP = 448.0


def _quantize_torch(w):
    """The backend's ``fp8_block_quantize`` in torch ops, for host tensors."""
    n = -(-w.shape[-1] // BLOCK)
    b = torch.nn.functional.pad(w.float(), (0, n * BLOCK - w.shape[-1])).view(*w.shape[:-1], n, BLOCK)
    finite = torch.isfinite(b).all(-1)
    amax = torch.where(finite, b.abs().amax(-1), torch.zeros((), device=w.device))
    m, e = torch.frexp(amax)
    e = torch.where(m > 0, e - 9 + (m > TOP / 512).int(), torch.full_like(e, -127)).clamp_min(-127)
    b = torch.where(finite.unsqueeze(-1), b, torch.zeros((), device=w.device))
    codes = torch.ldexp(b, -e.unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.nn.functional.pad(torch.where(finite, e + 127, torch.full_like(e, 255)), (0, -n % 4))
    return codes.view(*w.shape[:-1], n * BLOCK), scales.to(torch.uint8)


def quantize(w):
    """(codes uint8 [..., 128 n], scales uint8 [..., 4 ceil(n / 4)]) of w [..., in_f], n = ceil(in_f / 128)."""
    if w.dim() < 1 or w.shape[-1] < 1 or not w.is_floating_point():
        raise ValueError(f"quantize: floating point rows expected, got {w.dtype} {tuple(w.shape)}")
    with torch.no_grad():
        w = w.detach()
        if w.dtype not in (torch.float32, torch.bfloat16):
            w = w.float()
        return get_backend().fp8_block_quantize(w) if w.is_cuda else _quantize_torch(w)


def decode(codes, scales, in_f, dtype=torch.float32):
    """The values [..., in_f] that codes and scales stand for."""
    if codes.is_cuda:
        return get_backend().fp8_block_dequantize(codes, scales, in_f, dtype)
    n = codes.shape[-1] // BLOCK
    s = scales[..., :n].unsqueeze(-1)
    v = codes.view(torch.float8_e4m3fn).double().view(*codes.shape[:-1], n, BLOCK)
    v = v * torch.where(s == 255, math.nan, torch.pow(2.0, s.double() - 127))
    return v.reshape(codes.shape)[..., :in_f].to(dtype)


def _rows(x):
    """x, in a type that the backend reads."""
    return x if x.dtype in (torch.float32, torch.bfloat16) else x.float()


def _addends(x, residual):
    """x and residual in one type that the norm reads, and the type of their sum."""
    total = x.dtype if residual is None else torch.promote_types(x.dtype, residual.dtype)
    if not total.is_floating_point:
        total = torch.float32
    kind = total if total in (torch.float32, torch.bfloat16) else torch.float32
    return x.to(kind), None if residual is None else residual.to(kind), total


def _check_leaves(*leaves):
    """Refuses to record a pass under capture while a pass recorded outside holds one of its
    leaves: autograd orders the leaf's accumulation by the stream of the pass that first
    recorded it, and a captured backward pass that meets a stream outside its capture ends
    the process.  Returns what the caller holds until its pass is recorded: the leaves'
    nodes, which carry the mark."""
    leaves = [t for t in leaves if t is not None and t.requires_grad and t.is_leaf and t.is_cuda]
    if not leaves or not torch.is_grad_enabled():
        return []
    capturing = torch.cuda.is_current_stream_capturing()
    nodes = [torch.autograd.graph.get_gradient_edge(t).node for t in leaves]
    for node in nodes:
        if node.metadata.setdefault("smaul_captured", capturing) is False and capturing:
            raise RuntimeError("a pass recorded outside of this capture still holds a leaf of this one: free its "
                               "outputs before the capture")
    return nodes


class _Matmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, codes, scales, in_f, out_f):
        ctx.save_for_backward(codes, scales)
        ctx.dims = (in_f, out_f, x.dtype)
        y = get_backend().fp8_block_forward(_rows(x), codes, scales, in_f, out_f)
        return y.to(x.dtype if x.is_floating_point() else torch.float32)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        if not ctx.needs_input_grad[0]:
            return None, None, None, None, None
        codes, scales = ctx.saved_tensors
        in_f, out_f, dtype = ctx.dims
        dx = get_backend().fp8_block_backward_input(_rows(grad), codes, scales, in_f, out_f)
        return dx.to(dtype), None, None, None, None


class FP8BlockLinear(nn.Module):
    """Linear layer over frozen block codes: buffers ``w8`` / ``ws``, optional fp32 ``bias``."""

    def __init__(self, in_f, out_f, bias=False):
        super().__init__()
        if in_f <= 0 or out_f <= 0:
            raise ValueError(f"in_f/out_f must be positive, got {in_f}/{out_f}")
        self.in_f, self.out_f = in_f, out_f
        bound = 1.0 / math.sqrt(in_f)  # nn.Linear's default distribution
        w8, ws = quantize(torch.empty(out_f, in_f).uniform_(-bound, bound))
        self.register_buffer("w8", w8)
        self.register_buffer("ws", ws)
        self.bias = nn.Parameter(torch.zeros(out_f)) if bias else None

    @classmethod
    def from_float(cls, lin):
        """An FP8BlockLinear holding ``lin``'s weight (and bias) quantized."""
        m = cls(lin.in_features, lin.out_features, lin.bias is not None).to(lin.weight.device)
        m._set(lin.weight, lin.bias)
        return m

    @classmethod
    def from_fp8(cls, lin):
        """An FP8BlockLinear holding an ``FP8Linear``'s decoded weight (and bias) quantized."""
        m = cls(lin.in_f, lin.out_f, lin.bias is not None).to(lin.w8.device)
        m._set(decode_block(lin.w8, lin.sc.float(), 0, lin.out_f, lin.in_f, lin.tile), lin.bias)
        return m

    @torch.no_grad()
    def _set(self, weight, bias):
        w8, ws = quantize(weight)
        self.w8.copy_(w8)
        self.ws.copy_(ws)
        if bias is not None:
            self.bias.copy_(bias.detach())

    def forward(self, x):
        nodes = _check_leaves(x, self.bias)
        y = _Matmul.apply(x, self.w8, self.ws, self.in_f, self.out_f)
        if self.bias is not None:
            y = y + self.bias
        del nodes
        return y

    def extra_repr(self):
        return f"in_f={self.in_f}, out_f={self.out_f}, bias={self.bias is not None}"


class _AddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        s, y = get_backend().add_rms_norm(x, residual, weight, eps)
        ctx.eps, ctx.wtype = eps, None if weight is None else weight.dtype
        ctx.save_for_backward(s, weight)
        ctx.set_materialize_grads(False)  # a sum that nothing uses has no gradient to read
        if residual is None:
            s = s.view_as(s)  # an output of its own
        return y, s

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds):
        s, weight = ctx.saved_tensors
        need_dw = weight is not None and ctx.needs_input_grad[2]
        dy = torch.zeros_like(s) if dy is None else dy.to(s.dtype)
        ds = None if ds is None else ds.to(s.dtype)
        dx, dw = get_backend().add_rms_norm_backward(dy, s, weight, ctx.eps, ds, need_dw)
        return dx, dx if ctx.needs_input_grad[1] else None, dw.to(ctx.wtype) if need_dw else None, None


class AddRMSNorm(nn.Module):
    """(y, s): s = x + residual (x without one), y = RMSNorm(s) in x's type, one device pass.

    Rows of another type than fp32 or bf16 and addends of two types are cast first, s is in the
    type of their sum (which y is formed from in fp32 then, not rounded) and gradients in their own."""

    def __init__(self, d, eps=1e-6):
        super().__init__()
        if d <= 0:
            raise ValueError(f"d must be positive, got {d}")
        if not math.isfinite(eps) or eps <= 0:
            raise ValueError(f"RMSNorm eps must be positive finite, got {eps!r}")
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(d))

    def forward(self, x, residual=None):
        nodes = _check_leaves(x, residual, self.weight)
        a, b, total = _addends(x, residual)
        y, s = _AddRMSNorm.apply(a, b, self.weight, self.eps)
        del nodes
        return y.to(x.dtype if x.is_floating_point() else total), s.to(total)

    def extra_repr(self):
        return f"d={self.weight.numel()}, eps={self.eps}"


class _FFN(torch.autograd.Function):
    """The block on rows, or on the norm of a sum (eps given): (y, s)."""

    @staticmethod
    def forward(ctx, x, residual, norm_weight, eps, d, h, trainable, need, *weights):
        be = get_backend()
        ctx.wtypes = [w.dtype for w in weights] if trainable else None
        codes = [t for w in weights for t in be.fp8_block_quantize(_rows(w))] if trainable else list(weights)
        if eps is None:
            s, rows, xs = None, x, None
            if x.dtype != torch.bfloat16:  # rounded once, from its own type
                rows, xs = be.fp8_block_quantize(_rows(x))
        else:
            s, rows, xs = be.add_rms_norm(x, residual, norm_weight, eps, quantize=True)
        y = be.fp8_block_ffn_forward(rows, codes, d, h, xs=xs, save=need)
        if need:
            y, saved = y
            if not trainable:  # only the weights' gradients read the codes
                saved = (None, None, None, None, saved[4])
            ctx.dims, ctx.xtype, ctx.wtype = (d, h, eps), x.dtype, None if norm_weight is None else norm_weight.dtype
            ctx.save_for_backward(s, norm_weight, *codes, *saved)
            ctx.set_materialize_grads(False)
        y = y.to(x.dtype if x.is_floating_point() else torch.float32)
        if eps is None:
            return y
        return y, s.view_as(s) if residual is None else s

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds=None):
        be = get_backend()
        s, norm_weight, *rest = ctx.saved_tensors
        (d, h, eps), codes, saved = ctx.dims, rest[:6], rest[6:]
        need_dw = ctx.wtypes is not None and any(ctx.needs_input_grad[8:])
        need_norm = norm_weight is not None and ctx.needs_input_grad[2]
        need_dx = ctx.needs_input_grad[0] or ctx.needs_input_grad[1] or need_norm
        dy = torch.zeros_like(s, dtype=torch.bfloat16) if dy is None else dy.to(torch.bfloat16)
        dx, *dw = be.fp8_block_ffn_backward(dy, codes, saved, d, h, need_dx, need_dw)
        dn = None
        if need_dx:
            dx = dx.to(ctx.xtype)
            if eps is not None:
                ds = None if ds is None else ds.to(s.dtype)
                dx, dn = be.add_rms_norm_backward(dx, s, norm_weight, eps, ds, need_norm)
        dw = [g.to(t) for g, t in zip(dw, ctx.wtypes)] if need_dw else [None] * (3 if ctx.wtypes is not None else 6)
        return (dx if ctx.needs_input_grad[0] else None, dx if ctx.needs_input_grad[1] else None,
                dn.to(ctx.wtype) if need_norm else None, None, None, None, None, None, *dw)


class FP8BlockFFN(nn.Module):
    """down(silu(gate(x)) * up(x)) with 8-bit weights, rows and hidden rows.

    Frozen: buffers ``gate_w`` / ``gate_s``, ... in the format; ``trainable``: float
    parameters ``gate``, ``up`` and ``down``, rounded in every forward pass."""

    _NAMES = ("gate_w", "gate_s", "up_w", "up_s", "down_w", "down_s")

    def __init__(self, d, h, trainable=False):
        super().__init__()
        if d <= 0 or h <= 0:
            raise ValueError(f"d and h must be positive, got {d} and {h}")
        self.d, self.h, self.trainable = d, h, bool(trainable)
        for name, n, k in (("gate", h, d), ("up", h, d), ("down", d, h)):
            bound = 1.0 / math.sqrt(k)  # nn.Linear's default distribution
            self._hold(name, torch.empty(n, k).uniform_(-bound, bound))

    def _hold(self, name, weight):
        if self.trainable:
            setattr(self, name, nn.Parameter(weight))
        else:
            w, s = quantize(weight)
            self.register_buffer(name + "_w", w)
            self.register_buffer(name + "_s", s)

    @classmethod
    def from_swiffn(cls, ffn, trainable=False, **kw):
        """The block of a ``SwiFFN``'s decoded weights."""
        lins = (ffn.gate, ffn.up, ffn.down)
        m = cls(ffn.gate.in_f, ffn.gate.out_f, trainable, **kw).to(ffn.gate.w8.device)
        with torch.no_grad():
            for name, lin in zip(("gate", "up", "down"), lins):
                w = decode_block(lin.w8, lin.sc.float(), 0, lin.out_f, lin.in_f, lin.tile)
                if trainable:
                    getattr(m, name).copy_(w)
                else:
                    for suffix, t in zip(("_w", "_s"), quantize(w)):
                        getattr(m, name + suffix).copy_(t)
        return m

    def _weights(self):
        if self.trainable:
            return self.gate, self.up, self.down
        return tuple(getattr(self, n) for n in self._NAMES)

    def _apply_block(self, x, residual, norm_weight, eps):
        weights = self._weights()
        nodes = _check_leaves(x, residual, norm_weight, *weights)
        # a recorded pass keeps what its gradients need
        need = torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                               for t in (x, residual, norm_weight, *weights))
        a, b, total = (x, None, None) if eps is None else _addends(x, residual)
        y = _FFN.apply(a, b, norm_weight, eps, self.d, self.h, self.trainable, need, *weights)
        del nodes
        if eps is None:
            return y
        return y[0].to(x.dtype if x.is_floating_point() else total), y[1].to(total)

    def forward(self, x):
        return self._apply_block(x, None, None, None)

    def extra_repr(self):
        return f"d={self.d}, h={self.h}, trainable={self.trainable}"


class FP8BlockNormFFN(FP8BlockFFN):
    """(y, s): s = x + residual (x without one), y = the block on RMSNorm(s), whose codes
    the norm writes itself (rounded once, from fp32).  Types as ``AddRMSNorm``'s."""

    def __init__(self, d, h, trainable=False, eps=1e-6):
        super().__init__(d, h, trainable)
        if not math.isfinite(eps) or eps <= 0:
            raise ValueError(f"RMSNorm eps must be positive finite, got {eps!r}")
        self.eps = eps
        self.norm = nn.Parameter(torch.ones(d))

    def forward(self, x, residual=None):
        return self._apply_block(x, residual, self.norm, self.eps)

    def extra_repr(self):
        return super().extra_repr() + f", eps={self.eps}"
