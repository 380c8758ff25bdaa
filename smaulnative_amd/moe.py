"""``SwiFFN`` and ``SwiFFN_MoE`` with the reference's interface (model.py:282-290, 506-606).

``SwiFFN_MoE.forward(x)`` keeps the reference signature, output dtype and the
diagnostic attributes read by training logs and retention reports:
``last_prob``, ``last_topi``, ``last_executed``, ``expert_token_counts``,
``routing_stats()``, ``reset_routing_stats()``, ``balance_loss(prob)``.

The whole layer (router, dispatch, the expert SwiGLU GEMMs, combine) is one
call to the backend's ``moe_forward``; the per-expert Python loop with a host
sync per expert (model.py:574-582) is gone.  When autograd must record the
layer (grad mode on and the input or a parameter requiring grad, in train and
eval mode alike) it runs as device torch ops around the experts' FP8Linear
kernels instead, so gradients reach the input, the router and the experts'
weight gradients (``_forward_train``).  ``expert_token_counts`` and
``last_executed`` are materialised from the device counts only when read, so
a decode step does not force a device->host sync per layer.

Only the plain architecture's dense SwiGLU experts are on this path; the rawr
(sparse) experts are not (model.py:528-534).

Beyond the reference, a config may ask for another router (``router_*``: sigmoid
scores, groups, a balance bias, no renormalisation, a scale; the backend's
``moe_route`` in place of its softmax router) and for experts in 4 bits
(``precision="mx4"``, ``MX4Experts``).
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from smaulnative_amd.compute import get_backend
from smaulnative_amd.fp8_tile import FP8Linear


@dataclass
class MoEConfig:
    """The LinearConfig fields (model.py:18-40) the MoE layer reads.

    A reference ``LinearConfig`` instance works in its place (same names).
    """
    d_model: int = 512
    ffn_mult: float = 2.5
    tile: int = 64
    num_experts: int = 1
    num_experts_per_tok: int = 1
    precision: str = "fp8"  # "mx4": experts in microscaled 4-bit floating point
    architecture: str = "plain"
    # the router (RocmBackend.moe_route); a config without these has the softmax top-k
    router_score: str = "softmax"
    router_groups: int = 1
    router_top_groups: int | None = None
    router_group_best: int = 2
    router_renorm: bool = True
    router_scale: float = 1.0
    router_bias: bool = False  # a balance bias of the choice, moved by balance_step()
    expert_act: str = "keep"  # mx4 experts: "mx4" rounds their activations too

    def __post_init__(self):
        for name in ("d_model", "tile", "num_experts", "num_experts_per_tok"):
            v = getattr(self, name)
            if not isinstance(v, int) or v <= 0:
                raise ValueError(f"{name} must be a positive int, got {v!r}")
        if self.num_experts_per_tok > self.num_experts:
            raise ValueError(f"num_experts_per_tok ({self.num_experts_per_tok}) > "
                             f"num_experts ({self.num_experts})")


# of one call of the backend's layer entries and its dispatch
_CALL_EXPERTS, _CALL_SLOTS = 64, 8


def _router_fields(cfg) -> dict:
    """moe_route's arguments from a config's ``router_*`` fields, unchecked."""
    args = dict(score=getattr(cfg, "router_score", "softmax"), groups=getattr(cfg, "router_groups", 1),
                top_groups=getattr(cfg, "router_top_groups", None), group_best=getattr(cfg, "router_group_best", 2),
                renorm=getattr(cfg, "router_renorm", True), scale=getattr(cfg, "router_scale", 1.0))
    if args["top_groups"] is None:
        args["top_groups"] = args["groups"]
    return args


def is_plain_router(cfg) -> bool:
    """Whether a config's router is the reference's: softmax, top-k, renormalised."""
    args = _router_fields(cfg)
    return args["score"] == "softmax" and args["top_groups"] == args["groups"] and bool(args["renorm"]) and \
        args["scale"] == 1.0 and not getattr(cfg, "router_bias", False)


def _needs_grad(module: nn.Module, x: torch.Tensor) -> bool:
    """Whether the forward must record autograd: grad mode on and x or a
    parameter of ``module`` requiring grad, in train and eval mode alike (as
    with the reference's autograd function, kernel/fp8_tile.py:162-170; the
    module's training flag only decides whether FP8Linear accumulates ``_gw``).
    The fused device entries keep no activations, so they run only otherwise."""
    if not torch.is_grad_enabled():
        return False
    return x.requires_grad or any(p.requires_grad for p in module.parameters())


class _SwiGLU(torch.autograd.Function):
    """(silu(gate.float()) * up.float()).to(gate.dtype) and its gradients, a device
    pass each."""

    @staticmethod
    def forward(ctx, gate, up):
        ctx.save_for_backward(gate, up)
        return get_backend().swiglu(gate, up)

    @staticmethod
    def backward(ctx, dout):
        gate, up = ctx.saved_tensors
        if torch.is_grad_enabled():  # a graph of the gradients is wanted: tensor operations
            g, u, d = gate.float(), up.float(), dout.float()
            sig = torch.sigmoid(g)
            return (d * u * sig * (1 + g * (1 - sig))).to(gate.dtype), (d * (g * sig)).to(up.dtype)
        return tuple(get_backend().swiglu_backward(dout, gate, up))


def _swiglu(gate, up, dtype):
    """(silu(gate.float()) * up.float()).to(dtype) of a SwiFFN being trained."""
    if gate.is_cuda and gate.dtype == up.dtype == dtype and dtype in (torch.float32, torch.bfloat16) and \
            hasattr(get_backend(), "swiglu"):
        return _SwiGLU.apply(gate, up)
    return (F.silu(gate.float()) * up.float()).to(dtype)


def _sum_slots(y, at, weight=None):
    """[T, d]: the sum over each token's slots of y[at] (times weight [T, k, 1]);
    a slot with at < 0 has no row and adds nothing (``at`` is full: none has)."""
    at, full = at
    T, k = at.shape
    rows = (at if full else at.clamp_min(0)).view(-1)
    yk = y.index_select(0, rows).view(T, k, y.shape[1])
    if not full:  # before the product: a dropped slot's weight may be NaN, its gradients are zero
        has = (at >= 0).unsqueeze(-1)
        yk = torch.where(has, yk, torch.zeros_like(yk))
        weight = weight if weight is None else torch.where(has, weight, torch.zeros_like(weight))
    if weight is not None:
        yk = yk * weight
    return yk.sum(1)


class _GatherRows(torch.autograd.Function):
    """x[rows], every expert's rows; the gradient gathers a token's slots in order
    (index_select's own would add them up with atomics)."""

    @staticmethod
    def forward(ctx, x, rows, at, full):
        ctx.save_for_backward(at)
        ctx.full = full
        return x.index_select(0, rows)

    @staticmethod
    def backward(ctx, dy):
        return _sum_slots(dy, (ctx.saved_tensors[0], ctx.full)), None, None, None


class _Route(torch.autograd.Function):
    """(prob, topi, topw) of the backend's ``moe_route``, differentiable in the logits
    through the scores and the chosen weights (the choice is a constant)."""

    @staticmethod
    def forward(ctx, logits, bias, top_k, args):
        ctx.set_materialize_grads(False)
        prob, topi, topw = get_backend().moe_route(logits, top_k, bias=bias, **args)
        ctx.mark_non_differentiable(topi)
        ctx.save_for_backward(logits, topi)
        ctx.args = {n: args[n] for n in ("score", "renorm", "scale")}
        return prob, topi, topw

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dprob, dtopi, dtopw):
        logits, topi = ctx.saved_tensors
        if dtopw is None:
            if dprob is None:
                return None, None, None, None
            dtopw = torch.zeros(topi.shape, dtype=torch.float32, device=topi.device)
        return get_backend().moe_route_backward(dtopw, logits, topi, dprob=dprob, **ctx.args), None, None, None


class SwiFFN(nn.Module):
    """model.py:282-290: down((silu(gate(x).float()) * up(x).float()).to(x.dtype))."""

    def __init__(self, cfg):
        super().__init__()
        if cfg.precision != "fp8":
            raise ValueError("the rocm path implements precision='fp8' experts only")
        h = int(cfg.d_model * cfg.ffn_mult)
        self.gate = FP8Linear(cfg.d_model, h, cfg.tile)
        self.up = FP8Linear(cfg.d_model, h, cfg.tile)
        self.down = FP8Linear(h, cfg.d_model, cfg.tile)

    def forward(self, x):
        be = get_backend()
        if hasattr(be, "swiffn_forward") and not _needs_grad(self, x):
            xf = x if x.is_floating_point() else x.float()
            return be.swiffn_forward(xf, self.buffers6(), self.gate.tile)
        odt = x.dtype if x.is_floating_point() else torch.float32
        return self.down(_swiglu(self.gate(x), self.up(x), odt))

    def buffers6(self):
        # straight from the modules' dictionaries: nine attribute searches per
        # expert through nn.Module.__getattr__ take a decode call 3 us each expert
        try:
            mods = self._modules
            g, u, d = mods["gate"]._buffers, mods["up"]._buffers, mods["down"]._buffers
            return (g["w8"], g["sc"], u["w8"], u["sc"], d["w8"], d["sc"])
        except (KeyError, AttributeError):  # a buffer replaced by a plain attribute
            return (self.gate.w8, self.gate.sc, self.up.w8, self.up.sc, self.down.w8, self.down.sc)


class SwiFFN_MoE(nn.Module):
    """Top-k routed mixture of SwiFFN experts (model.py:506-606)."""

    def __init__(self, cfg, rawr_graph=None):
        super().__init__()
        if cfg.num_experts < 1 or cfg.num_experts_per_tok < 1:
            raise ValueError("num_experts and num_experts_per_tok must be >= 1")
        if cfg.num_experts_per_tok > cfg.num_experts:
            raise ValueError(
                f"num_experts_per_tok ({cfg.num_experts_per_tok}) > num_experts ({cfg.num_experts})")
        if getattr(cfg, "architecture", "plain") != "plain":
            raise ValueError("the rocm MoE path implements architecture='plain' (SwiFFN experts) only")
        self.top_k = cfg.num_experts_per_tok
        self.num_experts = cfg.num_experts
        self.architecture = "plain"
        self.tile = cfg.tile
        if cfg.precision == "mx4":
            from smaulnative_amd.mx4 import MX4Experts
            self.experts = MX4Experts(cfg.num_experts, cfg.d_model, int(cfg.d_model * cfg.ffn_mult),
                                      getattr(cfg, "expert_act", "keep"))
        else:
            self.experts = nn.ModuleList([SwiFFN(cfg) for _ in range(cfg.num_experts)])
        self.gate = nn.Linear(cfg.d_model, cfg.num_experts, bias=False)
        self.route_args = self._route_config(cfg)
        if getattr(cfg, "router_bias", False):
            self.register_buffer("balance_bias", torch.zeros(cfg.num_experts))
        else:
            self.balance_bias = None
        self.last_prob = None
        self.last_topi = None
        self._counts_dev = None
        self._counts_host = [0] * cfg.num_experts

    @staticmethod
    def _route_config(cfg):
        """moe_route's arguments from the config's ``router_*`` fields, or None for the
        reference's router (softmax, top-k, renormalised)."""
        E, k = cfg.num_experts, cfg.num_experts_per_tok
        args = _router_fields(cfg)
        if args["score"] not in ("softmax", "sigmoid"):
            raise ValueError(f"router_score must be 'softmax' or 'sigmoid', got {args['score']!r}")
        if args["groups"] < 1 or E % args["groups"] or not 1 <= args["top_groups"] <= args["groups"] or \
                args["top_groups"] * (E // args["groups"]) < k:
            raise ValueError(f"router_groups ({args['groups']}) must divide the {E} experts and router_top_groups "
                             f"({args['top_groups']}) of them hold {k}")
        if args["group_best"] not in (1, 2):
            raise ValueError(f"router_group_best must be 1 or 2, got {args['group_best']!r}")
        if is_plain_router(cfg) and cfg.precision != "mx4":
            return None
        if not 0.0 < args["scale"] < math.inf:
            raise ValueError(f"router_scale must be positive and finite, got {args['scale']!r}")
        if E > 512 or k > 16 or args["groups"] > 64:
            raise ValueError(f"the router takes up to 512 experts, 16 a token and 64 groups, got {E}, {k} and "
                             f"{args['groups']}")
        return args

    def __setstate__(self, state):
        super().__setstate__(state)
        # a layer pickled before there were other routers
        self.__dict__.setdefault("route_args", None)
        if "balance_bias" not in self._buffers:
            self.__dict__.setdefault("balance_bias", None)

    def _apply(self, fn, *args, **kwargs):
        kept = self.balance_bias
        super()._apply(fn, *args, **kwargs)
        # moves with the layer, but stays fp32: 16 bits would swallow balance_step's steps
        if kept is not None and self.balance_bias.dtype != kept.dtype and not kept.is_meta:
            self.balance_bias = kept.to(self.balance_bias.device)
        return self

    @torch.no_grad()
    def balance_step(self, rate: float) -> None:
        """Moves the balance bias by ``rate`` towards the experts that got fewer rows than
        their share in the last forward, and away from the others."""
        if self.balance_bias is None:
            raise RuntimeError("balance_step: the layer has no balance bias (router_bias)")
        counts = self._counts_dev
        counts = torch.tensor(self._counts_host, device=self.balance_bias.device) if counts is None else counts
        counts = counts.to(self.balance_bias.dtype)
        self.balance_bias.add_(torch.sign(counts.mean() - counts), alpha=rate)

    # -- diagnostics (model.py:538-543,583-584,587-606), materialised lazily --
    @property
    def expert_token_counts(self):
        if self._counts_dev is not None:
            self._counts_host = [int(c) for c in self._counts_dev.tolist()]
            self._counts_dev = None
        return self._counts_host

    @expert_token_counts.setter
    def expert_token_counts(self, value):
        self._counts_dev = None
        self._counts_host = list(value)

    @property
    def last_executed(self):
        return [c > 0 for c in self.expert_token_counts]

    @last_executed.setter
    def last_executed(self, value):
        # kept for interface compatibility; executed is derived from counts
        pass

    def balance_loss(self, prob: torch.Tensor) -> torch.Tensor:
        """Switch-style load-balancing aux loss (model.py:545-555)."""
        density = prob.mean(0)
        return (density * density * self.num_experts).sum()

    def forward(self, x):
        be = get_backend()
        if not hasattr(be, "moe_forward"):
            raise RuntimeError(f"compute backend {be.name!r} has no moe_forward entry")
        if _needs_grad(self, x):
            return self._forward_train(x)
        if self.route_args is not None or not isinstance(self.experts, nn.ModuleList):
            out, prob, topi, counts = self._forward_routed(be, x)
        else:
            experts = [ex.buffers6() for ex in self.experts]
            out, prob, topi, counts = be.moe_forward(x, self.gate.weight, self.gate.bias, experts,
                                                     self.top_k, self.tile)
        # plain attributes (or a subclass's properties), set past
        # nn.Module.__setattr__ (3 us each): none is a parameter, buffer or module
        for name, value in (("last_prob", prob), ("last_topi", topi), ("_counts_dev", counts)):
            object.__setattr__(self, name, value)
        return out

    def _logits(self, xs):
        bias = None if self.gate.bias is None else self.gate.bias.float()
        return F.linear(xs.float(), self.gate.weight.float(), bias)

    def _forward_routed(self, be, x):
        """(out, prob, topi, counts): the router's logits, ``moe_route``, and the experts on
        that routing."""
        lead, k = x.shape[:-1], self.top_k
        xs = x.reshape(-1, x.shape[-1])
        prob, topi, topw = be.moe_route(self._logits(xs), k, bias=self.balance_bias, **(self.route_args or {}))
        xs = xs if xs.is_floating_point() else xs.float()
        fp8 = isinstance(self.experts, nn.ModuleList)
        if k > _CALL_SLOTS or xs.shape[-1] % 8 or xs.dtype not in (torch.float32, torch.bfloat16) or \
                not (fp8 or self.experts.act == "keep" or xs.dtype == torch.bfloat16):
            # what the entries do not take runs expert by expert, as in training (with a
            # host synchronisation each: not to be captured)
            out, counts = self._experts_by_mask(xs, topi, topw)
            out, counts = out.to(xs.dtype), torch.tensor(counts, dtype=torch.int32, device=xs.device)
        else:
            # More experts than one call takes: equal parts, a call each.  The slots of other
            # parts are outside [0, E) there and add nothing; the parts' sums, each rounded
            # to x's type, are added in fp32.
            parts = -(-self.num_experts // _CALL_EXPERTS)
            step = -(-self.num_experts // parts)
            calls = [self._part(be, xs, prob, topi, topw, lo, min(lo + step, self.num_experts))
                     for lo in range(0, self.num_experts, step)]
            out, counts = calls[0]
            if parts > 1:
                out = sum((part.float() for part, _ in calls[1:]), out.float()).to(xs.dtype)
                counts = torch.cat([c for _, c in calls])
        return out.view(x.shape), prob.view(*lead, self.num_experts), topi.view(*lead, k), counts

    def _part(self, be, xs, prob, topi, topw, lo, hi):
        """(out, counts) of the experts lo to hi on a routing among all of them."""
        whole = hi - lo == self.num_experts
        topi = topi if whole else topi - lo
        if not isinstance(self.experts, nn.ModuleList):
            experts = self.experts.buffers6()
            return be.mx4_moe_forward(xs, topi, topw, experts if whole else tuple([b[lo:hi] for b in experts]),
                                      self.experts.act)
        experts = [ex.buffers6() for ex in self.experts]
        weight, bias = self.gate.weight, self.gate.bias
        if not whole:  # of the router's arguments only topi and topw are read
            weight, bias, experts = weight[lo:hi], None, experts[lo:hi]
            prob = prob.new_empty(prob.shape[0], hi - lo)
        out, _, _, counts = be.moe_forward(xs, weight, bias, experts, self.top_k, self.tile, routing=(prob, topi, topw))
        return out, counts

    def _forward_train(self, x):
        """The layer with autograd, for training.

        The router softmax, top-k and renormalisation of model.py:557-570 as
        torch ops on the device (gradient reaches the router through the
        selected probabilities only, as in the reference); each expert's rows
        gathered and run through its SwiFFN, whose FP8Linear modules compute
        the forward and the input gradient with the backend's kernels and
        accumulate their weight gradients in ``_gw``; the weighted outputs added
        back token by token in ascending expert order (model.py:571-585).  The
        fused moe_forward path has no backward, so training runs this one.
        """
        d = x.shape[-1]
        lead = x.shape[:-1]
        xs = x.reshape(-1, d)
        if self.route_args is not None or not isinstance(self.experts, nn.ModuleList):
            prob, topi, topv = _Route.apply(self._logits(xs), self.balance_bias, self.top_k,
                                            self.route_args or dict(score="softmax", renorm=True, scale=1.0))
        else:
            prob = torch.softmax(self.gate(xs.float()), -1)
            topv, topi = torch.topk(prob, self.top_k, -1)
            total = topv.sum(-1, keepdim=True)
            topv = torch.where(total < 1e-6, torch.full_like(topv, 1.0 / self.top_k), topv / total.clamp_min(1e-9))
        # kept with x's leading dimensions, as the reference's are (model.py:558-565)
        self.last_prob = prob.view(*lead, self.num_experts)
        self.last_topi = topi.detach().view(*lead, self.top_k)
        if xs.is_cuda and 0 < xs.shape[0] * self.top_k < 1 << 31 and self.num_experts <= _CALL_EXPERTS and \
                self.top_k <= _CALL_SLOTS and hasattr(get_backend(), "moe_dispatch"):
            out, counts = self._experts_dispatched(xs, topi, topv)
        else:
            out, counts = self._experts_by_mask(xs, topi, topv)
        self.expert_token_counts = counts
        return out.view(x.shape).to(x.dtype if x.is_floating_point() else torch.float32)

    def _experts_by_mask(self, xs, topi, topv):
        """The experts' weighted outputs [T, d] fp32 and token counts, each expert's
        rows found by its own mask (a host synchronisation per expert)."""
        out = torch.zeros(xs.shape, dtype=torch.float32, device=xs.device)
        counts = []
        for e, expert in enumerate(self.experts):
            weight = torch.where(topi == e, topv, torch.zeros_like(topv)).sum(-1)
            rows = torch.nonzero(weight > 0).squeeze(-1)
            counts.append(int(rows.numel()))
            if counts[-1]:
                y = expert(xs.index_select(0, rows)).float() * weight.index_select(0, rows).unsqueeze(-1)
                out = out.index_add(0, rows, y)
        return out, counts

    def _experts_dispatched(self, xs, topi, topv):
        """The same from the backend's dispatch: one synchronisation, one gather of
        every expert's rows (ascending tokens, as the masks give them) and, per
        token, its experts' outputs in ascending expert order."""
        T, k = topi.shape
        disp = get_backend().moe_dispatch(topi, topv.detach(), self.num_experts, 64)
        counts = disp["counts"].tolist()
        n = sum(counts)
        if n == 0:
            return torch.zeros(xs.shape, dtype=torch.float32, device=xs.device), counts
        order = topi.argsort(-1) if k > 1 else torch.zeros_like(topi)
        at = disp["inv"][:T * k].view(T, k).gather(1, order)  # the slots' rows, by expert
        full = n == T * k
        rows = _GatherRows.apply(xs, disp["perm_row"][:n], at, full).split(counts)
        y = torch.cat([expert(r) for expert, r in zip(self.experts, rows) if r.shape[0]]).float()
        return _sum_slots(y, (at, full), topv.gather(1, order).unsqueeze(-1)), counts

    def routing_stats(self) -> dict:
        counts = list(self.expert_token_counts)
        total = sum(counts)
        usage = [(c / total) if total else 0.0 for c in counts]
        return {
            "num_experts": self.num_experts,
            "top_k": self.top_k,
            "token_counts": counts,
            "usage_frac": usage,
            "executed": [c > 0 for c in counts],
            "inactive_experts": sum(1 for c in counts if c == 0),
            "max_usage_frac": max(usage) if usage else 0.0,
        }

    def reset_routing_stats(self) -> None:
        self.last_prob = None
        self.last_topi = None
        self._counts_dev = None
        self._counts_host = [0] * self.num_experts
