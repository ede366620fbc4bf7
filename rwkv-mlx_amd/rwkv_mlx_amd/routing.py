"""Routing of tokens to experts with the options that models of many experts
use, from logits: softmax or sigmoid scores, a bias that balances the experts'
load, groups of experts, renormalised and scaled gates.

``route_topk`` is the operator (``rwkvmoe_route``, differentiable through
``rwkvmoe_route_backward``); ``GroupRouter`` a router module around it with the
interface of ``Router`` (the reference's rwkv_mlx/moe.py:35-86, which is the
softmax case without groups and bias).
"""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .model import require_device

__all__ = ["route_topk", "GroupRouter"]

SCORES = {"softmax": 0, "sigmoid": 1}
GROUP_SCORES = {"max": 0, "top2": 1}


def _route(plan, logits, bias):
    desc, shape, k = plan
    inds = torch.empty(*shape, k, dtype=torch.int32, device=logits.device)
    gates = torch.empty(*shape, k, dtype=torch.float32, device=logits.device)
    _lib.launch(_lib.lib().rwkvmoe_route, "rwkvmoe_route", logits.device, desc, logits.data_ptr(),
                None if bias is None else bias.data_ptr(), inds.data_ptr(), gates.data_ptr())
    return inds, gates


class _RouteFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, plan):
        inds, gates = _route(plan, logits, bias)
        ctx.save_for_backward(logits, inds, gates)
        ctx.desc = plan[0]
        ctx.mark_non_differentiable(inds)
        ctx.set_materialize_grads(False)  # (no zeros for inds)
        return inds, gates

    @staticmethod
    @once_differentiable
    def backward(ctx, d_inds, d_gates):
        if d_gates is None:
            return None, None, None
        logits, inds, gates = ctx.saved_tensors
        d_gates = d_gates.to(torch.float32).contiguous()
        # (dense, whatever the strides of logits)
        d_logits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        _lib.launch(_lib.lib().rwkvmoe_route_backward, "rwkvmoe_route_backward", logits.device, ctx.desc,
                    logits.data_ptr(), inds.data_ptr(), gates.data_ptr(), d_gates.data_ptr(), d_logits.data_ptr())
        return d_logits, None, None


def route_topk(logits: torch.Tensor, top_k: int, *, bias: torch.Tensor | None = None, score: str = "softmax",
               n_groups: int = 1, top_groups: int | None = None, group_score: str = "max", renormalize: bool = True,
               scale: float = 1.0):
    """(inds (..., k) int32, gates (..., k) fp32) of logits (..., E).

    s = softmax(l) or sigmoid(l).  Experts are ranked by s + bias (compared in
    64 bits), without a bias by l; ``bias`` (E) only ranks.  With ``n_groups``
    > 1 the experts form consecutive groups, of which the best ``top_groups``
    (default: all) are ranked; a group counts as its best expert ("max") or as
    the sum of the scores (with the bias) of its two best ("top2").  inds are
    best first, ties to the lower index.  gates are s of the selected, divided
    by their sum with ``renormalize``, times ``scale``.

    An expert with a logit (or a bias) of -inf or NaN takes no part: it comes
    after the others of the chosen groups and its gate is 0; a row with nothing
    left has valid, distinct inds and gates of 0.  Differentiable with respect
    to logits (the selection is piecewise constant).  E up to 512, k up to 32,
    up to 64 groups."""
    require_device(logits, "route_topk")
    if logits.dim() < 1 or logits.dtype not in _lib.TORCH_DTYPE_CODE:
        raise TypeError(f"route_topk: logits (..., E) in float32, float16 or bfloat16 expected, got "
                        f"{tuple(logits.shape)} {logits.dtype}")
    if score not in SCORES or group_score not in GROUP_SCORES:
        raise ValueError(f"route_topk: score is one of {list(SCORES)} and group_score of {list(GROUP_SCORES)}; got "
                         f"{score!r}, {group_score!r}")
    E = logits.shape[-1]
    if bias is not None:
        if bias.shape != (E,) or bias.device != logits.device:
            raise ValueError(f"route_topk: bias ({E},) on {logits.device} expected, got {tuple(bias.shape)} on "
                             f"{bias.device}")
        if bias.requires_grad or bias.dtype is not torch.float32 or not bias.is_contiguous():
            bias = bias.detach().to(torch.float32).contiguous()
    shape = logits.shape[:-1]
    # rows of one stride are read in place
    if logits.dim() == 2 and logits.stride(1) == 1 and logits.stride(0) >= E:
        flat = logits
    else:
        flat = logits.reshape(-1, E).contiguous()
    rows = flat.shape[0]
    stride = flat.stride(0) if rows > 1 else E
    desc = _lib.route_desc(rows, E, top_k, n_groups, n_groups if top_groups is None else top_groups,
                           _lib.TORCH_DTYPE_CODE[logits.dtype], SCORES[score], GROUP_SCORES[group_score],
                           _lib.ROUTE_RENORM if renormalize else 0, scale, max(stride, E))
    plan = (desc, shape, top_k)
    if rows == 0:  # nothing to launch; the options are checked all the same
        _lib.check(_lib.lib().rwkvmoe_route(desc, None, None, None, None, None), "rwkvmoe_route")
        return (torch.empty(*shape, top_k, dtype=torch.int32, device=logits.device),
                logits.new_zeros((*shape, top_k), dtype=torch.float32) + logits.sum().to(torch.float32) * 0
                if logits.requires_grad else
                torch.empty(*shape, top_k, dtype=torch.float32, device=logits.device))
    if torch.is_grad_enabled() and flat.requires_grad:
        return _RouteFunction.apply(flat, bias, plan)
    return _route(plan, flat, bias)


class GroupRouter(nn.Module):
    """A router of many experts: gate.weight (E, C), ``route_topk``'s options,
    and a bias that balances the experts' load without a loss
    (``balance_bias``, a buffer: it ranks, it is not trained, and it stays
    float32 when the module is cast, as small steps add up in it).

    Returns what ``Router`` returns, (inds (B,T,k) int32, weights (B,T,k) in
    x's dtype, aux_loss, z_loss), both losses 0: ``update_balance`` takes their
    place.  It routes for ``Fp8MoE_CMix`` and for layers that call their router;
    the layers whose kernels route by themselves refuse it."""

    def __init__(self, d_model: int, n_experts: int, top_k: int = 2, score: str = "sigmoid", n_groups: int = 1,
                 top_groups: int | None = None, group_score: str = "top2", renormalize: bool = True,
                 scale: float = 1.0):
        super().__init__()
        self.gate = nn.Linear(d_model, n_experts, bias=False)
        self.n_experts = n_experts
        self.top_k = top_k
        self.options = dict(score=score, n_groups=n_groups, top_groups=top_groups, group_score=group_score,
                            renormalize=renormalize, scale=scale)
        self.register_buffer("balance_bias", torch.zeros(n_experts))

    @property
    def logit_bias(self):
        # the fused layers read their router's weights, not its result
        raise TypeError("this layer routes in its own kernels, by softmax and top-k; a GroupRouter goes with "
                        "Fp8MoE_CMix")

    def _apply(self, fn, recurse=True):
        bias = self.balance_bias
        super()._apply(fn, recurse)
        if self.balance_bias.dtype != bias.dtype:  # a cast goes past the bias, a move does not
            self.balance_bias = bias.to(self.balance_bias.device)
        return self

    def forward(self, x: torch.Tensor):
        require_device(x, "GroupRouter")
        # fp32 logits, also under autocast: which expert is taken hangs on small differences
        if torch.is_autocast_enabled("cuda"):
            with torch.autocast("cuda", enabled=False):
                return self.forward(x)
        logits = nn.functional.linear(x.to(torch.float32), self.gate.weight.to(torch.float32))
        inds, gates = route_topk(logits, self.top_k, bias=self.balance_bias, **self.options)
        zero = torch.zeros((), dtype=torch.float32, device=x.device)
        return inds, gates.to(x.dtype), zero, zero.clone()

    @torch.no_grad()
    def update_balance(self, inds: torch.Tensor, rate: float = 1e-3) -> None:
        """After a step: the bias of experts with fewer assignments than the
        mean rises by `rate`, that of the others falls."""
        load = torch.bincount(inds.reshape(-1).long(), minlength=self.n_experts).to(torch.float32)
        self.balance_bias.add_(torch.sign(load.mean() - load), alpha=rate)
