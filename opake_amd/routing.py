"""Routing of tokens to experts.

``route_topk`` turns router logits into each token's ``k`` experts and their
weights in one launch, and its backward is one launch too (``csrc/route.hip``).
The reference routes by softmax and top-k (packages/opake-patches/src/opake/api/
patches/kernels/moe.py:570-627).  Routers trained without a balancing loss have sigmoid
scores, a balancing bias and groups by the sum of their two best experts
(``group_score="top2"``); earlier ones groups by their best alone.
"""

from __future__ import annotations

import torch

from opake_amd import _native as nat
from opake_amd.exceptions import ConfigurationError, InputTypeError

MAX_EXPERTS = 1024
MAX_TOP_K = 64
_LARGEST = torch.finfo(torch.float32).max
_SCORES = {"softmax": nat.ROUTE_SOFTMAX, "sigmoid": nat.ROUTE_SIGMOID}
_GROUP_SCORES = {"max": 0, "top2": nat.ROUTE_GROUPS_BY_TWO}


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, options):
        code, k, score, groups, top_groups, group_score, renormalize, scale = options
        dev = logits.device
        z = logits.contiguous()
        lead, E = z.shape[:-1], z.shape[-1]
        weights = torch.empty((*lead, k), dtype=torch.float32, device=dev)
        experts = torch.empty((*lead, k), dtype=torch.int64, device=dev)
        nat.call_on(dev, "dpc_route_topk", z.data_ptr(), z.numel() // E, E, code,
                    0 if bias is None else bias.data_ptr(), k, score | group_score, groups,
                    top_groups, renormalize, scale, weights.data_ptr(), experts.data_ptr())
        ctx.mark_non_differentiable(experts)
        if ctx.needs_input_grad[0]:
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(logits, weights, experts)
            ctx.options = (code, k, score, renormalize, scale)
        return weights, experts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        if grad is None:
            return None, None, None
        logits, weights, experts = ctx.saved_tensors
        z = logits.contiguous()
        E = z.shape[-1]
        g = (grad if grad.dtype == torch.float32 else grad.float()).contiguous()
        dz = torch.empty_like(z)
        code, k, score, renormalize, scale = ctx.options
        nat.call_on(z.device, "dpc_route_topk_grad", z.data_ptr(), z.numel() // E, E, code, k,
                    score, renormalize, scale, experts.data_ptr(), weights.data_ptr(),
                    g.data_ptr(), dz.data_ptr())
        return dz, None, None


def route_topk(logits: torch.Tensor, k: int, *, score: str = "softmax",
               bias: torch.Tensor | None = None, groups: int = 1, top_groups: int | None = None,
               group_score: str = "max", renormalize: bool = True, scale: float = 1.0):
    """Experts and weights of every token: ``(weights float32 [..., k], experts int64 [..., k])``.

    ``logits`` [..., E] (float32, bfloat16 or float16, E <= 1024).  ``score``:
    ``"softmax"`` over the experts or ``"sigmoid"`` of each.  ``bias`` [E] (float32)
    is added to the scores for the choice only, as a balancing rule adjusts it; it
    has no gradient.  ``groups``: the experts form that many equal groups of
    consecutive ones, and only the ``top_groups`` best of them take part (all by
    default): by ``group_score`` those with the best expert (``"max"``) or with the
    largest sum of their two best experts' scores plus bias (``"top2"``; of one
    unmasked expert, that one's).  The ``k`` best come in descending order, ties to the
    lower index.  Their weights are the scores, divided by their sum if ``renormalize``,
    times ``scale``; gradients reach ``logits`` through them.

    An expert whose logit is -inf (masked) is never chosen: a token with fewer than
    ``k`` left gets expert -1 with weight 0 in its last places.  A NaN logit makes
    its token's weights NaN."""
    nat.require_device(logits, bias)
    for name, v in (("k", k), ("groups", groups), ("top_groups", top_groups)):
        if v is not None and (isinstance(v, bool) or not isinstance(v, int)):
            raise InputTypeError(f"{name} must be an int, got {type(v)}")
    if isinstance(scale, bool) or not isinstance(scale, (int, float)):
        raise InputTypeError(f"scale must be a number, got {type(scale)}")
    if score not in _SCORES:
        raise ConfigurationError(f"score must be one of {sorted(_SCORES)}, got {score!r}")
    if group_score not in _GROUP_SCORES:
        raise ConfigurationError(
            f"group_score must be one of {sorted(_GROUP_SCORES)}, got {group_score!r}")
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ConfigurationError(
            f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_EXPERTS:
        raise ConfigurationError(
            f"expected logits [..., E] with 1 <= E <= {MAX_EXPERTS}, got {tuple(logits.shape)}")
    E = logits.shape[-1]
    top_groups = groups if top_groups is None else top_groups
    if groups < 1 or E % groups or not 1 <= top_groups <= groups:
        raise ConfigurationError(
            f"{E} experts need groups that divide them and 1 <= top_groups <= groups, got "
            f"{groups} and {top_groups}")
    if not 1 <= k <= min(MAX_TOP_K, top_groups * (E // groups)):
        raise ConfigurationError(
            f"k must be between 1 and {min(MAX_TOP_K, top_groups * (E // groups))}, got {k}")
    if not abs(scale) <= _LARGEST:
        raise ConfigurationError(f"scale must be a finite float32, got {scale}")
    if bias is not None:
        if bias.dtype != torch.float32 or tuple(bias.shape) != (E,):
            raise ConfigurationError(f"bias must be float32 [{E}], got {bias.dtype} "
                                     f"{tuple(bias.shape)}")
        bias = bias.detach().contiguous()
    return _Route.apply(logits, bias,
                        (nat.dtype_code(logits.dtype, wide=True), k, _SCORES[score], groups,
                         top_groups, _GROUP_SCORES[group_score], int(bool(renormalize)),
                         float(scale)))


__all__ = ["MAX_EXPERTS", "MAX_TOP_K", "route_topk"]
