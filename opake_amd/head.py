"""Losses of a vocabulary head that never hold its logits.

``linear_cross_entropy`` is the softmax cross entropy of ``hidden @ weight.T``
against one target a token; ``topk_distillation`` is the Kullback-Leibler
divergence from a teacher of which only the top logits were kept.  Both return
one loss a token (float32), so a caller can reduce them per example as
per-example clipping needs, and both are differentiable with respect to ``hidden`` and, where it requires a gradient,
``weight``.

Forward, one matrix-core product leaves the maximum and the sum of
exponentials of every 256-wide piece of the vocabulary per token; backward,
the pieces are computed again and multiplied on at once
(``csrc/head.hip``).  No ``[tokens, vocabulary]`` tensor is kept: the
backward's workspace holds one piece of at most 256 MiB (one 256-wide column
block for more than half a million tokens).
"""

from __future__ import annotations

import math

import torch

from opake_amd import _native as nat
from opake_amd.exceptions import ConfigurationError, InputTypeError
from opake_amd.ops import _aligned


def _check_head(hidden: torch.Tensor, weight: torch.Tensor) -> int:
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ConfigurationError(
            f"expected hidden [..., D] and weight [V, D], got {tuple(hidden.shape)} and "
            f"{tuple(weight.shape)}")
    if hidden.dtype != weight.dtype:
        raise ConfigurationError(
            f"hidden and weight must share a dtype, got {hidden.dtype} and {weight.dtype}")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ConfigurationError(f"weight must not be empty, got {tuple(weight.shape)}")
    return nat.dtype_code(hidden.dtype)


def _integer(t: torch.Tensor, what: str) -> None:
    if t.dtype not in (torch.int64, torch.int32):
        raise InputTypeError(f"{what} must be int64 or int32, got {t.dtype}")


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, index, teacher, ignore_index, temperature):
        dev = nat.require_device(hidden, weight, index, teacher)
        code = nat.dtype_code(hidden.dtype)
        lead, D = hidden.shape[:-1], hidden.shape[-1]
        V = weight.shape[0]
        h = _aligned(hidden.detach().reshape(-1, D))
        w = _aligned(weight.detach())
        N, K = h.shape[0], 1 if teacher is None else index.shape[-1]
        index = index.to(torch.int64).contiguous()
        if teacher is not None:
            teacher = teacher.detach().to(torch.float32).contiguous()
        loss = torch.empty(lead, dtype=torch.float32, device=dev)
        rows = torch.empty(2 * N + 1, dtype=torch.int32, device=dev)
        lse = torch.empty(N, dtype=torch.float32, device=dev)
        cols = torch.empty((N, K), dtype=torch.int32, device=dev)
        corr = torch.empty((N, K), dtype=torch.float32, device=dev)
        with torch.cuda.device(dev):
            ws_bytes = nat.load().dpc_head_loss_workspace_bytes(N, D, V, K, code)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
            nat.call("dpc_head_loss", nat.ptr(h), nat.ptr(w), N, D, V, code, nat.ptr(index),
                     nat.ptr(teacher), K, ignore_index, temperature, nat.ptr(loss), nat.ptr(rows),
                     nat.ptr(lse), nat.ptr(cols), nat.ptr(corr), nat.ptr(ws), ws_bytes,
                     nat.stream_handle(dev))
        ctx.save_for_backward(hidden, weight, rows, lse, cols, corr)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, rows, lse, cols, corr = ctx.saved_tensors
        want_h, want_w = ctx.needs_input_grad[:2]
        if not want_h and not want_w:
            return (None,) * 6
        dev, code = hidden.device, nat.dtype_code(hidden.dtype)
        D, V = hidden.shape[-1], weight.shape[0]
        h = _aligned(hidden.detach().reshape(-1, D))
        w = _aligned(weight.detach())
        g = grad.to(torch.float32).contiguous()
        N, K = cols.shape
        dh = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if want_h else None
        dw = None
        if want_w:  # no token, no launch: the sum over none is zero
            dw = (torch.empty if N else torch.zeros)((V, D), dtype=weight.dtype, device=dev)
        with torch.cuda.device(dev):
            ws_bytes = nat.load().dpc_head_loss_grad_workspace_bytes(N, D, V, K, code, int(want_h),
                                                                     int(want_w))
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
            nat.call("dpc_head_loss_grad", nat.ptr(h), nat.ptr(w), N, D, V, code, nat.ptr(rows),
                     nat.ptr(cols), nat.ptr(corr), K, nat.ptr(lse), nat.ptr(g), ctx.temperature,
                     nat.ptr(dh), nat.ptr(dw), nat.ptr(ws), ws_bytes, nat.stream_handle(dev))
        return dh, dw, None, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100) -> torch.Tensor:
    """``-log softmax(hidden @ weight.T)[target]`` of every token, float32 [...].

    ``hidden`` [..., D] and ``weight`` [V, D] share a dtype (bfloat16 or
    float32); ``targets`` [...] are integers.  A token whose target is
    ``ignore_index`` has loss 0 and no part in any gradient.  A target outside
    the vocabulary makes that token's loss NaN."""
    nat.require_device(hidden, weight, targets)
    _check_head(hidden, weight)
    _integer(targets, "targets")
    if targets.shape != hidden.shape[:-1]:
        raise ConfigurationError(
            f"targets must be {tuple(hidden.shape[:-1])}, got {tuple(targets.shape)}")
    return _HeadLoss.apply(hidden, weight, targets, None, int(ignore_index), 1.0)


def topk_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_logits: torch.Tensor,
                      teacher_indices: torch.Tensor, *, temperature: float = 1.0) -> torch.Tensor:
    """``temperature^2 KL(q || p)`` of every token, float32 [...].

    ``p = softmax(hidden @ weight.T / temperature)`` over the whole vocabulary;
    ``q = softmax(teacher_logits / temperature)`` over the token's K kept
    entries, at the vocabulary's columns ``teacher_indices`` (both [..., K]).
    An entry whose index is negative is absent, so rows may hold fewer than K;
    a token with none left has loss 0 and no part in any gradient.  The factor
    ``temperature^2`` keeps the gradient's size when the temperature changes.
    No gradient reaches the teacher."""
    nat.require_device(hidden, weight, teacher_logits, teacher_indices)
    _check_head(hidden, weight)
    _integer(teacher_indices, "teacher_indices")
    if not teacher_logits.is_floating_point():
        raise InputTypeError(f"teacher_logits must be floating point, got {teacher_logits.dtype}")
    if (teacher_indices.shape != teacher_logits.shape or teacher_indices.dim() != hidden.dim()
            or teacher_indices.shape[:-1] != hidden.shape[:-1] or teacher_indices.shape[-1] < 1):
        raise ConfigurationError(
            f"expected teacher_logits and teacher_indices {tuple(hidden.shape[:-1])} + (K,), got "
            f"{tuple(teacher_logits.shape)} and {tuple(teacher_indices.shape)}")
    if isinstance(temperature, bool) or not isinstance(temperature, (int, float)):
        raise InputTypeError(f"temperature must be a number, got {type(temperature)}")
    if not (0.0 < temperature < 1e15 and math.isfinite(temperature)):
        raise ConfigurationError(f"temperature must be positive, got {temperature}")
    return _HeadLoss.apply(hidden, weight, teacher_indices, teacher_logits, 0, float(temperature))


__all__ = ["linear_cross_entropy", "topk_distillation"]
