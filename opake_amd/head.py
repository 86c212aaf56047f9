"""Losses of a vocabulary head that never hold its logits.

``linear_cross_entropy`` is the softmax cross entropy of ``hidden @ weight.T``
against one target a token; ``topk_distillation`` is the Kullback-Leibler
divergence from a teacher of which only the top logits were kept.  Both return
one loss a token (float32), so a caller can reduce them per example as
per-example clipping needs, and both are differentiable with respect to
``hidden`` and, where it requires a gradient, ``weight``.

Forward, one matrix-core product leaves the maximum and the sum of
exponentials of every 128 columns of the vocabulary per token
(``csrc/head.hip``).  Where only ``hidden`` requires a gradient -- a frozen head,
the usual case under per-example clipping -- the exponentials of up to 512 MiB
of tokens at a time become its gradient in the forward, which is kept in
float32 for the backward to scale.  A trained head keeps its exponentials (16
bits each, 32 for float32) where all of them fit in 512 MiB, and makes the
logits again, piece by piece of the vocabulary, where they do not.  With gradients
disabled the loss alone is made, whatever requires one.  So no more
than 512 MiB of any ``[tokens, vocabulary]`` kind are kept, and twice that exist
at a time (one 256-wide row or column block, where that is more).
"""

from __future__ import annotations

import torch

from opake_amd import _native as nat
from opake_amd.exceptions import ConfigurationError, InputTypeError
from opake_amd.ops import _aligned

MAX_VOCABULARY = 1 << 19
MAX_WIDTH = 1 << 20
MAX_ENTRIES = 1 << 16  # of the teacher, a token


def _check_head(hidden: torch.Tensor, weight: torch.Tensor) -> int:
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ConfigurationError(
            f"expected hidden [..., D] and weight [V, D], got {tuple(hidden.shape)} and "
            f"{tuple(weight.shape)}")
    if hidden.dtype != weight.dtype:
        raise ConfigurationError(
            f"hidden and weight must share a dtype, got {hidden.dtype} and {weight.dtype}")
    if not 1 <= weight.shape[0] <= MAX_VOCABULARY or not 1 <= weight.shape[1] <= MAX_WIDTH:
        raise ConfigurationError(
            f"weight must be [V, D] with 1 <= V <= {MAX_VOCABULARY} and 1 <= D <= {MAX_WIDTH}, "
            f"got {tuple(weight.shape)}")
    return nat.dtype_code(hidden.dtype)


def _integer(t: torch.Tensor, what: str) -> None:
    if t.dtype not in (torch.int64, torch.int32):
        raise InputTypeError(f"{what} must be int64 or int32, got {t.dtype}")


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, index, teacher, options):
        ignore_index, temperature, code, grad_enabled = options
        dev = hidden.device
        lead, D = hidden.shape[:-1], hidden.shape[-1]
        V = weight.shape[0]
        h, w = _aligned(hidden), _aligned(weight)
        N, K = h.numel() // D, 1 if teacher is None else index.shape[-1]
        index = index.to(torch.int64).contiguous()
        if teacher is not None:
            teacher = teacher.to(torch.float32).contiguous()
        # needs_input_grad is true of a parameter under no_grad too.
        want_h, want_w = (need and grad_enabled for need in ctx.needs_input_grad[:2])
        lib, sizes = nat.load(), (N, D, V, K, code, int(want_h), int(want_w))
        loss = torch.empty(lead, dtype=torch.float32, device=dev)
        state_bytes = lib.dpc_head_loss_state_bytes(*sizes)
        state = torch.empty(state_bytes, dtype=torch.uint8, device=dev)
        ws_bytes = lib.dpc_head_loss_workspace_bytes(*sizes)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        nat.call_on(dev, "dpc_head_loss", h.data_ptr(), w.data_ptr(), N, D, V, code,
                    index.data_ptr(), 0 if teacher is None else teacher.data_ptr(), K,
                    ignore_index, temperature, int(want_h), int(want_w), loss.data_ptr(),
                    state.data_ptr(), state_bytes, ws.data_ptr(), ws_bytes)
        if want_h or want_w:
            ctx.save_for_backward(hidden, weight, state)
            ctx.sizes, ctx.temperature = sizes, temperature
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, state = ctx.saved_tensors
        want_h, want_w = ctx.needs_input_grad[:2]
        sizes = ctx.sizes
        N, D, V, K, code, forward_h, forward_w = sizes
        if not want_h and not want_w:
            return (None,) * 5
        dev = hidden.device
        h, w = _aligned(hidden), _aligned(weight)
        g = (grad if grad.dtype == torch.float32 else grad.float()).contiguous()
        dh = torch.empty_like(h) if want_h else None
        dw = None
        if want_w:  # no token, no launch: the sum over none is zero
            dw = (torch.empty_like if N else torch.zeros_like)(w)
        ws_bytes = nat.load().dpc_head_loss_grad_workspace_bytes(*sizes)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        nat.call_on(dev, "dpc_head_loss_grad", h.data_ptr(), w.data_ptr(), N, D, V, code, K,
                    ctx.temperature, forward_h, forward_w, state.data_ptr(), state.numel(),
                    g.data_ptr(), 0 if dh is None else dh.data_ptr(),
                    0 if dw is None else dw.data_ptr(), ws.data_ptr(), ws_bytes)
        return dh, dw, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100) -> torch.Tensor:
    """``-log softmax(hidden @ weight.T)[target]`` of every token, float32 [...].

    ``hidden`` [..., D] and ``weight`` [V, D] share a dtype (bfloat16 or
    float32); ``targets`` [...] are integers.  A token whose target is
    ``ignore_index`` has loss 0 and no part in any gradient.  A target outside
    the vocabulary makes that token's loss NaN."""
    nat.require_device(hidden, weight, targets)
    code = _check_head(hidden, weight)
    _integer(targets, "targets")
    if targets.shape != hidden.shape[:-1]:
        raise ConfigurationError(
            f"targets must be {tuple(hidden.shape[:-1])}, got {tuple(targets.shape)}")
    return _HeadLoss.apply(hidden, weight, targets, None,
                           (int(ignore_index), 1.0, code, torch.is_grad_enabled()))


def topk_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_logits: torch.Tensor,
                      teacher_indices: torch.Tensor, *, temperature: float = 1.0) -> torch.Tensor:
    """``temperature^2 KL(q || p)`` of every token, float32 [...].

    ``p = softmax(hidden @ weight.T / temperature)`` over the whole vocabulary;
    ``q = softmax(teacher_logits / temperature)`` over the token's K kept
    entries, at the vocabulary's columns ``teacher_indices`` (both [..., K]).
    An entry whose index is negative is absent, so rows may hold fewer than K;
    a token with none left has loss 0 and no part in any gradient.  The factor
    ``temperature^2`` keeps the gradient's size when the temperature changes.
    No gradient reaches the teacher.  Entries of a row are compared pair by pair: a few
    thousand of them cost more than the products do."""
    nat.require_device(hidden, weight, teacher_logits, teacher_indices)
    code = _check_head(hidden, weight)
    _integer(teacher_indices, "teacher_indices")
    if not teacher_logits.is_floating_point():
        raise InputTypeError(f"teacher_logits must be floating point, got {teacher_logits.dtype}")
    if (teacher_indices.shape != teacher_logits.shape or teacher_indices.dim() != hidden.dim()
            or teacher_indices.shape[:-1] != hidden.shape[:-1]
            or not 1 <= teacher_indices.shape[-1] <= MAX_ENTRIES):
        raise ConfigurationError(
            f"expected teacher_logits and teacher_indices {tuple(hidden.shape[:-1])} + (K,), got "
            f"{tuple(teacher_logits.shape)} and {tuple(teacher_indices.shape)}")
    if isinstance(temperature, bool) or not isinstance(temperature, (int, float)):
        raise InputTypeError(f"temperature must be a number, got {type(temperature)}")
    if not 1e-15 < temperature < 1e15:  # its square and reciprocal are float32's
        raise ConfigurationError(
            f"temperature must be between 1e-15 and 1e15, got {temperature}")
    return _HeadLoss.apply(hidden, weight, teacher_indices, teacher_logits,
                           (0, float(temperature), code, torch.is_grad_enabled()))


__all__ = ["linear_cross_entropy", "topk_distillation"]
