"""Softmax attention that keeps nothing of size [queries, keys], with its gradients.

``attention`` takes queries, keys and values as the projections leave them ([B, T, heads,
h], any strides: places of a fused projection go in as they are), shares key heads among
groups of query heads, and masks by what a query sees: causal, a window, each example's
length and the position of its first query.  The forward keeps two numbers a query (for
bfloat16 one, and a byte an element of the output: what rounding took from it) for the
backward, which forms the probabilities again (``csrc/attention.hip``).  Results do not depend
on anything but the inputs: no sums whose order changes.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from opake_amd import _native as nat
from opake_amd._autograd import check_leaves, note_leaves
from opake_amd.exceptions import ConfigurationError, InputTypeError

MAX_HEAD = 256
MAX_HEADS = 1 << 16
MAX_TOKENS = 1 << 24
_MOST_BYTES = 0x7ff00000 - (1 << 20)


def _rows(t: torch.Tensor, odd: int, rep: int = 1, apart: int = 0) -> torch.Tensor:
    """Rows of whole 16-byte chunks (``odd`` zeros more, which add nothing to a score and come
    out as zeros), at least ``apart`` elements from each other, and tiles of 65 tokens
    within a buffer's range."""
    if odd:
        t = F.pad(t, (0, odd))
    size = t.element_size()
    b, n, head, last = t.stride()
    if (last == 1 and (n >= apart or t.shape[1] < 2) and t.data_ptr() % 16 == 0 and b * size % 16 == 0 and n * size % 16 == 0
            and head * size % 16 == 0 and (65 * n + rep * head) * size <= _MOST_BYTES):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _call(name, dev, tensors, strides, sizes, lengths, starts, options, *rest):
    causal, window, scale = options
    nat.call_on(dev, name, *(t.data_ptr() for t in tensors),
                (nat._c_i64 * len(strides))(*strides), *sizes,
                0 if lengths is None else lengths.data_ptr(),
                0 if starts is None else starts.data_ptr(), causal, window, scale, *rest)


class _Attention(torch.autograd.Function):
    """Of q, k and v as they are, so that the leaves among them are its own; its output has the
    copied rows' width."""

    @staticmethod
    def forward(ctx, q, k, v, lengths, starts, code, options, grad_enabled):
        dev = q.device
        B, T, H, h = q.shape
        S, KV = k.shape[1:3]
        odd = -h % (4 if q.dtype == torch.float32 else 8)
        h += odd
        qr, kr, vr = _rows(q, odd, H // KV), _rows(k, odd, 1, h), _rows(v, odd, 1, h)
        sizes = (B, T, S, H, KV, h, code)
        out = torch.empty((B, T, H, h), dtype=q.dtype, device=dev)
        lib, state, state_bytes = nat.load(), None, 0
        # needs_input_grad is true of a parameter under no_grad too.
        if grad_enabled and any(ctx.needs_input_grad[:3]):
            note_leaves(ctx)
            state_bytes = lib.dpc_attention_state_bytes(B, T, H, h, code)
            state = torch.empty(state_bytes, dtype=torch.uint8, device=dev)
            ctx.save_for_backward(q, k, v, out, state, lengths, starts)
            ctx.sizes, ctx.options, ctx.odd = sizes, options, odd
        ws_bytes = lib.dpc_attention_workspace_bytes(*sizes)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        _call("dpc_attention", dev, (qr, kr, vr),
              (*qr.stride()[:3], *kr.stride()[:3], *vr.stride()[:3]), sizes, lengths, starts,
              options, out.data_ptr(), 0 if state is None else state.data_ptr(), state_bytes,
              ws.data_ptr(), ws_bytes)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        check_leaves(ctx)
        q, k, v, out, state, lengths, starts = ctx.saved_tensors
        dev, sizes = q.device, ctx.sizes
        B, T, S, H, KV, h, _ = sizes
        rep, odd = H // KV, ctx.odd
        qr, kr, vr = _rows(q, odd, rep), _rows(k, odd, 1, h), _rows(v, odd, 1, h)
        gr = _rows(grad, 0, rep)
        dq = torch.empty((B, T, H, h), dtype=q.dtype, device=dev)
        dk = dv = None
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            dk, dv = (torch.empty((B, S, KV, h), dtype=q.dtype, device=dev) for _ in range(2))
        ws_bytes = nat.load().dpc_attention_grad_workspace_bytes(B, T, H)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        _call("dpc_attention_grad", dev, (qr, kr, vr, out, gr),
              (*qr.stride()[:3], *kr.stride()[:3], *vr.stride()[:3], *gr.stride()[:3]), sizes,
              lengths, starts, ctx.options, state.data_ptr(), state.numel(), dq.data_ptr(),
              *(0 if t is None else t.data_ptr() for t in (dk, dv)), ws.data_ptr(), ws_bytes)
        if odd:
            dq, dk, dv = (t if t is None else t[..., :h - odd] for t in (dq, dk, dv))
        return dq, dk, dv, None, None, None, None, None


def _whole(t, name: str, B: int):
    if t is None:
        return None
    if t.dtype not in (torch.int64, torch.int32):
        raise InputTypeError(f"{name} must be int64 or int32, got {t.dtype}")
    if tuple(t.shape) != (B,):
        raise ConfigurationError(f"{name} must be [{B}], got {tuple(t.shape)}")
    return t.detach().to(torch.int64).contiguous()


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = True,
              window: int | None = None, lengths: torch.Tensor | None = None,
              starts: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """``softmax(scale q k^T) v`` of every head over the keys a query sees: [B, T, H, h].

    ``q`` [B, T, H, h], ``k`` and ``v`` [B, S, KV, h] (bfloat16 or float32, any strides);
    query heads share key heads in consecutive groups of H / KV.  ``lengths`` (integers
    [B]): example b has that many keys, those behind are padding (all S by default).  Not
    ``causal``: a query sees them all.  ``causal``: token t of example b is at position
    ``starts[b] + t`` (integers; S - T + t by default, so the last query sees the last
    key) and sees the keys up to its own position, with ``window`` the last ``window`` of
    them; a token at a position below 0 or not below the length is padding.  ``scale``:
    positive, 1 / sqrt(h) by default.

    Scores, statistics and sums are float32.  bfloat16: probabilities and the gradients of
    scores are rounded to it (2^-8 of each at most) before their products, so that output and
    gradients are 2.0e-3 and 2.4e-3 from 64 bits in the mean square (2.8e-3 at most), where the
    rounding of either alone leaves 1.7e-3; float32: 2e-7 (2e-6 at most).

    A query that sees no key has output 0 and no part in any gradient; one whose scores are all
    -inf has NaN, as their softmax is.  What padding holds reaches nothing; what a token holds reaches its own example's head group alone, but there a
    value that is not finite may reach queries that do not see it.  Gradients reach ``q``,
    ``k`` and ``v``.  For one token of each of several sequences: T = 1, keys and values
    the caches [B, S, KV, h], ``lengths`` the sequences' and ``starts`` one less.  65 tokens of
    all heads of a tensor must take less than 2 GiB."""
    nat.require_device(q, k, v, lengths, starts)
    if (q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0]
            or q.shape[3] != k.shape[3]):
        raise ConfigurationError(
            f"expected q [B, T, H, h], k and v [B, S, KV, h], got {tuple(q.shape)}, "
            f"{tuple(k.shape)} and {tuple(v.shape)}")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise ConfigurationError(
            f"q, k and v must share a dtype, got {q.dtype}, {k.dtype} and {v.dtype}")
    code = nat.dtype_code(q.dtype)
    B, T, H, h = q.shape
    S, KV = k.shape[1:3]
    if not 1 <= h <= MAX_HEAD or KV < 1 or not 1 <= H <= MAX_HEADS or H % KV:
        raise ConfigurationError(
            f"heads must be 1 to {MAX_HEAD} wide and query heads (at most {MAX_HEADS}) a "
            f"multiple of key heads, got {H} and {KV} of {h}")
    if T > MAX_TOKENS or S > MAX_TOKENS:
        raise ConfigurationError(f"at most {MAX_TOKENS} tokens, got {T} and {S}")
    if window is not None:
        if isinstance(window, bool) or not isinstance(window, int):
            raise InputTypeError(f"window must be an int, got {type(window)}")
        if not causal or window < 1:
            raise ConfigurationError(f"a window is causal and at least 1, got {window}")
    if starts is not None and not causal:
        raise ConfigurationError("starts are for causal attention")
    if scale is None:
        scale = 1.0 / math.sqrt(h)
    elif isinstance(scale, bool) or not isinstance(scale, (int, float)):
        raise InputTypeError(f"scale must be a number, got {type(scale)}")
    if not 1e-30 < scale < 1e30:
        raise ConfigurationError(f"scale must be between 1e-30 and 1e30, got {scale}")
    options = (int(bool(causal)), min(window or 0, MAX_TOKENS), float(scale))
    out = _Attention.apply(q, k, v, _whole(lengths, "lengths", B), _whole(starts, "starts", B),
                           code, options, torch.is_grad_enabled())
    return out if out.shape[3] == h else out[..., :h]


__all__ = ["MAX_HEAD", "attention"]
