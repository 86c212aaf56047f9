"""Rotary positions of queries and keys, for either layout of the pairs, part of a
head, and frequencies scaled for contexts longer than a model was trained on.

``rotary`` rotates queries and keys in one launch; its backward is one launch too
(``csrc/rotary.hip``).  Angles are formed in float64 from the positions themselves:
there are no tables, and far positions are as exact as near ones.
"""

from __future__ import annotations

import math

import torch

from opake_amd import _native as nat
from opake_amd._autograd import check_leaves, note_leaves
from opake_amd.exceptions import ConfigurationError, InputTypeError

MAX_HEAD = 2048
MAX_HEADS_WIDTH = 1 << 22  # heads of queries and keys, times their width
_SCALINGS = {"linear": {"factor"}, "ntk": {"factor"},
             "bands": {"factor", "low", "high", "original"},
             "ramp": {"factor", "low", "high", "original"}}


def _number(value, name: str) -> float:
    if isinstance(value, bool) or not isinstance(value, (int, float)):
        raise InputTypeError(f"{name} must be a number, got {type(value)}")
    if not math.isfinite(value):
        raise ConfigurationError(f"{name} must be finite, got {value}")
    return float(value)


def rotary_frequencies(dims: int, base: float = 10000.0, *, scaling: dict | None = None,
                       device=None) -> tuple[torch.Tensor, float]:
    """Frequencies (radians a position, float64 [dims / 2]) and the amplitude for ``rotary``.

    ``freq_i = base ** (-2 i / dims)``.  ``scaling`` stretches them by ``factor`` (>= 1):

    ``{"kind": "linear", "factor"}``: every frequency divided by it (positions in between).
    ``{"kind": "ntk", "factor"}``: a larger base, so that the lowest frequency is divided by
    ``factor`` and the highest is kept.
    ``{"kind": "bands", "factor", "low", "high", "original"}``: pairs that turn more than
    ``high`` times within the ``original`` context are kept, those that turn less than
    ``low`` times divided by ``factor``, and between the two the frequencies are mixed
    linearly in the number of turns.
    ``{"kind": "ramp", ...}``: the same with the mix linear in the pair's index, from the
    pair that turns ``high`` times to the one that turns ``low`` times, and an amplitude of
    ``0.1 ln(factor) + 1``, which sharpens attention over the longer context (1 for the
    other kinds)."""
    if isinstance(dims, bool) or not isinstance(dims, int):
        raise InputTypeError(f"dims must be an int, got {type(dims)}")
    if dims < 2 or dims % 2 or dims > MAX_HEAD:
        raise ConfigurationError(f"dims must be even, from 2 to {MAX_HEAD}, got {dims}")
    base = _number(base, "base")
    if not base > 1.0:
        raise ConfigurationError(f"base must be above 1, got {base}")
    pair = torch.arange(0, dims, 2, dtype=torch.float64, device=device) / dims
    if scaling is None:
        return base ** -pair, 1.0
    options = dict(scaling)
    kind = options.pop("kind", None)
    if kind not in _SCALINGS or set(options) != _SCALINGS[kind]:
        raise ConfigurationError(
            "scaling must have a kind and its options, one of "
            f"{ {k: sorted(v) for k, v in _SCALINGS.items()} }, got {scaling!r}")
    options = {k: _number(v, k) for k, v in options.items()}
    factor = options["factor"]
    if factor < 1.0:
        raise ConfigurationError(f"factor must be at least 1, got {factor}")
    if kind == "linear":
        return base ** -pair / factor, 1.0
    if kind == "ntk":
        if dims == 2:
            raise ConfigurationError("ntk scaling needs more than one pair")
        return (base * factor ** (dims / (dims - 2))) ** -pair, 1.0
    low, high, original = options["low"], options["high"], options["original"]
    if not 0.0 < low < high or not original > 0.0:
        raise ConfigurationError(
            f"expected 0 < low < high and original > 0, got {low}, {high} and {original}")
    freq = base ** -pair
    if kind == "bands":
        keep = ((original * freq / (2.0 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        amplitude = 1.0
    else:
        def index(turns):  # of the pair that turns that often within the original context
            return dims * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        first = max(math.floor(index(high)), 0)
        last = min(math.ceil(index(low)), dims - 1)
        i = torch.arange(dims // 2, dtype=torch.float64, device=device)
        keep = 1.0 - ((i - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        amplitude = 0.1 * math.log(factor) + 1.0
    return freq * keep + freq / factor * (1.0 - keep), amplitude


def _heads(t: torch.Tensor) -> torch.Tensor:
    """Any strides of examples and tokens, but heads within 32 bits of each other and each one's
    elements side by side."""
    if t.stride(-1) == 1 and t.stride(2) < 1 << 31:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _rotate(tensors, positions, freqs, options, inverse: int):
    code, interleaved, amplitude = options
    q, k = tensors
    dev = q.device
    q = _heads(q)
    out = [torch.empty(q.shape, dtype=q.dtype, device=dev)]
    KV, kp, kop = 0, 0, 0
    strides = [*q.stride()[:3], 0, 0, 0]
    if k is not None:
        k = _heads(k)
        out.append(torch.empty(k.shape, dtype=k.dtype, device=dev))
        KV, kp, kop = k.shape[2], k.data_ptr(), out[1].data_ptr()
        strides[3:] = k.stride()[:3]
    B, T, H, h = q.shape
    pos, pb, pt = 0, 0, 0
    if positions is not None:
        pos, pt = positions.data_ptr(), positions.stride(-1)
        pb = positions.stride(0) if positions.dim() == 2 else 0
    nat.call_on(dev, "dpc_rotary", q.data_ptr(), kp, B, T, H, KV, h, code, (nat._c_i64 * 6)(*strides),
                pos, pb, pt, freqs.data_ptr(), freqs.numel(), interleaved, amplitude, inverse,
                out[0].data_ptr(), kop)
    return out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, freqs, options):
        note_leaves(ctx)
        out = _rotate((q, k), positions, freqs, options, 0)
        ctx.save_for_backward(positions, freqs)
        ctx.options = options
        return tuple(out) if k is not None else out[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk=None):
        check_leaves(ctx)
        positions, freqs = ctx.saved_tensors
        out = _rotate((gq, gk), positions, freqs, ctx.options, 1)
        return out[0], out[1] if gk is not None else None, None, None, None


def rotary(q: torch.Tensor, k: torch.Tensor | None, freqs: torch.Tensor, *,
           positions: torch.Tensor | None = None, interleaved: bool = False,
           amplitude: float = 1.0):
    """Queries [B, T, H, h] and keys [B, T, KV, h] (bfloat16 or float32, any strides),
    rotated to their positions: two new contiguous tensors (one, if ``k`` is None).

    ``freqs`` (float64 [n], 2 n <= h; ``rotary_frequencies``): pair i of a head turns by
    ``positions * freqs[i]``, and what lies behind the n pairs is copied.  Pairs are
    ``(x[i], x[n + i])``, or with ``interleaved`` the neighbours ``(x[2 i], x[2 i + 1])``.
    ``positions``: integers, [T] or [B, T]; 0, 1, ... by default.  ``amplitude`` multiplies
    what is rotated.  Gradients reach ``q`` and ``k``."""
    nat.require_device(q, k, freqs, positions)
    for t, what in ((q, "q"), (k, "k")):
        if t is not None and (t.dim() != 4 or t.shape[:2] != q.shape[:2] or t.shape[3] != q.shape[3]
                              or t.dtype != q.dtype):
            raise ConfigurationError(
                f"expected {what} [B, T, heads, h] like q, got {tuple(t.shape)} of {t.dtype} beside "
                f"{tuple(q.shape)} of {q.dtype}")
    B, T, H, h = q.shape
    heads = H + (0 if k is None else k.shape[2])
    if not 1 <= h <= MAX_HEAD or H < 1 or (k is not None and k.shape[2] < 1) \
            or heads * h > MAX_HEADS_WIDTH:
        raise ConfigurationError(
            f"heads must be 1 to {MAX_HEAD} wide, one at least and {MAX_HEADS_WIDTH} elements in "
            f"all, got {heads} of {h}")
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or not 1 <= freqs.numel() <= h // 2:
        raise ConfigurationError(
            f"freqs must be float64 [n] with 1 <= n <= {h // 2}, got {freqs.dtype} "
            f"{tuple(freqs.shape)}")
    if positions is not None:
        if positions.dtype not in (torch.int64, torch.int32):
            raise InputTypeError(f"positions must be int64 or int32, got {positions.dtype}")
        if tuple(positions.shape) not in ((T,), (B, T)):
            raise ConfigurationError(
                f"positions must be [{T}] or [{B}, {T}], got {tuple(positions.shape)}")
        positions = positions.to(torch.int64)
    amplitude = _number(amplitude, "amplitude")
    return _Rotary.apply(q, k, positions, freqs.detach().contiguous(),
                         (nat.dtype_code(q.dtype), int(bool(interleaved)), amplitude))


__all__ = ["MAX_HEAD", "rotary", "rotary_frequencies"]
