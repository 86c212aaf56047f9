"""A gated feed-forward layer's projections with the activation and the product.

``gated_linear(x, weight)`` is ``act(x Wg^T) * (x Wu^T)`` for ``weight = [Wg; Wu]``: one
matrix-core product whose tiles hold both projections of their columns, so the result is
formed before anything is written (``csrc/gated.hip``).  The backward makes the
projections' gradient in one pass and takes two products.  ``GatedLinear`` is the layer: a
bias-free ``nn.Linear`` [2 F, D] that returns the product, and that ghost clipping knows
(its operands are the layer's input and the projections' gradient).
"""

from __future__ import annotations

import torch
from torch import nn
from torch.autograd.forward_ad import unpack_dual

from opake_amd import _native as nat
from opake_amd._autograd import check_leaves, note_leaves
from opake_amd.exceptions import ConfigurationError
from opake_amd.ops import _aligned

MAX_TOKENS = 1 << 30
MAX_WIDTH = 1 << 20
MAX_INTER = 1 << 19
_ACTIVATIONS = {"silu": nat.ACT_SILU, "gelu": nat.ACT_GELU}


def _forward(x, weight, options, keep: bool):
    """``h``, and where kept the projections ``z`` and (bfloat16) what rounding took from them."""
    code, act = options
    dev = x.device
    xa, w = _aligned(x), _aligned(weight)
    D, F = w.shape[1], w.shape[0] // 2
    N = xa.numel() // D
    h = torch.empty((*x.shape[:-1], F), dtype=x.dtype, device=dev)
    z = torch.empty((*x.shape[:-1], 2 * F), dtype=x.dtype, device=dev) if keep else None
    rest = None
    if keep and x.dtype == torch.bfloat16:
        rest = torch.empty(z.shape, dtype=torch.int8, device=dev)
    ws_bytes = nat.load().dpc_gated_linear_workspace_bytes(N, D, F, code)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    nat.call_on(dev, "dpc_gated_linear", xa.data_ptr(), w.data_ptr(), N, D, F, code, act,
                h.data_ptr(), *(0 if t is None else t.data_ptr() for t in (z, rest)), ws.data_ptr(),
                ws_bytes)
    return h, z, rest


class _Project(torch.autograd.Function):
    """The projections, with the product made of them beside (``box``)."""

    @staticmethod
    def forward(ctx, x, weight, options, box):
        note_leaves(ctx)
        h, z, rest = _forward(x, weight, options, True)
        box += (h, rest)
        ctx.save_for_backward(x, weight)
        ctx.code = options[0]
        return z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dz):
        check_leaves(ctx)
        x, weight = ctx.saved_tensors
        want_x, want_w = ctx.needs_input_grad[:2]
        dev = x.device
        xa, w = _aligned(x), _aligned(weight)
        D, F = w.shape[1], w.shape[0] // 2
        N = xa.numel() // D
        dz = _aligned(dz)
        dx = torch.empty_like(xa) if want_x else None
        dw = None
        if want_w:  # no token, no launch: the sum over none is zero
            dw = (torch.empty_like if N else torch.zeros_like)(w)
        ws_bytes = nat.load().dpc_gated_linear_grad_workspace_bytes(N, D, F, ctx.code, int(want_x),
                                                                    int(want_w))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        nat.call_on(dev, "dpc_gated_linear_grad", xa.data_ptr(), w.data_ptr(), dz.data_ptr(), N, D,
                    F, ctx.code, dx.data_ptr() if want_x else 0, dw.data_ptr() if want_w else 0,
                    ws.data_ptr(), ws_bytes)
        return dx, dw, None, None


class _Product(torch.autograd.Function):
    """The product that ``_Project`` made, as a function of the projections."""

    @staticmethod
    def forward(ctx, z, options, box):
        h, rest = box
        box.clear()
        ctx.save_for_backward(z, rest)
        ctx.options = options
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        z, rest = ctx.saved_tensors
        code, act = ctx.options
        F = z.shape[-1] // 2
        z, dh = _aligned(z), _aligned(dh)
        dz = torch.empty_like(z)
        nat.call_on(z.device, "dpc_gated_linear_act_grad", z.data_ptr(),
                    0 if rest is None else rest.data_ptr(), dh.data_ptr(), dh.numel() // F, F, code,
                    act, dz.data_ptr())
        return dz, None, None


def _gated(x: torch.Tensor, weight: torch.Tensor, activation: str):
    """``(h, z)``; z, which h is differentiated through, is None without gradients."""
    nat.require_device(x, weight)
    if activation not in _ACTIVATIONS:
        raise ConfigurationError(
            f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.shape[0] % 2:
        raise ConfigurationError(
            f"expected x [..., D] and weight [2 F, D], got {tuple(x.shape)} and "
            f"{tuple(weight.shape)}")
    if x.dtype != weight.dtype:
        raise ConfigurationError(
            f"x and weight must share a dtype, got {x.dtype} and {weight.dtype}")
    D, F = weight.shape[1], weight.shape[0] // 2
    if not 1 <= D <= MAX_WIDTH or not 1 <= F <= MAX_INTER or x.numel() // D > MAX_TOKENS:
        raise ConfigurationError(
            f"expected 1 <= D <= {MAX_WIDTH}, 1 <= F <= {MAX_INTER} and at most {MAX_TOKENS} "
            f"tokens, got x {tuple(x.shape)} and weight {tuple(weight.shape)}")
    options = (nat.dtype_code(x.dtype), _ACTIVATIONS[activation])
    if not torch.is_grad_enabled() or not (x.requires_grad or weight.requires_grad):
        # Past the autograd functions, which refuse tangents themselves.
        if unpack_dual(x).tangent is not None or unpack_dual(weight).tangent is not None:
            raise NotImplementedError("gated_linear has no forward-mode derivative")
        return _forward(x, weight, options, False)[:2]
    box: list = []
    z = _Project.apply(x, weight, options, box)
    return _Product.apply(z, options, box), z


def gated_linear(x: torch.Tensor, weight: torch.Tensor, *,
                 activation: str = "silu") -> torch.Tensor:
    """``act(x @ weight[:F].T) * (x @ weight[F:].T)`` [..., F], rounded once.

    ``x`` [..., D] and ``weight`` [2 F, D] share a dtype (bfloat16 or float32).
    ``activation``: ``"silu"`` or ``"gelu"`` (with the normal distribution function).  Gradients
    reach both; for them the projections [..., 2 F] are kept, in the inputs' dtype (bfloat16: and 8
    bits more of each).  bfloat16: the projections' gradient is rounded to it before its products,
    so that gradients are 2.3e-3 from 64 bits in the mean square, 2.7e-3 at most (1.7e-3: the
    rounding of the results alone).  There is no forward-mode derivative."""
    return _gated(x, weight, activation)[0]


class GatedLinear(nn.Linear):
    """Bias-free ``nn.Linear(d, 2 * inter)`` whose forward is ``gated_linear``: [..., inter]."""

    def __init__(self, d: int, inter: int, *, activation: str = "silu", dtype=None, device=None):
        super().__init__(d, 2 * inter, bias=False, dtype=dtype, device=device)
        if activation not in _ACTIVATIONS:
            raise ConfigurationError(
                f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
        self.activation = activation
        # Ghost clipping clips a linear layer by the gradient of what x @ weight.T gives:
        # while it captures a forward, that is left here.
        self.dpc_keep_projections = False
        self.dpc_projections: torch.Tensor | None = None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        h, z = _gated(x, self.weight, self.activation)
        if self.dpc_keep_projections:
            self.dpc_projections = z
        return h


__all__ = ["GatedLinear", "gated_linear"]
