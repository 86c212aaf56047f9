"""Top-k mixture-of-experts SwiGLU FFN whose experts feed ghost clipping.

Forward semantics follow the reference's expert FFN
(packages/opake-patches/src/opake/api/patches/kernels/moe.py:74-103,
``opake_moe`` :570-627): per expert ``e``,
``h = silu(x W_gu[e][:I]^T) * (x W_gu[e][I:]^T)`` (the SiLU taken in float32
and cast back), ``y = h W_down[e]^T``, and each token's output is the
route-weighted sum over its top-k experts (accumulated in float32).  Routing
weights are the softmax over the top-k router logits.

Layout: each expert is its own module with two bias-free linear layers
(``experts.<e>.gate_up`` [2I, d] and ``experts.<e>.down`` [d, I]), so the
parameter pytree has one leaf per expert and projection and a ``PerGroup``
can put each expert in its own clipping group.  The router is a frozen
linear layer; ``forward`` also accepts router logits directly.  With ``routing``
the choice is ``routing.route_topk``'s instead: softmax or sigmoid scores, a
balancing bias (the buffer ``route_bias``), groups of experts, and masked experts
(a token left with fewer than ``k`` goes to those alone).

``RoutedLM`` puts such an FFN behind a transformer block, between a frozen
embedding and a frozen head, and takes its losses from the hidden states with
``head.linear_cross_entropy`` and ``head.topk_distillation``: no logits are kept.

With ``fused`` (on the GPU, bfloat16 or float32) an expert's ``gate_up`` is a
``gated.GatedLinear`` of the same parameter, which rounds the product once, and
``RoutedLM``'s block is a fused one (``transformer``).

Dispatch sorts the (token, slot) assignments by expert and, within an
expert, by token, so expert ``e``'s input rows are its examples' tokens in
example order.  Before calling an expert's layers the module sets
``dpc_row_segments`` on them to the per-example row counts, which is what
the model-level ghost clipping needs to form per-example (per-expert) norms
and clipped sums without materialising a gradient.  Computing the counts
takes one device-to-host copy of the [E, B] count table per forward (the
per-expert GEMM shapes need it anyway).
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn

from opake_amd.gated import GatedLinear
from opake_amd.head import linear_cross_entropy, topk_distillation
from opake_amd.routing import route_topk
from opake_amd.transformer import LlamaBlock


class SwiGLUExpert(nn.Module):
    fused = False  # (of blocks that were pickled before they could be)

    def __init__(self, d: int, inter: int, *, fused: bool = False, dtype=None, device=None):
        super().__init__()
        self.inter, self.fused = inter, fused
        kw = dict(dtype=dtype, device=device)
        self.gate_up = (GatedLinear(d, inter, **kw) if fused
                        else nn.Linear(d, 2 * inter, bias=False, **kw))
        self.down = nn.Linear(inter, d, bias=False, dtype=dtype, device=device)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.fused:
            return self.down(self.gate_up(x))
        gu = self.gate_up(x)
        h = F.silu(gu[:, : self.inter].float()).to(x.dtype) * gu[:, self.inter:]
        return self.down(h)


class TopKMoE(nn.Module):
    """``d``-wide top-``k`` MoE FFN with ``n_experts`` SwiGLU experts of width ``inter``.

    ``routing``: keyword arguments of ``route_topk`` (``score``, ``groups``, ``top_groups``,
    ``group_score``, ``renormalize``, ``scale``), which then routes."""

    def __init__(self, d: int, inter: int, n_experts: int, top_k: int = 2, *,
                 routing: dict | None = None, fused: bool = False, dtype=None, device=None):
        super().__init__()
        if not 1 <= top_k <= n_experts:
            raise ValueError("top_k must be between 1 and n_experts")
        self.d, self.inter, self.n_experts, self.top_k = d, inter, n_experts, top_k
        self.router = nn.Linear(d, n_experts, bias=False, dtype=dtype, device=device)
        self.router.weight.requires_grad_(False)
        self.experts = nn.ModuleList(
            SwiGLUExpert(d, inter, fused=fused, dtype=dtype, device=device)
            for _ in range(n_experts))
        self.routing = None if routing is None else dict(routing)
        if routing is not None:
            self.register_buffer("route_bias",
                                 torch.zeros(n_experts, dtype=torch.float32, device=device))
        self.last_counts: torch.Tensor | None = None  # [E, B] host copy of the last routing

    def _apply(self, fn, recurse=True):
        """Casts leave ``route_bias`` in float32: a balancing rule's steps are below what
        bfloat16 holds, and ``route_topk`` takes nothing else."""
        bias = self._buffers.get("route_bias")
        super()._apply(fn, recurse)
        if bias is not None and self.route_bias.dtype != torch.float32:
            self.route_bias = bias.to(self.route_bias.device)
        return self

    def route(self, x: torch.Tensor, router_logits: torch.Tensor | None = None):
        """Top-k expert indices and weights ([B, T, k] each); -1: none (``routing`` only)."""
        logits = self.router(x) if router_logits is None else router_logits
        if self.routing is not None:
            top_w, top_i = route_topk(logits, self.top_k, bias=self.route_bias, **self.routing)
            return top_i, top_w.to(x.dtype)
        top_v, top_i = torch.topk(logits.float(), self.top_k, dim=-1)
        return top_i, torch.softmax(top_v, dim=-1).to(x.dtype)

    def forward(self, x: torch.Tensor, router_logits: torch.Tensor | None = None):
        B, T, d = x.shape
        E, k = self.n_experts, self.top_k
        top_i, top_w = self.route(x, router_logits)
        expert = top_i.reshape(-1)
        token = torch.arange(B * T, device=x.device).repeat_interleave(k)
        weight = top_w.reshape(-1)
        if self.routing is not None:
            # A token whose logits are all NaN has NaN weights and no expert: any will do to
            # keep it NaN.
            chosen = (expert >= 0) | weight.isnan()
            expert, token, weight = expert[chosen].clamp(min=0), token[chosen], weight[chosen]
        order = torch.argsort(expert * (B * T) + token, stable=True)
        counts = torch.bincount(expert * B + token // T, minlength=E * B).view(E, B).cpu()
        self.last_counts = counts
        rows = counts.sum(dim=1).tolist()
        tok_sorted = token[order]
        xs = x.reshape(B * T, d)[tok_sorted]
        outs = []
        start = 0
        for e in range(E):
            n = rows[e]
            mod = self.experts[e]
            seg = counts[e].tolist()
            mod.gate_up.dpc_row_segments = seg
            mod.down.dpc_row_segments = seg
            outs.append(mod(xs[start:start + n]))
            start += n
        y = torch.cat(outs) * weight[order].unsqueeze(1)
        out = torch.zeros((B * T, d), dtype=torch.float32, device=x.device)
        out.index_add_(0, tok_sorted, y.float())
        return out.to(x.dtype).view(B, T, d)


class RoutedLM(nn.Module):
    """Frozen embedding -> ``LlamaBlock`` -> RMSNorm and ``TopKMoE`` (residual) ->
    frozen head.  ``forward`` returns hidden states [B, T, d]; ``loss`` takes them.

    For distillation the teacher's top logits and their columns ([B, T, K] each) go
    in with the tokens, and ``loss`` mixes ``distill`` of KL into the cross entropy:

        fn, state = ghost_clipped_grad(model, model.loss, clipping_norm=1.0)
        fn((ids, teacher_logits, teacher_indices), targets, state=state)
    """

    def __init__(self, vocab: int, d: int, n_heads: int, ffn: int, inter: int, n_experts: int,
                 top_k: int = 2, *, routing: dict | None = None, distill: float = 0.5,
                 temperature: float = 1.0, ignore_index: int = -100, fused: bool = False,
                 dtype=None, device=None):
        super().__init__()
        kw = dict(dtype=dtype, device=device)
        self.distill, self.temperature = distill, temperature
        self.ignore_index = ignore_index
        self.embed = nn.Embedding(vocab, d, **kw)
        self.block = LlamaBlock(d, n_heads, ffn, fused=fused, **kw)
        self.moe_norm = nn.RMSNorm(d, eps=1e-5, **kw)
        self.moe = TopKMoE(d, inter, n_experts, top_k, routing=routing or {}, fused=fused,
                           **kw)
        self.head = nn.Linear(d, vocab, bias=False, **kw)
        self.embed.weight.requires_grad_(False)
        self.head.weight.requires_grad_(False)

    def forward(self, ids: torch.Tensor, teacher_logits: torch.Tensor | None = None,
                teacher_indices: torch.Tensor | None = None):
        x = self.block(self.embed(ids))
        x = x + self.moe(self.moe_norm(x))
        return x if teacher_logits is None else (x, teacher_logits, teacher_indices)

    def loss(self, outputs, targets: torch.Tensor) -> torch.Tensor:
        """Each example's loss [B] (float32): the mean over its tokens.  A target of
        ``ignore_index`` makes its token's cross entropy zero, not its part of the KL,
        which goes by the teacher's entries: negative ``teacher_indices`` leave a token
        out of that too."""
        hidden, teacher = (outputs, None) if torch.is_tensor(outputs) else (outputs[0],
                                                                             outputs[1:])
        loss = linear_cross_entropy(hidden, self.head.weight, targets,
                                    ignore_index=self.ignore_index)
        if teacher is not None:
            kl = topk_distillation(hidden, self.head.weight, *teacher,
                                   temperature=self.temperature)
            loss = (1.0 - self.distill) * loss + self.distill * kl
        return loss.mean(dim=1)


def expert_groups(model: TopKMoE, prefix: str = "", clipping_norm: float = 1.0):
    """``PerGroup`` with one group per expert, ``C_e = C / sqrt(E)`` (so the
    effective bound is ``C``): the per-expert clipping of a MoE step."""
    import math

    from opake_amd.types import PerGroup

    groups, values = {}, {}
    bound = clipping_norm / math.sqrt(model.n_experts)
    for e in range(model.n_experts):
        name = f"expert{e}"
        values[name] = bound
        for proj in ("gate_up", "down"):
            groups[f"{prefix}experts.{e}.{proj}.weight"] = name
    return PerGroup(groups, values)


__all__ = ["RoutedLM", "SwiGLUExpert", "TopKMoE", "expert_groups"]
