"""The routed language model: head losses and routing under ghost clipping (GPU).

``ghost_clipped_grad`` on a ``RoutedLM`` against per-example gradients of the same
model in 64 bits on the CPU, with routing and losses written out plainly there.
Tolerance: about ten products of at most 64 terms forward and as many back, each
within 2^-21 of its size, so 2e-5 in all.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from opake_amd.clipping import ghost_clipped_grad
from opake_amd.moe import RoutedLM, TopKMoE
from oracle import clip_oracle, ghost_oracle

pytestmark = pytest.mark.gpu

TOL = 2e-5
V, D, HEADS, FFN, INTER, E, K = 61, 32, 4, 48, 40, 8, 3
ROUTING = dict(score="sigmoid", groups=4, top_groups=2, scale=1.5)


def _plain_route(moe, margin):
    """The 64-bit form of ``ROUTING``; ``margin`` collects the gap to the next choice."""

    def route(x, router_logits=None):
        score = torch.sigmoid(moe.router(x) if router_logits is None else router_logits)
        choice = score.detach() + moe.route_bias.double()
        best = choice.view(*choice.shape[:-1], 4, 2).amax(-1)
        order = best.sort(dim=-1, descending=True)
        margin.append((order.values[..., 1] - order.values[..., 2]).min().item())
        keep = torch.zeros_like(best, dtype=torch.bool).scatter(-1, order.indices[..., :2], True)
        choice = choice.masked_fill(~keep.repeat_interleave(2, dim=-1), -torch.inf)
        ranked = choice.sort(dim=-1, descending=True)
        gaps = ranked.values[..., :K] - ranked.values[..., 1:K + 1]
        margin.append(gaps.min().item())
        top = ranked.indices[..., :K]
        w = score.gather(-1, top)
        return top, 1.5 * w / w.sum(-1, keepdim=True)

    return route


def _plain_loss(model):
    def loss(outputs, targets):
        hidden, teacher, index = outputs
        z = model.head(hidden)
        ce = F.cross_entropy(z.flatten(0, 1), targets.flatten(), reduction="none",
                             ignore_index=-100).view(targets.shape)
        tau = model.temperature
        logq = torch.log_softmax(teacher.double() / tau, -1)
        logp = torch.log_softmax(z / tau, -1).gather(-1, index)
        kl = tau * tau * (logq.exp() * (logq - logp)).sum(-1)
        return ((1 - model.distill) * ce + model.distill * kl).mean(dim=1)

    return loss


def _case(B, T, seed):
    torch.manual_seed(seed)
    ref = RoutedLM(V, D, HEADS, FFN, INTER, E, K, routing=ROUTING, temperature=2.0,
                   dtype=torch.float64)
    with torch.no_grad():
        for n, p in ref.named_parameters():
            p.normal_(0.0, 0.25)
            p.copy_(p.float().double())
        ref.moe.route_bias.normal_(0.0, 0.02)
    g = torch.Generator().manual_seed(seed + 1)
    ids = torch.randint(0, V, (B, T), generator=g)
    tgt = torch.randint(0, V, (B, T), generator=g)
    tgt[0, :5] = -100
    index = torch.argsort(torch.rand(B, T, V, generator=g), dim=-1)[..., :6]
    teacher = 2 * torch.randn(B, T, 6, generator=g)
    return ref, ids, tgt, teacher, index


def _gpu_model(ref, dev):
    model = RoutedLM(V, D, HEADS, FFN, INTER, E, K, routing=ROUTING, temperature=2.0,
                     dtype=torch.float32).to(dev)
    model.load_state_dict({k: v.float() for k, v in ref.state_dict().items()})
    return model


@pytest.mark.parametrize("microbatch", [None, 2])
def test_clipped_gradients_match_per_example_ones(dev, microbatch):
    ref, ids, tgt, teacher, index = _case(3, 20, seed=6)
    model = _gpu_model(ref, dev)
    margin = []
    ref.moe.route = _plain_route(ref.moe, margin)
    per = ghost_oracle.per_example_grads_loop(ref, _plain_loss(ref), (ids, teacher, index), tgt)
    assert min(margin) > 1e-4  # no choice that float32 could make otherwise
    names = sorted(n for n, p in model.named_parameters() if p.requires_grad)
    want = clip_oracle.stream_clip_and_sum([per[n].float() for n in names],
                                           clip_oracle.conservative_bound(0.45),
                                           return_aux=True)
    fn, st = ghost_clipped_grad(model, model.loss, clipping_norm=0.45, normalize_by=3.0,
                                return_aux=True, microbatch_size=microbatch)
    inputs = tuple(t.to(dev) for t in (ids, teacher, index))
    (out, aux), _ = fn(inputs, tgt.to(dev), state=st)
    assert sorted(out.pytree) == names
    for i, n in enumerate(names):
        got, exp = out.pytree[n].double().cpu(), want.reduced[i].double() / 3.0
        assert ((got - exp).norm() / exp.norm().clamp_min(1e-300)).item() < TOL, n
    torch.testing.assert_close(aux.grad_norms.cpu().double(), want.norms.double(), rtol=TOL,
                               atol=0)


def test_tokens_with_fewer_experts_than_asked_for(dev):
    """Masked experts: a token goes to those it has left, or to none."""
    torch.manual_seed(1)
    moe = TopKMoE(D, INTER, 4, 2, routing={}, dtype=torch.float32).to(dev)
    x = torch.randn(2, 3, D, device=dev)
    logits = torch.randn(2, 3, 4, device=dev)
    logits[0, 0, 1:] = -torch.inf
    logits[1, 2] = -torch.inf
    y = moe(x, logits)
    torch.testing.assert_close(y[0, 0], moe.experts[0](x[0, :1])[0], rtol=1e-5, atol=1e-6)
    assert torch.equal(y[1, 2], torch.zeros_like(y[1, 2]))
    assert int(moe.last_counts.sum()) == 2 * 6 - 1 - 2
    plain = TopKMoE(D, INTER, 4, 2, dtype=torch.float32).to(dev)
    plain.load_state_dict({k: v for k, v in moe.state_dict().items() if k != "route_bias"})
    some = torch.randn(2, 3, 4, device=dev)
    torch.testing.assert_close(moe(x, some), plain(x, some), rtol=1e-5, atol=1e-6)


def test_loss_without_a_teacher(dev):
    ref, ids, tgt, _, _ = _case(2, 9, seed=9)
    model = _gpu_model(ref, dev)
    hidden = model(ids.to(dev))
    z = F.linear(hidden.double(), model.head.weight.double())
    want = F.cross_entropy(z.flatten(0, 1), tgt.to(dev).flatten(), reduction="none",
                           ignore_index=-100).view(tgt.shape).mean(dim=1)
    torch.testing.assert_close(model.loss(hidden, tgt.to(dev)).double(), want, rtol=1e-5,
                               atol=1e-5)


def test_ignored_targets_and_the_teacher(dev):
    """An ignored target takes its token out of the cross entropy alone; the teacher's KL
    there goes by the teacher's entries, and negative indices take it out as well."""
    ref, ids, tgt, teacher, index = _case(2, 9, seed=11)
    model = _gpu_model(ref, dev)
    ids, tgt, teacher, index = (x.to(dev) for x in (ids, tgt, teacher, index))
    tgt[1, 3] = -100
    ignored = (tgt == -100).unsqueeze(-1)
    other = torch.where(ignored, teacher + torch.randn_like(teacher), teacher)

    hidden = model(ids).detach().requires_grad_(True)

    def run(teacher, index):
        loss = model.loss((hidden, teacher, index), tgt)
        return loss, torch.autograd.grad(loss.sum(), [hidden])[0]

    a, b = run(teacher, index), run(other, index)
    assert (a[0] != b[0]).all() and not torch.equal(a[1], b[1])
    out = index.masked_fill(ignored, -1)
    c, d = run(teacher, out), run(other, out)
    assert torch.equal(c[0], d[0]) and torch.equal(c[1], d[1])
    want = _plain_loss(ref.double().to(dev))((hidden.double(), teacher, index), tgt)
    torch.testing.assert_close(a[0].double(), want, rtol=1e-5, atol=1e-5)


def test_a_cast_model_routes(dev):
    torch.manual_seed(3)
    moe = TopKMoE(D, INTER, 4, 2, routing=dict(score="sigmoid")).to(dev, torch.bfloat16)
    x = torch.randn(2, 3, D, device=dev, dtype=torch.bfloat16)
    assert moe(x).shape == x.shape and moe(x).dtype == torch.bfloat16


def test_nan_logits_reach_the_output(dev):
    """A token of which a logit, or every logit, is NaN has a NaN output, with or without
    ``routing``; the other tokens keep theirs."""
    torch.manual_seed(2)
    plain = TopKMoE(D, INTER, 4, 2, dtype=torch.float32).to(dev)
    moe = TopKMoE(D, INTER, 4, 2, routing={}, dtype=torch.float32).to(dev)
    moe.load_state_dict(plain.state_dict(), strict=False)
    x = torch.randn(2, 3, D, device=dev)
    logits = torch.randn(2, 3, 4, device=dev)
    want = moe(x, logits)
    logits[0, 1] = torch.nan
    logits[1, 2, 3] = torch.nan
    bad = torch.isnan(logits).any(-1)
    for m in (plain, moe):
        y = m(x, logits)
        assert torch.isnan(y[bad]).all()
        torch.testing.assert_close(y[~bad], want[~bad], rtol=1e-5, atol=1e-6)


def test_bfloat16(dev):
    """Every expert chosen, so that no rounding can change a choice.  About twenty roundings
    to 2^-8 (2^-9 on average) forward and back, half of them along one path: 8%."""
    torch.manual_seed(5)
    kw = dict(routing=dict(score="sigmoid", scale=1.5), temperature=2.0)
    ref = RoutedLM(V, D, HEADS, FFN, INTER, 4, 4, dtype=torch.float64, **kw)
    with torch.no_grad():
        for p in ref.parameters():
            p.normal_(0.0, 0.25)
            p.copy_(p.bfloat16().double())
    _, ids, tgt, teacher, index = _case(3, 20, seed=8)
    model = RoutedLM(V, D, HEADS, FFN, INTER, 4, 4, dtype=torch.bfloat16, **kw).to(dev)
    model.load_state_dict(ref.state_dict())

    def route(x, router_logits=None):
        score = torch.sigmoid(ref.moe.router(x))
        every = torch.arange(4).expand(score.shape)
        return every, 1.5 * score / score.sum(-1, keepdim=True)

    ref.moe.route = route
    per = ghost_oracle.per_example_grads_loop(ref, _plain_loss(ref), (ids, teacher, index), tgt)
    names = sorted(n for n, p in model.named_parameters() if p.requires_grad)
    want = clip_oracle.stream_clip_and_sum([per[n].float() for n in names],
                                           clip_oracle.conservative_bound(0.45),
                                           return_aux=True)
    fn, st = ghost_clipped_grad(model, model.loss, clipping_norm=0.45, return_aux=True)
    (out, aux), _ = fn(tuple(t.to(dev) for t in (ids, teacher, index)), tgt.to(dev), state=st)
    torch.testing.assert_close(aux.grad_norms.cpu().double(), want.norms.double(), rtol=0.08,
                               atol=0)
    for i, n in enumerate(names):
        got, exp = out.pytree[n].double().cpu(), want.reduced[i].double()
        assert ((got - exp).norm() / exp.norm()).item() < 0.08, n
