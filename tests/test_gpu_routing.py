"""Routing to experts: choice, weights and gradients against 64 bits (GPU).

Tolerances: the kernel's exponentials and divisions are within a few ulp and their
arguments are rounded once, so a score is within ``2^-20 (1 + |z - max z|)`` of itself
(relative); weights and gradients follow by sums of at most k of them.
"""

from __future__ import annotations

import math

import pytest
import torch

from opake_amd import routing
from opake_amd.exceptions import ConfigurationError, InputTypeError


def _reference(z, k, score, bias, groups, top_groups, renormalize, scale, up):
    """Plain 64-bit rounds of argmax (lowest index first) and autograd."""
    z0 = z.detach().double().reshape(-1, z.shape[-1])
    N, E = z0.shape
    x = z0.clone().requires_grad_(True)
    closed = ~(z0 > -math.inf)
    if score == "softmax":
        none = closed.all(1, keepdim=True)
        s = torch.softmax(torch.where(none, 0.0, torch.where(closed, -math.inf, x)), 1)
        s = torch.where(closed, 0.0, s)
    else:
        s = torch.where(closed, 0.0, torch.sigmoid(x))
    key = (s.detach() + bias.double()) if bias is not None else z0.clone()
    key = torch.where(closed, -math.inf, key)

    def first(v):
        top, n = v.amax(1, keepdim=True), v.shape[1]
        at = torch.where(v == top, torch.arange(n, device=v.device), n).amin(1)
        return at.clamp(max=n - 1), top.squeeze(1) > -math.inf

    if top_groups < groups:
        best = key.view(N, groups, -1).amax(2)
        kept = torch.zeros(N, groups, dtype=torch.bool, device=z.device)
        for _ in range(top_groups):
            at, there = first(best)
            kept[torch.arange(N, device=z.device)[there], at[there]] = True
            best = best.scatter(1, at[:, None], -math.inf)
        key = torch.where(kept.repeat_interleave(E // groups, 1), key, -math.inf)
    experts, chosen = [], []
    for _ in range(k):
        at, there = first(key)
        experts.append(torch.where(there, at, -1))
        chosen.append(torch.where(there, s.gather(1, at[:, None]).squeeze(1), 0.0))
        key = key.scatter(1, at[:, None], -math.inf)
    w = torch.stack(chosen, 1)
    experts = torch.stack(experts, 1)
    if renormalize and score == "softmax":
        # A softmax over the chosen: exactly no gradient elsewhere.
        there = experts >= 0
        zc = torch.where(there, x.gather(1, experts.clamp(min=0)), -math.inf)
        some = there.any(1, keepdim=True)
        w = torch.where(there, torch.softmax(torch.where(some, zc, 0.0), 1), 0.0)
    elif renormalize:
        tot = w.sum(1, keepdim=True)
        w = w / torch.where(tot > 0, tot, 1.0)
    w = w * scale
    (dz,) = torch.autograd.grad(w, [x], up.double().reshape(N, k))
    return w.detach(), experts, torch.where(closed, 0.0, dz)


def _check(z, k, score="softmax", bias=None, groups=1, top_groups=None, renormalize=True,
           scale=1.0, seed=0):
    g = torch.Generator(device=z.device).manual_seed(seed)
    up = torch.randn(*z.shape[:-1], k, generator=g, device=z.device)
    z = z.detach().requires_grad_(True)
    w, e = routing.route_topk(z, k, score=score, bias=bias, groups=groups, top_groups=top_groups,
                              renormalize=renormalize, scale=scale)
    assert w.shape == e.shape == (*z.shape[:-1], k)
    assert w.dtype == torch.float32 and e.dtype == torch.int64 and not e.requires_grad
    (dz,) = torch.autograd.grad(w, [z], up)
    assert dz.shape == z.shape and dz.dtype == z.dtype
    rw, re, rdz = _reference(z, k, score, bias, groups, groups if top_groups is None else top_groups,
                             renormalize, scale, up)
    assert torch.equal(e.reshape(re.shape), re)
    open_ = torch.where(z.detach().double() > -math.inf, z.detach().double(), math.nan)
    span = open_.reshape(-1, z.shape[-1]).abs().nan_to_num(0.0).amax(1, keepdim=True)
    rel = 2.0**-20 * (1 + 2 * span) * (k + 2)
    assert ((w.detach().double().reshape(rw.shape) - rw).abs() <= rel * rw.abs() + 1e-30).all()
    rnd = {torch.float32: 2.0**-23, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-10}[z.dtype]
    tiny = 2.0**-24 if z.dtype == torch.float16 else 1e-30
    # What the terms of a value can be off by: its own weight's and the row's sum of |g w|.
    s = (rw / scale).abs()
    gabs = up.double().reshape(rw.shape).abs() * abs(scale)
    if renormalize or score == "softmax":
        row = (gabs * s).sum(1, keepdim=True) + gabs.amax(1, keepdim=True)
    else:
        row = gabs.amax(1, keepdim=True)
    if score == "softmax" and not renormalize:
        zd = torch.where(torch.isnan(open_), -math.inf, open_).reshape(-1, z.shape[-1])
        size = torch.softmax(zd, 1).nan_to_num(0.0)
    else:
        # (Added up: an empty slot's place is expert 0's too.)
        size = torch.zeros_like(rdz).scatter_add_(1, re.clamp(min=0),
                                                  torch.where(re >= 0, 1.0, 0.0).double())
    tol = rel * row * size + rnd * rdz.abs() + tiny
    err = (dz.double().reshape(rdz.shape) - rdz).abs()
    assert (err <= tol).all(), (err / tol).max().item()


def _logits(dev, lead, E, dtype, seed=0, spread=1.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*lead, E, generator=g, device=dev) * spread).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16],
                         ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("lead,E,k", [
    ((1,), 1, 1), ((5,), 2, 1), ((3, 7), 8, 2), ((130,), 7, 4), ((257,), 60, 4), ((33,), 64, 16),
    ((65,), 65, 17), ((4097,), 256, 8), ((16,), 256, 8), ((50,), 255, 64), ((19,), 1000, 5),
    ((9,), 1024, 64),
])
def test_choice_weights_and_gradient(dev, lead, E, k, score, renormalize, dtype):
    """bfloat16 and float16 logits hold many exact ties."""
    _check(_logits(dev, lead, E, dtype, E + k), k, score, renormalize=renormalize, scale=2.5)


def _grid_bias(dev, E, seed):
    """Distinct biases between 0 and 3, in no order."""
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randperm(E, generator=g, device=dev).float() * (3.0 / E)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k,groups,top_groups", [
    (8, 2, 1, 1), (16, 3, 4, 2), (60, 4, 6, 3), (96, 6, 3, 1), (256, 8, 8, 4), (384, 8, 8, 3),
    (1024, 32, 64, 8), (12, 2, 12, 5),
])
def test_bias_and_groups(dev, E, k, groups, top_groups, score):
    """Rows in which two keys are nearer than float32 rounding of keys below 4 could
    swap (2^-21) are left out: there either choice is right."""
    z = _logits(dev, (700,), E, torch.float32, E)
    bias = _grid_bias(dev, E, k)
    s = torch.softmax(z.double(), 1) if score == "softmax" else torch.sigmoid(z.double())
    v = (s + bias.double()).sort(1).values
    z = z[(v[:, 1:] - v[:, :-1]).amin(1) > 2e-6]
    assert z.shape[0] >= 50
    _check(z, k, score, bias, groups, top_groups, scale=2.5)
    _check(z, k, score, bias, groups, top_groups, renormalize=False)
    _check(z, k, score, None, groups, top_groups)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_masks_that_leave_few_or_none(dev, score, renormalize):
    z = _logits(dev, (300,), 24, torch.float32, 4)
    g = torch.Generator(device=dev).manual_seed(1)
    z[torch.rand(300, 24, generator=g, device=dev) < 0.8] = -math.inf
    z[7] = -math.inf
    z[8, 1:] = -math.inf
    _check(z, 6, score, renormalize=renormalize)
    _check(z, 6, score, None, 4, 2, renormalize=renormalize)
    w, e = routing.route_topk(z, 6, score=score, renormalize=renormalize)
    assert (e[7] == -1).all() and (w[7] == 0).all()
    assert e[8].tolist() == [0 if z[8, 0] > -math.inf else -1, -1, -1, -1, -1, -1]
    one = torch.full((1, 24), -math.inf, device=dev)
    one[0, 17] = 0.25
    assert routing.route_topk(one, 6, score=score)[1].tolist() == [[17, -1, -1, -1, -1, -1]]
    # The type's lowest value is a logit like any other.
    z[9] = torch.finfo(torch.float32).min
    w, e = routing.route_topk(z[9], 2, score=score)
    assert e.tolist() == [0, 1] and torch.isfinite(w).all()


@pytest.mark.gpu
def test_all_equal_logits_choose_the_first(dev):
    for E, k in ((8, 4), (64, 16), (256, 8), (1000, 64)):
        z = torch.zeros(3, E, device=dev)
        z[1, ::2] = -0.0  # equal to 0
        w, e = routing.route_topk(z, k)
        assert (e == torch.arange(k, device=dev)).all()
        assert ((w - 1.0 / k).abs() <= 2.0**-20).all()


@pytest.mark.gpu
def test_extreme_and_nan_logits(dev):
    z = torch.tensor([[200.0, -200.0, 0.0, 199.0], [-300.0, -300.5, -301.0, -302.0],
                      [math.nan, 1.0, 2.0, 3.0]], device=dev)
    w, e = routing.route_topk(z, 2)
    assert e[:2].tolist() == [[0, 3], [0, 1]] and torch.isnan(w[2]).all()
    want = torch.softmax(torch.tensor([[200.0, 199.0], [-300.0, -300.5]]).double(), 1)
    assert ((w[:2].cpu().double() - want).abs() <= 2.0**-18).all()
    # Sigmoids that underflow: weights 0, not 0 / 0.
    w, _ = routing.route_topk(z[1:2], 2, score="sigmoid")
    assert (w == 0).all()


@pytest.mark.gpu
def test_views_streams_and_graph(dev):
    z = _logits(dev, (6, 50), 32, torch.float32, 3)
    want = routing.route_topk(z, 4)
    wide = torch.cat([z, z], -1)
    for view in (wide[..., :32], z.transpose(0, 1).contiguous().transpose(0, 1)):
        assert all(torch.equal(a, b) for a, b in zip(routing.route_topk(view, 4), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = routing.route_topk(z, 4)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    x = z.clone().requires_grad_(True)

    def step():
        w, e = routing.route_topk(x, 4)
        (dz,) = torch.autograd.grad(w, [x], torch.ones_like(w).cumsum(-1))
        return w.detach(), e, dz

    ref = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ref))


@pytest.mark.gpu
def test_differences(dev):
    """<gradient, d> against central differences of the kernel's own weights; with the
    softmax's own weights every logit counts.  Third derivatives of a softmax along d
    are at most range(d)^3, the weights' rounding 2^-20 of weights below 1."""
    z = _logits(dev, (200,), 16, torch.float32, 8).requires_grad_(True)
    g = torch.Generator(device=dev).manual_seed(2)
    up = torch.randn(200, 3, generator=g, device=dev)
    d = torch.randn(200, 16, generator=g, device=dev)
    eps = 2.0**-6
    w, e = routing.route_topk(z, 3, renormalize=False)
    (dz,) = torch.autograd.grad(w, [z], up)
    hi, eh = routing.route_topk(z + eps * d, 3, renormalize=False)
    lo, el = routing.route_topk(z - eps * d, 3, renormalize=False)
    same = ((eh == e) & (el == e)).all(1)
    assert same.sum() > 100
    slope = ((hi - lo).double() * up.double()).sum(1) / (2 * eps)
    want = (dz.double() * d.double()).sum(1)
    span = (d.amax(1) - d.amin(1)).double()
    size = up.abs().double().sum(1)
    step = 2.0**-24 * (z.detach().abs() + eps * d.abs()).double().amax(1) * 2 / eps
    tol = size * (eps**2 / 6 * span**3 + 2.0**-18 * 2 / (2 * eps) + step + 2.0**-18 * span)
    assert ((slope - want).abs() <= tol)[same].all()


@pytest.mark.gpu
def test_no_tokens_and_no_gradient(dev):
    z = torch.zeros(0, 8, device=dev, requires_grad=True)
    w, e = routing.route_topk(z, 2)
    assert w.shape == e.shape == (0, 2)
    (dz,) = torch.autograd.grad(w.sum(), [z])
    assert dz.shape == (0, 8)
    w, _ = routing.route_topk(torch.zeros(4, 8, device=dev), 2)
    assert not w.requires_grad


@pytest.mark.gpu
def test_refusals(dev):
    z = torch.zeros(4, 12, device=dev)
    bad = [
        (ConfigurationError, lambda: routing.route_topk(z, 0)),
        (ConfigurationError, lambda: routing.route_topk(z, 13)),
        (ConfigurationError, lambda: routing.route_topk(z, 5, groups=3, top_groups=1)),
        (ConfigurationError, lambda: routing.route_topk(z, 2, groups=5)),
        (ConfigurationError, lambda: routing.route_topk(z, 2, groups=3, top_groups=4)),
        (ConfigurationError, lambda: routing.route_topk(z, 2, score="relu")),
        (ConfigurationError, lambda: routing.route_topk(z.double(), 2)),
        (ConfigurationError, lambda: routing.route_topk(torch.zeros(1, 1025, device=dev), 2)),
        (ConfigurationError, lambda: routing.route_topk(torch.zeros(1, 100, device=dev), 65)),
        (ConfigurationError, lambda: routing.route_topk(z, 2, bias=torch.zeros(11, device=dev))),
        (ConfigurationError, lambda: routing.route_topk(z, 2, bias=z[0].bfloat16())),
        (ConfigurationError, lambda: routing.route_topk(z, 2, scale=math.inf)),
        (InputTypeError, lambda: routing.route_topk(z, 2.0)),
        (InputTypeError, lambda: routing.route_topk(z, 2, scale="1")),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def test_cpu_tensors_are_refused():
    with pytest.raises(ConfigurationError, match="ROCm device"):
        routing.route_topk(torch.zeros(4, 12), 2)


def _top2_reference(z, k, score, bias, groups, top_groups):
    """The choice in 64 bits, with the gap of every row's closest decision over the size
    of its keys."""
    N, E = z.shape
    zd = z.double()
    closed = ~(zd > -math.inf)
    s = torch.sigmoid(zd) if score == "sigmoid" else torch.softmax(zd, 1).nan_to_num(0.0)
    key = torch.where(closed, -math.inf, s if bias is None else s + bias.double())
    two = key.view(N, groups, -1).sort(dim=2, descending=True).values[..., :2]
    best = torch.where(two > -math.inf, two, 0.0).sum(2)
    best = torch.where(two[..., 0] > -math.inf, best, -math.inf)

    def ranked(v, n):
        v, at = v.sort(dim=1, descending=True, stable=True)
        gap = v[:, :n] - v[:, 1:n + 1] if v.shape[1] > n else v[:, :n - 1] - v[:, 1:n]
        return v, at, torch.where(gap.isnan(), math.inf, gap)

    v, at, gap = ranked(best, top_groups)
    near = gap[:, -1] if top_groups < groups else torch.full((N,), math.inf, device=z.device)
    keep = torch.zeros(N, groups, dtype=torch.bool, device=z.device)
    keep.scatter_(1, at[:, :top_groups], v[:, :top_groups] > -math.inf)
    key = torch.where(keep.repeat_interleave(E // groups, 1), key, -math.inf)
    v, at, gap = ranked(key, k)
    near = torch.minimum(near, gap.amin(1)) if gap.numel() else near
    size = torch.where(closed, 0.0, key).nan_to_num(0.0, neginf=0.0).abs().amax(1)
    return torch.where(v[:, :k] > -math.inf, at[:, :k], -1), near / size


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [True, False])
@pytest.mark.parametrize("N,E,k,groups,top_groups", [
    (700, 8, 2, 2, 1), (700, 16, 3, 4, 2), (700, 60, 4, 6, 3), (700, 256, 8, 8, 4),
    (5000, 256, 8, 8, 4), (5000, 128, 6, 2, 1), (5000, 192, 8, 3, 2), (700, 384, 8, 8, 3),
    (300, 1024, 32, 64, 8), (700, 12, 2, 12, 5), (700, 36, 5, 18, 7), (900, 64, 17, 4, 3),
])
def test_groups_by_the_sum_of_their_two_best(dev, N, E, k, groups, top_groups, score, biased):
    """Rows in which two of the keys or sums that the choice goes by are nearer than
    float32 rounding could swap are left out."""
    g = torch.Generator(device=dev).manual_seed(E + k)
    z = torch.randn(N, E, generator=g, device=dev) * 1.5
    z[torch.rand(N, E, generator=g, device=dev) < 0.2] = -math.inf
    z[0] = -math.inf
    z[1, 1:] = -math.inf
    bias = None
    if biased:
        bias = torch.randint(-60, 61, (E,), generator=g, device=dev).float() * 1e-3
    want, near = _top2_reference(z, k, score, bias, groups, top_groups)
    w, e = routing.route_topk(z, k, score=score, bias=bias, groups=groups,
                              top_groups=top_groups, group_score="top2")
    ok = ~(near <= 4e-6)
    assert ok.sum() >= 0.5 * N
    assert torch.equal(e[ok], want[ok])
    # The weights and their gradient are those of the same experts however chosen.
    up = torch.randn(N, k, generator=g, device=dev)
    x = z.clone().requires_grad_(True)
    w, e = routing.route_topk(x, k, score=score, bias=bias, groups=groups, scale=2.5,
                              top_groups=top_groups, group_score="top2")
    (dz,) = torch.autograd.grad(w, [x], up)
    xd = z.double().requires_grad_(True)
    there = e >= 0
    zc = xd.gather(1, e.clamp(min=0))
    s = torch.sigmoid(zc) if score == "sigmoid" else torch.exp(
        zc - torch.where(there, zc, -math.inf).amax(1, keepdim=True).nan_to_num(0.0, neginf=0.0))
    s = torch.where(there, s, 0.0)
    tot = s.sum(1, keepdim=True)
    wd = 2.5 * s / torch.where(tot > 0, tot, 1.0)
    (dd,) = torch.autograd.grad(wd, [xd], up.double())
    dd = torch.where(z > -math.inf, dd.nan_to_num(0.0), 0.0)
    span = z.nan_to_num(0.0, neginf=0.0).abs().amax(1, keepdim=True).double()
    rel = 2.0**-20 * (1 + 2 * span) * (k + 2)
    assert ((w.double() - wd).abs() <= rel * wd.abs() + 1e-30).all()
    row = 2.5 * up.double().abs().sum(1, keepdim=True)
    assert ((dz.double() - dd).abs() <= 2 * rel * row).all()


@pytest.mark.gpu
def test_the_group_rules_differ(dev):
    """A group with the largest key against one with two large ones; ties of sums go to the
    first group; a group of one open expert counts that alone."""
    inf = math.inf
    z = torch.tensor([[3.0, -3.0, 1.0, 1.0], [1.0, 0.0, 0.0, 1.0], [3.0, -inf, 0.0, 0.0],
                      [3.0, -inf, -9.0, -9.0]], device=dev)
    for score in ("softmax", "sigmoid"):
        kw = dict(score=score, groups=2, top_groups=1)
        assert routing.route_topk(z, 2, **kw)[1].tolist() == [[0, 1], [0, 1], [0, -1], [0, -1]]
        by_two = routing.route_topk(z, 2, group_score="top2", **kw)[1].tolist()
        # softmax: 3 against 1 + 1 is e^3 + e^-3 against 2 e
        first = [0, 1] if score == "softmax" else [2, 3]
        third = [0, -1] if score == "softmax" else [2, 3]
        assert by_two == [first, [0, 1], third, [0, -1]]
    with pytest.raises(ConfigurationError):
        routing.route_topk(z, 2, group_score="sum", **kw)


@pytest.mark.gpu
def test_scales_that_float32_cannot_hold_are_refused(dev):
    z = torch.zeros(4, 12, device=dev)
    for scale in (1e39, -1e300):
        with pytest.raises(ConfigurationError):
            routing.route_topk(z, 2, scale=scale)
