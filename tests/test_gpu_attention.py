"""Attention and its gradients (GPU) against softmax attention in 64 bits on the CPU.

Tolerances are elementwise and follow the roundings, with u = 2^-23 for a float32
operation in any order of its sum, K terms each (K + 8) u of the sum of their magnitudes.
A score is within es = (h + 8) u scale (|q| |k|) of its own, relative errors of
probabilities are then ep = 2 max es + 32 u (exponential, maximum, sum).  bf16: probabilities
and ds go to the products in bf16 (2^-8 of themselves more), and the results are rounded
(2^-8); D is taken of the output with what that took from it, within 2^-17.
"""

from __future__ import annotations

import math

import pytest
import torch

from opake_amd import _native as nat
from opake_amd.attention import attention
from opake_amd.exceptions import ConfigurationError, InputTypeError, OperationError

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
U = 2.0 ** -23


def _seen(B, T, S, causal, window, lengths, starts):
    j = torch.arange(S)
    n = torch.full((B, 1, 1), S) if lengths is None else lengths.cpu().long().view(-1, 1, 1)
    n = n.clamp(0, S)
    seen = (j < n).expand(B, T, S)
    if causal:
        first = torch.full((B, 1, 1), S - T) if starts is None else starts.cpu().long().view(
            -1, 1, 1)
        at = first + torch.arange(T).view(1, T, 1)
        seen = seen & (j <= at) & (at < n)
        if window:
            seen = seen & (j > at - window)
    return seen


def _reference(q, k, v, up, causal=True, window=None, lengths=None, starts=None, scale=None):
    """(value, tolerance) of out, dq, dk and dv."""
    half = 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0
    B, T, H, h = q.shape
    S, KV = k.shape[1:3]
    rep = H // KV
    scale = scale or h ** -0.5
    seen = _seen(B, T, S, causal, window, lengths, starts)[:, None]
    qd, kd, vd, gd = (t.detach().cpu().double().transpose(1, 2) for t in (q, k, v, up))
    some = seen.any(-1, keepdim=True)
    # Padding reaches nothing, whatever it is.
    used = seen.any(-2)[..., None]
    kd, vd = (torch.where(used, t, 0.0).repeat_interleave(rep, 1) for t in (kd, vd))
    qd, gd = torch.where(some, qd, 0.0), torch.where(some, gd, 0.0)
    z = torch.where(seen, scale * qd @ kd.mT, -math.inf)
    p = torch.where(some, torch.softmax(torch.where(some, z, 0.0), -1), 0.0)
    es = torch.where(seen, (h + 8) * U * scale * (qd.abs() @ kd.abs().mT), 0.0)
    ep = 2 * es.amax(-1, keepdim=True) + 32 * U if S else torch.zeros(B, H, T, 1).double()
    o = p @ vd
    pv = p @ vd.abs()
    eo = (ep + half + (S + 8) * U) * pv
    eD = eo + (2.0 ** -17 * o.abs() if half else 0.0)
    eo = eo + half * (o.abs() + eo)
    dp = gd @ vd.mT
    D = (gd * o).sum(-1, keepdim=True)
    edp = (h + 8) * U * (gd.abs() @ vd.abs().mT)
    eD = (gd.abs() * eD).sum(-1, keepdim=True) + (h + 8) * U * (gd.abs() * o.abs()).sum(
        -1, keepdim=True)
    ds = p * (dp - D)
    eds = p * (edp + eD) + (ep + half + 4 * U) * p * (dp.abs() + D.abs())
    full = ds.abs() + eds
    dq, edq = scale * ds @ kd, scale * (eds @ kd.abs() + (S + 8) * U * full @ kd.abs())
    rows = rep * T + 8
    dk, edk = scale * ds.mT @ qd, scale * (eds.mT @ qd.abs() + rows * U * full.mT @ qd.abs())
    dv = p.mT @ gd
    edv = ((ep + half) * p).mT @ gd.abs() + rows * U * p.mT @ gd.abs()

    def heads(t):
        return t.view(B, KV, rep, S, h).sum(2)

    out = []
    for w, e, shared in ((o, eo, False), (dq, edq, False), (dk, edk, True), (dv, edv, True)):
        w, e = (heads(w), heads(e)) if shared else (w, e)
        e = e if w is o else e + half * (w.abs() + e)
        out.append((w.transpose(1, 2), e.transpose(1, 2) + 1e-30))
    return out


def _check(got, refs):
    for name, t, (want, tol) in zip(("out", "dq", "dk", "dv"), got, refs):
        err = (t.detach().cpu().double() - want).abs()
        assert bool((err <= tol).all()), (name, (err / tol).max().item(), err.max().item())


def _inputs(B, T, S, H, KV, h, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed + T + 7 * S + h)
    if S == T:  # places of one tensor, as a fused projection leaves them
        x = torch.randn(B, T, H + 2 * KV, h, generator=g).to(dtype).to(dev)
        q, k, v = x[:, :, :H], x[:, :, H:H + KV], x[:, :, H + KV:]
    else:
        q = torch.randn(B, T, H, h, generator=g).to(dtype).to(dev)
        k, v = torch.randn(2, B, S, KV, h, generator=g).to(dtype).to(dev)
    up = torch.randn(B, T, H, h, generator=g).to(dtype).to(dev)
    return [t.detach().requires_grad_() for t in (q, k, v)] + [up]


def _run(q, k, v, up, **kw):
    out = attention(q, k, v, **kw)
    return (out, *torch.autograd.grad(out, [q, k, v], up))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,T,S,H,KV,h", [
    (1, 1, 1, 1, 1, 8), (2, 3, 3, 2, 1, 16), (1, 31, 31, 4, 4, 64), (2, 33, 33, 3, 1, 40),
    (1, 64, 64, 2, 2, 128), (1, 65, 65, 6, 2, 80), (1, 129, 129, 8, 2, 128),
    (2, 200, 200, 7, 1, 96), (1, 130, 130, 2, 1, 256), (1, 70, 70, 1, 1, 192),
    (1, 5, 77, 4, 2, 64), (3, 1, 300, 8, 2, 128), (1, 40, 500, 16, 1, 32), (1, 2, 130, 2, 2, 256),
    (2, 20, 20, 2, 1, 7), (1, 50, 20, 2, 2, 24), (1, 300, 300, 2, 2, 64), (1, 1, 2100, 4, 4, 64),
    (2, 3, 1500, 6, 2, 256), (1, 33, 700, 16, 1, 96), (1, 2, 900, 70, 1, 64), (1, 130, 130, 130, 1, 16),
    (16, 260, 260, 16, 16, 64), (3, 500, 500, 48, 24, 128)])
def test_causal(dev, dtype, B, T, S, H, KV, h):
    x = _inputs(B, T, S, H, KV, h, DTYPES[dtype], dev)
    _check(_run(*x), _reference(*x))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,S,h", [(1, 1, 64), (37, 90, 128), (130, 65, 64), (3, 700, 16)])
def test_all_keys(dev, dtype, T, S, h):
    x = _inputs(2, T, S, 4, 2, h, DTYPES[dtype], dev)
    _check(_run(*x, causal=False), _reference(*x, causal=False))
    n = torch.tensor([S // 2, 0], device=dev)
    _check(_run(*x, causal=False, lengths=n, scale=0.3),
           _reference(*x, causal=False, lengths=n, scale=0.3))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 1000])
@pytest.mark.parametrize("T,S", [(150, 150), (9, 333)])
def test_windows(dev, dtype, window, T, S):
    x = _inputs(2, T, S, 6, 2, 64, DTYPES[dtype], dev)
    n = torch.tensor([S, S - 3], device=dev)
    for kw in (dict(window=window), dict(window=window, lengths=n)):
        _check(_run(*x, **kw), _reference(*x, **kw))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T", [1, 63, 64, 130, 260])
def test_padding_reaches_nothing(dev, dtype, T):
    """Lengths from none to all, with NaN and infinities behind them."""
    lengths = torch.tensor([0, 1, T // 2, T - 1, T, T + 5, -2], device=dev)
    x = _inputs(7, T, T, 4, 2, 64, DTYPES[dtype], dev)
    refs = _reference(*x, lengths=lengths)
    with torch.no_grad():
        for i, t in enumerate(x):
            for b, n in enumerate(lengths.tolist()):
                t[b, max(n, 0):] = math.nan if i % 2 else math.inf
    got = _run(*x, lengths=lengths)
    _check(got, refs)
    for t in got:  # padding itself: exactly zero
        for b, n in enumerate(lengths.tolist()):
            assert not t[b, max(n, 0):].any()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,S", [(1, 600), (5, 600), (40, 333)])
def test_sequences_in_caches(dev, dtype, T, S):
    """The last tokens of sequences of different lengths, some longer than they are."""
    lengths = torch.tensor([S, S // 2, T, 1, 0, S - 1], device=dev)
    starts = lengths - T
    x = _inputs(6, T, S, 8, 2, 128, DTYPES[dtype], dev)
    for t in (lengths, lengths.int()):
        _check(_run(*x, lengths=t, starts=starts), _reference(*x, lengths=lengths, starts=starts))
    kw = dict(lengths=lengths, starts=starts - 2, window=50)
    _check(_run(*x, **kw), _reference(*x, **kw))
    far = torch.tensor([1 << 40, -(1 << 40), 0, 3, 3, 3], device=dev)
    _check(_run(*x, starts=far), _reference(*x, starts=far))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_large_and_masked_scores(dev, dtype):
    """Scores of hundreds, and rows whose largest ones are masked."""
    q, k, v, up = _inputs(1, 100, 100, 2, 1, 64, DTYPES[dtype], dev)
    with torch.no_grad():
        q *= 16
        k[:, 50:] *= 64
    _check(_run(q, k, v, up), _reference(q, k, v, up))


def test_no_queries_or_keys(dev):
    for B, T, S in ((0, 3, 3), (2, 0, 5), (2, 4, 0)):
        x = _inputs(B, T, S, 2, 1, 16, torch.float32, dev) if B else [
            torch.zeros(0, 3, n, 16, device=dev, requires_grad=True) for n in (2, 1, 1)] + [
            torch.zeros(0, 3, 2, 16, device=dev)]
        out, dq, dk, dv = _run(*x, causal=T <= S)
        assert not out.any() and not dq.any() and not dk.any() and not dv.any()


def test_strides(dev):
    """Transposed heads, unaligned starts, expanded keys, strided gradients."""
    g = torch.Generator().manual_seed(1)
    base = torch.randn(2, 4, 70, 41, generator=g).to(torch.bfloat16).to(dev)
    q = base[..., 1:].transpose(1, 2).detach().requires_grad_()
    k = torch.randn(1, 70, 1, 40, generator=g).to(torch.bfloat16).to(dev).expand(2, 70, 2, 40)
    k = k.detach().requires_grad_()
    v = torch.randn(2, 2, 70, 48, generator=g).to(torch.bfloat16).to(dev)[..., :40]
    v = v.transpose(1, 2).detach().requires_grad_()
    up = torch.randn(2, 4, 40, 70, generator=g).to(torch.bfloat16).to(dev).permute(0, 3, 1, 2)
    _check(_run(q, k, v, up), _reference(q, k, v, up))


def test_some_gradients_and_the_same_every_time(dev):
    q, k, v, up = _inputs(2, 190, 190, 8, 2, 64, torch.bfloat16, dev)
    want = _run(q, k, v, up)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(_run(q, k, v, up), want))
    out = attention(q, k.detach(), v.detach())
    (dq,) = torch.autograd.grad(out, [q], up, retain_graph=True)
    assert torch.equal(dq, want[1]) and torch.equal(torch.autograd.grad(out, [q], up)[0], dq)
    out = attention(q.detach(), k, v.detach())
    assert torch.equal(torch.autograd.grad(out, [k], up)[0], want[2])
    with torch.no_grad():
        out = attention(q, k, v)
    assert torch.equal(out, want[0]) and not out.requires_grad


def test_against_differences(dev):
    """The gradients in float32 against central differences of the forward in float64."""
    q, k, v, up = _inputs(1, 9, 9, 2, 1, 8, torch.float32, dev)
    grads = _run(q, k, v, up)[1:]
    for i, (t, g) in enumerate(zip((q, k, v), grads)):
        way = torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).to(dev)

        def loss(step):
            x = [q.detach(), k.detach(), v.detach()]
            x[i] = x[i].double() + step * way.double()
            return (_reference(*x, up)[0][0] * up.cpu().double()).sum().item()

        d = 1e-4  # third derivatives of order one: 1e-8
        slope = (loss(d) - loss(-d)) / (2 * d)
        assert abs(slope - (g * way).sum().item()) < 1e-5 * max(1.0, abs(slope))


def test_other_examples_are_not_reached(dev):
    for dtype in DTYPES.values():
        x = _inputs(3, 100, 100, 4, 2, 64, dtype, dev)
        want = _run(*x)
        with torch.no_grad():
            for t in x[:3]:
                t[1, 17] = math.nan
        got = _run(*x)
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
        assert bool(got[0][1, 17:].isnan().all())


def test_captured_and_refused_beside_a_living_eager_graph(dev):
    q, k, v, up = _inputs(2, 96, 96, 4, 2, 64, torch.bfloat16, dev)
    one = _inputs(2, 1, 900, 4, 2, 64, torch.bfloat16, dev)
    lengths = torch.tensor([900, 30], device=dev)
    alive = attention(q, k, v)

    def step():
        return (*_run(q, k, v, up), attention(*one[:3], lengths=lengths, starts=lengths - 1).detach())

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    with pytest.raises(OperationError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
            lengths.copy_(torch.tensor([700 - i, 5 * i], device=dev))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)


def test_on_another_stream(dev):
    x = _inputs(2, 1, 1500, 4, 1, 128, torch.bfloat16, dev)
    want = attention(*x[:3])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [attention(*x[:3]) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(t, want) for t in got)


def test_refusals(dev):
    q, k, v, _ = _inputs(2, 8, 8, 4, 2, 16, torch.float32, dev)
    n = torch.tensor([8, 8], device=dev)
    for args, kw in (
            ((q[0], k, v), {}), ((q, k, v[:, :4]), {}), ((q, k[:1], v[:1]), {}),
            ((q[..., :8], k, v), {}), ((q[:, :, :3], k, v), {}), ((q, k.bfloat16(), v), {}),
            ((q.half(), k.half(), v.half()), {}), ((q, k, v), dict(window=0)),
            ((q, k, v), dict(window=3, causal=False)), ((q, k, v), dict(starts=n, causal=False)),
            ((q, k, v), dict(lengths=n[:1])), ((q, k, v), dict(scale=0.0)),
            ((q, k, v), dict(scale=math.nan)), ((q.cpu(), k, v), {}),
            ((q[:, :, :0], k, v), {}), ((q, k[:, :, :0], v[:, :, :0]), {}),
            ((q.new_zeros(1, 2, 1, 264),) * 3, {})):
        with pytest.raises(ConfigurationError):
            attention(*args, **kw)
    for kw in (dict(window=1.5), dict(window=True), dict(lengths=n.float()), dict(scale="1")):
        with pytest.raises(InputTypeError):
            attention(q, k, v, **kw)


# One row tile and several, two waves a compute unit's SIMD, keys in splits.
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,T,S,H,KV,h", [
    (2, 2, 2, 2, 2, 16), (2, 70, 70, 4, 2, 64), (2, 130, 130, 2, 1, 256), (16, 260, 260, 16, 16, 64),
    (2, 1, 900, 8, 2, 128), (2, 3, 1500, 2, 2, 64)])
def test_scores_that_are_all_minus_infinity(dev, dtype, B, T, S, H, KV, h):
    """No probabilities come of them: NaN, as their softmax is, and not the zeros of a row that
    sees no key."""
    q, k, v, up = (t.detach().clone() for t in _inputs(B, T, S, H, KV, h, DTYPES[dtype], dev))
    k[..., 0] = k[..., 0].abs() + 1
    q[..., 0] = q[..., 0].abs()
    want = _run(*(t.requires_grad_() for t in (q, k, v)), up)
    t, head = T // 2, H - 1
    with torch.no_grad():
        q[0, t, head, 0] = -math.inf
    out, dq, dk, dv = got = _run(q, k, v, up)
    for x, w in zip(got[:2], want):
        assert bool(x[0, t, head].isnan().all())
        others = torch.ones(x.shape[:3], dtype=torch.bool, device=dev)
        others[0, t, head] = False
        assert torch.equal(x[others], w[others])
    seen = S - T + t + 1  # keys of the head's group
    assert bool(dk[0, :seen, -1].isnan().all()) and bool(dv[0, :seen, -1].isnan().all())
    for x, w in zip(got[2:], want[2:]):
        assert torch.equal(x[1:], w[1:]) and torch.equal(x[0, :, :-1], w[0, :, :-1])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("which", ["q", "k", "v", "up"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("B,T,S,h", [(2, 1, 1, 16), (2, 70, 70, 64), (2, 33, 33, 256),
                                     (64, 260, 260, 128), (2, 5, 700, 64)])
def test_one_key_of_values_that_are_not_finite(dev, dtype, which, bad, B, T, S, h):
    """A query that sees one key has no gradient of query and key, unless what it is formed of
    is not finite: then it is what the formula gives, and not zero."""
    x = [t.detach().clone() for t in _inputs(B, T, S, 4, 4, h, DTYPES[dtype], dev)]
    for t in x[:2]:
        t[..., 0] = t[..., 0].abs() + 1  # (a score is the infinity's, not NaN of its zero)
    want = _run(*(t.requires_grad_() for t in x[:3]), x[3], window=1)
    assert not want[1].any() and not want[2].any()
    t, i = T - 1, ["q", "k", "v", "up"].index(which)
    with torch.no_grad():  # the last token and its key
        x[i][1, -1, 2, 0] = bad
    out, dq, dk, dv = got = _run(*x, window=1)
    assert bool(dq[1, t, 2].isnan().all()) and bool(dk[1, -1, 2].isnan().all())
    assert bool(dv[1, -1, 2].isnan().all()) == (i < 2) and bool(out[1, t, 2].isnan().all()) == (i < 2)
    for a, b in zip(got, want):  # the other heads and examples
        others = torch.ones(a.shape[:3], dtype=torch.bool, device=dev)
        others[1, :, 2] = False
        assert torch.equal(a[others], b[others])
