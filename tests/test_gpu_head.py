"""Head losses without logits: values and gradients against 64 bits (GPU).

Error model the tolerances come from (u = 2^-23, one extra addend of slack per
16 products, as for the Gram kernels): a product sum of n terms is off by at
most 1.125 n u times the sum of the terms' magnitudes.  So a logit is off by
``zerr = 1.125 n u |h| |w|``; a loss by twice that and a few ulp of the log sum
exp; dz by its bf16 rounding (float32: two fp16 planes, 2^-24) and by what the logits'
error does to p; and a gradient by dz's error and the sum's own, rounded once.  With a
frozen head (bf16) dz goes through fp16 exponentials relative to a tile's maximum:
another 2^-12 of it, or 2^-25 where they are subnormal.
"""

from __future__ import annotations

import math

import pytest
import torch

from opake_amd import _native as nat
from opake_amd import head
from opake_amd.exceptions import ConfigurationError, InputTypeError

U = 2.0**-23


def _inputs(dev, lead, D, V, dtype, seed, spread=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    h = torch.randn(*lead, D, generator=g, device=dev).to(dtype)
    W = (torch.randn(V, D, generator=g, device=dev) * (spread / math.sqrt(D))).to(dtype)
    up = torch.rand(*lead, generator=g, device=dev) + 0.5
    return g, h, W, up


def _reference(h, W, q, ent, tau, up, frozen=False):
    """Losses and gradients in 64 bits from the dense target distribution q [N, V]
    (rows of zeros: no target) and its negative entropy, with error bounds."""
    D = h.shape[-1]
    hd, Wd, u = h.detach().double().reshape(-1, D), W.detach().double(), up.double().reshape(-1, 1)
    f32 = h.dtype == torch.float32
    used = q.sum(1, keepdim=True)
    z = hd @ Wd.t() / tau
    lse = torch.logsumexp(z, 1, keepdim=True)
    logp = z - lse
    loss = tau * tau * (ent - (q * logp).sum(1))
    n = (6 if f32 else 1) * (D + 64)
    zerr = 1.125 * n * U * hd.norm(dim=1, keepdim=True) * Wd.norm(dim=1).max() / tau
    sharp = 2 * zerr + 2.0**-19 * (1 + logp.abs().amin(1, keepdim=True) + lse.abs())
    loss_tol = tau * tau * (2 * sharp.squeeze(1) + 2.0**-20 * (1 + loss.abs() + ent.abs()))
    p = logp.exp() * used
    dz = (p - q) * (tau * u)
    rnd = 2.0**-22 if f32 else 2.0**-8
    # p's relative error: the logits' and the exponential's (its argument's rounding).
    perr = (p * (sharp + 2.0**-22 * logp.abs()) + 2.0**-21 * q) * (tau * u)
    dzerr = dz.abs() * rnd + perr
    if frozen and not f32:
        dzerr = dzerr + (p * 2.0**-11 + 2.0**-25 * used) * (tau * u)
    out = 2.0**-23 if f32 else 2.0**-8

    def product(x, xerr, y, terms):
        val = x @ y
        terms *= 6 if f32 else 1
        tol = (xerr + 1.125 * (terms + 64) * U * x.abs()) @ y.abs() + out * val.abs()
        return val, tol + 1e-30

    N, V = q.shape
    dh = product(dz, dzerr, Wd, V)
    dW = product(dz.t().contiguous(), dzerr.t().contiguous(), hd, N)
    return (loss, loss_tol), dh, dW


def _close(got, want, what):
    val, tol = want
    err = (got.detach().double().reshape(val.shape) - val).abs()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert torch.isfinite(got).all(), what
    assert worst <= 1.0, f"{what}: {worst:.3f} of its tolerance"


def _onehot(t, V, ignore):
    t = t.reshape(-1)
    q = torch.zeros(t.numel(), V, dtype=torch.float64, device=t.device)
    r = torch.nonzero(t != ignore).flatten()
    q[r, t[r].long()] = 1.0
    return q


SHAPES = [
    # lead, D, V: one of everything, odd ones, tile edges and past them, long K
    ((1,), 1, 1), ((1,), 8, 2), ((3,), 7, 5), ((2, 5), 64, 256), ((255,), 65, 257),
    ((256,), 128, 512), ((257,), 72, 511), ((1, 1), 264, 1000), ((4, 100), 200, 3001),
    ((700,), 24, 777), ((33,), 1000, 5003),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lead,D,V", SHAPES)
def test_cross_entropy(dev, lead, D, V, dtype):
    g, h, W, up = _inputs(dev, lead, D, V, dtype, seed=D + V)
    t = torch.randint(0, V, lead, generator=g, device=dev)
    if t.numel() > 2:
        t.view(-1)[::5] = -100
    h.requires_grad_(True)
    W.requires_grad_(True)
    loss = head.linear_cross_entropy(h, W, t)
    assert loss.shape == lead and loss.dtype == torch.float32
    dh, dW = torch.autograd.grad(loss, [h, W], up)
    assert dh.shape == h.shape and dh.dtype == dtype and dW.dtype == dtype
    q = _onehot(t, V, -100)
    L, DH, DW = _reference(h, W, q, torch.zeros(q.shape[0], dtype=torch.float64, device=dev), 1.0,
                           up)
    _close(loss, L, "loss")
    _close(dh, DH, "hidden_grad")
    _close(dW, DW, "weight_grad")
    ignored = (t == -100)
    assert (loss[ignored] == 0).all() and (dh[ignored] == 0).all()
    _frozen(lambda x, y: head.linear_cross_entropy(x, y, t), h, W, up, loss, q,
            torch.zeros(q.shape[0], dtype=torch.float64, device=dev), 1.0, ignored)


def _frozen(call, h, W, up, loss, q, ent, tau, empty):
    """The same with a frozen head, whose gradient is made in the forward."""
    frozen = call(h, W.detach())
    (dh,) = torch.autograd.grad(frozen, [h], up, retain_graph=True)
    assert torch.equal(frozen, loss)
    _, DH, _ = _reference(h, W, q, ent, tau, up, frozen=True)
    _close(dh, DH, "hidden_grad of a frozen head")
    assert (dh[empty] == 0).all()
    # A second backward of the same graph, with another gradient.
    (again,) = torch.autograd.grad(frozen, [h], 2 * up)
    assert torch.equal(again, 2 * dh)


def _teacher(g, dev, lead, V, K, duplicates=False):
    if duplicates:
        idx = torch.randint(0, max(1, V // 3), (*lead, K), generator=g, device=dev)
    else:
        idx = torch.rand(*lead, V, generator=g, device=dev).topk(K, -1).indices
    return torch.randn(*lead, K, generator=g, device=dev) * 2 + 3, idx


def _soft(tl, ti, V, tau):
    """Dense q and its negative entropy per entry (repeated entries add up in q)."""
    K = ti.shape[-1]
    tl, ti = tl.double().reshape(-1, K) / tau, ti.reshape(-1, K)
    there = (ti >= 0) & (tl > -math.inf)
    some = there.any(1, keepdim=True)
    e = torch.softmax(torch.where(there, tl, -math.inf), 1)
    e = torch.where(some, e, 0.0)
    ent = torch.special.xlogy(e, e).sum(1)
    q = torch.zeros(ti.shape[0], V, dtype=torch.float64, device=tl.device)
    q.scatter_add_(1, ti.clamp(min=0), e)
    return q, ent


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lead,D,V,K,tau,dup", [
    ((1,), 8, 1, 1, 1.0, False), ((5,), 16, 9, 9, 0.5, False), ((2, 130), 64, 300, 8, 2.0, False),
    ((129,), 40, 513, 64, 1.5, False), ((70,), 100, 700, 65, 4.0, False),
    ((31,), 64, 1025, 200, 1.0, True), ((300,), 33, 257, 6, 2.0, True),
])
def test_distillation(dev, lead, D, V, K, tau, dup, dtype):
    g, h, W, up = _inputs(dev, lead, D, V, dtype, seed=K + V)
    tl, ti = _teacher(g, dev, lead, V, K, dup)
    flat_i, flat_l = ti.view(-1, K), tl.view(-1, K)
    n = flat_i.shape[0]
    if n > 4:  # rows cut short, rows with none, entries the teacher rules out
        keep = torch.randint(0, K + 1, (n, 1), generator=g, device=dev)
        flat_i[torch.arange(K, device=dev) >= keep] = -1
        flat_i[0] = -1
        flat_l[1, :] = -math.inf
        flat_l[2, 0] = -math.inf
    h.requires_grad_(True)
    W.requires_grad_(True)
    loss = head.topk_distillation(h, W, tl, ti, temperature=tau)
    dh, dW = torch.autograd.grad(loss, [h, W], up)
    q, ent = _soft(tl, ti, V, tau)
    L, DH, DW = _reference(h, W, q, ent, tau, up)
    _close(loss, L, "loss")
    _close(dh, DH, "hidden_grad")
    _close(dW, DW, "weight_grad")
    empty = q.sum(1).view(lead) == 0
    assert (loss[empty] == 0).all() and (dh[empty] == 0).all()
    _frozen(lambda x, y: head.topk_distillation(x, y, tl, ti, temperature=tau), h, W, up, loss, q,
            ent, tau, empty)


@pytest.mark.gpu
def test_distillation_from_one_entry_is_cross_entropy(dev):
    g, h, W, _ = _inputs(dev, (90,), 64, 700, torch.bfloat16, 5)
    t = torch.randint(0, 700, (90,), generator=g, device=dev)
    a = head.linear_cross_entropy(h, W, t)
    b = head.topk_distillation(h, W, torch.full((90, 1), 7.0, device=dev), t[:, None])
    assert (a - b).abs().max() <= 2.0**-20 * (1 + a.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_many_pieces(dev, dtype):
    """Enough tokens that the backward takes the vocabulary in several pieces, and a frozen
    head's forward the tokens in several chunks."""
    N, D, V = 300_001, 8, 600
    g, h, W, up = _inputs(dev, (N,), D, V, dtype, 11)
    t = torch.randint(0, V, (N,), generator=g, device=dev)
    h.requires_grad_(True)
    W.requires_grad_(True)
    loss = head.linear_cross_entropy(h, W, t)
    dh, dW = torch.autograd.grad(loss, [h, W], up)
    q, zero = _onehot(t, V, -100), torch.zeros(N, dtype=torch.float64, device=dev)
    L, DH, DW = _reference(h, W, q, zero, 1.0, up)
    _close(loss, L, "loss")
    _close(dh, DH, "hidden_grad")
    _close(dW, DW, "weight_grad")
    del DH, DW
    _frozen(lambda x, y: head.linear_cross_entropy(x, y, t), h, W, up, loss, q, zero, 1.0, t == -100)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("grad_h", [True, False], ids=["both", "weight"])
def test_more_than_is_kept(dev, dtype, grad_h):
    """A trained head with more exponentials than the forward keeps: the backward makes
    the logits again, for both gradients or the weight's alone."""
    N, D, V = 150_001, 8, 1900
    g, h, W, up = _inputs(dev, (N,), D, V, dtype, 12)
    t = torch.randint(0, V, (N,), generator=g, device=dev)
    t[:7] = -100
    h.requires_grad_(grad_h)
    W.requires_grad_(True)
    loss = head.linear_cross_entropy(h, W, t)
    grads = torch.autograd.grad(loss, [h, W] if grad_h else [W], up)
    L, DH, DW = _reference(h, W, _onehot(t, V, -100),
                           torch.zeros(N, dtype=torch.float64, device=dev), 1.0, up)
    _close(loss, L, "loss")
    _close(grads[-1], DW, "weight_grad")
    if grad_h:
        _close(grads[0], DH, "hidden_grad")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_many_rows_of_broken_lines(dev, dtype):
    """Widths that are not whole 128-byte lines, with enough tokens to be copied."""
    N, D, V = 8200, 264, 130
    g, h, W, up = _inputs(dev, (N,), D, V, dtype, 21)
    t = torch.randint(0, V, (N,), generator=g, device=dev)
    t[::5] = -100
    q, zero = _onehot(t, V, -100), torch.zeros(N, dtype=torch.float64, device=dev)
    h.requires_grad_(True)
    W.requires_grad_(True)
    loss = head.linear_cross_entropy(h, W, t)
    dh, dW = torch.autograd.grad(loss, [h, W], up)
    L, DH, DW = _reference(h, W, q, zero, 1.0, up)
    _close(loss, L, "loss")
    _close(dh, DH, "hidden_grad")
    _close(dW, DW, "weight_grad")
    _frozen(lambda x, y: head.linear_cross_entropy(x, y, t), h, W, up, loss, q, zero, 1.0,
            t == -100)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("N,D,V", [(1, 4096, 300), (40, 2500, 1000), (300, 1544, 513)])
def test_few_tiles_and_a_long_sum(dev, N, D, V, dtype):
    """The logits' sums in slices: the loss alone, a frozen head, a trained one."""
    g, h, W, up = _inputs(dev, (N,), D, V, dtype, N)
    t = torch.randint(0, V, (N,), generator=g, device=dev)
    q, zero = _onehot(t, V, -100), torch.zeros(N, dtype=torch.float64, device=dev)
    L, DH, DW = _reference(h, W, q, zero, 1.0, up)
    alone = head.linear_cross_entropy(h, W, t)
    _close(alone, L, "loss")
    h.requires_grad_(True)
    W.requires_grad_(True)
    loss = head.linear_cross_entropy(h, W, t)
    assert torch.equal(loss, alone)
    dh, dW = torch.autograd.grad(loss, [h, W], up)
    _close(dh, DH, "hidden_grad")
    _close(dW, DW, "weight_grad")
    _frozen(lambda x, y: head.linear_cross_entropy(x, y, t), h, W, up, loss, q, zero, 1.0, t == -100)


@pytest.mark.gpu
def test_strided_and_unaligned_operands(dev):
    """Views: a transposed batch, a slice of a wider tensor, an odd element offset."""
    g, h, W, up = _inputs(dev, (6, 40), 64, 300, torch.bfloat16, 3)
    t = torch.randint(0, 300, (6, 40), generator=g, device=dev)
    want = head.linear_cross_entropy(h, W, t)
    hv = h.transpose(0, 1).contiguous().transpose(0, 1)
    Wv = torch.cat([W, W], 1)[:, :64]
    buf = torch.empty(h.numel() + 1, dtype=h.dtype, device=dev)
    ho = buf[1:].view(h.shape)
    ho.copy_(h)
    tv = t.to(torch.int32).t().contiguous().t()
    assert torch.equal(head.linear_cross_entropy(hv, Wv, tv), want)
    assert torch.equal(head.linear_cross_entropy(ho, W, t), want)
    grads = []
    for x, y in ((h, W), (hv, Wv), (ho, W)):
        x, y = x.detach().requires_grad_(True), y.detach().requires_grad_(True)
        # A broadcast upstream gradient (stride 0).
        grads.append(torch.autograd.grad(head.linear_cross_entropy(x, y, t).sum(), [x, y]))
    for got in grads[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got, grads[0]))


@pytest.mark.gpu
def test_only_what_is_asked_for(dev):
    g, h, W, up = _inputs(dev, (50,), 64, 300, torch.bfloat16, 9)
    t = torch.randint(0, 300, (50,), generator=g, device=dev)
    h1, W1 = h.clone().requires_grad_(True), W.clone().requires_grad_(True)
    both = torch.autograd.grad(head.linear_cross_entropy(h1, W1, t), [h1, W1], up)
    (dW,) = torch.autograd.grad(head.linear_cross_entropy(h, W1, t), [W1], up)
    (dh,) = torch.autograd.grad(head.linear_cross_entropy(h1, W1, t), [h1], up)
    assert torch.equal(dh, both[0]) and torch.equal(dW, both[1])
    assert not head.linear_cross_entropy(h, W, t).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_large_logits_and_nonfinite_rows(dev, dtype):
    """Logits of hundreds (one column takes all the mass); a NaN or infinite hidden row
    spoils its own loss and hidden gradient only; so does a target outside the vocabulary."""
    g, h, W, up = _inputs(dev, (40,), 64, 600, dtype, 21, spread=60.0)
    t = torch.randint(0, 600, (40,), generator=g, device=dev)
    h.requires_grad_(True)
    loss = head.linear_cross_entropy(h, W, t)
    (dh,) = torch.autograd.grad(loss, [h], up)
    q = _onehot(t, 600, -100)
    L, DH, _ = _reference(h, W, q, torch.zeros(40, dtype=torch.float64, device=dev), 1.0, up)
    _close(loss, L, "loss")
    _close(dh, DH, "hidden_grad")
    h2, t2 = h.detach().clone(), t.clone()
    h2[3, 5], h2[7, 0] = math.nan, math.inf
    t2[11], t2[12] = 600, -7
    h2.requires_grad_(True)
    loss2 = head.linear_cross_entropy(h2, W, t2)
    (dh2,) = torch.autograd.grad(loss2, [h2], up)
    bad = torch.zeros(40, dtype=torch.bool, device=dev)
    bad[[3, 7, 11, 12]] = True
    assert (~torch.isfinite(loss2[bad])).all() and torch.isnan(dh2[bad]).any(1).all()
    assert torch.equal(loss2[~bad], loss[~bad]) and torch.equal(dh2[~bad], dh[~bad])


@pytest.mark.gpu
def test_nan_in_rows_without_a_target_reaches_nothing(dev):
    """Padding rows may hold anything: ignored, they change no loss and no gradient."""
    g, h, W, up = _inputs(dev, (300,), 64, 600, torch.bfloat16, 2)
    t = torch.randint(0, 600, (300,), generator=g, device=dev)
    t[10:90] = -100
    h1, W1 = h.clone().requires_grad_(True), W.clone().requires_grad_(True)
    l1 = head.linear_cross_entropy(h1, W1, t)
    g1 = torch.autograd.grad(l1, [h1, W1], up)
    h2 = h.clone()
    h2[10:50], h2[50:90] = math.nan, math.inf
    h2.requires_grad_(True)
    up2 = up.clone()
    up2[10:90] = math.nan
    l2 = head.linear_cross_entropy(h2, W1, t)
    g2 = torch.autograd.grad(l2, [h2, W1], up2)
    assert torch.equal(l1, l2) and torch.equal(g1[0], g2[0]) and torch.equal(g1[1], g2[1])
    f1 = torch.autograd.grad(head.linear_cross_entropy(h1, W, t), [h1], up)
    f2 = torch.autograd.grad(head.linear_cross_entropy(h2, W, t), [h2], up2)
    assert torch.equal(f1[0], f2[0])


@pytest.mark.gpu
@pytest.mark.parametrize("power", [-60, 40, 90])
def test_float32_of_any_magnitude(dev, power):
    """float32 operands are held relative to their largest: powers of two that cancel
    in the logits change nothing, and come out of the gradients as they went in."""
    g, h, W, up = _inputs(dev, (130,), 72, 300, torch.float32, 11)
    t = torch.randint(0, 300, (130,), generator=g, device=dev)

    def run(h, W, both):
        h, W = h.clone().requires_grad_(), W.clone().requires_grad_(both)
        loss = head.linear_cross_entropy(h, W, t)
        loss.backward(up)
        return loss.detach(), h.grad, W.grad

    f = 2.0**power
    for both in (False, True):
        a, b = run(h, W, both), run(h * f, W / f, both)
        assert torch.equal(a[0], b[0])
        assert torch.equal(a[1], b[1] * f)
        if both:
            assert torch.equal(a[2], b[2] / f)


@pytest.mark.gpu
def test_float32_rows_keep_their_own_scale(dev):
    """A row far larger than the others does not change their losses or gradients."""
    g, h, W, up = _inputs(dev, (130,), 72, 300, torch.float32, 12)
    t = torch.randint(0, 300, (130,), generator=g, device=dev)
    big = h.clone()
    big[77] *= 2.0**60
    keep = torch.arange(130, device=dev) != 77
    for both in (False, True):
        res = []
        for x in (h, big):
            x, w = x.clone().requires_grad_(), W.clone().requires_grad_(both)
            loss = head.linear_cross_entropy(x, w, t)
            loss.backward(up)
            assert torch.isfinite(loss).all() and torch.isfinite(x.grad).all()
            res.append((loss.detach()[keep], x.grad[keep]))
        assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])


@pytest.mark.gpu
def test_no_tokens(dev):
    h = torch.zeros(0, 16, device=dev, requires_grad=True)
    W = torch.randn(30, 16, device=dev, requires_grad=True)
    loss = head.linear_cross_entropy(h, W, torch.zeros(0, dtype=torch.int64, device=dev))
    dh, dW = torch.autograd.grad(loss.sum(), [h, W])
    assert loss.shape == (0,) and dh.shape == (0, 16) and (dW == 0).all()


@pytest.mark.gpu
def test_differences(dev):
    """<gradient, d> against central differences of the kernel's own losses along d.
    The third derivative of a log sum exp along d is a third central moment of w.d,
    at most range^3 / (6 sqrt 3)."""
    N, D, V, eps = 40, 48, 350, 2.0**-5
    g, h, W, up = _inputs(dev, (N,), D, V, torch.float32, 31)
    tl, ti = _teacher(g, dev, (N,), V, 12)
    h.requires_grad_(True)
    loss = head.topk_distillation(h, W, tl, ti, temperature=1.0)
    (dh,) = torch.autograd.grad(loss, [h], up)
    d = torch.randn(N, D, generator=g, device=dev)
    with torch.no_grad():
        hi = head.topk_distillation(h + eps * d, W, tl, ti, temperature=1.0).double()
        lo = head.topk_distillation(h - eps * d, W, tl, ti, temperature=1.0).double()
    slope = (hi - lo) / (2 * eps)
    want = (dh.double() * d.double()).sum(1) / up.double()
    s = d.double() @ W.double().t()
    span = s.amax(1) - s.amin(1)
    q, ent = _soft(tl, ti, V, 1.0)
    (_, ltol), (_, gtol), _ = _reference(h, W, q, ent, 1.0, up)
    # The step itself rounds each coordinate of h by half an ulp.
    step = (h.detach().abs().double() + eps * d.abs().double()) * 2.0**-24
    tol = (2 * ltol / (2 * eps) + eps**2 / 6 * span**3 / (6 * 3**0.5)
           + (gtol * d.double().abs()).sum(1) / up.double()
           + (step * (2 * W.double().abs().amax(0))).sum(1) / eps)
    assert ((slope - want).abs() <= tol).all(), ((slope - want).abs() / tol).max().item()


@pytest.mark.gpu
def test_repeats_streams_and_graph(dev):
    """The same bits call after call, on another stream and from a replayed graph."""
    g, h, W, up = _inputs(dev, (3, 130), 64, 700, torch.bfloat16, 17)
    t = torch.randint(0, 700, (3, 130), generator=g, device=dev)
    h.requires_grad_(True)
    W.requires_grad_(True)

    def step():
        loss = head.linear_cross_entropy(h, W, t)
        frozen = head.linear_cross_entropy(h, W.detach(), t)
        return (loss.detach(), *torch.autograd.grad(loss, [h, W], up),
                *torch.autograd.grad(frozen, [h], up))

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        for x in out:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        torch.randn(1000, device=dev).sum().item()


@pytest.mark.gpu
def test_refusals(dev):
    h, W = torch.zeros(4, 16, device=dev), torch.zeros(9, 16, device=dev)
    t = torch.zeros(4, dtype=torch.int64, device=dev)
    tl, ti = torch.zeros(4, 3, device=dev), torch.zeros(4, 3, dtype=torch.int64, device=dev)
    bad = [
        (ConfigurationError, lambda: head.linear_cross_entropy(h, W[:, :8], t)),
        (ConfigurationError, lambda: head.linear_cross_entropy(h, W.bfloat16(), t)),
        (ConfigurationError, lambda: head.linear_cross_entropy(h.half(), W.half(), t)),
        (ConfigurationError, lambda: head.linear_cross_entropy(h, W, t[:3])),
        (ConfigurationError, lambda: head.linear_cross_entropy(h, W[:0], t)),
        (InputTypeError, lambda: head.linear_cross_entropy(h, W, t.float())),
        (ConfigurationError, lambda: head.topk_distillation(h, W, tl, ti[:, :2])),
        (ConfigurationError, lambda: head.topk_distillation(h, W, tl[:, :0], ti[:, :0])),
        (InputTypeError, lambda: head.topk_distillation(h, W, tl.long(), ti)),
        (InputTypeError, lambda: head.topk_distillation(h, W, tl, tl)),
        (ConfigurationError, lambda: head.topk_distillation(h, W, tl, ti, temperature=0.0)),
        (ConfigurationError, lambda: head.topk_distillation(h, W, tl, ti, temperature=math.nan)),
        (InputTypeError, lambda: head.topk_distillation(h, W, tl, ti, temperature="2")),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def test_cpu_tensors_are_refused():
    h, W = torch.zeros(4, 16), torch.zeros(9, 16)
    with pytest.raises(ConfigurationError, match="ROCm device"):
        head.linear_cross_entropy(h, W, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ConfigurationError, match="ROCm device"):
        head.topk_distillation(h, W, torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_without_grad_mode_only_the_loss_is_made(dev, dtype, mode):
    """A parameter, or hidden states that require a gradient, evaluated with gradients
    off: the loss-only plan's memory, and its bits."""
    N, D, V = 512, 64, 5000
    g, h, W, _ = _inputs(dev, (N,), D, V, dtype, 41)
    t = torch.randint(0, V, (N,), generator=g, device=dev)

    def peak(h, W):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        with mode():
            loss = head.linear_cross_entropy(h, W, t)
        return loss, torch.cuda.max_memory_allocated() - before

    want, least = peak(h, W)
    for x, w in ((h, W.requires_grad_()), (h.requires_grad_(), W), (h, W.detach())):
        loss, most = peak(x, w)
        assert torch.equal(loss, want) and not loss.requires_grad
        assert most == least
    tl, ti = torch.randn(N, 8, device=dev), torch.arange(8, device=dev).expand(N, 8)
    with mode():
        a = head.topk_distillation(h, W, tl, ti)
        b = head.topk_distillation(h.detach(), W.detach(), tl, ti)
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("tau", [0.5, 1.0, 1.5, 3.0])
def test_teacher_entries_at_the_lowest_value(dev, tau):
    """Masks of the type's lowest value: beside other entries they weigh nothing, and a
    row that holds nothing else is uniform over them.  Logits of any size are weighed by
    their differences."""
    V, K = 300, 5
    low = torch.finfo(torch.float32).min
    tl = torch.tensor([[1.0, 2.0, 3.0, low, low], [low] * 5, [3e38, 3e38, low, low, 1.0],
                       [1e30, 1e30, 1e30, -1e30, 0.0], [-1e8, -1e8 - 8, -1e8 + 8, low, -2e8]],
                      device=dev)
    n = tl.shape[0]
    g, h, W, up = _inputs(dev, (n,), 64, V, torch.float32, 43)
    ti = torch.arange(K, device=dev) * 7 + torch.arange(n, device=dev)[:, None]
    h.requires_grad_(True)
    loss = head.topk_distillation(h, W, tl, ti, temperature=tau)
    (dh,) = torch.autograd.grad(loss, [h], up)
    q, ent = _soft(tl, ti, V, tau)
    L, DH, _ = _reference(h, W, q, ent, tau, up, frozen=True)
    _close(loss, L, "loss")
    _close(dh, DH, "hidden_grad")


@pytest.mark.gpu
def test_temperatures_that_float32_cannot_square_are_refused(dev):
    h, W = torch.zeros(4, 16, device=dev), torch.zeros(9, 16, device=dev)
    tl, ti = torch.zeros(4, 3, device=dev), torch.zeros(4, 3, dtype=torch.int64, device=dev)
    for tau in (1e-16, 1e-40, 1e16):
        with pytest.raises(ConfigurationError):
            head.topk_distillation(h, W, tl, ti, temperature=tau)


def _planes(x, top):
    """x as the two fp16 planes of the kernels over the power of two of `top`: [first,
    second], in 64 bits."""
    s = 2.0 ** (14 - math.floor(math.log2(top)))
    x0 = (x * s).to(torch.float16).double()
    x1 = (x * s - x0).to(torch.float16).double()
    return x0 / s, x1 / s


def _plane_case(dev):
    g = torch.Generator(device=dev).manual_seed(51)
    N, D, V = 24, 8, 24
    h = torch.randn(N, D, generator=g, device=dev)
    W = torch.randn(V, D, generator=g, device=dev)
    t = torch.randint(0, V, (N,), generator=g, device=dev)
    up = torch.rand(N, generator=g, device=dev) + 0.5
    return h, W, t, up


def _plane_reference(h, W, t, up):
    """Values in 64 bits and bounds of float32 accuracy.  A value is 2^-23 of itself away
    from its planes and a product of two low planes is below 2^-22 of the product, so with
    both operands' planes a term is off by 2^-21; a sum of 3 n products by 1.125 u (3 n)
    of the terms (u = 2^-23); log sum exp, exponentials and logs add 2^-21 of what they
    hold."""
    h, W, up = h.double(), W.double(), up.double()[:, None]
    N, D, V = h.shape[0], h.shape[1], W.shape[0]
    q = _onehot(t, V, -100)

    def product(x, xerr, y):  # x @ y, and how far it may be off
        terms = x.abs() @ y.abs()
        return x @ y, xerr @ y.abs() + (2.0**-21 + 1.125 * U * 3 * x.shape[1]) * terms

    z, zerr = product(h, torch.zeros_like(h), W.t())
    lse = torch.logsumexp(z, 1, keepdim=True)
    logp = z - lse
    perr = zerr + zerr.amax(1, keepdim=True) + 2.0**-21 * (1 + z.abs() + lse.abs())
    p = logp.exp()
    loss, loss_tol = -(q * logp).sum(1), (q * perr).sum(1)
    dz, dzerr = p - q, p * perr + 2.0**-22 * (p - q).abs()
    dh, dh_tol = product(dz, dzerr, W)
    dW, dW_tol = product((dz * up).t(), (dzerr * up).t(), h)
    rounded = 2.0**-23
    return ((loss, loss_tol), (dh * up, dh_tol * up + rounded * (dh * up).abs()),
            (dW, dW_tol + rounded * dW.abs()))


@pytest.mark.gpu
def test_float32_accuracy(dev):
    """Few terms a sum, so that a plane or a plane product left out would be seen (below)."""
    h, W, t, up = _plane_case(dev)
    L, DH, DW = _plane_reference(h, W, t, up)
    h.requires_grad_(True)
    frozen = head.linear_cross_entropy(h, W, t)
    _close(frozen, L, "loss")
    _close(torch.autograd.grad(frozen, [h], up)[0], DH, "hidden_grad of a frozen head")
    W.requires_grad_(True)
    loss = head.linear_cross_entropy(h, W, t)
    dh, dW = torch.autograd.grad(loss, [h, W], up)
    _close(loss, L, "loss")
    _close(dh, DH, "hidden_grad")
    _close(dW, DW, "weight_grad")


def _with_planes(h, W, t, up, pairs):
    """The loss and gradients with products over the given plane pairs only, in 64 bits."""
    def product(x, y):
        xp, yp = _planes(x, x.abs().max().item()), _planes(y, y.abs().max().item())
        return sum(xp[a] @ yp[b] for a, b in pairs)

    h, W, up = h.double(), W.double(), up.double()[:, None]
    z = product(h, W.t())
    logp = z - torch.logsumexp(z, 1, keepdim=True)
    q = _onehot(t, W.shape[0], -100)
    dz = logp.exp() - q
    return -(q * logp).sum(1), product(dz, W) * up, product(dz.t(), h * up)


def test_float32_bounds_tell_the_planes_apart():
    case = _plane_case(torch.device("cpu"))
    want = _plane_reference(*case)

    def worst(pairs):
        got = _with_planes(*case, pairs)
        return [((g - v).abs() / tol).max().item() for g, (v, tol) in zip(got, want)]

    assert max(worst([(1, 0), (0, 1), (0, 0)])) <= 1.0
    for lost in ([(0, 0)], [(1, 0), (0, 0)], [(0, 1), (0, 0)]):
        assert min(worst(lost)) > 1.0, lost


@pytest.mark.gpu
@pytest.mark.parametrize("path", ["frozen", "trained"])
def test_small_exponentials_keep_their_bits(dev, path):
    """Every half tile's largest column stands 15.6875 above the others (e^-15.6875 = 2.58
    times 2^-24), whose probabilities alone make up one column of the hidden gradient.  An
    exponential is off by 2^-11 of itself and 2^-39 of the largest (held without a power of
    two it would be 3 or 2 times 2^-24), dz in bf16 by 2^-8, the gradient by its own
    rounding."""
    dtype = torch.bfloat16
    N, D, V = 70, 8, 300
    h = torch.zeros(N, D, device=dev, dtype=dtype)
    h[:, 1] = 1.0
    W = torch.zeros(V, D, device=dev, dtype=dtype)
    W[:, 0], W[:, 1] = 1.0, -15.6875
    W[::128] = 0.0
    t = torch.zeros(N, dtype=torch.int64, device=dev)
    h.requires_grad_(True)
    W.requires_grad_(path == "trained")
    (dh,) = torch.autograd.grad(head.linear_cross_entropy(h, W, t).sum(), [h])
    tops = W[::128].shape[0]
    low = math.exp(-15.6875)
    want = (V - tops) * low / (tops + (V - tops) * low)
    tol = 2.0**-39 / low + 2.0**-11 + 2 * 2.0**-8
    assert ((dh[:, 0].double() - want).abs() <= tol * want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("kept", [0.01, 0.6, 1.0])
def test_chunks_and_pieces(dev, dtype, kept):
    """A frozen head's forward in several chunks of rows and a trained head's backward in
    several pieces of the vocabulary, with all rows, with so few that the last chunk holds
    a part or nothing, and (1%) with dH's pieces in slices."""
    N, D, V = 150_001, 8, 1900
    lib, code = nat.load(), nat.dtype_code(dtype)
    planes = 2 if dtype == torch.float32 else 1
    rows = -(-N // 256) * 256
    whole = planes * rows * -(-V // 256) * 512  # exponentials, or dz, of all
    assert whole > 512 << 20
    sizes = (N, D, V, 1, code)
    exponentials = (lib.dpc_head_loss_workspace_bytes(*sizes, 1, 0)
                    - lib.dpc_head_loss_workspace_bytes(*sizes, 1, 1))
    assert 0 < exponentials < whole
    assert lib.dpc_head_loss_state_bytes(*sizes, 1, 1) < whole
    assert lib.dpc_head_loss_grad_workspace_bytes(*sizes, 1, 1) < whole
    g, h, W, up = _inputs(dev, (N,), D, V, dtype, 61)
    t = torch.randint(0, V, (N,), generator=g, device=dev)
    t[torch.rand(N, generator=g, device=dev) >= kept] = -100
    on = t != -100
    L, DH, DW = _reference(h[on], W, _onehot(t[on], V, -100),
                           torch.zeros(int(on.sum()), dtype=torch.float64, device=dev), 1.0,
                           up[on], frozen=True)
    h.requires_grad_(True)
    frozen = head.linear_cross_entropy(h, W, t)
    (dh,) = torch.autograd.grad(frozen, [h], up)
    _close(frozen[on], L, "loss")
    _close(dh[on], DH, "hidden_grad of a frozen head")
    assert (frozen[~on] == 0).all() and (dh[~on] == 0).all()
    W.requires_grad_(True)
    loss = head.linear_cross_entropy(h, W, t)
    dh, dW = torch.autograd.grad(loss, [h, W], up)
    assert torch.equal(loss, frozen)
    _close(dh[on], DH, "hidden_grad")
    _close(dW, DW, "weight_grad")
    assert (dh[~on] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("N,D,V", [(5, 8, 1 << 19), (3, 1 << 20, 9), (130, 24, (1 << 17) + 3)])
def test_the_largest_sizes(dev, N, D, V, dtype):
    """The widest vocabulary and hidden state that are taken; one more of either is not."""
    g, h, W, up = _inputs(dev, (N,), D, V, dtype, 71)
    t = torch.randint(0, V, (N,), generator=g, device=dev)
    t[0] = V - 1
    q, zero = _onehot(t, V, -100), torch.zeros(N, dtype=torch.float64, device=dev)
    L, DH, DW = _reference(h, W, q, zero, 1.0, up, frozen=True)
    h.requires_grad_(True)
    W.requires_grad_(True)
    loss = head.linear_cross_entropy(h, W, t)
    dh, dW = torch.autograd.grad(loss, [h, W], up)
    _close(loss, L, "loss")
    _close(dh, DH, "hidden_grad")
    _close(dW, DW, "weight_grad")
    frozen = head.linear_cross_entropy(h, W.detach(), t)
    _close(torch.autograd.grad(frozen, [h], up)[0], DH, "hidden_grad of a frozen head")
    for more in ((1, 8, (1 << 19) + 1), (1, (1 << 20) + 1, 2)):
        with pytest.raises(ConfigurationError):
            head.linear_cross_entropy(torch.zeros(1, more[1], device=dev, dtype=dtype),
                                      torch.zeros(more[2], more[1], device=dev, dtype=dtype),
                                      torch.zeros(1, dtype=torch.int64, device=dev))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("N,D,V", [(40, 64, 300), (300, 1544, 513), (700, 100, 3001)])
def test_no_token_has_a_target(dev, N, D, V, dtype):
    """Losses and both gradients are zeros, whatever the rows hold."""
    _, h, W, up = _inputs(dev, (N,), D, V, dtype, 72)
    h[::2] = math.nan
    t = torch.full((N,), -100, device=dev)
    h.requires_grad_(True)
    for w in (W, W.clone().requires_grad_(True)):
        for loss in (head.linear_cross_entropy(h, w, t),
                     head.topk_distillation(h, w, torch.zeros(N, 3, device=dev),
                                            torch.full((N, 3), -1, device=dev))):
            assert (loss == 0).all()
            grads = torch.autograd.grad(loss, [h, w] if w.requires_grad else [h], up)
            assert all((x == 0).all() for x in grads)


@pytest.mark.gpu
def test_thousands_of_teacher_entries(dev):
    N, D, V, K, tau = 19, 64, 9000, 3001, 2.0
    g, h, W, up = _inputs(dev, (N,), D, V, torch.bfloat16, 73)
    tl = torch.randn(N, K, generator=g, device=dev) * 2
    ti = torch.randint(0, V, (N, K), generator=g, device=dev)  # some of them repeated
    ti[:, ::7] = -1
    ti[3, 1:] = -1
    h.requires_grad_(True)
    W.requires_grad_(True)
    loss = head.topk_distillation(h, W, tl, ti, temperature=tau)
    dh, dW = torch.autograd.grad(loss, [h, W], up)
    q, ent = _soft(tl, ti, V, tau)
    L, DH, DW = _reference(h, W, q, ent, tau, up, frozen=True)
    _close(loss, L, "loss")
    _close(dh, DH, "hidden_grad")
    _close(dW, DW, "weight_grad")


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1, 64])
def test_bfloat16_gradients_in_norm(dev, K):
    """dz's rounding to bf16 and the gradient's own, independent and at most 2^-8 / sqrt(3)
    each in the mean square: 0.82 times 2^-8 together, and fp16 exponentials add 2^-11."""
    N, D, V, tau = 400, 256, 3000, 1.5
    g, h, W, up = _inputs(dev, (N,), D, V, torch.bfloat16, 81)
    tl, ti = _teacher(g, dev, (N,), V, K)
    q, ent = _soft(tl, ti, V, tau)
    _, (DH, _), (DW, _) = _reference(h, W, q, ent, tau, up)
    h.requires_grad_(True)
    for trained in (False, True):
        W.requires_grad_(trained)
        loss = head.topk_distillation(h, W, tl, ti, temperature=tau)
        grads = torch.autograd.grad(loss, [h, W] if trained else [h], up)
        for got, want in zip(grads, (DH, DW)):
            assert (got.double() - want).norm() <= 2.0**-8 * want.norm()
