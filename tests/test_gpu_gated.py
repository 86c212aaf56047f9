"""Gated projections (GPU) against the same formulas in 64 bits on the CPU.

Tolerances are elementwise and follow the roundings.  A product of K terms is within
(K 2^-23 + 2^-21) sum |a b| of its own: float32 sums in any order, and for float32 operands
the two planes' 2^-21 a term.  act is 1.13-Lipschitz and act' 0.8-Lipschitz (SiLU: 1.1 and
0.5; GELU: 1.13 and 0.8); act, act' and the products round a few times more (16 x 2^-23
covers them, and the fast exponential and reciprocal of bf16 inputs).  bf16: the result, dz
and the gradients are rounded to it, 2^-8 of each; the projections are kept within 2^-17.
"""

from __future__ import annotations

import math

import pytest
import torch

from opake_amd import _native as nat
from opake_amd.exceptions import ConfigurationError, OperationError
from opake_amd.gated import GatedLinear, gated_linear

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
FEW = 16 * 2.0 ** -23


def _act(g, kind):
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    s = 0.5 * torch.erfc(-g * math.sqrt(0.5))
    return g * s, s + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def _sum_error(a, b, k):
    return (k * 2.0 ** -23 + 2.0 ** -21) * (a.abs() @ b.abs())


def _rounded(want, err, half):
    return err + (half * (want.abs() + err) if half else 0.0)


def _reference(x, w, up, act, dtype):
    """(value, tolerance) of h, dx and dw."""
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    x, w, up = (t.detach().cpu().double() for t in (x, w, up))
    F, D = w.shape[0] // 2, w.shape[1]
    x, up = x.reshape(-1, D), up.reshape(-1, F)
    z, ez = x @ w.T, _sum_error(x, w.T, D)
    g, u, eg, eu = z[:, :F], z[:, F:], ez[:, :F], ez[:, F:]
    a, slope = _act(g, act)
    h = a * u
    eh = 1.13 * eg * (u.abs() + eu) + a.abs() * eu + FEW * h.abs()
    # The backward reads z as it was kept.
    kept = 2.0 ** -17 if half else 0.0
    eg, eu = _rounded(g, eg, kept), _rounded(u, eu, kept)
    dz = torch.cat([up * u * slope, up * a], 1)
    es, ea = 0.8 * eg + FEW * (slope.abs() + g.abs()), 1.13 * eg + FEW * a.abs()
    edz = torch.cat([up.abs() * ((u.abs() + eu) * es + slope.abs() * eu), up.abs() * ea], 1)
    edz = _rounded(dz, edz + FEW * dz.abs(), half)
    full = dz.abs() + edz
    dx, dw = dz @ w, dz.T @ x
    edx = edz @ w.abs() + _sum_error(full, w, 2 * F)
    edw = edz.T @ x.abs() + _sum_error(full.T, x, x.shape[0])
    return [(v, _rounded(v, e, half)) for v, e in ((h, eh), (dx, edx), (dw, edw))]


def _check(got, ref):
    want, tol = ref
    err = (got.detach().cpu().double().reshape(want.shape) - want).abs()
    assert bool((err <= tol).all()), ((err - tol).max().item(), err.max().item())


def _inputs(shape, F, dtype, dev, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    D = shape[-1]
    x = torch.randn(*shape, generator=g).to(dtype).to(dev)
    w = (torch.randn(2 * F, D, generator=g) * (spread / math.sqrt(D))).to(dtype).to(dev)
    up = torch.randn(*shape[:-1], F, generator=g).to(dtype).to(dev)
    return x.requires_grad_(), w.requires_grad_(), up


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("shape,F", [
    ((1, 1), 1), ((3, 7), 2), ((2, 5, 8), 3), ((17, 64), 64), ((1, 256), 127), ((300, 100), 129),
    ((256, 130), 260), ((5, 2048), 100), ((1100, 40), 50), ((2, 301, 72), 300), ((33, 96), 4),
    ((16, 1032), 513), ((64, 520), 31), ((65, 264), 132)])
def test_values_and_gradients(dev, dtype, shape, F, act):
    x, w, up = _inputs(shape, F, DTYPES[dtype], dev, seed=F + len(shape))
    h = gated_linear(x, w, activation=act)
    assert h.shape == (*shape[:-1], F) and h.dtype == x.dtype
    dx, dw = torch.autograd.grad(h, [x, w], up)
    for got, ref in zip((h, dx, dw), _reference(x, w, up, act, x.dtype)):
        _check(got, ref)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_one_gradient_alone_and_none(dev, dtype):
    x, w, up = _inputs((70, 136), 90, DTYPES[dtype], dev, seed=3)
    h = gated_linear(x, w)
    dx, dw = torch.autograd.grad(h, [x, w], up, retain_graph=True)
    again = torch.autograd.grad(h, [x, w], up)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])
    (only_x,) = torch.autograd.grad(gated_linear(x, w.detach()), [x], up)
    (only_w,) = torch.autograd.grad(gated_linear(x.detach(), w), [w], up)
    assert torch.equal(dx, only_x) and torch.equal(dw, only_w)
    with torch.no_grad():
        assert torch.equal(gated_linear(x, w), h)
    assert not gated_linear(x.detach(), w.detach()).requires_grad


def test_no_token(dev):
    for dtype in DTYPES.values():
        x, w, up = _inputs((0, 16), 8, dtype, dev, seed=1)
        h = gated_linear(x, w)
        dx, dw = torch.autograd.grad(h, [x, w], up)
        assert h.shape == (0, 8) and dx.shape == x.shape and not dw.any()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("D,F", [(2048, 8192), (1024, 1408), (1001, 512), (64, 512)])
def test_no_token_at_the_widths_of_a_block(dev, dtype, D, F):
    """Sums long enough to be cut in slices, of no tiles."""
    x, w, up = _inputs((0, D), F, DTYPES[dtype], dev, seed=1)
    h = gated_linear(x, w)
    assert h.shape == (0, F) and gated_linear(x.detach(), w.detach()).shape == (0, F)
    for want in ([x, w], [x], [w]):
        got = torch.autograd.grad(h, want, up, retain_graph=True)
        assert all(t.shape == o.shape and not t.any() for t, o in zip(got, want))


def test_strided_and_unaligned_operands(dev):
    g = torch.Generator().manual_seed(5)
    base = torch.randn(40, 3, 65, generator=g).to(torch.bfloat16).to(dev)
    wide = (torch.randn(48, 130, generator=g) / 8).to(torch.bfloat16).to(dev)
    up = torch.randn(24, 40, generator=g).to(torch.bfloat16).to(dev)
    x = base[:, 1, 1:].detach().requires_grad_()
    w = wide[:, 1:129:2].detach().requires_grad_()
    h = gated_linear(x, w)
    dx, dw = torch.autograd.grad(h, [x, w], up.T)
    for got, ref in zip((h, dx, dw), _reference(x, w, up.T, "silu", torch.bfloat16)):
        _check(got, ref)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_saturated_gates(dev, dtype, act):
    """Gates far into either side: the activation is the identity or nothing."""
    dt = DTYPES[dtype]
    x = torch.tensor([[1.0], [-1.0], [30.0], [-30.0], [0.0], [1e30]], device=dev).to(dt)
    w = torch.tensor([[100.0], [2.0]], device=dev).to(dt)
    x.requires_grad_(), w.requires_grad_()
    up = torch.ones(6, 1, device=dev, dtype=dt)
    h = gated_linear(x[:5], w, activation=act)
    want = torch.tensor([200.0, 0.0, 180000.0, 0.0, 0.0], dtype=torch.float64)
    torch.testing.assert_close(h[:, 0].double().cpu(), want, rtol=2.0 ** -8, atol=1e-30)
    dx, dw = torch.autograd.grad(h, [x, w], up[:5])
    assert bool(dx.isfinite().all()) and bool(dw.isfinite().all())
    assert gated_linear(x, w, activation=act)[5].item() == math.inf


def test_float32_rows_of_very_different_sizes(dev):
    """A token's outlier costs the others nothing, forward, in dx and (against the largest
    contribution) in dw."""
    x, w, up = _inputs((64, 48), 40, torch.float32, dev, seed=9)
    scale = torch.ones(64, 1, device=dev)
    scale[3], scale[5] = 1e12, 1e-12
    xs = (x * scale).detach().requires_grad_()
    h, hs = gated_linear(x, w), gated_linear(xs, w)
    keep = [i for i in range(64) if i not in (3, 5)]
    torch.testing.assert_close(hs[keep], h[keep], rtol=1e-6, atol=1e-7)
    ups = up / scale
    dx = torch.autograd.grad(hs, [xs, w], ups)
    for got, ref in zip((hs, *dx), _reference(xs, w, ups, "silu", torch.float32)):
        _check(got, ref)


def test_nonfinite_tokens_stay_their_own(dev):
    for dtype in DTYPES.values():
        x, w, up = _inputs((20, 24), 12, dtype, dev, seed=2)
        h = gated_linear(x, w)
        with torch.no_grad():
            y = x.clone()
            y[4] = math.nan
            y[7, 3] = math.inf
        y.requires_grad_()
        hy = gated_linear(y, w)
        (dx,), (dy,) = (torch.autograd.grad(a, [b], up) for a, b in ((h, x), (hy, y)))
        keep = [i for i in range(20) if i not in (4, 7)]
        assert torch.equal(h[keep], hy[keep]) and torch.equal(dx[keep], dy[keep])
        assert bool(hy[4].isnan().all()) and not bool(hy[7].isfinite().any())


def test_captured_and_refused_beside_a_living_eager_graph(dev):
    x, w, up = _inputs((96, 64), 80, torch.bfloat16, dev, seed=4)
    alive = gated_linear(x, w)

    def step():
        h = gated_linear(x, w)
        return (h, *torch.autograd.grad(h, [x, w], up))

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
    for _ in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)


def test_on_another_stream(dev):
    x, w, up = _inputs((257, 72), 136, torch.float32, dev, seed=6)
    want = gated_linear(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [gated_linear(x, w) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(t, want) for t in got)


def test_layer(dev):
    layer = GatedLinear(24, 40, activation="gelu", dtype=torch.float32, device=dev)
    x = torch.randn(3, 5, 24, device=dev)
    assert torch.equal(layer(x), gated_linear(x, layer.weight, activation="gelu"))
    layer(x).sum().backward()
    assert layer.weight.grad.shape == (80, 24) and layer.dpc_projections is None


def test_refusals(dev):
    x, w, _ = _inputs((4, 16), 8, torch.float32, dev, seed=1)
    for args, kw in (((x, w[:15]), {}), ((x[:, :8], w), {}), ((x, w.bfloat16()), {}),
                     ((x.half(), w.half()), {}), ((x, w[0]), {}), ((x, w), dict(activation="tanh")),
                     ((x.cpu(), w), {}), ((x, w[:0]), {}), ((x[:, :0], w[:, :0]), {})):
        with pytest.raises(ConfigurationError):
            gated_linear(*args, **kw)
    with pytest.raises(ConfigurationError):
        GatedLinear(4, 4, activation="tanh")


def test_entry_points_refuse(dev):
    lib = nat.load()
    x, w, _ = _inputs((4, 16), 8, torch.float32, dev, seed=1)
    h = torch.empty(4, 8, device=dev)
    n = lib.dpc_gated_linear_workspace_bytes(4, 16, 8, nat.DPC_F32)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)

    def call(N=4, D=16, F=8, code=nat.DPC_F32, act=0, xp=x.data_ptr(), size=n):
        return lib.dpc_gated_linear(xp, w.data_ptr(), N, D, F, code, act, h.data_ptr(), 0, 0,
                                    ws.data_ptr(), size, 0)

    assert call(size=n - 1) == nat.DPC_ENOSPC
    for bad in (dict(N=-1), dict(D=0), dict(F=0), dict(code=nat.DPC_F16), dict(act=2), dict(xp=0),
                dict(xp=x.data_ptr() + 4)):
        assert call(**bad) == nat.DPC_EINVAL, bad


def test_tangents_are_refused(dev):
    """Forward-mode differentiation, with gradients and without."""
    x, w, _ = _inputs((4, 16), 8, torch.float32, dev, seed=1)
    layer = GatedLinear(16, 8, dtype=torch.float32, device=dev)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
            for call in (lambda: gated_linear(dual, w), lambda: gated_linear(dual, w.detach()),
                         lambda: layer(dual)):
                with pytest.raises(NotImplementedError):
                    call()


def test_what_is_kept_of_projections(dev):
    """bfloat16: z and its rest give the float32 sum within 2^-16, half a step of 8 bits more;
    within 2^-15 (a step) where the rest would pass its byte, |z - bf16(z)| >= 127.5 / 128 of half
    a bf16 step.  Sums of a pair are exact here, so what is off is the rest alone."""
    F, D, N = 64, 8, 300  # (tiles; the few tokens' kernel takes the first 5)
    g = torch.Generator().manual_seed(8)
    x = torch.zeros(N, D)
    x[:, 0] = 1.0
    x[:, 1] = torch.randint(-256, 257, (N,), generator=g) * 2.0 ** -16  # up to half a bf16 step
    w = torch.zeros(2 * F, D)
    w[:, 0] = 1 + torch.randint(0, 128, (2 * F,), generator=g) / 128
    w[:, 1] = 1.0
    x, w = x.bfloat16(), w.bfloat16()
    z = x.double() @ w.double().T
    assert torch.equal(z.float().double(), z)  # exact in float32
    near = (z - z.float().bfloat16().double()).abs() >= 127.5 / 128 * 2.0 ** -8
    assert near.any() and not near.all()
    lib, xd, wd = nat.load(), x.to(dev), w.to(dev)
    for n in (5, N):
        h, kept = (torch.empty(n, c, dtype=torch.bfloat16, device=dev) for c in (F, 2 * F))
        rest = torch.empty(n, 2 * F, dtype=torch.int8, device=dev)
        size = lib.dpc_gated_linear_workspace_bytes(n, D, F, nat.DPC_BF16)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        nat.call_on(xd.device, "dpc_gated_linear", xd.data_ptr(), wd.data_ptr(), n, D, F,
                    nat.DPC_BF16, nat.ACT_SILU, h.data_ptr(), kept.data_ptr(), rest.data_ptr(),
                    ws.data_ptr(), size)
        bits = (kept.view(torch.int16).int() << 16) + (rest.int() << 8)
        off = (bits.view(torch.float32).cpu().double() - z[:n]).abs() / z[:n]
        assert torch.equal(kept.cpu(), z[:n].float().bfloat16())
        assert bool((off <= torch.where(near[:n], 2.0 ** -15, 2.0 ** -16)).all())
