"""Rotary positions (GPU) against the same rotation in 64 bits on the CPU.

Tolerance: sine and cosine are within 1.5 x 2^-23 of theirs (the reduced angle's rounding
2^-25, the series 2^-29 and six roundings of at most 2^-24 of partial sums below one) and the
amplitude, two products and their sum round four times more, so an element of a pair (a, b)
is within 5 x 2^-23 amplitude (|a| + |b|); bfloat16 results are rounded once more, 2^-8 of
themselves.
"""

from __future__ import annotations

import math

import pytest
import torch

from opake_amd import _native as nat
from opake_amd.exceptions import ConfigurationError, InputTypeError
from opake_amd.rotary import rotary, rotary_frequencies

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _pairs(x, n, interleaved):
    """The two halves of every pair, and the indices they lie at."""
    i = torch.arange(n)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, n + i)
    return x[..., a], x[..., b], a, b


def _want(x, positions, freqs, interleaved, amplitude, sign=1.0):
    x = x.detach().cpu().double()
    n = freqs.numel()
    turn = positions.cpu().double().unsqueeze(-1) * freqs.cpu() * sign
    c, s = (torch.cos(turn) * amplitude).unsqueeze(-2), (torch.sin(turn) * amplitude).unsqueeze(-2)
    a, b, ia, ib = _pairs(x, n, interleaved)
    out, size = x.clone(), torch.zeros_like(x)
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = abs(amplitude) * (a.abs() + b.abs())
    return out, size


def _check(got, want, size):
    tol = 5 * 2.0 ** -23 * size
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    err = (got.detach().cpu().double() - want).abs()
    assert bool((err <= tol).all()), (err - tol).max().item()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,H,KV,h,dims", [
    (1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 16, 16), (3, 7, 5, 1, 80, 40), (2, 5, 3, 3, 96, 24),
    (1, 33, 8, 2, 128, 128), (2, 9, 2, 1, 128, 64), (1, 4, 3, 2, 37, 10), (2, 2, 2, 1, 7, 6),
    (1, 2, 40, 8, 256, 256), (1, 1, 1, 1, 2048, 2048)])
def test_rotation_and_gradient(dev, dtype, interleaved, B, T, H, KV, h, dims):
    g = torch.Generator().manual_seed(B + 10 * T + 100 * h)
    dt = DTYPES[dtype]
    # Places of one tensor, as a fused projection leaves them.
    x = torch.randn(B, T, H + KV + 1, h, generator=g).to(dt).to(dev)
    q, k = (t.detach().requires_grad_() for t in (x[:, :, :H], x[:, :, H:H + KV]))
    freqs, _ = rotary_frequencies(dims, 10000.0, device=dev)
    pos = torch.randint(0, 1 << 20, (B, T), generator=g)
    oq, ok = rotary(q, k, freqs, positions=pos.to(dev), interleaved=interleaved, amplitude=1.25)
    assert oq.is_contiguous() and ok.is_contiguous()
    up = [torch.randn(t.shape, generator=g).to(dt).to(dev) for t in (oq, ok)]
    grads = torch.autograd.grad([oq, ok], [q, k], up)
    for t, got in ((q, oq), (k, ok)):
        _check(got, *_want(t, pos, freqs, interleaved, 1.25))
    for t, got in zip(up, grads):
        _check(got, *_want(t, pos, freqs, interleaved, 1.25, -1.0))


@pytest.mark.parametrize("positions", [None, "T", "int32"])
def test_positions(dev, positions):
    x = torch.randn(3, 300, 4, 64, device=dev)
    freqs, _ = rotary_frequencies(64, device=dev)
    at = torch.arange(300)
    arg = None
    if positions is not None:
        at = at * 7 - 50
        arg = at.to(dev) if positions == "T" else at.int().to(dev).expand(3, -1)
    out = rotary(x, None, freqs, positions=arg)
    _check(out, *_want(x, at.expand(3, -1), freqs, False, 1.0))


def test_the_angle_of_a_far_position(dev):
    """A million turns on, the angle is the near one's: frequencies of whole turns."""
    freqs = torch.full((8,), 2 * math.pi / 64, dtype=torch.float64, device=dev)
    x = torch.randn(1, 2, 1, 16, device=dev)
    pos = torch.tensor([3, 3 + 64 * 10 ** 6], device=dev)
    out = rotary(x[:, :1].expand(1, 2, 1, 16), None, freqs, positions=pos)
    torch.testing.assert_close(out[:, 0], out[:, 1], rtol=0, atol=1e-6)


def test_strides_and_unaligned_starts(dev):
    freqs, _ = rotary_frequencies(32, device=dev)
    base = torch.randn(2, 5, 6, 40, device=dev).to(torch.bfloat16)
    at = torch.arange(5).expand(2, -1)
    for x in (base[..., 1:33], base[..., ::1][:, :, ::2, 3:35], base.transpose(1, 2)[:, :5, :, :32],
              base[..., :32].flip(-1), base[:, :, :1, :32].expand(2, 5, 6, 32)):
        _check(rotary(x, None, freqs), *_want(x, at[:, :x.shape[1]], freqs, False, 1.0))


def test_transposed_gradients_and_one_output_alone(dev):
    freqs, _ = rotary_frequencies(32, device=dev)
    q = torch.randn(2, 5, 3, 32, device=dev, requires_grad=True)
    k = torch.randn(2, 5, 2, 32, device=dev, requires_grad=True)
    oq, ok = rotary(q, k, freqs)
    up = torch.randn(2, 3, 5, 32, device=dev)
    (gq,) = torch.autograd.grad(oq.transpose(1, 2), [q], up)
    _check(gq, *_want(up.transpose(1, 2), torch.arange(5).expand(2, -1), freqs, False, 1.0, -1.0))
    oq, ok = rotary(q, k.detach(), freqs)
    (gq2,) = torch.autograd.grad(oq.transpose(1, 2), [q], up)
    assert torch.equal(gq, gq2)


def test_nothing_to_rotate(dev):
    freqs, _ = rotary_frequencies(8, device=dev)
    q = torch.empty(0, 4, 2, 8, device=dev)
    assert rotary(q, q, freqs)[0].shape == q.shape
    q = torch.empty(2, 0, 2, 8, device=dev)
    assert rotary(q, None, freqs).shape == q.shape


def test_captured_forward_and_backward(dev):
    freqs, _ = rotary_frequencies(64, device=dev)
    q = torch.randn(2, 16, 4, 64, device=dev, requires_grad=True)
    up = torch.randn(2, 16, 4, 64, device=dev)

    def step():
        out = rotary(q, None, freqs)
        return out, torch.autograd.grad(out, [q], up)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)


def test_refusals(dev):
    q = torch.randn(2, 3, 4, 16, device=dev)
    freqs, _ = rotary_frequencies(16, device=dev)
    bad = [((q[0], None, freqs), {}), ((q, q[:, :2], freqs), {}), ((q, q.bfloat16(), freqs), {}),
           ((q, q[..., :8], freqs), {}), ((q.half(), None, freqs), {}),
           ((q, None, freqs.float()), {}), ((q[..., :8], None, freqs), {}),
           ((q, None, freqs[:0]), {}), ((q, q[:, :, :0], freqs), {}),
           ((q, None, freqs), dict(positions=torch.arange(4, device=dev))),
           ((q, None, freqs), dict(amplitude=math.inf)), ((q.cpu(), None, freqs), {})]
    for args, kw in bad:
        with pytest.raises(ConfigurationError):
            rotary(*args, **kw)
    with pytest.raises(InputTypeError):
        rotary(q, None, freqs, positions=torch.rand(3, device=dev))
    with pytest.raises(InputTypeError):
        rotary(q, None, freqs, amplitude="1")
    lib = nat.load()
    strides = (nat._c_i64 * 6)(*([0, 0, 1 << 40] * 2))
    assert lib.dpc_rotary(q.data_ptr(), 0, 2, 3, 4, 0, 16, nat.DPC_F32, strides, 0, 0, 0,
                          freqs.data_ptr(), 8, 0, 1.0, 0, q.data_ptr(), 0, 0) == nat.DPC_EINVAL


def test_heads_far_from_each_other(dev):
    """Strides past 32 bits, of which one head alone takes no memory."""
    freqs, _ = rotary_frequencies(16, device=dev)
    base = torch.randn(2, 5, 16, device=dev)
    q = base.as_strided((2, 5, 1, 16), (80, 16, 1 << 40, 1))
    want = rotary(base.view(2, 5, 1, 16), None, freqs)
    assert torch.equal(rotary(q, None, freqs), want)
    for got in rotary(base.view(2, 5, 1, 16), q, freqs):
        assert torch.equal(got, want)
