"""The block's operators (GPU): differences, few tokens, two streams, captured blocks.

References and their tolerances are those of the operators' own test files.
"""

from __future__ import annotations

import pytest
import torch

from opake_amd.attention import attention
from opake_amd.clipping import ghost_clipped_grad
from opake_amd.exceptions import OperationError
from opake_amd.gated import gated_linear
from opake_amd.lora import LoRABlock
from opake_amd.rotary import rotary, rotary_frequencies
from opake_amd.transformer import BlockLM, LlamaBlock, per_example_lm_loss
from test_gpu_gated import DTYPES, _act, _check, _inputs, _reference

pytestmark = pytest.mark.gpu


# Up to 32 tokens in bfloat16 and 64 in float32 have a kernel of their own: one to four blocks of 16
# tokens, whole runs along D and rests of them (a run is 128 or 64 wide, eight at a time), rows
# of F that end in a block, and widths that are not whole chunks, which it does not take.
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("N", [1, 15, 16, 17, 32, 33, 64, 65])
@pytest.mark.parametrize("D,F", [(8, 5), (1024, 16), (1160, 17), (4, 36), (100, 50), (2176, 33)])
def test_few_tokens(dev, dtype, N, D, F):
    x, w, up = _inputs((N, D), F, DTYPES[dtype], dev, seed=N + D)
    with torch.no_grad():
        alone = gated_linear(x, w)
    h = gated_linear(x, w)
    assert torch.equal(alone, h)
    dx, dw = torch.autograd.grad(h, [x, w], up)
    for got, ref in zip((h, dx, dw), _reference(x, w, up, "silu", x.dtype)):
        _check(got, ref)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_few_tokens_stay_their_own(dev, dtype):
    """Neither another token nor another weight row's infinities and NaN."""
    x, w, _ = _inputs((20, 200), 24, DTYPES[dtype], dev, seed=2)
    want = gated_linear(x, w).detach()
    with torch.no_grad():
        x[3, 7] = float("nan")
        x[19, 199] = float("inf")
        w[5, 0] = float("inf")
        got = gated_linear(x, w)
    keep = torch.ones(20, dtype=torch.bool, device=dev)
    keep[[3, 19]] = False
    cols = torch.ones(24, dtype=torch.bool, device=dev)
    cols[5] = False
    assert torch.equal(got[keep][:, cols], want[keep][:, cols])
    assert bool(got[3].isnan().all()) and not bool(got[19].isfinite().any())


def test_gated_gradients_against_differences(dev):
    """In float32, against central differences of the formula in float64."""
    for act in ("silu", "gelu"):
        x, w, up = _inputs((5, 12), 7, torch.float32, dev, seed=9)
        grads = torch.autograd.grad(gated_linear(x, w, activation=act), [x, w], up)
        for i, g in enumerate(grads):
            way = torch.randn(g.shape, generator=torch.Generator().manual_seed(i)).double()

            def loss(step):
                t = [x.detach().cpu().double(), w.detach().cpu().double()]
                t[i] = t[i] + step * way
                z = t[0] @ t[1].T
                return (_act(z[:, :7], act)[0] * z[:, 7:] * up.cpu().double()).sum().item()

            d = 1e-4  # third derivatives of order one: 1e-8
            slope = (loss(d) - loss(-d)) / (2 * d)
            assert abs(slope - (g.cpu().double() * way).sum().item()) < 1e-5 * max(1.0, abs(slope))


def test_rotary_gradients_against_differences(dev):
    """The rotation is linear: its differences are its derivative, 2^-22 of either value off."""
    g = torch.Generator().manual_seed(4)
    for interleaved in (False, True):
        q, way, up = (torch.randn(2, 9, 3, 24, generator=g).to(dev) for _ in range(3))
        q.requires_grad_()
        freqs, amplitude = rotary_frequencies(16, scaling={"kind": "linear", "factor": 3.0},
                                              device=dev)
        turn = lambda t: rotary(t, None, freqs, interleaved=interleaved,  # noqa: E731
                                amplitude=1.25 * amplitude)
        (dq,) = torch.autograd.grad(turn(q), [q], up)
        slope = ((turn(q + way) - turn(q)).double() * up.double()).sum().item()
        size = (up.double() ** 2).sum().sqrt().item() * (q.double() ** 2).sum().sqrt().item()
        assert abs(slope - (dq.double() * way.double()).sum().item()) < 2.0 ** -18 * size


def test_one_tensor_as_queries_keys_and_values(dev):
    g = torch.Generator().manual_seed(6)
    x = torch.randn(2, 77, 4, 32, generator=g).to(dev).requires_grad_()
    up = torch.randn(2, 77, 4, 32, generator=g).to(dev)
    (got,) = torch.autograd.grad(attention(x, x, x), [x], up)
    parts = [x.detach().clone().requires_grad_() for _ in range(3)]
    want = torch.autograd.grad(attention(*parts), parts, up)
    torch.testing.assert_close(got, want[0] + want[1] + want[2], rtol=2.0 ** -20, atol=1e-6)
    freqs, _ = rotary_frequencies(32, device=dev)
    a, b = rotary(x, x, freqs)
    assert torch.equal(a, b)
    (got,) = torch.autograd.grad((a, b), [x], (up, up))
    (once,) = torch.autograd.grad(rotary(x, None, freqs), [x], up)
    assert torch.equal(got, 2 * once)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("h", [16, 128, 256])
def test_a_query_that_sees_one_key(dev, dtype, h):
    """Its probability is one whatever the score: no gradient of query or key, exactly."""
    g = torch.Generator().manual_seed(h)
    for B, T, S, options in ((2, 300, 300, dict(window=1)), (1, 1, 1, {}), (2, 70, 1, dict(causal=False)),
                             (20, 900, 900, dict(window=1)), (2, 40, 90, dict(window=1))):
        q, k, v, up = (torch.randn(B, n, heads, h, generator=g).to(DTYPES[dtype]).to(dev)
                       for n, heads in ((T, 4), (S, 2), (S, 2), (T, 4)))
        q, k, v = (t.requires_grad_() for t in (q, k, v))
        out = attention(q, k, v, **options)
        dq, dk, dv = torch.autograd.grad(out, [q, k, v], up)
        assert not dq.any() and not dk.any() and dv.any()
        own = v[:, -T:].repeat_interleave(2, 2) if S > 1 else v.repeat_interleave(2, 2).expand_as(q)
        # (p v) (1 / p): three float32 roundings, 3 x 2^-24 of v; in bfloat16 rounded away.
        off = 3 * 2.0 ** -24 if dtype == "fp32" else 0.0
        assert bool(((out.double() - own.double()).abs() <= off * own.double().abs()).all())
    # The first token of a sequence, and a sequence of one.
    q, k, v, up = (torch.randn(2, 150, 2, h, generator=g).to(DTYPES[dtype]).to(dev).requires_grad_()
                   for _ in range(4))
    lengths = torch.tensor([150, 1], device=dev)
    dq, dk, _ = torch.autograd.grad(
        attention(q, k, v, lengths=lengths, starts=torch.zeros_like(lengths)), [q, k, v], up)
    assert not dq[:, 0].any() and not dk[1].any() and dq[0, 1:].any() and dk[0].any()


def test_two_streams_at_once(dev):
    """Calls beside each other have their own workspaces, and answer as one by one."""
    torch.manual_seed(1)
    blocks = [LlamaBlock(128, 2, 192, fused=True, dtype=torch.bfloat16).to(dev) for _ in range(2)]
    xs = [torch.randn(2, 300, 128, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    caches = [torch.randn(4, 3000, 2, 64, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    ones = [torch.randn(4, 1, 8, 64, dtype=torch.bfloat16, device=dev) for _ in range(2)]

    def work(i):
        x = xs[i].detach().requires_grad_()
        y = blocks[i](x)
        (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
        return y.detach(), dx, attention(ones[i], caches[i], caches[i])

    want = [work(0), work(1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_captured_block(dev, dtype):
    """A fused block's forward and its input's gradient in one graph, replayed."""
    torch.manual_seed(2)
    block = LlamaBlock(128, 2, 192, fused=True, dtype=DTYPES[dtype]).to(dev)
    block.requires_grad_(False)
    x = torch.randn(2, 150, 128, dtype=DTYPES[dtype], device=dev)
    up = torch.randn_like(x)

    def step():
        leaf = x.detach().requires_grad_()
        y = block(leaf)
        return y.detach(), torch.autograd.grad(y, [leaf], up)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)


def test_frequencies_follow_the_block(dev):
    """Casts leave them in float64, and moves take them along."""
    for make in (lambda: LlamaBlock(64, 2, 24, fused=True),
                 lambda: LoRABlock(64, 2, 1, 24, 4, fused=True)):
        block = make().to(torch.bfloat16).to(dev)
        want, _ = rotary_frequencies(32, device=dev)
        assert torch.equal(block.rope.freqs, want) and not any("rope" in n for n in block.state_dict())
        x = torch.randn(1, 5, 64, dtype=torch.bfloat16, device=dev)
        assert torch.isfinite(block(x)).all()


def test_a_failed_capture_leaves_the_layer_as_it_was(dev):
    model = BlockLM(11, 32, 2, 24, fused=True, dtype=torch.float32).to(dev)
    ids = torch.zeros(2, 4, dtype=torch.int64, device=dev)
    layer = model.block.gate_up

    def broken(logits, targets):
        raise RuntimeError("no loss")

    fn, st = ghost_clipped_grad(model, broken, clipping_norm=1.0)
    with pytest.raises(RuntimeError, match="no loss"):
        fn(ids, ids, state=st)
    assert not layer.dpc_keep_projections and layer.dpc_projections is None
    model(ids)
    assert layer.dpc_projections is None
    fn, st = ghost_clipped_grad(model, per_example_lm_loss, clipping_norm=1.0)
    out, _ = fn(ids, ids, state=st)
    assert all(torch.isfinite(t).all() for t in out.pytree.values())


def test_caches_past_32_bits(dev):
    """Keys whose elements lie past 2^31: a window at the end of the last of three sequences."""
    B, S, KV, h, window = 3, 1 << 20, 8, 128, 90
    g = torch.Generator().manual_seed(8)
    q = torch.randn(B, 2, 16, h, generator=g).to(torch.bfloat16).to(dev)
    k, v = (torch.zeros(B, S, KV, h, dtype=torch.bfloat16, device=dev) for _ in range(2))
    assert k.numel() > 2 ** 31
    for t in (k, v):
        t[:, -400:] = torch.randn(B, 400, KV, h, generator=g).to(torch.bfloat16).to(dev)
    lengths = torch.tensor([S, S - 300, S - 7], device=dev)
    got = attention(q, k, v, window=window, lengths=lengths, starts=lengths - 2)
    near = attention(q, k[:, -400:].contiguous(), v[:, -400:].contiguous(), window=window,
                     lengths=lengths - (S - 400), starts=lengths - 2 - (S - 400))
    # Either rounds p to 2^-8 of itself and the result once more, in an order of its own.
    assert ((got.double() - near.double()).abs() <= 2.0 ** -6 * v[:, -400:].abs().max()).all()
    assert torch.isfinite(got).all() and got.abs().max() > 0.1


def test_tokens_past_32_bits(dev):
    """Results whose elements lie past 2^31, against a few of the last tokens by themselves."""
    N, D, F, few = 70001, 64, 16384, 65
    x, w, _ = _inputs((N, D), F, torch.bfloat16, dev, seed=5)
    h = gated_linear(x, w)
    up = torch.randn_like(h)
    (dx,) = torch.autograd.grad(h, [x], up)
    assert N * 2 * F > 2 ** 31
    last = x.detach()[-few:].clone().requires_grad_()
    want = gated_linear(last, w.detach())
    (dlast,) = torch.autograd.grad(want, [last], up[-few:])
    for got, ref in zip((h[-few:], dx[-few:]), (want, dlast)):
        # The same operands in other tiles: float32 sums in another order, one rounding each.
        off = 2.0 ** -7 * ref.double().abs() + 2.0 ** -12 * ref.double().abs().max()
        assert bool(((got.double() - ref.double()).abs() <= off).all())
    del h, up, dx
    T = 270001
    q = torch.randn(1, T, 64, 128, dtype=torch.bfloat16, device=dev)
    assert q.numel() > 2 ** 31
    freqs, _ = rotary_frequencies(128, device=dev)
    far = rotary(q, None, freqs)
    positions = torch.arange(T - 9, T, device=dev)
    assert torch.equal(far[:, -9:], rotary(q[:, -9:], None, freqs, positions=positions))


def test_more_sequences_than_a_launch_takes(dev):
    """2^23 key heads of one token, 512 threads each: they go out in two launches."""
    B, KV, h = 1 << 21, 4, 8
    g = torch.Generator(device=dev).manual_seed(3)
    q, k, v, up = (torch.randn(B, 1, KV, h, generator=g, device=dev, dtype=torch.bfloat16)
                   for _ in range(4))
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out = attention(q, k, v)
    dq, dk, dv = torch.autograd.grad(out, [q, k, v], up)
    assert torch.equal(out, v) and torch.equal(dv, up) and not dq.any() and not dk.any()


def test_more_tokens_than_a_launch_takes(dev):
    """2^24 tokens of a workgroup each: they go out in two launches."""
    N, h = (1 << 24) + 3, 1026
    g = torch.Generator(device=dev).manual_seed(3)
    q = torch.randn(1, 1, 1, h, generator=g, device=dev, dtype=torch.bfloat16)
    freqs, _ = rotary_frequencies(h, device=dev)
    positions = (torch.arange(N, device=dev) % 7).view(N, 1)
    out = rotary(q.expand(N, 1, 1, h), None, freqs, positions=positions)
    want = rotary(q.expand(7, 1, 1, h), None, freqs, positions=positions[:7])
    for at in range(0, N, 7 << 18):
        part = out[at:at + (7 << 18)]
        assert torch.equal(part, want[positions[at:at + (7 << 18), 0]])


def test_odd_widths_are_refused_beside_a_living_eager_graph_too(dev):
    """Heads that are no whole chunks, whose rows are copied: the leaves are seen all the same."""
    g = torch.Generator().manual_seed(7)
    q, k, v, up = (torch.randn(2, 30, 2, 7, generator=g).to(dev) for _ in range(4))
    q, k, v = (t.requires_grad_() for t in (q, k, v))

    def step():
        out = attention(q, k, v)
        return (out, *torch.autograd.grad(out, [q, k, v], up))

    alive = attention(q, k, v)
    assert len(alive.grad_fn.next_functions[0][0].accumulators) == 3
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
            q.copy_(torch.randn_like(q))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)
