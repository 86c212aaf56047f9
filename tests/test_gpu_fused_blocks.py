"""The fused transformer blocks (GPU): rotary, attention and gated projections together.

Each model with ``fused`` against the default one in 64 bits on the CPU: ordinary gradients,
clipped gradients against per-example ones, and a sequence taken token by token with a cache.
Tolerances: in float32 about twenty products and sums, forward and back, each within 2^-21 of
its size: 2e-5 in all, as for the routed model.  In bfloat16 a gradient passes some thirty
roundings of at most 2^-8; their signs are independent, so they add as sqrt(30) 2^-8 / sqrt(3)
(a rounding's error is uniform over the step, and over a binade half as large in the mean):
1.2e-2 at most in norm, 2e-2 with what the norms and the residuals multiply it by.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from opake_amd import ops
from opake_amd.attention import attention
from opake_amd.clipping import auto_ghost_clipped_grad, ghost_clipped_grad
from opake_amd.exceptions import OpakeError
from opake_amd.gated import GatedLinear
from opake_amd.lora import LoRABlock
from opake_amd.moe import RoutedLM, TopKMoE, expert_groups
from opake_amd.noise import gaussian_noise
from opake_amd.random import key
from opake_amd.rotary import rotary, rotary_frequencies
from opake_amd.transformer import BlockLM, LlamaBlock, per_example_lm_loss
from opake_amd.types import PerGroup
from oracle import clip_oracle, ghost_oracle

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2e-5, torch.bfloat16: 2e-2}


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    return ((got - want).norm() / want.norm().clamp_min(1e-300)).item()


def _pair(make, dtype, dev, std=0.05, seed=0):
    """The default model in 64 bits and the fused one on the device, of equal weights."""
    torch.manual_seed(seed)
    ref = make(dtype=torch.float64, fused=False)
    with torch.no_grad():
        for p in ref.parameters():
            p.normal_(0.0, std)
            p.copy_(p.to(dtype).double())
    model = make(dtype=dtype, fused=True)
    model.load_state_dict({k: v.to(dtype) for k, v in ref.state_dict().items()})
    return ref, model.to(dev)


def _oracle(ref, loss, inputs, tgt, C, names):
    per = ghost_oracle.per_example_grads_loop(ref, loss, inputs, tgt)
    leaves = [per[n].float() for n in names]
    if isinstance(C, PerGroup):
        values = {k: clip_oracle.conservative_bound(v) for k, v in C.values.items()}
        return clip_oracle.stream_clip_and_sum(leaves, None, groups=[C.groups[(n,)] for n in names],
                                               group_values=values, return_aux=True)
    return clip_oracle.stream_clip_and_sum(leaves, clip_oracle.conservative_bound(C),
                                           return_aux=True)


def _names(model):
    return sorted(n for n, p in model.named_parameters() if p.requires_grad)


def _sq(out, t):
    return ((out - t.to(out.dtype)).to(torch.promote_types(out.dtype, torch.float32)) ** 2).sum(
        dim=(1, 2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,d,heads,ffn", [(3, 20, 32, 4, 48), (2, 129, 96, 2, 72),
                                             (2, 1, 64, 1, 8), (1, 257, 128, 1, 200)])
def test_block_output_and_ordinary_gradients(dev, dtype, B, T, d, heads, ffn):
    ref, model = _pair(lambda **kw: LlamaBlock(d, heads, ffn, **kw), dtype, dev, std=0.1, seed=T)
    g = torch.Generator().manual_seed(T + 1)
    x = torch.randn(B, T, d, generator=g).to(dtype)
    t = torch.randn(B, T, d, generator=g).to(dtype)
    xr = x.double().requires_grad_()
    xd = x.to(dev).requires_grad_()
    want, got = ref(xr), model(xd)
    assert _rel(got, want) < TOL[dtype]
    (want * t.double()).sum().backward()
    (got * t.to(dev)).sum().backward()
    assert _rel(xd.grad, xr.grad) < TOL[dtype]
    for (n, p), (m, q) in zip(model.named_parameters(), ref.named_parameters()):
        assert n == m
        if T > 1 or n != "qkv.weight":
            assert _rel(p.grad, q.grad) < TOL[dtype], n
    if T == 1:  # one key: nothing reaches queries and keys
        w = ref.qkv.weight.grad
        assert _rel(model.qkv.weight.grad[2 * d:], w[2 * d:]) < TOL[dtype]
        assert model.qkv.weight.grad[:2 * d].abs().max().item() < 1e-2 * w.abs().max().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_token_has_no_gradient_of_queries_and_keys(dev, dtype):
    """Exactly zero: one key's probability is one, and rotary and the layer keep zeros."""
    d = 64
    block = LlamaBlock(d, 1, 8, fused=True, dtype=dtype, device=dev)
    lora = LoRABlock(d, 2, 1, 8, 2, fused=True, dtype=dtype, device=dev)
    with torch.no_grad():
        for n, p in lora.named_parameters():
            if p.requires_grad:
                p.normal_(0.0, 0.1)
    g = torch.Generator().manual_seed(18)
    x, up = (torch.randn(2, 1, d, generator=g).to(dtype).to(dev) for _ in range(2))
    for model in (block, lora):
        (model(x) * up).sum().backward()
    grad = block.qkv.weight.grad
    assert not grad[:2 * d].any() and grad[2 * d:].any()
    for n, p in lora.named_parameters():
        if p.requires_grad:
            assert bool(p.grad.any()) == (n.split(".")[0] not in ("q", "k")), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("per_group", [False, True])
def test_clipped_block_matches_per_example_oracle(dev, dtype, per_group):
    V, d, B, T = 61, 64, 3, 40
    ref, model = _pair(lambda **kw: BlockLM(V, d, 4, 96, **kw), dtype, dev, seed=4)
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, V, (B, T), generator=g)
    tgt = torch.randint(0, V, (B, T), generator=g)
    names = _names(model)
    C = 0.1
    if per_group:
        C = PerGroup({n: "mlp" if "gate_up" in n or "down" in n else "rest" for n in names},
                     {"mlp": 0.1, "rest": 0.2})
    res = _oracle(ref, per_example_lm_loss, (ids,), tgt, C, names)
    fn, st = ghost_clipped_grad(model, per_example_lm_loss, clipping_norm=C, normalize_by=3.0,
                                return_aux=True, dtype=torch.float32)
    (out, aux), _ = fn(ids.to(dev), tgt.to(dev), state=st)
    assert sorted(out.pytree) == names
    for i, n in enumerate(names):
        assert _rel(out.pytree[n], res.reduced[i] / 3.0) < TOL[dtype], n
    assert _rel(aux.grad_norms, res.norms) < TOL[dtype]
    layer = model.block.gate_up
    assert isinstance(layer, GatedLinear) and not layer.dpc_keep_projections
    assert layer.dpc_projections is None


def test_clipped_block_noise_and_microbatches(dev):
    """The fused noise, microbatches and the automatic clipping see the same gradients."""
    V, d, B, T = 61, 64, 4, 33
    _, model = _pair(lambda **kw: BlockLM(V, d, 2, 96, **kw), torch.float32, dev, seed=6)
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, V, (B, T), generator=g).to(dev)
    tgt = torch.randint(0, V, (B, T), generator=g).to(dev)
    fn, st = ghost_clipped_grad(model, per_example_lm_loss, clipping_norm=0.1)
    plain, _ = fn(ids, tgt, state=st)
    again, _ = fn(ids, tgt, state=st)
    half, st2 = ghost_clipped_grad(model, per_example_lm_loss, clipping_norm=0.1,
                                   microbatch_size=2)
    parts, _ = half(ids, tgt, state=st2)
    noise_fn, nstate = gaussian_noise(noise_multiplier=0.7, key=key(11))
    noisy, _, _ = fn(ids, tgt, state=st, noise_fn=noise_fn, noise_state=nstate)
    separate, _ = noise_fn(plain, nstate)
    auto, ast = auto_ghost_clipped_grad(model, per_example_lm_loss, R=0.1, gamma=0.01)
    scaled, _ = auto(ids, tgt, state=ast)
    for n in _names(model):
        assert torch.equal(plain.pytree[n], again.pytree[n]), n
        assert torch.equal(noisy.pytree[n], separate.pytree[n]), n
        assert _rel(parts.pytree[n], plain.pytree[n]) < TOL[torch.float32], n
        assert torch.isfinite(scaled.pytree[n]).all(), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clipped_lora_block_matches_per_example_oracle(dev, dtype):
    ref, model = _pair(lambda **kw: LoRABlock(d=64, n_heads=4, n_kv_heads=2, ffn=96, r=4, **kw),
                       dtype, dev, std=0.1, seed=8)
    g = torch.Generator().manual_seed(9)
    x = torch.randn(3, 64, 64, generator=g).to(dtype)
    t = torch.randn(3, 64, 64, generator=g).to(dtype)
    names = _names(model)
    assert len(names) == 14
    res = _oracle(ref, _sq, (x.double(),), t.double(), 0.5, names)
    fn, st = ghost_clipped_grad(model, _sq, clipping_norm=0.5, normalize_by=2.0, return_aux=True,
                                dtype=torch.float32)
    (out, aux), _ = fn(x.to(dev), t.to(dev), state=st)
    for i, n in enumerate(names):
        assert _rel(out.pytree[n], res.reduced[i] / 2.0) < TOL[dtype], n
    assert _rel(aux.grad_norms, res.norms) < TOL[dtype]


@pytest.mark.parametrize("dtype,d,inter,T", [(torch.float32, 48, 40, 50),
                                             (torch.bfloat16, 128, 192, 160)])
@pytest.mark.parametrize("starved", [False, True])
def test_clipped_experts_match_per_example_oracle(dev, dtype, d, inter, T, starved):
    """Row-segmented experts; ``starved``: one gets no token at all, one none of an example."""
    E, B = 4, 3
    ref, model = _pair(lambda **kw: TopKMoE(d, inter, E, 2, **kw), dtype, dev, std=0.05, seed=10)
    g = torch.Generator().manual_seed(11)
    x = torch.randn(B, T, d, generator=g).to(dtype)
    logits = torch.randn(B, T, E, generator=g)
    if starved:
        logits[..., 3] = -50.0
        logits[0, :, 2] = -40.0
    t = torch.randn(B, T, d, generator=g).to(dtype)
    names = _names(model)
    C = expert_groups(model, clipping_norm=0.5)
    res = _oracle(ref, _sq, (x.double(), logits.double()), t.double(), C, names)
    fn, st = ghost_clipped_grad(model, _sq, clipping_norm=C, return_aux=True, dtype=torch.float32)
    (out, aux), _ = fn((x.to(dev), logits.to(dev)), t.to(dev), state=st)
    if starved:
        assert model.last_counts[3].sum() == 0 and model.last_counts[2][0] == 0
    for i, n in enumerate(names):
        if starved and "experts.3" in n:
            assert out.pytree[n].abs().max() == 0, n
        else:
            assert _rel(out.pytree[n], res.reduced[i]) < TOL[dtype], n
    for name in C.values:
        assert _rel(aux.group_norms[name], res.group_norms[name]) < TOL[dtype], name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_of_the_input_beside_an_expert_without_tokens(dev, dtype):
    """Widths at which the products' sums are cut in slices."""
    d, inter, E = 64, 1024, 4
    ref, model = _pair(lambda **kw: TopKMoE(d, inter, E, 2, **kw), dtype, dev, std=0.05, seed=16)
    g = torch.Generator().manual_seed(17)
    x = torch.randn(2, 9, d, generator=g).to(dtype)
    logits = torch.randn(2, 9, E, generator=g)
    logits[..., 3] = -50.0
    xr, xd = x.double().requires_grad_(), x.to(dev).requires_grad_()
    _sq(ref(xr, logits.double()), torch.zeros(2, 9, d)).sum().backward()
    _sq(model(xd, logits.to(dev)), torch.zeros(2, 9, d, device=dev)).sum().backward()
    assert model.last_counts[3].sum() == 0
    assert _rel(xd.grad, xr.grad) < TOL[dtype]
    for (n, p), (_, q) in zip(model.named_parameters(), ref.named_parameters()):
        if "experts.3" in n:
            assert not p.grad.any(), n
        elif p.requires_grad:
            assert _rel(p.grad, q.grad) < TOL[dtype], n


def test_clipped_routed_model_equals_the_default_one(dev):
    """The whole model, all three operators with the head's loss and the router's choice."""
    V, d = 61, 32
    torch.manual_seed(12)
    make = lambda fused: RoutedLM(V, d, 4, 48, 40, 8, 3,  # noqa: E731
                                  routing=dict(score="sigmoid", groups=4, top_groups=2),
                                  dtype=torch.float32, fused=fused).to(dev)
    model, fused = make(False), make(True)
    with torch.no_grad():
        for p in model.parameters():
            p.normal_(0.0, 0.25)
    fused.load_state_dict(model.state_dict())
    g = torch.Generator().manual_seed(13)
    ids = torch.randint(0, V, (3, 37), generator=g).to(dev)
    tgt = torch.randint(0, V, (3, 37), generator=g).to(dev)
    outs = []
    for m in (model, fused):
        fn, st = ghost_clipped_grad(m, m.loss, clipping_norm=0.3, return_aux=True)
        outs.append(fn(ids, tgt, state=st)[0])
    assert torch.equal(model.moe.last_counts, fused.moe.last_counts)
    (want, waux), (got, gaux) = outs
    for n in _names(model):
        assert _rel(got.pytree[n], want.pytree[n]) < 2 * TOL[torch.float32], n
    assert _rel(gaux.grad_norms, waux.grad_norms) < 2 * TOL[torch.float32]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_by_token_with_a_cache_equals_the_whole_sequence(dev, dtype):
    """Sequences of unequal lengths: the first tokens together, the rest one by one."""
    B, T, S, d, heads, ffn = 3, 70, 96, 128, 2, 192
    _, block = _pair(lambda **kw: LlamaBlock(d, heads, ffn, **kw), dtype, dev, std=0.1, seed=14)
    h = d // heads
    freqs, _ = rotary_frequencies(h, device=dev)
    x = torch.randn(B, T, d, generator=torch.Generator().manual_seed(15)).to(dtype).to(dev)
    first = [64, 1, 37]
    cache = torch.full((2, B, S, heads, h), float("nan"), dtype=dtype, device=dev)

    def step(x, positions, lengths, starts, into):
        b, t, _ = x.shape
        qkv = block.qkv(block.attn_norm(x)).view(b, t, 3, heads, h)
        q, k = rotary(qkv[:, :, 0], qkv[:, :, 1], freqs, positions=positions)
        into(k, qkv[:, :, 2])
        a = attention(q, cache[0, :b], cache[1, :b], lengths=lengths, starts=starts)
        x = x + block.o(a.view(b, t, d))
        return x + block.down(block.gate_up(block.mlp_norm(x)))

    with torch.no_grad():
        want = block(x)
        # The first tokens, padded to the longest; what the padding computes is not used.
        n = torch.tensor(first, device=dev)
        pos = torch.arange(64, device=dev).expand(B, 64).contiguous()

        def fill(k, v):
            for b, m in enumerate(first):
                cache[0, b, :m], cache[1, b, :m] = k[b, :m], v[b, :m]

        got = step(x[:, :64], pos, n, torch.zeros_like(n), fill)
        for b, m in enumerate(first):
            assert _rel(got[b, :m], want[b, :m]) < TOL[dtype], b
        rows = torch.arange(B, device=dev)
        for i in range(6):
            at = n + i

            def put(k, v):
                cache[0][rows, at], cache[1][rows, at] = k[:, 0], v[:, 0]

            got = step(x[rows, at][:, None], at[:, None], at + 1, at, put)
            assert _rel(got[:, 0], want[rows, at]) < TOL[dtype], i


def test_fused_modules_keep_parameters_and_refuse_the_cpu():
    kw = dict(dtype=torch.float32)
    for make in (lambda **o: BlockLM(7, 8, 2, 6, **o, **kw),
                 lambda **o: LoRABlock(8, 2, 1, 6, 2, **o, **kw),
                 lambda **o: RoutedLM(7, 8, 2, 6, 5, 3, **o, **kw)):
        a, b = make(), make(fused=True)
        assert {k: v.shape for k, v in a.state_dict().items()} == {
            k: v.shape for k, v in b.state_dict().items()}
    with pytest.raises(OpakeError):
        LlamaBlock(8, 2, 6, fused=True, **kw)(torch.zeros(1, 2, 8))


def test_widths_the_default_block_takes(dev):
    """Head widths of every kind that ``d / n_heads`` gives: even ones only."""
    for d, heads in ((24, 4), (20, 2), (264, 4)):
        ref, model = _pair(lambda **kw: LlamaBlock(d, heads, 24, **kw), torch.float32, dev)
        x = torch.randn(2, 9, d, generator=torch.Generator().manual_seed(d))
        assert _rel(model(x.to(dev)), ref(x.double())) < TOL[torch.float32]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 0, 64), (0, 5, 64)])
def test_blocks_of_no_tokens(dev, dtype, shape):
    """An empty batch or sequence, forward and backward, at widths whose sums are cut in slices."""
    kw = dict(fused=True, dtype=dtype, device=dev)
    for model in (LlamaBlock(64, 1, 1024, **kw), LoRABlock(64, 2, 1, 96, 4, **kw),
                  TopKMoE(64, 1024, 4, 2, **kw)):
        x = torch.zeros(shape, dtype=dtype, device=dev, requires_grad=True)
        y = model(x)
        y.sum().backward()
        assert y.shape == shape and x.grad.shape == shape
        assert not any(p.grad is not None and p.grad.any() for p in model.parameters())
