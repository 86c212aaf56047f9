"""The operators of a transformer block that a user of the package calls, as measurable cases.

``attn``   ``attention.attention``: softmax attention with shared key heads, causal, windowed
           and ragged, with the gradients of queries, keys and values
``rope``   ``rotary.rotary``: rotary positions of queries and keys, with their gradients
``gated``  ``gated.gated_linear``: both projections of a gated feed-forward layer, the
           activation and the product, with the gradients of the input and the weight

``listed()`` names twelve cases, ``draw(rng)`` gives more of the same ranges.  With
``own`` false ``run`` computes each operator in plain torch, in 32 bits (the angles of
rotary positions in 64); with ``own`` true it calls the package.  ``exact`` restates them
in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------


def _attn(name, B, T, S, H, KV, h, dtype="bf16", causal=True, window=0, ragged="", grad=False):
    """``window``: 0 for none.  ``ragged``: "" (all of it), "padded" (examples of different
    lengths in one batch, an empty one among them) or "cache" (the last T tokens of
    sequences of different lengths)."""
    return dict(name=name, kind="attn", B=B, T=T, S=S, H=H, KV=KV, h=h, dtype=dtype,
                causal=causal, window=window, ragged=ragged, grad=grad)


def _rope(name, B, T, H, KV, h, dims, dtype="bf16", interleaved=False, far=0, base=10000.0,
          amplitude=1.0, grad=False):
    """``far``: positions are given, and begin below that many; 0: they count from zero."""
    return dict(name=name, kind="rope", B=B, T=T, H=H, KV=KV, h=h, dims=dims, dtype=dtype,
                interleaved=interleaved, far=far, base=base, amplitude=amplitude, grad=grad)


def _gated(name, B, T, D, F, dtype="bf16", activation="silu", grad="both"):
    """``grad``: "none", "hidden" (a frozen weight) or "both"."""
    return dict(name=name, kind="gated", B=B, T=T, D=D, F=F, dtype=dtype, activation=activation,
                grad=grad)


def listed():
    return [
        # The smallest block's heads in float32, where launches and host time are all there is.
        _attn("attn_tiny", 4, 24, 24, 4, 4, 16, dtype="fp32", grad=True),
        # The Llama-style block's training step: d = 2048 in 16 heads, B = 16, T = 1024.
        _attn("attn_block", 16, 1024, 1024, 16, 16, 128, grad=True),
        # The LoRA block's: d = 4096 in 32 heads that share 8 key heads, B = 8, T = 2048.
        _attn("attn_lora", 8, 2048, 2048, 32, 8, 128, grad=True),
        # Evaluation of one long document.
        _attn("attn_long", 1, 16384, 16384, 16, 16, 128),
        # One decoding step of a batch of sequences of different lengths.
        _attn("attn_step", 16, 1, 8192, 32, 8, 128, ragged="cache"),
        # A padded batch in odd sizes, one example empty, each token sees 200 others.
        _attn("attn_odd", 9, 443, 443, 6, 2, 80, window=200, ragged="padded", grad=True),
        # The positions of one decoding step's tokens, far into their sequences.
        _rope("rope_step", 16, 1, 32, 8, 128, 128, far=120000, base=500000.0),
        # The Llama-style block's.
        _rope("rope_block", 16, 1024, 16, 16, 128, 128, grad=True),
        # Neighbouring pairs, half of each head, odd sizes, stretched for long contexts.
        _rope("rope_part", 5, 1999, 32, 8, 128, 64, interleaved=True, far=100000,
              amplitude=1.1, grad=True),
        # One decoding step: the LoRA block's feed-forward weights, read once.
        _gated("gated_step", 16, 1, 4096, 14336, grad="none"),
        # The Llama-style block's training step.
        _gated("gated_block", 16, 1024, 2048, 8192),
        # Odd sizes in float32, the weight frozen.
        _gated("gated_odd", 9, 197, 1000, 2731, dtype="fp32", activation="gelu", grad="hidden"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "rope", "gated"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    B = rng.randint(1, 32)
    if kind == "attn":
        while True:
            h = rng.choice([16, 32, 40, 64, 80, 96, 128, 192, 256])
            KV, rep = rng.randint(1, 8), rng.choice([1, 1, 2, 3, 4, 8])
            H = KV * rep
            step = rng.random() < 0.3
            T = rng.randint(1, 8) if step else _log(rng, 2, 4096)
            S = _log(rng, 16, 32768) if step else T + rng.choice([0, 0, 0, rng.randint(1, 500)])
            grad = not step and rng.random() < 0.7
            if (B * H * T * S * h * (6 if grad else 2) <= 3e11 and B * H * T * S <= 2 ** 30
                    and B * KV * S * h <= 2 ** 28 and S >= T):
                break
        causal = step or rng.random() < 0.85
        window = rng.randint(1, S) if causal and rng.random() < 0.3 else 0
        ragged = rng.choice(["", "cache"]) if step else "padded" if (
            causal and S == T and rng.random() < 0.4) else ""
        c = _attn("", B, T, S, H, KV, h, dtype, causal, window, ragged, grad)
    elif kind == "rope":
        T, KV, rep = _log(rng, 1, 4096), rng.randint(1, 16), rng.choice([1, 2, 4])
        h = rng.choice([16, 40, 64, 80, 96, 128, 192, 256])
        dims = rng.choice([h, h, h // 2, h // 4])
        while B * T * KV * (rep + 1) * h > 2 ** 27:
            T = max(1, T // 2)
        c = _rope("", B, T, KV * rep, KV, h, dims // 2 * 2, dtype, rng.random() < 0.4,
                  rng.choice([0, 0, 1000, 1000000]), rng.choice([10000.0, 500000.0]),
                  rng.choice([1.0, 1.1]), rng.random() < 0.6)
    else:
        while True:
            T = _log(rng, 1, 2048)
            D, F = _log(rng, 48, 4608), _log(rng, 48, 15000)
            if rng.random() < 0.6:
                D, F = max(64, D // 64 * 64), max(64, F // 64 * 64)
            if 12.0 * B * T * D * F <= 2e12 and B * T * F <= 2 ** 28:
                break
        c = _gated("", B, T, D, F, dtype, rng.choice(["silu", "silu", "gelu"]),
                   rng.choice(["none", "hidden", "both"]))
    del c["name"]
    return c


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _heads(c, g, T, H, KV, S=None):
    """Queries, keys and values as a fused projection leaves them: places of one tensor
    (keys and values of another length lie in one of their own)."""
    B, h, dt = c["B"], c["h"], DTYPES[c["dtype"]]
    if S is None or S == T:
        x = _randn(g, B, T, H + 2 * KV, h).to(dt)
        return x[:, :, :H], x[:, :, H:H + KV], x[:, :, H + KV:]
    x = _randn(g, B, S, 2 * KV, h).to(dt)
    return _randn(g, B, T, H, h).to(dt), x[:, :, :KV], x[:, :, KV:]


def _lengths(c, g):
    """Valid keys of each example, and the position of its first query."""
    B, T, S = c["B"], c["T"], c["S"]
    if not c["ragged"]:
        return None, None
    lo = 0 if c["ragged"] == "padded" else min(T, S)
    n = torch.randint(lo, S + 1, (B,), generator=g, device="cuda")
    n[0] = S
    if c["ragged"] == "padded":
        if B > 1:
            n[1] = 0
        return n, None
    return n, n - T


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] == "attn":
        q, k, v = _heads(c, g, c["T"], c["H"], c["KV"], c["S"])
        s = dict(zip("qkv", (t.detach().requires_grad_(c["grad"]) for t in (q, k, v))))
        s["lengths"], s["starts"] = _lengths(c, g)
        s["up"] = _randn(g, *q.shape).to(q.dtype) if c["grad"] else None
    elif c["kind"] == "rope":
        B, T, n = c["B"], c["T"], c["dims"]
        q, k, _ = _heads(c, g, T, c["H"], c["KV"])
        s = dict(zip("qk", (t.detach().requires_grad_(c["grad"]) for t in (q, k))))
        s["freqs"] = c["base"] ** (-torch.arange(0, n, 2, device="cuda", dtype=torch.float64) / n)
        s["positions"] = None
        if c["far"]:
            first = torch.randint(0, c["far"], (B, 1), generator=g, device="cuda")
            s["positions"] = first + torch.arange(T, device="cuda")
        if c["grad"]:
            s["up"] = tuple(_randn(g, *t.shape).to(t.dtype) for t in (q, k))
    else:
        B, T, D, F, dt = c["B"], c["T"], c["D"], c["F"], DTYPES[c["dtype"]]
        x = _randn(g, B, T, D)
        x = (x * x.square().mean(-1, keepdim=True).rsqrt()).to(dt)  # normed, as its layer's are
        w = (_randn(g, 2 * F, D) / math.sqrt(D)).to(dt)
        s = dict(x=x.requires_grad_(c["grad"] != "none"), w=w.requires_grad_(c["grad"] == "both"))
        s["up"] = _randn(g, B, T, F).to(dt) if c["grad"] != "none" else None
    s["case"] = dict(c)
    return s


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------


def _own_attn(c, s):
    from opake_amd import attention

    o = attention.attention(s["q"], s["k"], s["v"], causal=c["causal"],
                            window=c["window"] or None, lengths=s["lengths"], starts=s["starts"])
    out = {"out": o.detach()}
    if c["grad"]:
        grads = torch.autograd.grad(o, [s["q"], s["k"], s["v"]], s["up"])
        out.update(zip(("q_grad", "k_grad", "v_grad"), grads))
    return out


def _own_rope(c, s):
    from opake_amd import rotary

    q, k = rotary.rotary(s["q"], s["k"], s["freqs"], positions=s["positions"],
                         interleaved=c["interleaved"], amplitude=c["amplitude"])
    out = {"q": q.detach(), "k": k.detach()}
    if c["grad"]:
        grads = torch.autograd.grad([q, k], [s["q"], s["k"]], s["up"])
        out.update(zip(("q_grad", "k_grad"), grads))
    return out


def _own_gated(c, s):
    from opake_amd import gated

    y = gated.gated_linear(s["x"], s["w"], activation=c["activation"])
    out = {"out": y.detach()}
    if c["grad"] == "hidden":
        (out["x_grad"],) = torch.autograd.grad(y, [s["x"]], s["up"])
    elif c["grad"] == "both":
        out["x_grad"], out["weight_grad"] = torch.autograd.grad(y, [s["x"], s["w"]], s["up"])
    return out


def _visible(c, lengths, starts, device):
    """[B or 1, T, S]: the keys that a query sees."""
    T, S = c["T"], c["S"]
    j = torch.arange(S, device=device)
    n = torch.full((1, 1, 1), S, device=device) if lengths is None else lengths.view(-1, 1, 1)
    seen = (j < n).expand(-1, T, -1)
    if c["causal"]:
        first = torch.full((1, 1, 1), S - T, device=device) if starts is None else starts.view(
            -1, 1, 1)
        at = first + torch.arange(T, device=device).view(1, T, 1)
        seen = seen & (j <= at) & (at < n)
        if c["window"]:
            seen = seen & (j > at - c["window"])
    return seen


def _plain_attn(c, s):
    B, T, S, H, KV, h = (c[x] for x in ("B", "T", "S", "H", "KV", "h"))
    rep, scale = H // KV, 1.0 / math.sqrt(h)
    seen = _visible(c, s["lengths"], s["starts"], s["q"].device)

    def rows(t, n):  # [B, KV, n * T or S, h], query heads that share a key head after another
        t = t.detach().float()
        return t.view(B, -1, KV, n, h).permute(0, 2, 3, 1, 4).reshape(B, KV, -1, h)

    q, k, v = rows(s["q"], rep), rows(s["k"], 1), rows(s["v"], 1)
    up = rows(s["up"], rep) if c["grad"] else None
    o, dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.empty_like(k), \
        torch.empty_like(v)
    per = max(1, 2 ** 29 // (rep * T * S))  # key heads at a time
    for b in range(B):
        see = seen[b if seen.shape[0] > 1 else 0].repeat(rep, 1)
        for a in range(0, KV, per):
            at = (b, slice(a, a + per))
            z = (q[at] @ k[at].transpose(1, 2)) * scale
            z = torch.where(see, z, -math.inf)
            m = z.amax(-1, keepdim=True)
            e = torch.exp(z - torch.where(m > -math.inf, m, 0.0))
            total = e.sum(-1, keepdim=True)
            p = e / torch.where(total > 0, total, 1.0)
            o[at] = p @ v[at]
            if c["grad"]:
                dv[at] = p.transpose(1, 2) @ up[at]
                dp = up[at] @ v[at].transpose(1, 2)
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                dq[at] = ds @ k[at]
                dk[at] = ds.transpose(1, 2) @ q[at]

    def back(t, like, n):
        t = t.view(B, KV, n, -1, h).permute(0, 3, 1, 2, 4).reshape(like.shape)
        return t.to(like.dtype)

    out = {"out": back(o, s["q"], rep)}
    if c["grad"]:
        out.update(q_grad=back(dq, s["q"], rep), k_grad=back(dk, s["k"], 1),
                   v_grad=back(dv, s["v"], 1))
    return out


def _plain_rope(c, s):
    n = c["dims"]
    at = s["positions"]
    if at is None:
        at = torch.arange(c["T"], device="cuda").view(1, -1)
    turn = at.double().unsqueeze(-1) * s["freqs"]
    cos = (torch.cos(turn) * c["amplitude"]).float().unsqueeze(2)
    sin = (torch.sin(turn) * c["amplitude"]).float().unsqueeze(2)

    def rotate(x, sin):
        y = x.detach().float().clone()
        if c["interleaved"]:
            a, b = y[..., 0:n:2].clone(), y[..., 1:n:2].clone()
            y[..., 0:n:2], y[..., 1:n:2] = a * cos - b * sin, a * sin + b * cos
        else:
            a, b = y[..., :n // 2].clone(), y[..., n // 2:n].clone()
            y[..., :n // 2], y[..., n // 2:n] = a * cos - b * sin, a * sin + b * cos
        return y.to(x.dtype)

    out = {"q": rotate(s["q"], sin), "k": rotate(s["k"], sin)}
    if c["grad"]:
        out["q_grad"], out["k_grad"] = (rotate(t, -sin) for t in s["up"])
    return out


def _plain_gated(c, s):
    D, F = c["D"], c["F"]
    x, w = s["x"].detach().float().view(-1, D), s["w"].detach().float()
    z = x @ w.t()
    g, u = z[:, :F], z[:, F:]
    if c["activation"] == "silu":
        gate = 1.0 / (1.0 + torch.exp(-g))
        slope = gate * (1.0 + g * (1.0 - gate))
    else:
        gate = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        slope = gate + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    act = g * gate
    out = {"out": (act * u).to(s["x"].dtype).view(*s["x"].shape[:-1], F)}
    if c["grad"] != "none":
        up = s["up"].float().view(-1, F)
        dz = torch.cat([up * u * slope, up * act], 1)
        out["x_grad"] = (dz @ w).to(s["x"].dtype).view(s["x"].shape)
        if c["grad"] == "both":
            out["weight_grad"] = (dz.t() @ x).to(s["w"].dtype)
    return out


def run(state):
    c = state["case"]
    f = {"attn": (_plain_attn, _own_attn), "rope": (_plain_rope, _own_rope),
         "gated": (_plain_gated, _own_gated)}[c["kind"]]
    return f[bool(own)](c, state)


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------


def _pairs(c):
    """Visible (query, key) pairs of a head and the keys read, over the batch: of ragged
    batches for the mean length."""
    B, T, S = c["B"], c["T"], c["S"]
    n, t = float(S), float(T)
    if c["ragged"] == "padded":
        n = t = max(1.0, S / 2)
    elif c["ragged"] == "cache":
        n = (T + S) / 2
    if not c["causal"]:
        return B * t * n, B * n
    w = min(n, c["window"] or n)
    # Query i of t sees min(n - t + i + 1, w) keys.
    first = n - t + 1
    rising = min(t, max(0.0, w - first))
    pairs = rising * (first + first + rising) / 2 + (t - rising) * w
    return B * pairs, B * min(n, w + t)


def work(case):
    c, b = case, BYTES[case["dtype"]]
    if c["kind"] == "attn":
        pairs, keys = _pairs(c)
        q, kv = c["B"] * c["T"] * c["H"] * c["h"], 2 * keys * c["KV"] * c["h"]
        moved = (2 * q + kv) * b
        flops = 4.0 * pairs * c["H"] * c["h"]
        if c["grad"]:  # the output's gradient in, three gradients out; four products
            moved += (2 * q + kv) * b
            flops *= 3
        return {"bytes": moved, "flops": flops}
    if c["kind"] == "rope":
        n = c["B"] * c["T"] * (c["H"] + c["KV"])
        passes = 2 if c["grad"] else 1
        return {"bytes": passes * 2 * n * c["h"] * b, "flops": passes * 3 * n * c["dims"]}
    N, D, F = c["B"] * c["T"], c["D"], c["F"]
    products = {"none": 1, "hidden": 2, "both": 3}[c["grad"]]
    moved = (N * D + 2 * F * D + N * F) * b
    if c["grad"] != "none":
        moved += (N * F + N * D) * b
    if c["grad"] == "both":
        moved += 2 * F * D * b
    return {"bytes": moved, "flops": 4.0 * N * D * F * products}


# --------------------------------------------------------------------------
# The definitions in 64 bits
# --------------------------------------------------------------------------


def _exact_attn(c, s):
    """Head by head: softmax over the visible keys, gradients by automatic differentiation."""
    H, KV, T, S, h = c["H"], c["KV"], c["T"], c["S"], c["h"]
    out = {"out": torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")}
    if c["grad"]:
        for x in "qkv":
            out[x + "_grad"] = torch.zeros(s[x].shape, dtype=torch.float64, device="cuda")
    t, j = torch.arange(T, device="cuda")[:, None], torch.arange(S, device="cuda")[None, :]
    lengths = [S] * c["B"] if s["lengths"] is None else s["lengths"].tolist()
    starts = [S - T] * c["B"] if s["starts"] is None else s["starts"].tolist()
    rows = T if c["grad"] else max(1, 2 ** 27 // S)
    for b in range(c["B"]):
        hidden = (j >= lengths[b]).expand(T, S).clone()
        if c["causal"]:
            at = t + starts[b]
            hidden |= (j > at) | (at >= lengths[b])
            if c["window"]:
                hidden |= at - j >= c["window"]
        alone = hidden.all(1, keepdim=True)  # a row that sees nothing
        bias = torch.zeros(T, S, dtype=torch.float64, device="cuda")
        bias.masked_fill_(hidden & ~alone, -math.inf)
        for i in range(H):
            g = i * KV // H
            q, k, v = (s[x][b, :, n].detach().double().requires_grad_(c["grad"])
                       for x, n in (("q", i), ("k", g), ("v", g)))
            for r in range(0, T, rows):
                e = min(T, r + rows)
                p = torch.softmax(torch.matmul(q[r:e], k.T) * h ** -0.5 + bias[r:e], -1)
                o = torch.matmul(p, v).masked_fill(alone[r:e], 0.0)
                out["out"][b, r:e, i] = o.detach()
                if c["grad"]:
                    grads = torch.autograd.grad(o, [q, k, v], s["up"][b, :, i].double())
                    for x, n, d in zip("qkv", (i, g, g), grads):
                        out[x + "_grad"][b, :, n] += d
    return out


def _exact_rope(c, s):
    """Pairs as complex numbers."""
    n = c["dims"]
    at = s["positions"]
    if at is None:
        at = torch.arange(c["T"], device="cuda")[None, :]
    turn = torch.polar(torch.full_like(s["freqs"], c["amplitude"]).expand(*at.shape, -1),
                       at[..., None] * s["freqs"])[:, :, None, :]

    def rotate(x, turn):
        y = x.detach().double()
        head, rest = y[..., :n], y[..., n:]
        shape = (*head.shape[:-1], n // 2, 2)
        two = head.reshape(shape) if c["interleaved"] else head.unflatten(-1, (2, n // 2)).mT
        z = torch.view_as_real(torch.view_as_complex(two.contiguous()) * turn)
        z = z.flatten(-2) if c["interleaved"] else z.mT.flatten(-2)
        return torch.cat([z, rest], -1)

    out = {"q": rotate(s["q"], turn), "k": rotate(s["k"], turn)}
    if c["grad"]:
        out["q_grad"], out["k_grad"] = (rotate(x, turn.conj()) for x in s["up"])
    return out


def _exact_gated(c, s):
    F, want = c["F"], c["grad"]
    x = s["x"].detach().double().requires_grad_(want != "none")
    w = s["w"].detach().double().requires_grad_(want == "both")
    act = torch.nn.functional.silu if c["activation"] == "silu" else torch.nn.functional.gelu
    y = act(torch.matmul(x, w[:F].T)) * torch.matmul(x, w[F:].T)
    out = {"out": y.detach()}
    if want == "hidden":
        (out["x_grad"],) = torch.autograd.grad(y, [x], s["up"].double())
    elif want == "both":
        out["x_grad"], out["weight_grad"] = torch.autograd.grad(y, [x, w], s["up"].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "rope": _exact_rope, "gated": _exact_gated}[case["kind"]](case, s)
