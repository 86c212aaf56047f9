"""The language-model operators that a user of the package calls, as measurable cases.

``ce``       ``head.linear_cross_entropy``: the loss of a vocabulary head from the hidden
             states and the head's weight, with its gradients
``distill``  ``head.topk_distillation``: the same head against a teacher's top logits
``route``    ``routing.route_topk``: experts and weights of every token from router logits,
             with the gradient of the logits

``listed()`` names twelve cases, ``draw(rng)`` gives more of the same ranges.  With
``own`` false ``run`` computes each operator in plain torch, in 32 bits; with ``own`` true
it calls the package.  ``exact`` restates them in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}
IGNORE = -100


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------


def _ce(name, B, T, D, V, dtype="bf16", grad="both", ignored=0.0):
    """``grad``: "none" (the loss alone), "hidden" (a frozen head) or "both"."""
    return dict(name=name, kind="ce", B=B, T=T, D=D, V=V, dtype=dtype, grad=grad, ignored=ignored)


def _distill(name, B, T, D, V, K, tau, dtype="bf16", grad="hidden", short=False):
    """``short``: rows with fewer than K teacher entries, a few of them with none."""
    return dict(name=name, kind="distill", B=B, T=T, D=D, V=V, K=K, tau=tau, dtype=dtype,
                grad=grad, short=short)


def _route(name, B, T, E, k, score="softmax", dtype="fp32", bias=False, groups=1, top_groups=1,
           renormalize=True, scale=1.0, masked=False, grad=True):
    return dict(name=name, kind="route", B=B, T=T, E=E, k=k, score=score, dtype=dtype, bias=bias,
                groups=groups, top_groups=top_groups, renormalize=renormalize, scale=scale,
                masked=masked, grad=grad)


def listed():
    return [
        # The smallest head: a byte vocabulary on a short batch, where launches and host
        # time are all there is.
        _ce("ce_tiny", 4, 24, 64, 256),
        # The Llama-style block's step: B = 16, T = 1024, d = 2048, vocabulary 32000, the head
        # frozen.
        _ce("ce_block", 16, 1024, 2048, 32000, grad="hidden"),
        # Evaluation of a wide model over a large vocabulary: the loss alone.
        _ce("ce_eval", 2, 1024, 4096, 131072, grad="none"),
        # A trained head with odd sizes, prompts ignored.
        _ce("ce_odd_head", 9, 443, 1000, 50001, ignored=0.3),
        # Training in float32, head included.
        _ce("ce_fp32", 16, 128, 768, 8001, dtype="fp32"),
        # The smallest distillation: a short float32 batch.
        _distill("distill_tiny", 4, 24, 64, 256, 8, 1.0, dtype="fp32"),
        # The block distilled from a teacher's 64 stored logits a token, the head frozen.
        _distill("distill_block", 8, 1024, 2048, 32000, 64, 2.0),
        # A trained head, odd sizes, top-p storage: rows of different lengths, some empty.
        _distill("distill_odd", 5, 197, 1000, 32001, 50, 1.5, grad="both", short=True),
        # The router of the top-2 MoE FFN: 8 experts, B = 16, T = 1024.
        _route("route_top2", 16, 1024, 8, 2, dtype="bf16"),
        # One decoding step of a batch: single tokens, many experts.
        _route("route_step", 16, 1, 256, 8, score="sigmoid", bias=True, groups=8, top_groups=4,
               scale=2.5, grad=False),
        # Training with many experts in groups, a balancing bias.
        _route("route_groups", 16, 4096, 256, 8, score="sigmoid", bias=True, groups=8,
               top_groups=4, scale=2.5),
        # Odd sizes, experts masked out, tokens with none left; the softmax's own weights.
        _route("route_masked", 9, 1109, 60, 4, renormalize=False, masked=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["ce", "ce", "distill", "route"])
    if kind == "route":
        E = rng.choice([4, 8, 16, 33, 60, 64, 128, 160, 256, 384])
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if E % g == 0 and E // g >= 2])
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(8, top_groups * (E // groups)))
        B, T = rng.randint(1, 32), _log(rng, 1, 2048)
        c = _route("", B, T, E, k, score=rng.choice(["softmax", "sigmoid"]),
                   dtype=rng.choice(["bf16", "fp32"]), bias=rng.random() < 0.5, groups=groups,
                   top_groups=top_groups, renormalize=rng.random() < 0.6,
                   scale=rng.choice([1.0, 2.5]), masked=rng.random() < 0.3,
                   grad=rng.random() < 0.7)
    else:
        while True:
            B, T = rng.randint(1, 32), _log(rng, 1, 2048)
            D, V = _log(rng, 48, 4608), _log(rng, 200, 140000)
            if rng.random() < 0.6:
                D = max(64, D // 64 * 64)
            if 2 * B * T * D * V <= 5e11 and B * T * V <= 4e8:
                break
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        grad = rng.choice(["none", "hidden", "both"])
        if kind == "ce":
            c = _ce("", B, T, D, V, dtype, grad, rng.choice([0.0, 0.2, 0.7]))
        else:
            c = _distill("", B, T, D, V, _log(rng, 1, 128), rng.choice([1.0, 1.5, 4.0]), dtype,
                         grad, rng.random() < 0.5)
    del c["name"]
    return c


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _head_inputs(c, g, likely):
    """Normed hidden states, a head that gives logits of a trained model's spread (standard
    deviation 2.5), and the weight that each token's loss has in the step's loss: one over
    its example's tokens.  Half of the tokens lean towards the head's row of what they are to
    answer (``likely``), as after some training; the others are surprises."""
    B, T, D, V, dt = c["B"], c["T"], c["D"], c["V"], DTYPES[c["dtype"]]
    h = torch.randn(B, T, D, generator=g, device="cuda")
    h = h * h.square().mean(-1, keepdim=True).rsqrt()
    W = (torch.randn(V, D, generator=g, device="cuda") * (2.5 / math.sqrt(D))).to(dt)
    lean = 2.0 * (torch.rand(B, T, 1, generator=g, device="cuda") < 0.5)
    h = (h + lean * W[likely]).to(dt)
    up = torch.full((B, T), 1.0 / T, device="cuda")
    h.requires_grad_(c["grad"] != "none")
    W.requires_grad_(c["grad"] == "both")
    return dict(h=h, W=W, up=up)


def _route_keys(c, z, bias):
    """What the choice compares, in 64 bits: the logits themselves where that is the same order
    as the scores', else scores plus bias."""
    z = z.double()
    if c["score"] == "softmax" and bias is None:
        return z
    m = z.amax(-1, keepdim=True)
    s = torch.sigmoid(z) if c["score"] == "sigmoid" else torch.exp(z - m) / torch.exp(
        z - m).sum(-1, keepdim=True)
    s = torch.where(z == -math.inf, -math.inf, s)
    return s if bias is None else s + bias.double()


def _route_settled(c, z, bias):
    """Rows whose choice no rounding to 32 bits can change: among the keys that the choice
    goes through, every gap between neighbours is exactly zero (equal logits, no bias: a tie
    that goes to the lower index) or wide enough."""
    N, G = c["B"] * c["T"], c["groups"]
    keys = _route_keys(c, z, bias).view(N, -1)
    if c["score"] == "softmax" and bias is None:
        return torch.ones(N, dtype=torch.bool, device=z.device)

    def wide(v, first, last):
        v = v.sort(dim=-1, descending=True).values[:, first:last + 1]
        gap = torch.where(v[:, 1:] == -math.inf, math.inf, v[:, :-1] - v[:, 1:])
        tied = (gap == 0) if bias is None else torch.zeros_like(gap, dtype=torch.bool)
        return (tied | (gap > 4e-6)).all(-1)

    ok = torch.ones(N, dtype=torch.bool, device=z.device)
    if G > 1:
        best = keys.view(N, G, -1).amax(-1)
        ok &= wide(best, c["top_groups"] - 1, c["top_groups"])
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        keys = torch.where(open_.repeat_interleave(c["E"] // G, 1), keys, -math.inf)
    return ok & wide(keys, 0, c["k"])


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] == "ce":
        t = torch.randint(0, c["V"], (c["B"], c["T"]), generator=g, device="cuda")
        s = _head_inputs(c, g, t)
        drop = torch.rand(c["B"], c["T"], generator=g, device="cuda") < c["ignored"]
        s["t"] = torch.where(drop, IGNORE, t)
    elif c["kind"] == "distill":
        B, T, V, K = c["B"], c["T"], c["V"], c["K"]
        # A teacher's K largest logits, descending, at distinct places of the vocabulary.
        step = torch.randint(1, max(2, V // K), (B, T, K), generator=g, device="cuda")
        ti = (step.cumsum(-1) + torch.randint(0, V, (B, T, 1), generator=g, device="cuda")) % V
        s = _head_inputs(c, g, ti[..., 0])
        fall = torch.rand(B, T, K, generator=g, device="cuda") * (8.0 / K)
        s["tl"] = 12.0 - fall.cumsum(-1)
        if c["short"]:
            n = torch.randint(0, K + 1, (B, T, 1), generator=g, device="cuda")
            ti = torch.where(torch.arange(K, device="cuda") < n, ti, -1)
        s["ti"] = ti
    else:
        B, T, E = c["B"], c["T"], c["E"]
        s = {}
        bias = None
        if c["bias"]:
            # What a balancing rule has added up in steps of a thousandth.
            bias = torch.randint(-60, 61, (E,), generator=g, device="cuda").float() * 1e-3
        mask = None
        if c["masked"]:
            mask = torch.rand(B, T, E, generator=g, device="cuda") < 0.3
            mask |= torch.rand(B, T, 1, generator=g, device="cuda") < 0.01
        z = None
        for _ in range(4):  # the few rows whose choice hangs on the last bits are drawn again
            new = (torch.randn(B, T, E, generator=g, device="cuda") * 1.5).to(DTYPES[c["dtype"]])
            if mask is not None:
                new = new.masked_fill(mask, -math.inf)
            z = new if z is None else torch.where(
                _route_settled(c, z, bias).view(B, T, 1), z, new)
        ok = _route_settled(c, z, bias).view(B * T)
        # Any that are left repeat their nearest settled row.
        at = torch.arange(B * T, device="cuda")
        near = torch.where(ok, at, 0).cummax(0).values
        z = z.view(B * T, E)[near].view(B, T, E).contiguous()
        s["z"] = z.requires_grad_(c["grad"])
        s["bias"] = bias
        s["up"] = torch.randn(B, T, c["k"], generator=g, device="cuda")
    s["case"] = dict(c)
    return s


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------


def _named(loss, dh, dW):
    out = {"loss": loss}
    if dh is not None:
        out["hidden_grad"] = dh
    if dW is not None:
        out["weight_grad"] = dW
    return out


def _own_head(c, s):
    from opake_amd import head

    if c["kind"] == "ce":
        loss = head.linear_cross_entropy(s["h"], s["W"], s["t"], ignore_index=IGNORE)
    else:
        loss = head.topk_distillation(s["h"], s["W"], s["tl"], s["ti"], temperature=c["tau"])
    dh = dW = None
    if c["grad"] == "hidden":
        (dh,) = torch.autograd.grad(loss, [s["h"]], s["up"])
    elif c["grad"] == "both":
        dh, dW = torch.autograd.grad(loss, [s["h"], s["W"]], s["up"])
    return _named(loss.detach(), dh, dW)


def _own_route(c, s):
    from opake_amd import routing

    w, i = routing.route_topk(s["z"], c["k"], score=c["score"], bias=s["bias"],
                              groups=c["groups"], top_groups=c["top_groups"],
                              renormalize=c["renormalize"], scale=c["scale"])
    out = {"weights": w.detach(), "experts": i}
    if c["grad"]:
        (out["logits_grad"],) = torch.autograd.grad(w, [s["z"]], s["up"])
    return out


def _plain_head(c, s):
    D, V = c["D"], c["V"]
    h = s["h"].detach().float().view(-1, D)
    W = s["W"].detach().float()
    up = s["up"].view(-1, 1)
    N = h.shape[0]
    inv_tau = 1.0 if c["kind"] == "ce" else 1.0 / c["tau"]
    z = h @ W.t()
    if inv_tau != 1.0:
        z = z * inv_tau
    m = z.amax(1, keepdim=True)
    p = torch.exp(z - m)
    total = p.sum(1, keepdim=True)
    lse = m + torch.log(total)
    if c["kind"] == "ce":
        t = s["t"].view(-1, 1)
        used = t != IGNORE
        at = torch.where(used, t, 0)
        q = used.float()
        loss = torch.where(used, lse - z.gather(1, at), 0.0)
        coef = 1.0
    else:
        ti, tl = s["ti"].view(N, -1), s["tl"].view(N, -1) * inv_tau
        there = ti >= 0
        at = torch.where(there, ti, 0)
        tl = torch.where(there, tl, -math.inf)
        tm = tl.amax(1, keepdim=True)
        used = tm > -math.inf
        e = torch.where(there, torch.exp(tl - torch.where(used, tm, 0.0)), 0.0)
        es = torch.where(used, e.sum(1, keepdim=True), 1.0)
        q = e / es
        logq = torch.where(there, tl - tm - torch.log(es), 0.0)
        loss = (q * (logq - z.gather(1, at) + lse)).sum(1, keepdim=True)
        loss = torch.where(used, loss, 0.0) * c["tau"] ** 2
        coef = c["tau"]
    dh = dW = None
    if c["grad"] != "none":
        p = p / total
        p = p * used.float()
        p.scatter_add_(1, at, -q)
        p = p * (up * coef)
        dh = (p @ W).to(s["h"].dtype).view(s["h"].shape)
        if c["grad"] == "both":
            dW = (p.t() @ h).to(s["W"].dtype)
    return _named(loss.view(s["up"].shape), dh, dW)


def _plain_route(c, s):
    k, G = c["k"], c["groups"]
    raw = s["z"].detach()
    z = raw.float().view(-1, c["E"])
    N, E = z.shape
    open_ = z > -math.inf
    m = z.amax(1, keepdim=True)
    m = torch.where(m > -math.inf, m, 0.0)
    if c["score"] == "softmax":
        e = torch.exp(z - m)
        tot = e.sum(1, keepdim=True)
        sc = e / torch.where(tot > 0, tot, 1.0)
    else:
        sc = 1.0 / (1.0 + torch.exp(-z))
    if s["bias"] is not None:
        key = sc + s["bias"]
    else:
        key = z if c["score"] == "softmax" else sc
    key = torch.where(open_, key, -math.inf)
    if G > 1:
        best = key.view(N, G, -1).amax(2)
        order = best.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        kept = torch.zeros(N, G, dtype=torch.bool, device=z.device).scatter_(1, order, True)
        key = torch.where(kept.repeat_interleave(E // G, 1), key, -math.inf)
    val, idx = key.sort(dim=1, descending=True, stable=True)
    there = val[:, :k] > -math.inf
    at = idx[:, :k]
    cs = torch.where(there, sc.gather(1, at), 0.0)
    if c["renormalize"]:
        tot = cs.sum(1, keepdim=True)
        w = cs / torch.where(tot > 0, tot, 1.0)
    else:
        w = cs
    out = {"weights": (w * c["scale"]).view(s["up"].shape),
           "experts": torch.where(there, at, -1).view(s["up"].shape)}
    if c["grad"]:
        gw = torch.where(there, s["up"].view(N, k), 0.0) * c["scale"]
        if c["renormalize"]:
            tot = torch.where(tot > 0, tot, 1.0)
            gs = (gw - (gw * w).sum(1, keepdim=True)) / tot
        else:
            gs = gw
        full = torch.zeros_like(z).scatter_add_(1, at, torch.where(there, gs, 0.0))
        if c["score"] == "softmax":
            dz = sc * (full - (full * sc).sum(1, keepdim=True))
        else:
            dz = full * sc * (1.0 - sc)
        out["logits_grad"] = dz.to(raw.dtype).view(raw.shape)
    return out


def run(state):
    c = state["case"]
    if c["kind"] == "route":
        return _own_route(c, state) if own else _plain_route(c, state)
    return _own_head(c, state) if own else _plain_head(c, state)


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------


def work(case):
    c = case
    N = c["B"] * c["T"]
    if c["kind"] == "route":
        n, b = N * c["E"], BYTES[c["dtype"]]
        moved = n * b + N * c["k"] * 12
        flops = 6 * n
        if c["grad"]:
            moved += n * b + N * c["k"] * 4
            flops += 6 * n
        return {"bytes": moved, "flops": flops}
    b, D, V = BYTES[c["dtype"]], c["D"], c["V"]
    products = {"none": 1, "hidden": 2, "both": 3}[c["grad"]]
    moved = (N * D + V * D) * b + 4 * N
    moved += 8 * N if c["kind"] == "ce" else 12 * N * c["K"]
    if c["grad"] != "none":
        moved += N * D * b + 4 * N
    if c["grad"] == "both":
        moved += V * D * b
    return {"bytes": moved, "flops": 2.0 * N * D * V * products}


# --------------------------------------------------------------------------
# The definitions in 64 bits
# --------------------------------------------------------------------------


def _exact_head(c, s):
    """Rows in slices: log softmax in float64, the target as a dense distribution q, then
    the gradient (sum(q) softmax - q) of every row's loss."""
    V, tau = c["V"], c.get("tau", 1.0)
    W = s["W"].detach().double()
    h = s["h"].detach().double().flatten(0, 1)
    up = s["up"].double().flatten()
    N = h.shape[0]
    loss = torch.empty(N, dtype=torch.float64, device=h.device)
    dh = torch.empty_like(h) if c["grad"] != "none" else None
    dW = torch.zeros_like(W) if c["grad"] == "both" else None
    rows = max(1, int(2e8 // V))
    for a in range(0, N, rows):
        b = min(N, a + rows)
        logp = torch.log_softmax(torch.matmul(h[a:b], W.T) / tau, -1)
        q = torch.zeros_like(logp)
        if c["kind"] == "ce":
            t = s["t"].flatten()[a:b]
            r = torch.nonzero(t != IGNORE).flatten()
            q[r, t[r]] = 1.0
            loss[a:b] = -(q * logp).sum(-1)
        else:
            ti, tl = s["ti"].flatten(0, 1)[a:b], s["tl"].flatten(0, 1)[a:b].double() / tau
            some = (ti >= 0).any(-1, keepdim=True)
            tq = torch.softmax(torch.where(ti >= 0, tl, -math.inf), -1)
            tq = torch.where(some, tq, 0.0)
            ent = torch.special.xlogy(tq, tq).sum(-1)
            for i in range(c["K"]):
                r = torch.nonzero(ti[:, i] >= 0).flatten()
                q[r, ti[r, i]] += tq[r, i]
            loss[a:b] = tau * tau * (ent - (q * logp).sum(-1))
        if dh is not None:
            d = (logp.exp() * q.sum(-1, keepdim=True) - q) * (tau * up[a:b, None])
            dh[a:b] = torch.matmul(d, W)
            if dW is not None:
                dW += torch.matmul(d.T, h[a:b])
    shape = s["h"].shape
    return _named(loss.view(shape[:2]), None if dh is None else dh.view(shape), dW)


def _exact_route(c, s):
    z0 = s["z"].detach().double().flatten(0, 1)
    z = z0.clone().requires_grad_(True)
    N, E = z.shape
    G, k = c["groups"], c["k"]
    closed = z0 == -math.inf
    none = closed.all(1, keepdim=True)
    if c["score"] == "softmax":
        sc = torch.softmax(torch.where(none, 0.0, z), -1)
        sc = torch.where(none | closed, 0.0, sc)
    else:
        sc = torch.sigmoid(z)
    key = _route_keys(c, z0, s["bias"])
    key = torch.where(closed, -math.inf, key)
    left = torch.ones(N, E, dtype=torch.bool, device=z.device)
    place = torch.arange(E, device=z.device)

    def first_largest(v):
        top = v.amax(1, keepdim=True)
        n = v.shape[1]
        return torch.where(v == top, place[:n], n).amin(1), top.squeeze(1) > -math.inf

    if G > 1:
        best = key.view(N, G, E // G).amax(2)
        left[:] = False
        for _ in range(c["top_groups"]):
            at, _there = first_largest(best)
            at = torch.clamp(at, max=G - 1)
            left.view(N, G, E // G)[torch.arange(N, device=z.device), at] = True
            best = best.scatter(1, at[:, None], -math.inf)
    key = torch.where(left, key, -math.inf)
    picks, weights = [], []
    for _ in range(k):
        at, there = first_largest(key)
        at = torch.clamp(at, max=E - 1)
        picks.append(torch.where(there, at, -1))
        weights.append(torch.where(there, sc.gather(1, at[:, None]).squeeze(1), 0.0))
        key = key.scatter(1, at[:, None], -math.inf)
    w = torch.stack(weights, 1)
    if c["renormalize"]:
        tot = w.sum(1, keepdim=True)
        w = w / torch.where(tot > 0, tot, 1.0)
    w = w * c["scale"]
    shape = s["up"].shape
    out = {"weights": w.detach().view(shape), "experts": torch.stack(picks, 1).view(shape)}
    if c["grad"]:
        (dz,) = torch.autograd.grad(w, [z], s["up"].double().flatten(0, 1))
        out["logits_grad"] = torch.where(closed, 0.0, dz).view(s["z"].shape)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_route(case, s) if case["kind"] == "route" else _exact_head(case, s)
