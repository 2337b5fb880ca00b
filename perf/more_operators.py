"""The workloads by which the operators of a mixture of experts are followed: routing tokens to experts, and the experts' products.

Each case is a dict of plain values.  `prepare` makes what a program holds before the call, `run` is one pass through an operator - in its
plain form, elementary torch operations in 32 bits, or with `own` through the framework's entry points - `exact` the same outputs in 64 bits
from the definition, `work` the bytes and operations one pass cannot do without.

Kinds:
  route    logits z [N, E] -> the k experts of each token, best first, with their weights; with `grad` also the mean probabilities and the logits' gradient
  mlp      tokens x [N, C] through the experts chosen for them: out_n = sum_j w_nj Wd[e] (silu(g) * u), [g | u] = Wgu[e] x_n, e = idx_nj; with `grad` all gradients

Routing.  A logit of NaN counts as -inf, an expert at -inf is not there.  Scores s: softmax over the experts, or a sigmoid each.  Experts are chosen by z, or, with a bias or
groups, by s + b in 64 bits; equal ones by the lowest index.  Of `groups` equal groups the `top` best stay, by the sum of their two best s + b.  Weights are
scale * s, with `renorm` divided by the sum over the chosen.  Too few experts: index -1, weight 0.  Mean probabilities: softmax, or s / sum of s, over all tokens.
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
NEG = float("-inf")
TYPES = {"bf16": BF16, "f32": F32}


# ------------------------------------------------------------------ the cases
def listed():
    route = dict(kind="route", score="softmax", bias=False, groups=1, top=1, renorm=True, scale=1.0, dtype="bf16", grad=False, pad=0)
    mlp = dict(kind="mlp", gates="f32", grad=False, skew=0.5, drop=0)
    return [
        # a decoding step of 16 sequences: latency
        dict(route, name="route_step", N=16, E=64, k=6, renorm=False),
        # prompts: many experts in groups, chosen by sigmoids with a bias that balances them
        dict(route, name="route_groups", N=8192, E=256, k=8, score="sigmoid", bias=True, groups=8, top=4, scale=2.5, dtype="f32"),
        # a training step of the 12-layer / 768-wide decoder with eight experts a layer
        dict(route, name="route_train", N=16384, E=8, k=2, grad=True),
        # a training step with an odd number of tokens, some of them padding, and of experts
        dict(route, name="route_odd", N=5001, E=60, k=4, renorm=False, dtype="f32", grad=True, pad=100),
        # one token of one sequence through 6 of 64 small experts of a 2048-wide decoder
        dict(mlp, name="mlp_one", N=1, E=64, k=6, C=2048, I=1376),
        # a decoding step of 16 sequences, one of them not in use, through 2 of 8 large experts
        dict(mlp, name="mlp_step", N=16, E=8, k=2, C=2048, I=5504, drop=1),
        # a short prompt: fewer tokens than fill a tile, for most experts
        dict(mlp, name="mlp_short", N=301, E=64, k=6, C=2048, I=1376, gates="bf16"),
        # prompts of eight windows through the 768-wide decoder's experts
        dict(mlp, name="mlp_prompts", N=8192, E=8, k=2, C=768, I=2048),
        # a training step of the 12-layer / 768-wide decoder with eight experts a layer, one layer of it
        dict(mlp, name="mlp_train", N=16384, E=8, k=2, C=768, I=2048, gates="bf16", grad=True),
        # many small experts, some of them much more in demand than others
        dict(mlp, name="mlp_train_many", N=4096, E=64, k=6, C=2048, I=1376, gates="bf16", grad=True, skew=1.0),
        # odd sizes, tokens that go nowhere, and so few tokens for some experts that a tile is mostly empty
        dict(mlp, name="mlp_train_odd", N=1003, E=20, k=3, C=336, I=208, gates="bf16", grad=True, skew=1.0, drop=37),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.45:
        groups = rng.choice([1, 1, 2, 4, 8])
        E = groups * max(1, log(2, 512) // groups)
        top = rng.randint(1, groups)
        k = rng.randint(1, min(8, top * (E // groups)))
        N, grad = log(1, max(1, min(16384, 4_000_000 // E))), rng.random() < 0.5
        return dict(kind="route", N=N, E=E, k=k, score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups, top=top, renorm=rng.random() < 0.5,
                    scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["bf16", "f32"]), grad=grad, pad=rng.choice([0, 0, N // 10]))
    grad = rng.random() < 0.5
    C, I = 16 * log(4, 128), 16 * log(4, 128)
    E = log(1, max(2, min(64, 400_000_000 // (3 * C * I))))
    k = rng.randint(1, min(8, E))
    N = log(1, max(1, min(16384, 40_000_000_000 // (k * C * I))))
    return dict(kind="mlp", N=N, E=E, k=k, C=C, I=I, gates="bf16" if grad else rng.choice(["bf16", "f32"]), grad=grad, skew=rng.choice([0.0, 0.5, 1.5]), drop=rng.choice([0, 0, N // 20]))


# ------------------------------------------------------------------ prepare
def _normal(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=F32) * std).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return dict(case, **(_prepare_route if case["kind"] == "route" else _prepare_mlp)(case, g))


def _prepare_route(c, g):
    N, E, k, t = c["N"], c["E"], c["k"], TYPES[c["dtype"]]
    z = _normal(g, N, E, std=1.5) + _normal(g, E, std=0.5)
    if c["pad"]:
        z[torch.randperm(N, generator=g, device="cuda")[:c["pad"]]] = NEG
    s = dict(logits=z.to(t), bias_=_normal(g, E, std=0.05) if c["bias"] else None)
    if c["grad"]:
        s["logits"].requires_grad_()
        s.update(dweights=_normal(g, N, k, dtype=t), dmean=_normal(g, E) * E)
    else:
        s.update(weights=torch.empty(N, k, dtype=t, device="cuda"), idx=torch.empty(N, k, dtype=I32, device="cuda"))
    return s


def _prepare_mlp(c, g):
    N, E, k, C, I = (c[n] for n in ("N", "E", "k", "C", "I"))
    z = _normal(g, N, E) + _normal(g, E, std=c["skew"])
    top, idx = torch.topk(z, k, dim=1)
    idx, w = idx.to(I32), torch.softmax(top, 1)
    if c["drop"]:
        lost = torch.randperm(N, generator=g, device="cuda")[:c["drop"]]
        idx[lost], w[lost] = -1, 0.0
    gate_up, down = (torch.empty(E, *s, dtype=BF16, device="cuda") for s in ((2 * I, C), (C, I)))
    for e in range(E):
        gate_up[e], down[e] = _normal(g, 2 * I, C, std=C ** -0.5), _normal(g, C, I, std=I ** -0.5)
    s = dict(x=_normal(g, N, C, dtype=BF16), idx=idx, weights=w.to(TYPES[c["gates"]]), gate_up=gate_up, down=down)
    if c["grad"]:
        for n in ("x", "weights", "gate_up", "down"):
            s[n].requires_grad_()
        s["dout"] = _normal(g, N, C, dtype=BF16)
    else:
        s["out"] = torch.empty_like(s["x"])
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return globals()[("_own_" if own else "_plain_") + state["kind"]](state)


def _own_route(s):
    how = dict(bias=s["bias_"], score=s["score"], groups=s["groups"], top_groups=s["top"], renorm=s["renorm"], scale=s["scale"])
    if not s["grad"]:
        from ml_b200 import ops
        ops.moe_route(s["weights"], s["idx"], None, s["logits"], **how)
        return s["weights"], s["idx"]
    from ml_b200.ops import autograd as F
    weights, idx, mean = F.moe_route(s["logits"], s["k"], **how)
    dlogits, = torch.autograd.grad([weights, mean], [s["logits"]], [s["dweights"], s["dmean"]])
    return weights.detach(), idx, mean.detach(), dlogits


def _plain_route(s):
    z = s["logits"].detach().float().requires_grad_(s["grad"])
    zn = torch.where(torch.isnan(z), NEG, z)
    there = zn > NEG
    score = lambda t: _scores(t, there, s["score"])
    key = zn.detach() if s["bias_"] is None and s["groups"] == 1 else _keys(s, score(zn.detach().double()))
    key = torch.where(there, key, NEG)
    best, idx = torch.sort(key, dim=1, descending=True, stable=True)
    idx, has = idx[:, :s["k"]], best[:, :s["k"]] > NEG
    sc = score(zn)
    w = torch.where(has, sc.gather(1, idx), 0.0)
    if s["renorm"]:
        total = w.sum(1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    w = (w * s["scale"]).to(s["logits"].dtype)
    idx = torch.where(has, idx, -1).to(I32)
    if not s["grad"]:
        return w, idx
    if s["score"] == "sigmoid":
        total = sc.sum(1, keepdim=True)
        sc = sc / torch.where(total > 0, total, 1.0)
    mean = sc.mean(0)
    dz, = torch.autograd.grad([w, mean], [z], [s["dweights"], s["dmean"]])
    return w.detach(), idx, mean.detach(), dz.to(s["logits"].dtype)


def _scores(z, there, kind):
    """Scores of logits without NaN; 0 where there is no expert."""
    if kind == "sigmoid":
        return torch.where(there, torch.sigmoid(torch.where(there, z, 0.0)), 0.0)
    m = torch.where(there, z.detach(), NEG).amax(1, keepdim=True)
    e = torch.where(there, torch.exp(torch.where(there, z - torch.where(m > NEG, m, 0.0), 0.0)), 0.0)
    total = e.sum(1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _keys(s, sc):
    """What experts are chosen by, in 64 bits: scores and bias, -inf outside of the chosen groups."""
    t = sc if s["bias_"] is None else sc + s["bias_"].double()
    t = torch.where(torch.isneginf(s["logits"].detach()) | torch.isnan(s["logits"].detach()), NEG, t)
    if s["groups"] == 1:
        return t
    N, E, n = s["N"], s["E"], s["groups"]
    two = torch.sort(t.view(N, n, E // n), dim=2, descending=True).values[..., :2]
    two = torch.where((two > NEG) | (torch.arange(two.shape[2], device=t.device) == 0), two, 0.0)      # (one expert that is there counts alone)
    at = torch.sort(two.sum(2), dim=1, descending=True, stable=True).indices[:, :s["top"]]
    stays = torch.zeros(N, n, dtype=torch.bool, device=t.device).scatter_(1, at, True)
    return torch.where(stays[..., None], t.view(N, n, E // n), NEG).view(N, E)


def _own_mlp(s):
    if not s["grad"]:
        from ml_b200 import ops
        ops.moe_mlp(s["out"], s["x"], s["weights"], s["idx"], s["gate_up"], s["down"])
        return s["out"]
    from ml_b200.ops import autograd as F
    leaves = [s[n] for n in ("x", "weights", "gate_up", "down")]
    out = F.moe_mlp(leaves[0], leaves[1], s["idx"], *leaves[2:])
    return (out.detach(), *torch.autograd.grad([out], leaves, [s["dout"]]))


def _plain_mlp(s):
    N, E, k, C = s["N"], s["E"], s["k"], s["C"]
    x, w, gate_up, down = (s[n].detach().float().requires_grad_(s["grad"]) if s["grad"] or n in ("x", "weights") else s[n] for n in ("x", "weights", "gate_up", "down"))
    e = s["idx"].view(-1).long()
    held = e >= 0
    if not s["grad"] and N * k <= E:                                                  # fewer copies of tokens than experts: the experts to the tokens
        at = e.clamp(min=0)
        g, u = (gate_up[at].float() @ x.repeat_interleave(k, 0)[..., None]).squeeze(-1).chunk(2, -1)
        y = (down[at].float() @ (g * torch.sigmoid(g) * u)[..., None]).squeeze(-1)
    else:                                                                             # the tokens to the experts, in places of equal number
        onehot = (e[:, None] == torch.arange(E, device=e.device)).to(I32)
        nth = (onehot.cumsum(0) * onehot).sum(1) - 1
        room = max(1, int(onehot.sum(0).amax()))
        place = torch.where(held, e * room + nth, E * room)
        token = torch.arange(N * k, device=e.device) // k
        filled = torch.zeros(E * room + 1, C, device=e.device).index_copy(0, place[held], x[token[held]])[:-1].view(E, room, C)
        g, u = (filled @ gate_up.float().transpose(1, 2)).chunk(2, -1)
        y = ((g * torch.sigmoid(g) * u) @ down.float().transpose(1, 2)).reshape(-1, C)[place.clamp(max=E * room - 1)]
    y = torch.where(held[:, None], y, 0.0).view(N, k, C)
    out = (y * w[..., None]).sum(1)
    if not s["grad"]:
        return out.to(BF16)
    grads = torch.autograd.grad([out], [x, w, gate_up, down], [s["dout"].float()])
    return (out.detach().to(BF16), *(d.to(s[n].dtype) for d, n in zip(grads, ("x", "weights", "gate_up", "down"))))


# ------------------------------------------------------------------ 64 bits, from the definitions
def exact(case, seed):
    return (_exact_route if case["kind"] == "route" else _exact_mlp)(prepare(case, seed))


def _exact_route(s):
    z = s["logits"].detach().double()
    N, E, k = s["N"], s["E"], s["k"]
    out = z.isnan() | z.isneginf()
    softmax = s["score"] == "softmax"
    zs = z.masked_fill(out, -1e300)
    sc = (torch.softmax(zs, 1) if softmax else 1 / (1 + torch.exp(-zs))).masked_fill(out, 0.0)
    if s["bias_"] is None and s["groups"] == 1:
        t = zs.clone()
    else:
        t = sc + (0.0 if s["bias_"] is None else s["bias_"].double())
    t = t.masked_fill(out, NEG)
    if s["groups"] > 1:
        parts = t.view(N, s["groups"], -1)
        first = parts.amax(2)
        score = first.clone()
        if parts.shape[2] > 1:
            second = parts.topk(2, 2).values[..., 1]
            score = score + second.masked_fill(second.isneginf(), 0.0)
        order = torch.argsort(-score, dim=1, stable=True)
        rank = torch.empty_like(order).scatter_(1, order, torch.arange(s["groups"], device=z.device).expand(N, -1))
        t = parts.masked_fill((rank >= s["top"])[..., None], NEG).reshape(N, E)
    at = torch.argsort(-t, dim=1, stable=True)[:, :k]
    has = ~t.gather(1, at).isneginf()
    chosen = torch.zeros(N, E, dtype=torch.bool, device=z.device).scatter_(1, at, has)
    w = sc * chosen
    total = w.sum(1, keepdim=True).clamp(min=1e-300)
    q = w / total
    w = (q if s["renorm"] else w) * s["scale"]
    back = lambda full: full.gather(1, at) * has
    if not s["grad"]:
        return back(w), None
    p = sc / sc.sum(1, keepdim=True).clamp(min=1e-300)
    h = s["dmean"].double() / N
    gw = torch.zeros_like(z).scatter_(1, at, s["dweights"].double() * has) * s["scale"]
    rest = 1 - sc
    if s["renorm"]:
        dz = q * (gw - (q * gw).sum(1, keepdim=True)) * (1 if softmax else rest)
    else:
        dz = sc * (gw - (sc * gw).sum(1, keepdim=True)) if softmax else sc * rest * gw
    dz = dz + p * (h - (p * h).sum(1, keepdim=True)) * (1 if softmax else rest)
    return back(w), None, p.mean(0), dz


def _exact_mlp(s):
    x, w, idx = s["x"].detach().double(), s["weights"].detach().double(), s["idx"].long()
    out, dx, dw = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w)
    if s["grad"]:
        dgu, dd = (torch.zeros(s[n].shape, dtype=F64, device=x.device) for n in ("gate_up", "down"))
        dout = s["dout"].double()
    for e in range(s["E"]):
        n, j = (idx == e).nonzero(as_tuple=True)
        if not len(n):
            continue
        Wg, Wu = s["gate_up"][e].detach().double().chunk(2)
        Wd = s["down"][e].detach().double()
        xe, we = x[n], w[n, j][:, None]
        g, u = xe @ Wg.T, xe @ Wu.T
        sg = 1 / (1 + torch.exp(-g))
        h = g * sg * u
        out.index_add_(0, n, we * (h @ Wd.T))
        if not s["grad"]:
            continue
        back = dout[n] @ Wd
        dw[n, j] = (back * h).sum(1)
        dd[e] = dout[n].T @ (we * h)
        dh = we * back
        dg, du = dh * u * sg * (1 + g * (1 - sg)), dh * g * sg
        dgu[e] = torch.cat([dg.T @ xe, du.T @ xe])
        dx.index_add_(0, n, dg @ Wg + du @ Wu)
    return (out, dx, dw, dgu, dd) if s["grad"] else out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, N, E, k = case, case["N"], case["E"], case["k"]
    if c["kind"] == "route":
        b = 2 if c["dtype"] == "bf16" else 4
        bytes_ = N * E * b + N * k * (b + 4) + (4 * E if c["bias"] else 0)
        if c["grad"]:
            bytes_ += N * E * b + N * k * b + 8 * E                                   # the logits' gradient; those of weights and means
        return dict(bytes=bytes_, flops=(8 if c["grad"] else 4) * N * E)
    C, I = c["C"], c["I"]
    copies = (N - c["drop"]) * k
    used = E * (1 - (1 - k / E) ** (N - c["drop"]))                                   # experts with a token, on average
    w = N * k * (4 + (2 if c["gates"] == "bf16" else 4))
    if not c["grad"]:
        return dict(bytes=6 * used * C * I + 4 * N * C + w, flops=6 * copies * C * I)
    return dict(bytes=6 * used * C * I + 6 * E * C * I + 8 * N * C + w + 2 * N * k, flops=18 * copies * C * I)
