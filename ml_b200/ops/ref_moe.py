"""The operators of a mixture of experts in plain PyTorch: routing tokens to experts, and the experts' products.

Signatures and checks are those of `ops.native_moe`; what CPU tensors get and what the kernels are compared with.  (The reference's prototype has a softmax router and
expert kernels that nothing calls, csrc/kernels/moe_kernels.cu:18-194.)

Routing.  A logit of NaN counts as -inf, and an expert at -inf, or with a bias of NaN or -inf, is not there for the choice.  Scores s are a softmax over the experts or a sigmoid each.  A token's k experts are those of
the largest logits, or, with `bias` (fp32 [E]; for the choice only) or groups, of the largest s + bias in 64 bits; equal ones go to the lowest index.  Of `groups` equal
groups of neighbouring experts the `top_groups` best stay, by the sum of their two best s + bias.  Weights are scale * s, with `renorm` scale * s / (sum of the chosen
experts' s).  Where fewer than k experts are left, the index is -1 and the weight 0.  `mean` is the mean over all tokens of softmax(z), or of s / (sum of s).

The experts.  idx int32 [N, k], negative: none; gate_up [E, 2 I, C], the gate's rows first; down [E, C, I]:  out_n = sum_j w_nj down[e] (silu(g) * u), [g | u] = gate_up[e] x_n.
"""
from __future__ import annotations

import torch

F32, I32 = torch.float32, torch.int32
NEG = float("-inf")
SCORES = ("softmax", "sigmoid")
MAX_E, MAX_K, MAX_GROUPS = 1024, 32, 32


# ------------------------------------------------------------------ checks
def _need(t, shape, what, dtypes):
    if tuple(t.shape) != tuple(shape) or t.dtype not in dtypes:
        raise ValueError(f"{what} {tuple(t.shape)} {t.dtype}: need {tuple(shape)} {' or '.join(str(d) for d in dtypes)}")


def check_route(weights, idx, mean, logits, bias, score, groups, top_groups):
    """(N, E, k)"""
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, F32):
        raise ValueError(f"logits {tuple(logits.shape)} {logits.dtype}: need bfloat16 or float32 [tokens, experts]")
    N, E = logits.shape
    if score not in SCORES:
        raise ValueError(f"score {score!r}: one of {SCORES}")
    if not 1 <= E <= MAX_E:
        raise ValueError(f"{E} experts: 1 to {MAX_E}")
    if not (1 <= groups <= MAX_GROUPS and E % groups == 0 and 1 <= top_groups <= groups):
        raise ValueError(f"{top_groups} of {groups} groups of {E} experts: groups divide the experts, at most {MAX_GROUPS}")
    k = idx.shape[1] if idx.dim() == 2 else 0
    if not 1 <= k <= min(MAX_K, top_groups * (E // groups)):
        raise ValueError(f"idx {tuple(idx.shape)}: need [{N}, k], k from 1 to {min(MAX_K, top_groups * (E // groups))}")
    _need(idx, (N, k), "idx", (I32,))
    _need(weights, (N, k), "weights", (torch.bfloat16, F32))
    if mean is not None:
        _need(mean, (E,), "mean", (F32,))
    if bias is not None:
        _need(bias, (E,), "bias", (F32,))
    return N, E, k


def check_route_bwd(dlogits, dweights, dmean, logits, idx, score):
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, F32):
        raise ValueError(f"logits {tuple(logits.shape)} {logits.dtype}: need bfloat16 or float32 [tokens, experts]")
    N, E = logits.shape
    k = idx.shape[1] if idx.dim() == 2 else 0
    if score not in SCORES or not 1 <= E <= MAX_E or not 1 <= k <= min(MAX_K, E):
        raise ValueError(f"score {score!r}, {E} experts, idx {tuple(idx.shape)}: need one of {SCORES}, 1 to {MAX_E} and [{N}, k], k from 1 to {min(MAX_K, E)}")
    _need(idx, (N, k), "idx", (I32,))
    _need(dweights, (N, k), "dweights", (torch.bfloat16, F32))
    _need(dlogits, (N, E), "dlogits", (logits.dtype,))
    if dmean is not None:
        _need(dmean, (E,), "dmean", (F32,))
    return N, E, k


def check_plan(idx, E):
    if idx.dim() != 2 or idx.dtype != I32 or idx.shape[1] < 1:
        raise ValueError(f"idx {tuple(idx.shape)} {idx.dtype}: need int32 [tokens, experts of a token]")
    if not 1 <= E <= MAX_E:
        raise ValueError(f"{E} experts: 1 to {MAX_E}")
    N, k = idx.shape
    if N * k + 32 * E >= 1 << 31:
        raise ValueError(f"{N} tokens to {k} of {E} experts: rows are 32-bit numbers")
    return N, k


def check_mlp(x, weights, idx, gate_up, down):
    """(N, k, E, C, I)"""
    if gate_up.dim() != 3 or down.dim() != 3 or x.dim() != 2:
        raise ValueError(f"x {tuple(x.shape)}, gate_up {tuple(gate_up.shape)}, down {tuple(down.shape)}: need [N, C], [E, 2 I, C], [E, C, I]")
    E, C, I = down.shape
    N, k = check_plan(idx, E)
    _need(x, (N, C), "x", (gate_up.dtype,))
    _need(gate_up, (E, 2 * I, C), "gate_up", (down.dtype,))
    _need(weights, (N, k), "weights", (x.dtype, F32))
    return N, k, E, C, I


# ------------------------------------------------------------------ routing
def _scores(z, score):
    """Scores of logits without NaN; 0 where there is no expert."""
    there = z > NEG
    if score == "sigmoid":
        return torch.where(there, torch.sigmoid(z), 0.0)
    m = z.amax(1, keepdim=True)
    e = torch.where(z == m, 1.0, torch.exp(z - m))
    e = torch.where(there, e, 0.0)
    return _shares(e)


def _shares(e):
    total = e.sum(1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _relative(z):
    """Sigmoids of a row's logits over exp(top), top the largest of them that is not above 0: sums of small scores do not vanish."""
    there = z > NEG
    top = torch.clamp(z.amax(1, keepdim=True), max=0.0)
    e = torch.where(z >= 0, torch.sigmoid(z), torch.exp(torch.where(there, z - top, NEG)) * torch.sigmoid(-z))
    return torch.where(there, e, 0.0)


def _mean_scores(z, score):
    return _scores(z, score) if score == "softmax" else _shares(_relative(z))


def _seen(logits, dtype=F32):
    z = logits.to(dtype)
    return torch.where(torch.isnan(z), NEG, z)


def _chosen(z, idx, score, renorm):
    """Of the chosen experts: there or not, score, weight / scale."""
    has = (idx >= 0) & (idx < z.shape[1])
    at = torch.where(has, idx, 0).long()
    zj = torch.where(has, z.gather(1, at), NEG)
    has = zj > NEG
    s = torch.where(has, _scores(z, score).gather(1, at), 0.0)
    if not renorm:
        return has, at, s, s
    if score == "softmax":
        return has, at, s, _scores(zj, "softmax")
    return has, at, s, _shares(_relative(zj))


def moe_route(weights, idx, mean, logits, bias=None, score="softmax", groups=1, top_groups=1, renorm=True, scale=1.0):
    """The experts of each token and their weights: `weights` [N, k] (bf16 or fp32), `idx` int32 [N, k], `mean` fp32 [E] or None, from `logits` [N, E]."""
    N, E, k = check_route(weights, idx, mean, logits, bias, score, groups, top_groups)
    if N == 0:
        if mean is not None:
            mean.zero_()
        return
    z = _seen(logits)
    if bias is None and groups == 1:
        t = z
    else:
        zd = _seen(logits, torch.float64)
        t = _scores(zd, score) + (0.0 if bias is None else bias.double())
        t = torch.where((zd > NEG) & ~torch.isnan(t), t, NEG)
    if groups > 1:
        parts = t.view(N, groups, -1)
        two = parts.sort(dim=2, descending=True).values[..., :2]
        two = torch.cat([two[..., :1], torch.where(two[..., 1:] > NEG, two[..., 1:], 0.0)], 2).sum(2)
        best = two.sort(dim=1, descending=True, stable=True).indices[:, :top_groups]
        stays = torch.zeros(N, groups, dtype=torch.bool, device=z.device).scatter_(1, best, True)
        t = torch.where(stays[..., None], parts, NEG).reshape(N, E)
    best, at = t.sort(dim=1, descending=True, stable=True)
    idx.copy_(torch.where(best[:, :k] > NEG, at[:, :k], -1))
    weights.copy_(_chosen(z, idx, score, renorm)[3] * scale)
    if mean is not None:
        mean.copy_(_mean_scores(z, score).mean(0))


def moe_route_bwd(dlogits, dweights, dmean, logits, idx, score="softmax", renorm=True, scale=1.0):
    """`dlogits` [N, E] from the gradients of the weights and, where it is not None, of the means."""
    N, E, k = check_route_bwd(dlogits, dweights, dmean, logits, idx, score)
    if N == 0:
        return
    z = _seen(logits)
    s = _scores(z, score)
    rest = 1.0 if score == "softmax" else torch.where(z > NEG, torch.sigmoid(-z), 0.0)
    has, at, sj, q = _chosen(z, idx, score, renorm)
    g = torch.where(has, dweights.float() * scale, 0.0)
    if renorm:
        own = q * (g - (q * g).sum(1, keepdim=True))
        d = torch.zeros_like(z).scatter_add_(1, at, own) * rest
    elif score == "softmax":
        d = torch.zeros_like(z).scatter_add_(1, at, sj * g) - s * (sj * g).sum(1, keepdim=True)
    else:
        d = torch.zeros_like(z).scatter_add_(1, at, sj * g) * rest
    if dmean is not None:
        p, h = _mean_scores(z, score), dmean / N
        d = d + p * (h - (p * h).sum(1, keepdim=True)) * rest
    dlogits.copy_(d)


# ------------------------------------------------------------------ the experts
def _experts(x, weights, idx, gate_up, down):
    """Token, place and weight of each expert's copies, and its matrices."""
    for e in range(down.shape[0]):
        n, j = (idx == e).nonzero(as_tuple=True)
        if n.numel():
            yield e, n, j, x[n].float(), weights[n, j].float()[:, None], gate_up[e].float(), down[e].float()


def _check_idx(idx, E):
    if idx.numel() and int(idx.max()) >= E:
        raise ValueError(f"idx has expert {int(idx.max())} of {E}")


def moe_mlp(out, x, weights, idx, gate_up, down):
    """`out` [N, C]: the tokens through their experts."""
    N, k, E, C, I = check_mlp(x, weights, idx, gate_up, down)
    _need(out, (N, C), "out", (x.dtype,))
    _check_idx(idx, E)
    total = torch.zeros(N, C, dtype=F32, device=x.device)
    for e, n, _, xe, w, Wgu, Wd in _experts(x, weights, idx, gate_up, down):
        g, u = (xe @ Wgu.T).chunk(2, 1)
        total.index_add_(0, n, w * ((g * torch.sigmoid(g) * u) @ Wd.T))
    out.copy_(total)


def moe_mlp_fwd(out, x, weights, idx, gate_up, down):
    """The same for training: what `moe_mlp_bwd` needs besides the inputs, as a tuple of tensors."""
    moe_mlp(out, x, weights, idx, gate_up, down)
    return ()


def moe_mlp_bwd(dx, dweights, dgate_up, ddown, dout, x, weights, idx, gate_up, down, saved):
    """The gradients; those that are None are not formed (`dweights` always is)."""
    N, k, E, C, I = check_mlp(x, weights, idx, gate_up, down)
    _need(dout, (N, C), "dout", (x.dtype,))
    sx, sw = torch.zeros(N, C, dtype=F32, device=x.device), torch.zeros(N, k, dtype=F32, device=x.device)
    for t in (dgate_up, ddown):
        if t is not None:
            t.zero_()
    for e, n, j, xe, w, Wgu, Wd in _experts(x, weights, idx, gate_up, down):
        g, u = (xe @ Wgu.T).chunk(2, 1)
        s = torch.sigmoid(g)
        h, d = g * s * u, dout[n].float()
        dh = d @ Wd
        sw[n, j] = (dh * h).sum(1)
        if ddown is not None:
            ddown[e].copy_(d.T @ (w * h))
        dh = w * dh
        dgu = torch.cat([dh * u * s * (1 + g * (1 - s)), dh * g * s], 1)
        if dgate_up is not None:
            dgate_up[e].copy_(dgu.T @ xe)
        sx.index_add_(0, n, dgu @ Wgu)
    if dx is not None:
        dx.copy_(sx)
    dweights.copy_(sw)
