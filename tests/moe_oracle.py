"""Routing and experts in 64 bits, from the definitions, a token at a time."""
import math

import torch

F64 = torch.float64


def route(logits, k, bias=None, score="softmax", groups=1, top_groups=1, renorm=True, scale=1.0):
    """(weights [N, k], idx [N, k], mean [E]) in 64 bits; differentiable in `logits` (64 bits)."""
    N, E = logits.shape
    z = torch.where(torch.isnan(logits), -math.inf, logits)
    weights, idx, mean = [], torch.full((N, k), -1, dtype=torch.int32), torch.zeros(E, dtype=F64)
    for n in range(N):
        there = [e for e in range(E) if z[n, e] > -math.inf]
        if not there:
            weights.append(torch.zeros(k, dtype=F64))
            continue
        zt = z[n, there]
        s = torch.softmax(zt, 0) if score == "softmax" else torch.sigmoid(zt)
        p = s / s.sum()
        mean = mean + torch.zeros(E, dtype=F64).index_add(0, torch.tensor(there), p) / N
        key = {e: (float(z[n, e].detach()) if bias is None and groups == 1 else float(s[i].detach()) + (0.0 if bias is None else float(bias[e]))) for i, e in enumerate(there)}
        if groups > 1:
            size = E // groups
            of = {}
            for g in range(groups):
                best = sorted((key[e] for e in there if e // size == g), reverse=True)[:2]
                of[g] = sum(best) if best else -math.inf
            kept = sorted(range(groups), key=lambda g: (-of[g], g))[:top_groups]
            key = {e: t for e, t in key.items() if e // size in kept}
        chosen = sorted(key, key=lambda e: (-key[e], e))[:k]
        w = s[[there.index(e) for e in chosen]] if chosen else s[:0]
        if renorm and chosen:
            zc = z[n, chosen]
            w = torch.softmax(zc, 0) if score == "softmax" else w / w.sum()
        weights.append(torch.cat([w * scale, torch.zeros(k - len(chosen), dtype=F64)]))
        idx[n, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return torch.stack(weights) if N else torch.zeros(0, k, dtype=F64), idx, mean


def mlp(x, weights, idx, gate_up, down):
    """[N, C] in 64 bits; differentiable in all but idx."""
    out = torch.zeros(x.shape, dtype=F64, device=x.device)
    for e in range(down.shape[0]):
        n, j = (idx == e).nonzero(as_tuple=True)
        if len(n):
            g, u = (x[n] @ gate_up[e].T).chunk(2, 1)
            out = out.index_add(0, n, weights[n, j][:, None] * ((g * torch.sigmoid(g) * u) @ down[e].T))
    return out


def mlp_grads(dout, x, weights, idx, gate_up, down):
    """(out, dx, dweights, dgate_up, ddown) in 64 bits, of tensors of any type."""
    leaves = [t.detach().double().requires_grad_() for t in (x, weights, gate_up, down)]
    out = mlp(leaves[0], leaves[1], idx, leaves[2], leaves[3])
    grads = torch.autograd.grad(out, leaves, dout.double(), allow_unused=True) if out.requires_grad else [None] * 4
    return (out.detach(), *(torch.zeros_like(l) if g is None else g for g, l in zip(grads, leaves)))


def mlp_sizes(dout, x, weights, idx, gate_up, down):
    """The five with absolute values in place of all factors: a term's relative error, whatever its sign, comes to no more than that share of these."""
    x, weights, gate_up, down, dout = (t.detach().double() for t in (x, weights, gate_up, down, dout))
    out, dx, dw, dgu, dd = (torch.zeros_like(t) for t in (x, x, weights, gate_up, down))
    for e in range(down.shape[0]):
        n, j = (idx == e).nonzero(as_tuple=True)
        if not len(n):
            continue
        g, u = (x[n] @ gate_up[e].T).chunk(2, 1)
        s, w, Wd = torch.sigmoid(g), weights[n, j].abs()[:, None], down[e].abs()
        h, back = (g * s * u).abs(), dout[n].abs() @ Wd
        out.index_add_(0, n, w * (h @ Wd.T))
        dw[n, j] = (back * h).sum(1)
        dd[e] = dout[n].abs().T @ (w * h)
        # silu' passes 0, and a step of g moves it by |g silu''| of a step all the same: sums without signs of silu' and of g silu'', of silu and of g silu'
        d1 = s * (1 + g.abs() * (1 - s)) + g.abs() * s * (1 - s) * (2 + g.abs())
        d = torch.cat([w * back * u.abs() * d1, w * back * g.abs() * s * (1 + g.abs() * (1 - s))], 1)
        dgu[e] = d.T @ x[n].abs()
        dx.index_add_(0, n, d @ gate_up[e].abs())
    return out, dx, dw, dgu, dd
