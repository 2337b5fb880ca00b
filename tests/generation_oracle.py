"""The operators of generation in 64 bits, element by element from their definitions: what the kernels and the plain forms are compared with."""
import math

import numpy as np
import torch

TINY = 2.0 ** -120


def bf16(x):
    return torch.tensor(x, dtype=torch.float64).float().bfloat16()


def quantised(x):
    """float64 [..., hd] -> (codes, scales [..., hd / 32]); x has to be exact in fp32."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    hi, lo = g.max(-1), g.min(-1)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        s = bf16(np.where(hi > -lo, hi, lo) / -8).double().numpy()
        s = np.where(np.abs(s) < TINY, 0.0, s)
        s = np.where(np.isfinite(g).all(-1), s, np.nan)
        ok = (s != 0) & np.isfinite(s)
        q = np.rint((np.where(ok[..., None], g, 0) / np.where(ok, s, 1.0)[..., None]).astype(np.float32).astype(np.float64))
    c = np.where(ok[..., None], np.clip(q + 8, 0, 15), 8).astype(np.int64)
    return c.reshape(x.shape), s


def values(c, s):
    return (c - 8) * np.repeat(s, 32, -1)


def block_fields(pages):
    """uint8 [..., 18 hd] -> key and value codes [..., 16, hd] (int64), key and value scales [..., 16, hd / 32] (float64), by the layout's words."""
    p = pages.cpu().numpy()
    hd = p.shape[-1] // 18
    ng = hd // 32
    kc, vc = (np.zeros(p.shape[:-1] + (16, hd), dtype=np.int64) for _ in range(2))
    for t in range(16):
        for d in range(hd):
            g, e = d // 32, d % 32
            kb = t * hd // 2 + 4 * ((e // 8) * ng + g) + (e % 8) // 2
            vb = 8 * hd + t * hd // 2 + 2 * ((e // 4) * ng + g) + (e % 4) // 2
            kc[..., t, d] = p[..., kb] >> (4 * (e % 2)) & 15
            vc[..., t, d] = p[..., vb] >> (4 * (e % 2)) & 15
    sc = lambda a: torch.from_numpy(p[..., a * hd:(a + 1) * hd].copy()).view(torch.bfloat16).double().numpy().reshape(p.shape[:-1] + (16, ng))
    return kc, vc, sc(16), sc(17)


def rotated(x, cos, sin):
    """x float64 [N, heads, hd], cos / sin float64 [N, hd / 2]"""
    a, b = np.split(x, 2, -1)
    c, s = cos[:, None], sin[:, None]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def random_pages(n, Hkv, page, hd, seed, spread=1.0):
    """Pages of random codes with scales of both signs around `spread`."""
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, 256, (n, Hkv, page // 16, 18 * hd), generator=g, dtype=torch.uint8)
    s = (torch.rand(n, Hkv, page // 16, hd, generator=g) * 0.2 + 0.05) * spread
    s = torch.where(torch.rand(s.shape, generator=g) < 0.5, -s, s).bfloat16()
    p[..., 16 * hd:] = s.view(torch.uint8)      # hd scales of keys and values: 2 hd bytes
    return p


def attention(q, pages, table, lens, Tq, H, Hkv, hd, scale=None):
    """out [B, Tq, H, hd], lse [B, H, Tq], and bounds on how far a kernel in 32 bits with weights rounded to bf16 once may be off.

    The bounds: a score is a sum of products with codes shifted by 128, so of magnitude A = scale sum_d |q_d| 280 |s|, in fp32: off by E = 2^-20 A at most
    (16 roundings or truncations of 2^-24 each).  That shifts a weight by a factor of 1 +- 2 E; rounding to bf16 (8 significant bits) shifts it by 2^-8 at most, and so it does
    with the result; the sums over tokens by 2^-18.  So |out - o| <= (2 E + 2^-8 + 2^-18) sum_t p_t |v_t| + 2^-8 |o| (1 + small); |lse - l| <= 2 E + 2^-20 (1 + |l|)."""
    B, page, G = len(lens), pages.shape[2] * 16, H // Hkv
    scale = 1 / math.sqrt(hd) if scale is None else scale
    kc, vc, ks, vs = block_fields(pages)
    K, V = values(kc, ks), values(vc, vs)
    q = q.double().cpu().numpy().reshape(B, Tq, H, hd)
    out, lse = np.zeros((B, Tq, H, hd)), np.full((B, H, Tq), -np.inf)
    tol, ltol = np.zeros_like(out), np.zeros_like(lse)
    for b in range(B):
        for i in range(Tq):
            n = lens[b] - Tq + i + 1
            if n <= 0:
                continue
            at = np.arange(n)
            ids = table[b][at // page]
            k, v, s = (x[ids, :, at % page // 16, at % 16] for x in (K, V, ks))      # [n, Hkv, ...]
            for h in range(H):
                kv = h // G
                z = scale * (k[:, kv] @ q[b, i, h])
                m = z.max()
                e = np.exp(z - m)
                p = e / e.sum()
                lse[b, h, i] = m + math.log(e.sum())
                out[b, i, h] = p @ v[:, kv]
                E = 2.0 ** -20 * abs(scale) * 280 * (np.abs(s[:, kv]) @ np.abs(q[b, i, h]).reshape(-1, 32).sum(-1)).max()
                tol[b, i, h] = (2 * E + 2.0 ** -8 + 2.0 ** -18) * (p @ np.abs(v[:, kv])) + 2.0 ** -7.98 * np.abs(out[b, i, h])
                ltol[b, h, i] = 2 * E + 2.0 ** -20 * (1 + abs(lse[b, h, i]))
    return out, lse, tol, ltol


def tables(table, lens, new, stack, n_free, page, rows):
    """(table, slots, pos, starts, new_lens, left) as lists"""
    table, width = [list(r) for r in table], len(table[0])
    slots, pos, starts, out = [-1] * rows, [0] * rows, [0], []
    asked = taken = 0
    for r, (l, n) in enumerate(zip(lens, new)):
        at = starts[-1]
        starts.append(at + n)
        has = (l + page - 1) // page
        fits = l + n <= width * page
        want = (l + n + page - 1) // page - has if fits else 0
        asked += want
        if not fits or asked > n_free:
            out.append(l)
            continue
        for p in range(want):
            table[r][has + p] = stack[n_free - 1 - (asked - want) - p]
        taken = asked
        for i in range(n):
            t = l + i
            slots[at + i] = table[r][t // page] * page + t % page
            pos[at + i] = t
        out.append(l + n)
    return table, slots, pos, starts, out, n_free - taken


def selected(logits, prev, done, eos):
    """Every candidate's score in 64 bits [B, K V] (NaN and what has no score: -inf)."""
    B, K = prev.shape
    z = logits.double().view(B, K, -1).clone()
    V = z.shape[-1]
    z[torch.isnan(z)] = -math.inf
    out = torch.full((B, K, V), -math.inf, dtype=torch.float64)
    for b in range(B):
        for k in range(K):
            if done[b, k]:
                if 0 <= eos < V:
                    out[b, k, eos] = prev[b, k].double()
            else:
                l = torch.logsumexp(z[b, k], 0)
                if torch.isfinite(l):
                    out[b, k] = prev[b, k].double() + (z[b, k] - l)
    return out.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).view(B, K * V)
