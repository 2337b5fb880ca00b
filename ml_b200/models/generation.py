"""Generation from a `GPT` with its keys and values cached in 4 bits, sampling or with beams.

`GPT.generate` runs the training forward pass over the whole window for every token; here a token costs one pass over itself.  The prompt goes
through the training kernels (attention over its unrounded keys and values) and leaves its keys and values in the cache; after it every step reads the
cache: slots for the new tokens (`ops.block_tables`), keys and values into them (`ops.kv4_append`), attention over what is there (`ops.kv4_attn`), and with beams
the choice of continuations (`ops.beam_select`) and their state in the order of their parents (`ops.beam_reorder`).  Nothing is read back by the
host before the end, except to sample; there the kernels' error words are (`CachedDecoder.check`).
"""
from __future__ import annotations

import torch

from .. import ops
from ..ops.ref_gen import HEADS, PAGES


class Cache4:
    """Pool of pages for `layers` layers, block tables of `rows` sequences of up to `tokens` tokens, and one spare page a sequence where they are beams; `shared`:
    full pages of a sequence that are another one's too (a prompt's, of all beams of a request but the first), for `sharing` sequences."""

    def __init__(self, layers: int, rows: int, tokens: int, Hkv: int, hd: int, page: int = 64, device="cpu", spares: bool = False, shared: int = 0, sharing: int = 0):
        if page not in PAGES:
            raise ValueError(f"pages of {page} tokens: the 4-bit cache has {PAGES}")
        if hd not in HEADS:
            raise ValueError(f"head size {hd}: the 4-bit cache has {HEADS}")
        i32 = dict(dtype=torch.int32, device=device)
        self.page, self.width = page, -(-tokens // page)
        n = rows * (self.width + int(spares)) - shared * sharing
        self.pages = torch.empty(layers, n, Hkv, page // 16, 18 * hd, dtype=torch.uint8, device=device)
        self.table = torch.full((rows, self.width), -1, **i32)
        self.lens = torch.zeros(rows, **i32)
        self.free = torch.arange(n, **i32)
        self.spare = self.free[n - rows:].clone() if spares else None
        self.n_free = torch.tensor([n - rows if spares else n], **i32)

    def grow(self, new: torch.Tensor, places: int):
        """Slots, positions and first places of new[row] more tokens a row, `places` in all."""
        t = lambda *s: torch.empty(*s, dtype=torch.int32, device=self.table.device)
        slots, pos, starts = t(places), t(places), t(new.numel() + 1)
        ops.block_tables(self.table, slots, pos, starts, self.lens, self.n_free, self.lens, new, self.free, self.n_free, self.page)
        return slots, pos, starts

    def reorder(self, hist, parents, tokens, copy: bool = True):
        """Every row as its parent, `tokens` behind its history; returns the histories.  copy=False: the histories alone matter any more."""
        table, spare, h = torch.empty_like(self.table), torch.empty_like(self.spare), torch.zeros_like(hist)
        ops.beam_reorder(self.pages if copy else None, table, spare, h, self.table, self.spare, self.lens, hist, parents, tokens, self.page)
        self.table, self.spare = table, spare
        return h


class CachedDecoder:
    """A `GPT`'s weights behind a 4-bit cache of `rows` sequences."""

    def __init__(self, gpt, rows: int, tokens: int, page: int = 64, spares: bool = False, shared: int = 0, sharing: int = 0):
        c = gpt.cfg
        if gpt.sharded or gpt.cp is not None:
            raise ValueError("generation from the cache needs the whole model on this device")
        if tokens > c.T:
            raise ValueError(f"{tokens} tokens: the model's window has {c.T}")
        self.gpt, self.c, self.dev, self.dtype = gpt, c, gpt.device, gpt.dtype
        self.cache = Cache4(c.L, rows, tokens, c.H, c.hd, page, gpt.device, spares, shared, sharing)

    def _new(self, *shape, dtype=None):
        return torch.empty(*shape, dtype=dtype or self.dtype, device=self.dev)

    def _layers(self, ids, attention, rows=None):
        """Logits of tokens `ids` (of those at `rows` if given); attention(l, out, qkv) is a layer's attention over rows of queries, keys and values."""
        g, c, Lo = self.gpt, self.c, self.gpt.layout
        N, C, I = ids.numel(), c.C, c.I
        x, h, rstd = self._new(N, C), self._new(N, C), self._new(N, dtype=torch.float32)
        qkv, a, gu, sw, y = self._new(N, 3 * C), self._new(N, C), self._new(N, 2 * I), self._new(N, I), self._new(N, C)
        x1 = self._new(N, C)
        ops.embed_fwd(x, g.P(Lo.off_wte, c.V, C), ids)
        ops.rmsnorm_fwd(h, rstd, x, g.P(Lo.layer(0).ln1, C), c.eps)
        for l in range(c.L):
            o = Lo.layer(l)
            ops.linear_fwd(qkv, h, g.P(o.qkv, 3 * C, C))
            attention(l, a, qkv)
            ops.linear_fwd(y, a, g.P(o.o, C, C))
            ops.add_rmsnorm_fwd(x1, h, rstd, x, y, g.P(o.ln2, C), c.eps)
            ops.linear_fwd(gu, h, g.P(o.gate, 2 * I, C))
            ops.swiglu_fwd(sw, gu)
            ops.linear_fwd(y, sw, g.P(o.down, C, I))
            ops.add_rmsnorm_fwd(x, h, rstd, x1, y, g.P(Lo.layer(l + 1).ln1 if l + 1 < c.L else Lo.off_lnf, C), c.eps)
        if rows is not None:
            h = h[rows].contiguous()
        logits = self._new(h.shape[0], c.V)
        ops.linear_fwd(logits, h, g.P(Lo.off_lm, c.V, C))
        return logits

    def prompt(self, ids: torch.Tensor, slots: torch.Tensor):
        """ids [b, P] through the model, their keys and values into slots[b P]; the last tokens' logits [b, V]."""
        c, g = self.c, self.gpt
        b, P = ids.shape
        lse = self._new(b, c.H, P, dtype=torch.float32)

        def attention(l, out, qkv):
            ops.rope_fwd(qkv, g.cos, g.sin, b, P, c.H, c.hd)
            ops.attn_fwd(out, lse, qkv, b, P, c.H, c.hd)
            ops.kv4_append(self.cache.pages[l], None, qkv, slots, None, None, None, c.H, c.H, c.hd)

        last = torch.arange(1, b + 1, device=self.dev) * P - 1
        return self._layers(ids.reshape(-1), attention, last)

    def step(self, ids: torch.Tensor):
        """One token a row: ids [rows]; its logits [rows, V]."""
        c, g, k = self.c, self.gpt, self.cache
        rows = ids.numel()
        slots, pos, _ = k.grow(torch.ones(rows, dtype=torch.int32, device=self.dev), rows)
        q = self._new(rows, c.C)

        def attention(l, out, qkv):
            ops.kv4_append(k.pages[l], q, qkv, slots, pos, g.cos, g.sin, c.H, c.H, c.hd)
            ops.kv4_attn(out, None, q, k.pages[l], k.table, k.lens, 1, c.H, c.H, c.hd)

        return self._layers(ids, attention)

    def check(self):
        """Waits for the steps so far, and raises what their kernels have reported (CPU tensors raise where they stand)."""
        if self.dev.type == "cuda":
            torch.cuda.current_stream(self.dev).synchronize()
            ops.native_module().raise_error("generation")


@torch.no_grad()
def sample(gpt, prompt, n_new, choose, page=64):
    """`prompt` [b, P] and n_new tokens more, the next one of every row by choose(logits fp32 [b, V], new tokens so far) -> int64 [b]."""
    b, P = prompt.shape
    m = CachedDecoder(gpt, b, P + n_new, page)
    out = prompt.to(m.dev).long()
    slots, _, _ = m.cache.grow(torch.full((b,), P, dtype=torch.int32, device=m.dev), b * P)
    logits = m.prompt(out.int(), slots)
    for k in range(n_new):
        nxt = choose(logits.float(), out[:, P:])
        out = torch.cat([out, nxt.view(b, 1)], dim=1)
        if k + 1 < n_new:
            logits = m.step(nxt.int())
    m.check()
    return out


@torch.no_grad()
def beam_search(gpt, prompt, n_new, beams, eos=-1, page=64, length_penalty=0.0):
    """`prompt` [b, P] continued by n_new tokens with `beams` beams each: (tokens [b, beams, P + n_new], log-probabilities [b, beams]), best first.  A beam that
    has chosen `eos` is filled up with it; beams are compared by log-probability / length^length_penalty at the end (length: up to and with the first eos)."""
    b, P = prompt.shape
    rows = b * beams
    m = CachedDecoder(gpt, rows, P + n_new, page, True, P // page, rows - b)
    k, dev = m.cache, m.dev
    i32 = dict(dtype=torch.int32, device=dev)
    ids = prompt.to(dev).int()
    # a request's first beam gets the prompt; the others share its full pages and have a page of their own where the next one begins
    lead = torch.arange(rows, device=dev) % beams == 0
    k.lens = torch.where(lead, 0, P // page * page).int()
    slots, _, starts = k.grow(torch.where(lead, P, P % page).int(), b * P + (rows - b) * (P % page))
    table = k.table.view(b, beams, -1)
    table[:, 1:, :P // page] = table[:, :1, :P // page].clone()      # (a beam that the first choice leaves without a continuation reads them too)
    at = starts[:-1].view(b, beams)[:, :1] + torch.arange(P, **i32)
    logits = m.prompt(ids, slots[at.long()].view(-1).contiguous())
    logits = logits.repeat_interleave(beams, 0)
    hist = torch.zeros(rows, P + n_new, **i32)
    hist[:, :P] = ids.repeat_interleave(beams, 0)
    scores = torch.full((b, beams), float("-inf"), device=dev)
    scores[:, 0] = 0
    done, tokens, parents = (torch.zeros(b, beams, **i32) for _ in range(3))
    for n in range(n_new):
        ops.beam_select(scores, tokens, parents, done, logits, scores, done, eos)
        more = n + 1 < n_new
        hist = k.reorder(hist, parents, tokens, copy=more)
        if more:
            logits = m.step(tokens.view(-1))
    m.check()
    hist = hist.view(b, beams, -1)
    if length_penalty:
        new = hist[:, :, P:]
        ended = (new == eos).int().cumsum(-1) > 0
        length = (n_new - ended.sum(-1) + ended.any(-1)).float()
        order = (scores / length ** length_penalty).sort(dim=1, descending=True, stable=True).indices
        hist, scores = hist.gather(1, order[..., None].expand_as(hist)), scores.gather(1, order)
    return hist.long(), scores
