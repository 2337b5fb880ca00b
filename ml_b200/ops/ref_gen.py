"""The operators of generation in plain PyTorch: the 4-bit key / value cache and attention over it, block tables, beams.

Signatures and checks are those of `ops.native_gen`; what CPU tensors get and what the kernels are compared with.  The reference trainer
has nothing of this kind.

The cache: `pages` uint8 [n_pages, Hkv, page / 16, 18 hd] of one layer.  A block of 16 tokens of one key / value head is 16 rows of key codes
(hd / 2 bytes each), 16 rows of value codes, 16 rows of key scales (hd / 32 bf16) and 16 rows of value scales.  32 neighbouring elements g of a
row share a scale s, code c stands for (c - 8) s.  Of a key row, 32-bit word j NG + g (NG = hd / 32) holds the elements 32 g + 8 j + e, e = 0..7, in its e-th
four bits; of a value row, 16-bit word i NG + g the elements 32 g + 4 i + e, e = 0..3.  A slot is page number * page + place in the page.
"""
from __future__ import annotations

import math

import torch

TOK = 16             # tokens of a block
TINY = 2.0 ** -120   # a smaller scale is held as 0
HEADS, PAGES = (32, 64, 96, 128), (16, 32, 64, 128)      # head sizes, tokens of a page


# ------------------------------------------------------------------ checks
def pages_shape(pages, hd=None):
    """(n_pages, Hkv, page, hd) of one layer's pages."""
    if pages.dim() != 4 or pages.dtype != torch.uint8 or pages.shape[3] % 18 or (hd is not None and pages.shape[3] != 18 * hd):
        raise ValueError(f"pages {tuple(pages.shape)} {pages.dtype}: need uint8 [n_pages, Hkv, page / 16, 18 hd]" + (f" with hd = {hd}" if hd else ""))
    n, Hkv, blocks, b = pages.shape
    if b // 18 not in HEADS:
        raise ValueError(f"head size {b // 18}: the 4-bit cache has {HEADS}")
    if TOK * blocks not in PAGES:
        raise ValueError(f"pages of {TOK * blocks} tokens: the 4-bit cache has {PAGES}")
    if n * blocks * TOK >= 1 << 31:
        raise ValueError(f"{n} pages of {16 * blocks} tokens: slots are 32-bit numbers")
    return n, Hkv, TOK * blocks, b // 18


def need(t, shape, what, dtype=None):
    if tuple(t.shape) != tuple(shape) or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{what} {tuple(t.shape)} {t.dtype}: need {tuple(shape)}" + (f" {dtype}" if dtype is not None else ""))


def _row_tokens(table, page):
    if table.shape[1] * page >= 1 << 31:
        raise ValueError(f"rows of {table.shape[1]} pages of {page} tokens: places in a sequence are 32-bit numbers")


def check_append(pages, q_out, qkv, slots, pos, cos, sin, H, Hkv, hd):
    n, heads, page, _ = pages_shape(pages, hd)
    if H < 0 or heads != Hkv:
        raise ValueError(f"{H} query and {Hkv} key / value heads, pages of {heads}")
    N = slots.numel()
    need(qkv, (N, (H + 2 * Hkv) * hd), "qkv")
    need(slots, (N,), "slots", torch.int32)
    if q_out is not None:
        need(q_out, (N, H * hd), "q_out", qkv.dtype)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        need(pos, (N,), "pos", torch.int32)
        need(cos, (cos.shape[0], hd // 2), "cos", torch.float32)
        need(sin, cos.shape, "sin", torch.float32)
    return n, page, N


def check_read(k, v, pages, slots):
    n, Hkv, page, hd = pages_shape(pages)
    N = slots.numel()
    need(slots, (N,), "slots", torch.int32)
    need(k, (N, Hkv * hd), "k")
    need(v, (N, Hkv * hd), "v", k.dtype)
    return n, Hkv, page, hd, N


def check_attn(out, lse, q, pages, table, lens, Tq, H, Hkv, hd, scale):
    if scale is not None and not abs(scale) <= 2.0 ** 127:      # (times log2 e it still is an fp32 number)
        raise ValueError(f"scale = {scale}: need 2^127 at most")
    n, heads, page, _ = pages_shape(pages, hd)
    if Hkv < 1 or heads != Hkv or H % Hkv or H < 1 or Tq < 1:
        raise ValueError(f"{H} query heads over {Hkv} key / value heads (pages of {heads}), {Tq} tokens a sequence")
    B = lens.numel()
    need(lens, (B,), "lens", torch.int32)
    if table.dim() != 2 or table.shape[0] != B or table.dtype != torch.int32:
        raise ValueError(f"table {tuple(table.shape)} {table.dtype}: need int32 [{B}, pages of a sequence]")
    _row_tokens(table, page)
    need(q, (B * Tq, H * hd), "q")
    need(out, (B * Tq, H * hd), "out", q.dtype)
    if lse is not None:
        need(lse, (B, H, Tq), "lse", torch.float32)
    return n, page, B


def check_tables(table, slots, pos, starts, new_lens, left, lens, new, free, n_free, page):
    B = lens.numel()
    if B < 1 or B > 4096 or page < 1 or slots.numel() > 1 << 22:
        raise ValueError(f"{B} requests, {slots.numel()} places, pages of {page}: 1 to 4096 requests and 2^22 places at most")
    if table.dim() != 2 or table.shape[0] != B or table.shape[1] < 1:
        raise ValueError(f"table {tuple(table.shape)}: need [{B}, pages of a request]")
    _row_tokens(table, page)
    for t, s, n in ((table, table.shape, "table"), (slots, (slots.numel(),), "slots"), (pos, (slots.numel(),), "pos"), (starts, (B + 1,), "starts"), (new_lens, (B,), "new_lens"),
                    (left, (1,), "left"), (lens, (B,), "lens"), (new, (B,), "new"), (free, (free.numel(),), "free"), (n_free, (1,), "n_free")):
        need(t, s, n, torch.int32)
    return B


def check_select(scores, tokens, parents, done_out, logits, prev, done):
    if prev.dim() != 2:
        raise ValueError(f"prev {tuple(prev.shape)}: need [requests, beams]")
    B, K = prev.shape
    if not 1 <= K <= 32:
        raise ValueError(f"{K} beams: 1 to 32 a request")
    if logits.dim() != 2 or logits.shape[0] != B * K or logits.shape[1] < 1 or logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"logits {tuple(logits.shape)} {logits.dtype}: need bfloat16 or float32 [{B * K}, V]")
    if K * logits.shape[1] >= 0xFFFFFFFF or logits.shape[1] >= 1 << 31:
        raise ValueError(f"{K} beams of {logits.shape[1]} logits: their product has to stay below 2^32, and the logits below 2^31")
    for t, n, d in ((scores, "scores", torch.float32), (prev, "prev", torch.float32), (tokens, "tokens", torch.int32), (parents, "parents", torch.int32),
                    (done_out, "done_out", torch.int32), (done, "done", torch.int32)):
        need(t, (B, K), n, d)
    return B, K, logits.shape[1]


def check_reorder(pages, table_out, spare_out, hist_out, table, spare, lens, hist, parents, tokens, page):
    """(layers, n_pages, Hkv, page, bytes of a block, B, K)"""
    if parents.dim() != 2:
        raise ValueError(f"parents {tuple(parents.shape)}: need [requests, beams]")
    B, K = parents.shape
    rows = B * K
    if table.dim() != 2 or hist.dim() != 2 or table.shape[1] < 1:
        raise ValueError(f"table {tuple(table.shape)}, hist {tuple(hist.shape)}: need [{rows}, pages] and [{rows}, tokens]")
    for t, s, n in ((parents, (B, K), "parents"), (tokens, (B, K), "tokens"), (table, (rows, table.shape[1]), "table"), (table_out, table.shape, "table_out"),
                    (spare, (rows,), "spare"), (spare_out, (rows,), "spare_out"), (lens, (rows,), "lens"), (hist, (rows, hist.shape[1]), "hist"),
                    (hist_out, hist.shape, "hist_out")):
        need(t, s, n, torch.int32)
    if any(a.data_ptr() == b.data_ptr() for a, b in ((table, table_out), (spare, spare_out), (hist, hist_out)) if a.numel()):
        raise ValueError("table, spare and hist are read while the others are written: give other tensors for the outputs")
    if pages is None:
        if page is None or page < 16 or page % 16:
            raise ValueError(f"page = {page}: without pages the tokens of a page have to be given, a multiple of 16")
        _row_tokens(table, page)
        return 0, 0, 0, page, 16, B, K
    if pages.dim() != 5:
        raise ValueError(f"pages {tuple(pages.shape)}: need [layers, n_pages, Hkv, page / 16, 18 hd]")
    n, Hkv, size, hd = pages_shape(pages[0] if pages.shape[0] else pages.new_empty(pages.shape[1:]))
    if page is not None and page != size:
        raise ValueError(f"page = {page}, and pages of {size} tokens")
    _row_tokens(table, size)
    return pages.shape[0], n, Hkv, size, 18 * hd, B, K


# ------------------------------------------------------------------ 4-bit blocks
def kv4_codes(x):
    """x fp32 [..., hd] -> codes 0..15 (int64 [..., hd]) and scales (bf16 [..., hd / 32])."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    hi, lo = g.amax(-1), g.amin(-1)
    s = (torch.where(hi > -lo, hi, lo) * -0.125).to(torch.bfloat16)
    fine = torch.isfinite(g).all(-1)
    s = torch.where(s.float().abs() < TINY, torch.zeros_like(s), s)
    s = torch.where(fine, s, torch.full_like(s, float("nan")))
    some = (fine & (s != 0))[..., None]
    c = torch.clamp(torch.round(torch.where(some, g, 0.0) / torch.where(some, s.float()[..., None], 1.0)) + 8, 0, 15)
    return c.long().view(x.shape), s


def _row_bytes(c, run):
    """Codes [N, Hkv, hd] -> the bytes of their rows [N, Hkv, hd / 2], `run` elements (8: keys, 4: values) in a word."""
    n, h, hd = c.shape
    c = c.view(n, h, hd // 32, 32 // run, run // 2, 2).transpose(2, 3)
    return (c[..., 0] | c[..., 1] << 4).to(torch.uint8).reshape(n, h, hd // 2)


def _row_codes(b, run):
    n, h, half = b.shape
    b = b.view(n, h, 32 // run, half // 16, run // 2).transpose(2, 3).long()
    return torch.stack([b & 15, b >> 4], -1).reshape(n, h, 2 * half)


def _places(pages, slots, page):
    """Views of the pool by slot: key rows, value rows, key scales, value scales, each [slots, Hkv, bytes]."""
    hd = pages.shape[3] // 18
    b, r = slots // page, slots % page
    blk = pages[b, :, r // TOK]                  # [N, Hkv, 18 hd], a copy
    r = r % TOK
    at = [(0, hd // 2), (8 * hd, hd // 2), (16 * hd, hd // 16), (17 * hd, hd // 16)]
    cols = [(o + r * w)[:, None] + torch.arange(w, device=pages.device) for o, w in at]
    return blk, cols


def kv4_append(pages, q_out, qkv, slots, pos, cos, sin, H, Hkv, hd):
    """New tokens' keys and values written to the cache in 4 bits.  qkv [N, (H + 2 Hkv) hd]; with tables cos, sin [T, hd / 2] queries and keys are rotated to
    the positions pos[N] (rotate-half RoPE; None: they are as they come), the queries go to q_out [N, H hd] (None: nowhere), keys and values to slots[N]
    of `pages`; a negative slot is none.  Two rows of one call do not share a slot."""
    n, page, N = check_append(pages, q_out, qkv, slots, pos, cos, sin, H, Hkv, hd)
    if N == 0:
        return
    x = qkv.float().view(N, H + 2 * Hkv, hd)
    qk, v = x[:, :H + Hkv], x[:, H + Hkv:]
    if cos is not None:
        if int(pos.min()) < 0 or int(pos.max()) >= cos.shape[0]:
            raise IndexError("position outside the rotary tables (4-bit cache)")
        a, b = qk.chunk(2, -1)
        c, s = (t[pos.long()][:, None] for t in (cos, sin))
        qk = torch.cat([a * c - b * s, b * c + a * s], -1)
    if q_out is not None:
        q_out.copy_(qk[:, :H].reshape(N, H * hd))
    if int(slots.max()) >= n * page:
        raise IndexError("slot outside the pool (4-bit cache)")
    keep = slots >= 0
    s = slots[keep].long()
    (ck, sk), (cv, sv) = kv4_codes(qk[keep, H:].contiguous()), kv4_codes(v[keep].contiguous())
    rows = [_row_bytes(ck, 8), _row_bytes(cv, 4), sk.contiguous().view(torch.uint8), sv.contiguous().view(torch.uint8)]
    b, r = s // page, s % page
    _, cols = _places(pages, s, page)
    for col, val in zip(cols, rows):
        h = torch.arange(Hkv, device=pages.device)[None, :, None]
        pages[b[:, None, None], h, (r // TOK)[:, None, None], col[:, None]] = val


def kv4_read(k, v, pages, slots):
    """What the slots of the cache hold: k, v [N, Hkv hd]; zeros for a negative slot."""
    n, Hkv, page, hd, N = check_read(k, v, pages, slots)
    if N == 0:
        return
    if int(slots.max()) >= n * page:
        raise IndexError("slot outside the pool (4-bit cache)")
    blk, cols = _places(pages, slots.clamp(min=0).long(), page)
    part = [torch.gather(blk, 2, c[:, None].expand(N, Hkv, c.shape[1])) for c in cols]
    for out, b, run, s in ((k, part[0], 8, part[2]), (v, part[1], 4, part[3])):
        val = (_row_codes(b, run).float() - 8).view(N, Hkv, -1, 32) * s.contiguous().view(torch.bfloat16).float()[..., None]
        out.copy_(torch.where((slots >= 0)[:, None], val.view(N, -1), torch.zeros(())))


def kv4_attn(out, lse, q, pages, table, lens, Tq, H, Hkv, hd, scale=None):
    """Attention of the newest Tq tokens of every sequence over its cached keys and values.  q, out [B Tq, H hd]; table int32 [B, pages of a sequence] has the
    page numbers of a sequence's tokens in order, lens int32 [B] how many tokens it has, the Tq newest (already appended) among them: query token i
    sees the tokens before lens - Tq + i + 1.  Every key / value head serves H / Hkv consecutive query heads; scale: 1 / sqrt(hd).  A query
    that sees nothing gets zeros.  lse fp32 [B, H, Tq] (or None): log of the sum of the exponentials, -inf where nothing is seen.

    The kernel adds up in 32 bits.  It rounds to fewer: weights times values' scales to bf16, once, and of queries what lies below 2^-23 of a row's largest element; a score
    is off by some 2^-16 of max |q| times a scale.  Values of any size that the cache holds come out, but what is below 2^-81 beside more than 2^-50 in its
    group, or than 2^50 in another."""
    n, page, B = check_attn(out, lse, q, pages, table, lens, Tq, H, Hkv, hd, scale)
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    G = H // Hkv
    for b in range(B):
        t = int(lens[b])
        if t > table.shape[1] * page:
            raise IndexError("sequence longer than its row of the block table (attention over the 4-bit cache)")
        rows = slice(b * Tq, (b + 1) * Tq)
        out[rows] = 0
        if lse is not None:
            lse[b] = float("-inf")
        if t <= 0:
            continue
        at = torch.arange(t, device=q.device)
        ids = table[b, at // page].long()
        if int(ids.min()) < 0 or int(ids.max()) >= n:
            raise IndexError("page outside the pool (attention over the 4-bit cache)")
        k, v = (torch.empty(t, Hkv * hd, device=q.device) for _ in range(2))
        kv4_read(k, v, pages, (ids * page + at % page).int())
        k, v = (x.view(t, Hkv, hd).transpose(0, 1) for x in (k, v))
        x = q[rows].float().view(Tq, Hkv, G, hd).permute(1, 2, 0, 3)                     # [Hkv, G, Tq, hd]
        seen = at[None] < t - Tq + torch.arange(1, Tq + 1, device=q.device)[:, None]
        z = torch.where(seen, torch.einsum("kgid,ktd->kgit", x, k) * scale, float("-inf"))
        any_ = seen.any(-1)
        m = torch.where(any_, z.amax(-1), 0.0)
        e = torch.where(seen, torch.exp(z - m[..., None]), 0.0)
        l = e.sum(-1)
        o = torch.zeros(Hkv, G, Tq, hd, device=q.device)
        for i in range(Tq):
            d = t - Tq + i + 1
            if d > 0:
                o[:, :, i] = torch.einsum("kgt,ktd->kgd", e[:, :, i, :d], v[:, :d]) / l[:, :, i, None]
        out[rows] = o.permute(2, 0, 1, 3).reshape(Tq, H * hd).to(out.dtype)
        if lse is not None:
            lse[b] = torch.where(any_, m + torch.log(l), float("-inf")).reshape(H, Tq)


# ------------------------------------------------------------------ block tables
def block_tables(table, slots, pos, starts, new_lens, left, lens, new, free, n_free, page):
    """Pages and cache slots for the new tokens of a batch of requests; all tensors int32.

    Request r holds lens[r] tokens, in the pages that table[r] names, and gets new[r] more.  free[:n_free[0]] is a stack of free pages; requests take
    theirs from its top, in order, as long as it lasts: a request is refused if the needs of the requests up to it, its own included, pass what lies there, or
    if it would outgrow its row of the table.  Written: the fresh pages' numbers in `table`; starts[r] = sum of new[:r]; for the i-th new token
    of request r, in place starts[r] + i, its slot in `slots` and its position lens[r] + i in `pos` (refused, and behind the last one: -1 and 0); new_lens[r]
    = lens[r] + new[r], or lens[r] where refused; left[0] = pages that stay on the stack.  new_lens may be lens, left may be n_free."""
    B = check_tables(table, slots, pos, starts, new_lens, left, lens, new, free, n_free, page)
    width, rows = table.shape[1], slots.numel()
    L, N, f = lens.tolist(), new.tolist(), int(n_free)
    if min(L) < 0 or min(N) < 0 or max(N) > rows or not 0 <= f <= free.numel():
        raise IndexError("request of negative length, of more new tokens than the slot map has places, or more free pages than the stack (block tables)")
    if sum(N) > rows:
        raise IndexError("more new tokens than the slot map has places (block tables)")
    slots.fill_(-1)
    pos.zero_()
    at, asked, taken = 0, 0, 0
    stack = free.tolist()
    for r in range(B):
        starts[r] = at
        fits = L[r] + N[r] <= width * page
        has = -(-L[r] // page)
        want = -(-(L[r] + N[r]) // page) - has if fits else 0
        asked += want
        if fits and asked <= f:
            for p in range(want):
                table[r, has + p] = stack[f - 1 - (asked - want + p)]
            taken = max(taken, asked)
            t = torch.arange(L[r], L[r] + N[r], device=table.device)
            ids = table[r, t // page]
            slots[at:at + N[r]] = torch.where(ids < 0, -1, (ids.long() * page + t % page).clamp(max=(1 << 31) - 1)).int()
            pos[at:at + N[r]] = t.int()
            L[r] += N[r]
        at += N[r]
    starts[B] = at
    new_lens.copy_(torch.tensor(L, dtype=torch.int32))
    left.fill_(f - taken)


# ------------------------------------------------------------------ beams
def beam_select(scores, tokens, parents, done_out, logits, prev, done, eos):
    """One step's choice of continuations: of the scores prev[b, k] + log softmax(logits[b K + k])[v] over beams k and vocabulary v the K largest of every
    request b, equal ones by the lowest k V + v.  logits bf16 or fp32 [B K, V]; prev fp32 [B, K] (-inf: no beam); done int32 [B, K]: a beam that has ended
    goes on as (prev, eos).  Written [B, K]: scores fp32; tokens, parents (the beam continued) and done_out (ended, or eos) int32.  NaN counts as -inf; a
    beam without a finite logarithm of its sum has no continuation.  scores may be prev, done_out may be done."""
    B, K, V = check_select(scores, tokens, parents, done_out, logits, prev, done)
    ninf = float("-inf")
    z = logits.float().view(B, K, V)
    z = torch.where(torch.isnan(z), torch.full_like(z, ninf), z)
    m = z.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(z - m).sum(-1, keepdim=True))
    s = prev[..., None] + (z - lse)
    s = torch.where(torch.isnan(s) | ~torch.isfinite(lse), torch.full_like(s, ninf), s)
    kept = torch.where(torch.arange(V, device=z.device) == eos, prev[..., None], torch.full_like(s, ninf))
    s = torch.where((done != 0)[..., None], torch.where(torch.isnan(kept), torch.full_like(s, ninf), kept), s).view(B, K * V)
    best, at = torch.sort(s, dim=1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    par, tok = at // V, at % V
    ended = (done != 0).gather(1, par) | (tok == eos)
    for out, x in ((scores, best), (tokens, tok), (parents, par), (done_out, ended)):
        out.copy_(x)


def beam_reorder(pages, table_out, spare_out, hist_out, table, spare, lens, hist, parents, tokens, page=None):
    """The beams' state in the order of their parents, and their tokens appended; all index tensors int32.  Row b K + k continues row b K + parents[b, k]:

    hist_out[row] = the parent's first lens[row] tokens of hist [rows, T], then tokens[b, k];
    table_out[row] = the parent's numbers of full pages in table [rows, pages], then the row's own.  The page that is being filled belongs to one row: a row that continues
    another gets the parent's tokens in it copied to its page spare[row] in all layers of `pages` [layers, n_pages, Hkv, page / 16, 18 hd] (up to a whole block of
    16 tokens), which becomes its page, and the page it had becomes spare_out[row].
    The rows of a request have one length.  pages None (with page = its tokens): no cache to copy in."""
    layers, n, Hkv, page, _, B, K = check_reorder(pages, table_out, spare_out, hist_out, table, spare, lens, hist, parents, tokens, page)
    rows, width = table.shape
    if rows and (int(parents.min()) < 0 or int(parents.max()) >= K):
        raise IndexError("parent that is no beam of the request (beam reordering)")
    par = parents.reshape(-1).tolist()
    for r in range(rows):
        src = r // K * K + par[r]
        t = min(max(int(lens[r]), 0), width * page)
        full, rest = t // page, t % page
        table_out[r] = table[r]
        table_out[r, :full] = table[src, :full]
        spare_out[r] = spare[r]
        if rest and src != r:
            table_out[r, full], spare_out[r] = spare[r], table[r, full]
            if pages is not None:
                a, b = int(table[src, full]), int(spare[r])
                if not (0 <= a < n and 0 <= b < n):
                    raise IndexError("page outside the pool (beam reordering)")
                pages[:, b, :, :-(-rest // TOK)] = pages[:, a, :, :-(-rest // TOK)]
        h = min(t, hist.shape[1])
        hist_out[r, :h] = hist[src, :h]
        if t < hist.shape[1]:
            hist_out[r, t] = tokens.view(-1)[r]
