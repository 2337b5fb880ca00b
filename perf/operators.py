"""The workloads by which the operators of generation from a 4-bit key / value cache are followed.

Each case is a dict of plain values.  `prepare` makes what a program holds before the call, `run` is one pass through an operator - in its
plain form, elementary torch operations in 32 bits, or with `own` through the framework's entry points - `exact` the same outputs in 64 bits
from the definition, `work` the bytes and operations one pass cannot do without.

Kinds:
  attn     attention of the newest tokens of every sequence over its cached keys and values
  append   rotary embedding of new tokens' queries and keys, keys and values written to the cache in 4 bits and read back as what they stand for
  tables   cache slots and pages for the new tokens of a batch of requests
  select   one step's choice of the best continuations over beams and vocabulary
  reorder  the beams' block tables, token histories and half-filled pages in the order of their parents

The cache: `pages` uint8 [..., n_pages, Hkv, page / 16, 18 hd], a block of 16 tokens of one head being 16 rows of key codes (hd / 2 bytes each), 16 rows of
value codes, 16 rows of key scales (hd / 32 bf16) and 16 rows of value scales.  32 neighbouring elements g of a row share a scale s; code c stands for
(c - 8) s.  Of a key row, 32-bit word j NG + g (NG = hd / 32) holds the elements 32 g + 8 j + e, e = 0..7, in its e-th four bits; of a value row, 16-bit
word i NG + g the elements 32 g + 4 i + e, e = 0..3.  Token t of a sequence is row t % 16 of block (t % page) / 16 of page table[t / page].
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
NEG = float("-inf")


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one sequence's next token in the 12-layer / 768-wide decoder, its window nearly full: latency
        dict(name="attn_one", kind="attn", B=1, Tq=1, H=12, Hkv=12, hd=64, ctx=1000, page=64, empty=0),
        # samples from a checkpoint of the 2048-wide decoder, sequences of all lengths, two places of the batch not in use
        dict(name="attn_batch", kind="attn", B=16, Tq=1, H=16, Hkv=16, hd=128, ctx=2048, page=64, empty=2),
        # many long sequences of a model with grouped key / value heads
        dict(name="attn_long", kind="attn", B=64, Tq=1, H=32, Hkv=8, hd=128, ctx=8192, page=64, empty=0),
        # several tokens at once behind a long prompt: proposed ones that are checked together
        dict(name="attn_tokens", kind="attn", B=7, Tq=5, H=12, Hkv=4, hd=64, ctx=4001, page=16, empty=0),
        # a decoding step's new tokens, one of them padding
        dict(name="append_step", kind="append", N=16, H=16, Hkv=16, hd=128, page=64, T=2048, skip=1),
        # prompts of eight windows
        dict(name="append_prompts", kind="append", N=8192, H=12, Hkv=12, hd=64, page=64, T=1024, skip=0),
        # a decoding step of 64 requests
        dict(name="tables_step", kind="tables", B=64, old=1000, new=1, page=64, width=32),
        # requests that arrive with their prompts, of which the last find no page
        dict(name="tables_prompts", kind="tables", B=300, old=0, new=1024, page=16, width=64),
        # one request with four beams
        dict(name="select_one", kind="select", B=1, K=4, V=50304, dtype="bf16", done=0),
        # a batch of requests with eight beams each, some of which have ended
        dict(name="select_batch", kind="select", B=32, K=8, V=50304, dtype="bf16", done=1),
        # one request with four beams in the 12-layer / 768-wide decoder
        dict(name="reorder_one", kind="reorder", B=1, K=4, L=12, Hkv=12, hd=64, ctx=500, page=64, T=1024),
        # a batch of requests with eight beams each
        dict(name="reorder_batch", kind="reorder", B=16, K=8, L=12, Hkv=12, hd=64, ctx=500, page=64, T=1024),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.choice(["attn", "attn", "append", "tables", "select", "select", "reorder"])
    hd, page = rng.choice([32, 64, 96, 128]), rng.choice([16, 32, 64, 128])
    if kind == "attn":
        Hkv, G, Tq = log(1, 16), rng.choice([1, 1, 2, 3, 4, 6, 8]), rng.choice([1, 1, 1, 2, 3, 5, 8])
        ctx = log(Tq + 3, 16384)
        B = log(1, max(1, min(64, 2_000_000 // (ctx * Hkv))))
        return dict(kind="attn", B=B, Tq=Tq, H=G * Hkv, Hkv=Hkv, hd=hd, ctx=ctx, page=page, empty=rng.choice([0, 1]) if B > 2 else 0)
    if kind == "append":
        Hkv, G = log(1, 16), rng.choice([1, 1, 2, 4])
        N = log(1, 8192)
        return dict(kind="append", N=N, H=G * Hkv, Hkv=Hkv, hd=hd, page=page, T=rng.choice([512, 1024, 4096]), skip=min(N - 1, rng.choice([0, 1, 3])))
    if kind == "tables":
        B, new, old = log(1, 512), rng.choice([1, 1, log(1, 600)]), rng.choice([0, log(1, 4000)])
        return dict(kind="tables", B=B, old=old, new=new, page=page, width=-(-(old + new) // page) + rng.choice([0, 1, 7]))
    if kind == "select":
        B, K, V = log(1, 32), rng.choice([1, 2, 3, 4, 5, 8]), log(50, 50304)
        return dict(kind="select", B=B, K=K, V=V, dtype=rng.choice(["bf16", "f32"]) if B <= 16 else "bf16", done=rng.choice([0, 1]))
    K, L, Hkv, B = rng.choice([2, 3, 4, 8]), log(1, 12), log(1, 12), log(1, 16)
    return dict(kind="reorder", B=B, K=K, L=L, Hkv=Hkv, hd=rng.choice([32, 64]), ctx=log(2, 500), page=rng.choice([16, 32, 64]), T=1024)


# ------------------------------------------------------------------ sizes that follow from a case
def _lengths(c):
    """Lengths of the sequences of an attention case: from an eighth of the longest to the longest, `empty` of them nothing."""
    B = c["B"]
    n = [max(c["Tq"], c["ctx"] * (B + 7 * (b + 1)) // (8 * B)) for b in range(B)]
    return [0] * c["empty"] + n[c["empty"]:]


def _news(c):
    """New tokens of the requests of a tables case."""
    return [1 + (c["new"] - 1) * ((7 * b) % c["B"] + 1) // c["B"] for b in range(c["B"])]


def _olds(c):
    return [c["old"] * ((5 * b) % c["B"] + 1) // c["B"] for b in range(c["B"])]


def _rows_of(c):
    """Places of the slot map of a tables case: every new token, and some places behind them."""
    return sum(_news(c)) + 5


def _stack(c):
    """Pages on the free stack of a tables case: a tenth fewer than the requests ask for where each asks for many, else enough."""
    p = c["page"]
    pages = lambda n: -(-n // p)
    need = sum(pages(o + n) - pages(o) for o, n in zip(_olds(c), _news(c)))
    return max(1, need * 9 // 10 if c["new"] > 4 * p else need + 3)


# ------------------------------------------------------------------ the cache in 4 bits, as torch operations
def _codes(x):
    """x fp32 [..., hd] -> codes [..., hd / 32, 32] as fp32 and scales [..., hd / 32] in bf16."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    hi, lo = g.amax(-1), g.amin(-1)
    m = torch.where(hi > -lo, hi, lo)
    s = (m * -0.125).to(BF16)
    fine = torch.isfinite(hi) & torch.isfinite(lo)
    some = s.float().abs() >= 2.0 ** -120
    s = torch.where(fine, torch.where(some, s, torch.zeros_like(s)), torch.full_like(s, float("nan")))
    use = (fine & some)[..., None]
    c = torch.where(use, torch.clamp(torch.round(g / torch.where(use, s.float()[..., None], torch.ones_like(g))) + 8, 0, 15), torch.full_like(g, 8.0))
    return c, s


def _blocks(k, v):
    """Keys and values fp32 [blocks, 16, hd] -> uint8 [blocks, 18 hd]."""
    n, _, hd = k.shape
    ng = hd // 32
    (ck, sk), (cv, sv) = _codes(k), _codes(v)
    nib = lambda e: (16 ** torch.arange(e, device=k.device)).to(torch.int64)
    wk = (ck.to(torch.int64).view(n, 16, ng, 4, 8) * nib(8)).sum(-1).transpose(2, 3)
    wk = torch.where(wk >= 1 << 31, wk - (1 << 32), wk).to(I32).contiguous()
    wv = (cv.to(torch.int64).view(n, 16, ng, 8, 4) * nib(4)).sum(-1).transpose(2, 3)
    wv = torch.where(wv >= 1 << 15, wv - (1 << 16), wv).to(torch.int16).contiguous()
    raw = lambda t: t.contiguous().view(torch.uint8).reshape(n, -1)
    return torch.cat([raw(wk), raw(wv), raw(sk), raw(sv)], 1)


def _values(blocks):
    """uint8 [..., 18 hd] -> keys and values fp32 [..., 16, hd]."""
    hd, lead = blocks.shape[-1] // 18, blocks.shape[:-1]
    ng = hd // 32
    cut = lambda a, b: blocks[..., a * hd:b * hd].contiguous()
    nibbles = lambda t: torch.stack([t & 15, t >> 4], -1).float() - 8
    scale = lambda t: t.view(BF16).view(*lead, 16, ng, 1, 1).float()
    k = nibbles(cut(0, 8)).view(*lead, 16, 4, ng, 8).transpose(-3, -2) * scale(cut(16, 17))
    v = nibbles(cut(8, 16)).view(*lead, 16, 8, ng, 4).transpose(-3, -2) * scale(cut(17, 18))
    return k.reshape(*lead, 16, hd), v.reshape(*lead, 16, hd)


# ------------------------------------------------------------------ prepare
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return dict(case, **{"attn": _prepare_attn, "append": _prepare_append, "tables": _prepare_tables, "select": _prepare_select,
                         "reorder": _prepare_reorder}[case["kind"]](case, g))


def _normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=F32).to(dtype)


def _prepare_attn(c, g):
    B, Tq, H, Hkv, hd, page = (c[k] for k in ("B", "Tq", "H", "Hkv", "hd", "page"))
    order = torch.randperm(B, generator=g, device="cuda")
    lens = torch.tensor(_lengths(c), dtype=I32, device="cuda")[order]
    width = -(-c["ctx"] // page)
    used = -(-lens // page)
    at = torch.arange(width, device="cuda")[None] < used[:, None]
    n_pages = int(at.sum()) + 2
    ids = torch.randperm(n_pages, generator=g, device="cuda")[:n_pages - 2].to(I32)
    table = torch.full((B, width), -1, dtype=I32, device="cuda")
    table[at] = ids
    per_channel = 1 + 2 * torch.rand(Hkv, 1, hd, generator=g, device="cuda") ** 4      # keys have channels of larger values
    pages = torch.empty(n_pages, Hkv, page // 16, 18 * hd, dtype=torch.uint8, device="cuda")
    part = max(1, 32_000_000 // (Hkv * page * hd))
    for p in range(0, n_pages, part):
        n = min(part, n_pages - p)
        k = (_normal(g, n, Hkv, page, hd) * per_channel).to(BF16).float()
        v = _normal(g, n, Hkv, page, hd, dtype=BF16).float()
        pages[p:p + n] = _blocks(k.view(-1, 16, hd), v.view(-1, 16, hd)).view(n, Hkv, page // 16, 18 * hd)
    q = _normal(g, B * Tq, H * hd, dtype=BF16)
    return dict(pages=pages, table=table, lens=lens, q=q, out=torch.empty_like(q), lse=torch.empty(B, H, Tq, device="cuda"))


def _prepare_append(c, g):
    N, H, Hkv, hd, page, T = (c[k] for k in ("N", "H", "Hkv", "hd", "page", "T"))
    n_pages = N + 1 if N <= 256 else -(-N // page) + 1            # few: the next tokens of as many sequences; many: whole prompts
    pages = torch.zeros(n_pages, Hkv, page // 16, 18 * hd, dtype=torch.uint8, device="cuda")
    qkv = _normal(g, N, (H + 2 * Hkv) * hd, dtype=BF16)
    slots = torch.randperm(n_pages, generator=g, device="cuda")[:, None] * page
    if N <= 256:
        slots = slots[:N] + torch.randint(0, page, (N, 1), generator=g, device="cuda")
    else:
        slots = slots + torch.arange(page, device="cuda")
    slots = slots.view(-1)[:N].to(I32)
    if c["skip"]:
        slots[torch.randperm(N, generator=g, device="cuda")[:c["skip"]]] = -1
    first = torch.randint(0, T, (1,), generator=g, device="cuda")
    pos = ((torch.arange(N, device="cuda") + first) % T).to(I32)
    ang = torch.arange(T, device="cuda", dtype=F32)[:, None] * 10000.0 ** (-2.0 * torch.arange(hd // 2, device="cuda", dtype=F32) / hd)
    new = lambda h: torch.empty(N, h * hd, dtype=BF16, device="cuda")
    return dict(pages=pages, qkv=qkv, slots=slots, pos=pos, cos=torch.cos(ang), sin=torch.sin(ang), q=new(H), k=new(Hkv), v=new(Hkv))


def _prepare_tables(c, g):
    B, page, width, cap = c["B"], c["page"], c["width"], _rows_of(c)
    ints = lambda *s: torch.empty(*s, dtype=I32, device="cuda")
    turn = torch.randperm(B, generator=g, device="cuda")
    lens, new = (torch.tensor(f(c), dtype=I32, device="cuda")[turn] for f in (_olds, _news))
    n_free, held = _stack(c), -(-lens // page)
    at = torch.arange(width, device="cuda")[None] < held[:, None]
    ids = torch.randperm(int(at.sum()) + n_free, generator=g, device="cuda").to(I32)
    table = torch.full((B, width), -1, dtype=I32, device="cuda")
    table[at] = ids[n_free:]
    return dict(lens=lens, new=new, table=table, free=ids[:n_free].clone(), n_free=torch.tensor([n_free], dtype=I32, device="cuda"),
                slots=ints(cap), pos=ints(cap), starts=ints(B + 1), new_lens=ints(B), left=ints(1))


def _prepare_select(c, g):
    B, K, V = c["B"], c["K"], c["V"]
    # logits of a trained model: a few likely tokens above a broad rest
    z = _normal(g, B * K, V) * 2
    top = torch.randint(0, V, (B * K, 8), generator=g, device="cuda")
    z.scatter_add_(1, top, 6 + 3 * torch.rand(B * K, 8, generator=g, device="cuda"))
    prev = -20 * torch.rand(B, K, generator=g, device="cuda")
    done = torch.rand(B, K, generator=g, device="cuda") < (0.25 if c["done"] else -1.0)
    new = lambda t: torch.empty(B, K, dtype=t, device="cuda")
    return dict(logits=z.to(BF16 if c["dtype"] == "bf16" else F32), prev=prev.sort(1, descending=True).values, done_in=done.to(I32), eos=V // 2,
                scores=new(F32), tokens=new(I32), parents=new(I32), done_out=new(I32))


def _prepare_reorder(c, g):
    B, K, L, Hkv, hd, page, T, ctx = (c[k] for k in ("B", "K", "L", "Hkv", "hd", "page", "T", "ctx"))
    width, held = T // page, -(-(ctx + 1) // page)
    rows = B * K
    n_pages = rows * (held + 1)
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(I32)
    table = torch.full((rows, width), -1, dtype=I32, device="cuda")
    table[:, :held] = ids[:rows * held].view(rows, held)
    pages = torch.randint(0, 256, (L, n_pages, Hkv, page // 16, 18 * hd), generator=g, device="cuda", dtype=torch.uint8)
    lens = torch.full((rows,), ctx, dtype=I32, device="cuda")
    rand = lambda n, *s: torch.randint(0, n, s, generator=g, device="cuda", dtype=I32)
    hist, spare = rand(50304, rows, T), ids[rows * held:].clone()
    # about half of the beams go on, the others take the place of one that is left
    parents = torch.where(torch.rand(B, K, generator=g, device="cuda") < 0.5, torch.arange(K, device="cuda", dtype=I32), rand(K, B, K))
    return dict(pages=pages, table=table, spare=spare, lens=lens, hist=hist, parents=parents, tokens=rand(50304, B, K), table_out=torch.empty_like(table),
                spare_out=torch.empty_like(spare), hist_out=torch.zeros_like(hist))


# ------------------------------------------------------------------ one pass
def run(state):
    return globals()[("_own_" if own else "_plain_") + state["kind"]](state)


def _own_attn(s):
    from ml_b200 import ops
    ops.kv4_attn(s["out"], s["lse"], s["q"], s["pages"], s["table"], s["lens"], s["Tq"], s["H"], s["Hkv"], s["hd"])
    return s["out"], s["lse"]


def _plain_attn(s):
    B, Tq, H, Hkv, hd, page = (s[k] for k in ("B", "Tq", "H", "Hkv", "hd", "page"))
    width = s["table"].shape[1]
    blocks = s["pages"][s["table"].clamp(min=0).long()].transpose(1, 2)              # [B, Hkv, width, page / 16, 18 hd]
    k, v = (t.reshape(B, Hkv, width * page, hd) for t in _values(blocks))
    q = s["q"].float().view(B, Tq, Hkv, H // Hkv, hd).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, hd)
    z = (q @ k.transpose(-1, -2) / math.sqrt(hd)).view(B, Hkv, H // Hkv, Tq, -1)
    last = s["lens"][:, None] - Tq + torch.arange(Tq, device=z.device)                # the last token that a query sees
    seen = torch.arange(width * page, device=z.device) <= last[..., None]             # [B, Tq, tokens]
    z = torch.where(seen[:, None, None], z, NEG)
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(m == NEG, 0.0, m))
    l = e.sum(-1, keepdim=True)
    v = torch.where(seen.any(1)[:, None, :, None], v, 0.0)                            # (what lies behind a sequence may be anything)
    o = (e / torch.where(l == 0, 1.0, l)).view(B, Hkv, -1, width * page) @ v
    o = o.view(B, Hkv, H // Hkv, Tq, hd).permute(0, 3, 1, 2, 4).reshape(B * Tq, H * hd)
    return o.to(BF16), (torch.log(l) + m).reshape(B, H, Tq)


def _own_append(s):
    from ml_b200 import ops
    ops.kv4_append(s["pages"], s["q"], s["qkv"], s["slots"], s["pos"], s["cos"], s["sin"], s["H"], s["Hkv"], s["hd"])
    ops.kv4_read(s["k"], s["v"], s["pages"], s["slots"])
    return s["q"], s["k"], s["v"]


def _plain_append(s):
    N, H, Hkv, hd = s["N"], s["H"], s["Hkv"], s["hd"]
    q, k, v = (t.reshape(N, -1, hd) for t in s["qkv"].float().split([H * hd, Hkv * hd, Hkv * hd], 1))
    cos, sin = (s[n][s["pos"].long()][:, None] for n in ("cos", "sin"))

    def turned(x):
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    def held(x):
        c, sc = _codes(x)
        return torch.where((s["slots"] >= 0)[:, None], ((c - 8) * sc.float()[..., None]).reshape(N, -1), 0.0).to(BF16)

    return turned(q).reshape(N, -1).to(BF16), held(turned(k)), held(v)


def _own_tables(s):
    from ml_b200 import ops
    ops.block_tables(s["table"], s["slots"], s["pos"], s["starts"], s["new_lens"], s["left"], s["lens"], s["new"], s["free"], s["n_free"], s["page"])
    return s["table"], s["slots"], s["pos"], s["starts"], s["new_lens"], s["left"]


def _plain_tables(s):
    page, table, lens, new, n_free = s["page"], s["table"], s["lens"], s["new"], s["n_free"]
    dev, width = table.device, table.shape[1]
    fits = lens + new <= width * page
    has = -(-lens // page)
    need = torch.where(fits, -(-(lens + new) // page) - has, 0)
    upto = need.cumsum(0).to(I32)
    got = fits & (upto <= n_free)
    new_lens = torch.where(got, lens + new, lens)
    left = n_free - torch.where(got, upto, 0).amax().to(I32)
    starts = torch.cat([torch.zeros_like(n_free), new.cumsum(0).to(I32)])
    p = torch.arange(width, device=dev, dtype=I32)
    nth = (upto - need)[:, None] + p - has[:, None]
    fresh = got[:, None] & (p >= has[:, None]) & (p < (has + need)[:, None])
    table.copy_(torch.where(fresh, s["free"][(n_free - 1 - nth).clamp(0, s["free"].numel() - 1).long()], table))
    row = torch.arange(s["slots"].numel(), device=dev, dtype=I32)
    r = torch.searchsorted(starts[1:], row, right=True).clamp(max=lens.numel() - 1)
    at = lens[r] + row - starts[r]
    here = got[r] & (row < starts[-1])
    slot = table[r, (at // page).clamp(0, width - 1).long()] * page + at % page
    return table, torch.where(here, slot, -1), torch.where(here, at, 0), starts, new_lens, left


def _own_select(s):
    from ml_b200 import ops
    ops.beam_select(s["scores"], s["tokens"], s["parents"], s["done_out"], s["logits"], s["prev"], s["done_in"], s["eos"])
    return s["scores"], s["tokens"], s["parents"], s["done_out"]


def _plain_select(s):
    B, K, V, eos = s["B"], s["K"], s["V"], s["eos"]
    z = s["logits"].float().view(B, K, V)
    z = torch.where(torch.isnan(z), NEG, z)
    m = z.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(z - m).sum(-1, keepdim=True))
    score = s["prev"][..., None] + (z - lse)
    score = torch.where(torch.isnan(score), NEG, score)
    kept = torch.where(torch.arange(V, device=z.device) == eos, s["prev"][..., None], NEG)
    score = torch.where((s["done_in"] != 0)[..., None], kept, score).view(B, K * V)
    best, at = torch.sort(score, dim=1, descending=True, stable=True)
    best, at = best[:, :K].contiguous(), at[:, :K]
    parents, tokens = (at // V).to(I32), (at % V).to(I32)
    return best, tokens, parents, ((s["done_in"].gather(1, parents.long()) != 0) | (tokens == eos)).to(I32)


def _own_reorder(s):
    from ml_b200 import ops
    ops.beam_reorder(s["pages"], s["table_out"], s["spare_out"], s["hist_out"], s["table"], s["spare"], s["lens"], s["hist"], s["parents"], s["tokens"])
    return s["pages"], s["table_out"], s["spare_out"], s["hist_out"]


def _plain_reorder(s):
    page, table, spare, lens, hist, pages = (s[k] for k in ("page", "table", "spare", "lens", "hist", "pages"))
    B, K = s["parents"].shape
    dev = table.device
    src = (s["parents"] + K * torch.arange(B, device=dev, dtype=I32)[:, None]).view(-1).long()
    row = torch.arange(B * K, device=dev)
    full, rest = (lens // page).long(), lens % page
    moved = (rest > 0) & (src != row)
    p = torch.arange(table.shape[1], device=dev)
    out = torch.where(p < full[:, None], table[src], table)
    at = (row, full.clamp(max=table.shape[1] - 1))
    mine, theirs = table[at], table[src, at[1]]
    out[at] = torch.where(moved, spare, out[at])
    n = -(-rest // 16)
    some = torch.arange(page // 16, device=dev)[None] < n[:, None]                    # blocks of 16 tokens that hold any
    some = (some & moved[:, None])[None, :, None, :, None]
    to, fr = spare.long(), theirs.clamp(min=0).long()
    pages[:, to] = torch.where(some, pages[:, fr], pages[:, to])
    t = torch.arange(hist.shape[1], device=dev)
    h = torch.where(t < lens[:, None], hist[src], s["hist_out"])
    h = torch.where(t == lens[:, None], s["tokens"].view(-1, 1), h)
    return pages, out, torch.where(moved, mine, spare), h


# ------------------------------------------------------------------ 64 bits, from the definitions
def exact(case, seed):
    c = prepare(case, seed)
    if case["kind"] == "attn":
        return _exact_attn(c)
    if case["kind"] == "append":
        return _exact_append(c)
    if case["kind"] == "select":
        return _exact_select(c)
    return None      # (tables, reorder: nothing but whole numbers)


def _exact_attn(s):
    Tq, H, Hkv, hd, page = (s[k] for k in ("Tq", "H", "Hkv", "hd", "page"))
    ng, dev = hd // 32, s["q"].device
    d = torch.arange(hd, device=dev)
    g, e = d // 32, d % 32
    kb, ks = ((e // 8) * ng + g) * 4 + (e % 8) // 2, e % 2                            # byte and half of a key row, of a value row
    vb, vs = ((e // 4) * ng + g) * 2 + (e % 4) // 2, e % 2
    out = torch.zeros(s["B"], Tq, H, hd, dtype=F64, device=dev)
    lse = torch.full((s["B"], H, Tq), NEG, dtype=F64, device=dev)
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        pg = s["pages"][s["table"][b, :-(-n // page)].long()].transpose(0, 1).reshape(Hkv, -1, 18 * hd)
        part = lambda a, w: pg[..., a * hd:a * hd + 16 * w].reshape(Hkv, -1, w)[:, :n]
        scale = lambda a: part(a, 2 * ng).contiguous().view(BF16).double()[..., g]
        k = (((part(0, hd // 2)[..., kb] >> (4 * ks)) & 15).double() - 8) * scale(16)
        v = (((part(8, hd // 2)[..., vb] >> (4 * vs)) & 15).double() - 8) * scale(17)
        q = s["q"].view(s["B"], Tq, H, hd)[b].double()
        for i in range(Tq):
            t = n - Tq + i + 1
            z = torch.einsum("kgd,ktd->kgt", q[i].view(Hkv, -1, hd), k[:, :t]) / math.sqrt(hd)
            lse[b, :, i] = torch.logsumexp(z, -1).view(-1)
            out[b, i] = torch.einsum("kgt,ktd->kgd", torch.softmax(z, -1), v[:, :t]).reshape(H, hd)
    return out.view(-1, H * hd), lse


def _exact_append(s):
    N, H, Hkv, hd = s["N"], s["H"], s["Hkv"], s["hd"]
    x = s["qkv"].double().view(N, -1, hd)
    cos, sin = (s[n][s["pos"].long()].double()[:, None] for n in ("cos", "sin"))
    qk, h = x[:, :H + Hkv], hd // 2
    qk = torch.cat([qk[..., :h] * cos - qk[..., h:] * sin, qk[..., h:] * cos + qk[..., :h] * sin], -1)

    def held(x):
        g = x.reshape(N, -1, 32)
        top, low = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
        top = torch.where(top > low.abs(), top, low)
        sc = (-top / 8).to(BF16).double()
        v = torch.clamp(torch.round(g / sc), -8, 7) * sc
        return torch.where((s["slots"] >= 0)[:, None], v.reshape(N, -1), 0.0)

    return qk[:, :H].reshape(N, -1), held(qk[:, H:]), held(x[:, H + Hkv:])


def _exact_select(s):
    B, K, V = s["B"], s["K"], s["V"]
    best = []
    for b in range(B):
        z = torch.log_softmax(s["logits"].view(B, K, V)[b].double(), -1) + s["prev"][b, :, None].double()
        for k in range(K):
            if int(s["done_in"][b, k]):
                z[k] = NEG
                z[k, s["eos"]] = s["prev"][b, k].double()
        best.append(torch.topk(z.view(-1), K).values)
    return torch.stack(best), None, None, None


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "attn":
        tokens, B, Tq, H, Hkv, hd = sum(_lengths(c)), c["B"], c["Tq"], c["H"], c["Hkv"], c["hd"]
        pages = sum(-(-n // c["page"]) for n in _lengths(c))
        return dict(bytes=tokens * Hkv * hd * 9 // 8 + 4 * B * Tq * H * hd + 4 * B * H * Tq + 4 * (pages + B), flops=4 * tokens * Tq * H * hd)
    if c["kind"] == "append":
        N, H, Hkv, hd = c["N"], c["H"], c["Hkv"], c["hd"]
        kept = (N - c["skip"]) * Hkv * hd * 9 // 8                  # written, and read again
        return dict(bytes=2 * N * (H + 2 * Hkv) * hd + 2 * N * H * hd + 2 * kept + 4 * N * Hkv * hd + 8 * N + 4 * min(N, c["T"]) * hd,
                    flops=3 * N * (H + Hkv) * hd + 4 * N * 2 * Hkv * hd)
    if c["kind"] == "tables":
        return dict(bytes=8 * _rows_of(c) + 16 * c["B"] + 8 * min(_stack(c), c["B"] * c["width"]), flops=0)
    if c["kind"] == "select":
        n = c["B"] * c["K"] * c["V"]
        return dict(bytes=n * (2 if c["dtype"] == "bf16" else 4) + 24 * c["B"] * c["K"], flops=3 * n)
    rows, rest = c["B"] * c["K"], c["ctx"] % c["page"]
    moved = rows * (c["K"] - 1) / (2 * c["K"])                      # beams whose parent is another, on average
    return dict(bytes=2 * moved * c["L"] * c["Hkv"] * rest * c["hd"] * 9 / 8 + rows * (8 * c["T"] // c["page"] + 8 * c["ctx"] + 24), flops=0)
