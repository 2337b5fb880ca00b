"""Plain forms of the operators of generation against their definitions in 64 bits, and generation from the cache on CPU tensors."""
import math
import re

import numpy as np
import pytest
import torch

from ml_b200 import Config, ops
from ml_b200.models import GPT, generation
from ml_b200.ops import ref, ref_gen
from tests import generation_oracle as oracle

I32 = torch.int32


def ints(x):
    return torch.tensor(x, dtype=I32)


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_codes_are_those_of_the_definition(hd):
    torch.manual_seed(hd)
    N, Hkv, page = 40, 2, 16
    x = torch.randn(N, 3 * Hkv * hd)
    x[0] = 0
    x[1, -1], x[2, -3], x[3, -hd:] = math.inf, math.nan, 1e-39
    x[4, -32:] = torch.linspace(-2, 2, 32)
    pages = torch.zeros(4, Hkv, 1, 18 * hd, dtype=torch.uint8)
    slots = torch.randperm(64)[:N].int()
    slots[9] = -1
    ops.kv4_append(pages, None, x, slots, None, None, None, Hkv, Hkv, hd)
    kc, vc, ks, vs = oracle.block_fields(pages)
    for codes, scales, part in ((kc, ks, x[:, Hkv * hd:2 * Hkv * hd]), (vc, vs, x[:, 2 * Hkv * hd:])):
        c, s = oracle.quantised(part.double().numpy().reshape(N, Hkv, hd))
        for n in range(N):
            if (t := int(slots[n])) >= 0:
                assert np.array_equal(codes[t // 16, :, 0, t % 16], c[n]) and np.array_equal(scales[t // 16, :, 0, t % 16], s[n], equal_nan=True)
    k, v = torch.empty(N, Hkv * hd), torch.empty(N, Hkv * hd)
    ops.kv4_read(k, v, pages, slots)
    for got, codes, scales in ((k, kc, ks), (v, vc, vs)):
        want = oracle.values(codes, scales)[:, :, 0].transpose(0, 2, 1, 3).reshape(64, Hkv * hd)[slots.clamp(min=0).long()]
        want[9] = 0
        assert np.array_equal(got.double().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("lens,Tq,H,Hkv,hd,page", [([1], 1, 1, 1, 32, 16), ([0, 17, 64], 2, 4, 2, 64, 32), ([2, 50], 4, 3, 1, 96, 16)])
def test_plain_attention(lens, Tq, H, Hkv, hd, page):
    torch.manual_seed(0)
    B, width = len(lens), max(-(-n // page) for n in lens)
    pages = oracle.random_pages(B * width, Hkv, page, hd, 1)
    table = torch.randperm(B * width).view(B, width).int()
    q = torch.randn(B * Tq, H * hd).bfloat16().float()
    out, lse = torch.empty_like(q), torch.empty(B, H, Tq)
    ops.kv4_attn(out, lse, q, pages, table, ints(lens), Tq, H, Hkv, hd)
    o, l, _, ltol = oracle.attention(q, pages, table.numpy(), lens, Tq, H, Hkv, hd)
    assert np.abs(out.double().numpy().reshape(o.shape) - o).max() <= 2e-5
    assert np.array_equal(np.isinf(l), np.isinf(lse.numpy())) and (np.abs(np.where(np.isinf(l), 0, lse.numpy() - np.where(np.isinf(l), 0, l))) <= ltol + 1e-6).all()


@pytest.mark.parametrize("B,page,width,old,new,free", [(1, 16, 2, 0, 5, 3), (9, 16, 4, 60, 9, 6), (30, 5, 6, 20, 12, 40)])
def test_plain_tables(B, page, width, old, new, free):
    rng = np.random.default_rng(B)
    lens, news = rng.integers(0, old + 1, B).tolist(), rng.integers(0, new + 1, B).tolist()
    held = [-(-n // page) for n in lens]
    ids = rng.permutation(sum(held) + free).tolist()
    stack = [ids.pop() for _ in range(free)]
    table = [[ids.pop() for _ in range(h)] + [-1] * (width - h) for h in held]
    rows = sum(news) + 2
    t, l, nf = ints(table), ints(lens), ints([free])
    slots, pos, starts = torch.empty(rows, dtype=I32), torch.empty(rows, dtype=I32), torch.empty(B + 1, dtype=I32)
    ops.block_tables(t, slots, pos, starts, l, nf, l, ints(news), ints(stack), nf, page)
    assert (t.tolist(), slots.tolist(), pos.tolist(), starts.tolist(), l.tolist(), int(nf)) == oracle.tables(table, lens, news, stack, free, page, rows)


def test_sizes_past_32_bits_are_refused():
    """A place in a sequence, a slot and a token are 32-bit numbers."""
    one, wide = torch.zeros(1, dtype=I32), lambda n: torch.empty(1, n, dtype=I32)
    x = torch.zeros(1, 64)
    pages = torch.zeros(4, 1, 8, 18 * 64, dtype=torch.uint8)
    attn = lambda n: ref_gen.check_attn(x, None, x, pages, wide(n), one, 1, 1, 1, 64, None)
    tables = lambda n, page: ref_gen.check_tables(wide(n), one, one, ints([0, 0]), one, one, one, one, one, one, page)
    order = lambda n, pool, page: ref_gen.check_reorder(pool, wide(n), one, ints([[0]]), wide(n), ints([0]), one, ints([[0]]), ints([[0]]), ints([[0]]), page)
    select = lambda V: ref_gen.check_select(torch.zeros(1, 1), one[None], one[None], one[None], torch.empty(1, V, device="meta"), torch.zeros(1, 1), one[None])
    for f in (attn, lambda n: tables(n, 128), lambda n: order(n, pages[None], None), lambda n: order(n, None, 128)):
        f((1 << 24) - 1)
        with pytest.raises(ValueError, match="32-bit"):
            f(1 << 24)
    tables(1, (1 << 31) - 1)
    with pytest.raises(ValueError, match="32-bit"):
        tables(1, 1 << 31)
    select((1 << 31) - 1)
    with pytest.raises(ValueError, match="below 2\\^31"):
        select(1 << 31)


def test_a_page_number_whose_slot_passes_32_bits_gets_a_slot_of_no_pool():
    """... and not another page's."""
    table, slots, pos = ints([[-1, -1]]), ints([0] * 70), ints([0] * 70)
    ops.block_tables(table, slots, pos, ints([0, 0]), ints([0]), ints([0]), ints([0]), ints([70]), ints([1 << 26, 1 << 24]), ints([2]), 64)
    assert table.tolist() == [[1 << 24, 1 << 26]]
    assert slots.tolist() == [(1 << 30) + t for t in range(64)] + [(1 << 31) - 1] * 6


@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 3), (3, 5, 200)])
def test_plain_selection(B, K, V):
    torch.manual_seed(V)
    z, prev, done = torch.randn(B * K, V), -torch.rand(B, K), torch.zeros(B, K, dtype=I32)
    if K > 2:
        done[:, 1], prev[:, 2] = 1, -math.inf
        z[0, 0], z[3] = math.nan, -math.inf
    s, t, p, e = torch.empty(B, K), *(torch.empty(B, K, dtype=I32) for _ in range(3))
    ops.beam_select(s, t, p, e, z, prev, done, V // 2)
    best, at = torch.sort(oracle.selected(z, prev, done, V // 2), dim=1, descending=True, stable=True)
    n = min(K, K * V)
    assert torch.equal(p[:, :n].long() * V + t[:, :n].long(), at[:, :n]) and torch.allclose(s[:, :n].double(), best[:, :n], atol=1e-5)


def test_generation_entry_points_have_one_signature():
    """What ctypes declares, what the extension module calls and what the kernel library's sources define are the same, parameter by parameter."""
    from ml_b200 import build
    from ml_b200.ops import native
    assert native.bridge().generation_signatures() == {"mlb_" + k: v for k, v in native._GEN_KINDS.items()}
    letter = {"void*": "p", "float*": "f", "int*": "i", "uint8_t*": "u", "int": "n", "long": "l", "float": "d", "cudaStream_t": "s"}
    defined = {}
    for src in (build.CSRC / "kernels").glob("*.cu"):
        for name, args in re.findall(r"^MLB_API [\w ]+? (mlb_\w+)\(([^)]*)\)", src.read_text(), re.M):
            types = [re.sub(r"\s*\w+$", "", a.replace("const ", "").strip()).replace(" *", "*") for a in args.split(",")]
            defined[name] = "".join(letter.get(t, "?") for t in types)
    for name, kinds in native._GEN_KINDS.items():
        assert len(defined["mlb_" + name]) == len(kinds), name
        assert all(d == k or (d == "p" and k in "bfiu") for d, k in zip(defined["mlb_" + name], kinds)), name


def test_entries_refuse_addresses_off_16_bytes():
    """The kernels read and write 16 bytes at a time: -7, before anything is launched (without a device a launch answers with another code)."""
    from ml_b200.ops import native
    if torch.cuda.is_available():
        pytest.skip("the addresses are nobody's memory: asked only where no kernel can run")
    L, ok, off = native.lib(), 1 << 20, (1 << 20) + 2
    append = lambda **kw: L.mlb_kv4_append(*{**dict(pages=ok, q=ok, qkv=ok, slots=ok, pos=ok, cos=ok, sin=ok), **kw}.values(), 4, 16, 3, 512, 4, 2, 64, 9, None)
    read = lambda **kw: L.mlb_kv4_read(*{**dict(k=ok, v=ok, pages=ok, slots=ok), **kw}.values(), 4, 16, 3, 2, 64, None)
    attn = lambda **kw: L.mlb_kv4_attn(*{**dict(out=ok, lse=None, q=ok, pages=ok, table=ok, lens=ok, part=ok, count=ok), **kw}.values(), 4, 256, 1, 1, 4, 2, 64, 1, 16, 0.125, None)
    order = lambda **kw: L.mlb_beam_reorder(*{**dict(pages=ok), **kw}.values(), *[ok] * 9, 1, 4, 2, 16, 18 * 64, 1, 2, 2, 9, None)
    for call, names in ((append, ("pages", "q", "qkv", "cos", "sin")), (read, ("k", "v", "pages")), (attn, ("out", "q", "pages", "part")), (order, ("pages",))):
        assert call() > 0      # (no device)
        for name in names:
            assert call(**{name: off}) == -7, name


@pytest.mark.parametrize("B,Tq,H,Hkv,hd", [(8, 1024, 32, 8, 128), (1, 8192, 32, 8, 128), (2, 5000, 4, 4, 32), (64, 300, 12, 4, 96), (2100, 16, 8, 2, 64)])
def test_attention_workspace_is_that_of_the_blocks_that_run(B, Tq, H, Hkv, hd):
    """Two shares a thread block, of which all tiles of rows together have no more than the machine holds (8 an SM at most) and one more a tile."""
    from ml_b200.ops import native
    L, rows = native.lib(), H // Hkv * Tq
    tiles, share = -(-rows // 16), 16 * (hd + 2)
    for width in (1, 3, 512):
        got = L.mlb_kv4_attn_scratch(B, Tq, H, Hkv, hd, width, 16)
        assert tiles * 2 * share <= got <= (8 * 148 + tiles) * 2 * share


def test_attention_entries_refuse_no_tokens_and_no_heads():
    """... with their code, and do not divide by what there is none of."""
    from ml_b200.ops import native
    L, ok = native.lib(), 1 << 20
    for Tq, H, Hkv in ((0, 4, 2), (1, 0, 2), (-1, 4, 2), (1, 4, 0)):
        assert L.mlb_kv4_attn_scratch(1, Tq, H, Hkv, 64, 1, 16) == -7
        if not torch.cuda.is_available():
            assert L.mlb_kv4_attn(ok, None, ok, ok, ok, ok, ok, ok, 4, 256, 1, Tq, H, Hkv, 64, 1, 16, 0.125, None) == -7


@pytest.mark.parametrize("scale", [2e38, -1e300, math.inf, math.nan])
def test_scales_past_32_bits_are_refused(scale):
    """A kernel has the scale times log2 e as an fp32 number: one that becomes infinite there is none."""
    x, pages = torch.zeros(1, 64), torch.zeros(4, 1, 1, 18 * 64, dtype=torch.uint8)
    with pytest.raises(ValueError, match="scale"):
        ops.kv4_attn(torch.empty_like(x), None, x, pages, ints([[0]]), ints([1]), 1, 1, 1, 64, scale)
    ops.kv4_attn(torch.empty_like(x), None, x, pages, ints([[0]]), ints([1]), 1, 1, 1, 64, 2.0 ** 127)


def test_tensors_off_16_bytes_are_refused_by_name():
    """Views that begin in the middle of a buffer, before anything else is asked of them."""
    from ml_b200.ops import native_gen
    bf, hd = torch.bfloat16, 64
    whole = lambda *s, dtype=bf: torch.zeros(*s, dtype=dtype)
    off = lambda t: torch.zeros(t.numel() + 1, dtype=t.dtype)[1:].view(t.shape)
    pages, x, slots, pos = whole(4, 2, 1, 18 * hd, dtype=torch.uint8), whole(3, 8 * hd), ints([0, 1, 2]), ints([0, 1, 2])
    a = dict(pages=pages, q_out=whole(3, 4 * hd), qkv=x, slots=slots, pos=pos, cos=whole(9, hd // 2, dtype=torch.float32), sin=whole(9, hd // 2, dtype=torch.float32))
    r = dict(k=whole(3, 2 * hd), v=whole(3, 2 * hd), pages=pages, slots=slots)
    t = dict(out=whole(1, 4 * hd), lse=None, q=whole(1, 4 * hd), pages=pages, table=ints([[0]]), lens=ints([1]))
    calls = ((lambda **kw: native_gen.kv4_append(**{**a, **kw}, H=4, Hkv=2, hd=hd), a, ("q_out", "cos", "sin")),
             (lambda **kw: native_gen.kv4_read(**{**r, **kw}), r, ("k", "v")),
             (lambda **kw: native_gen.kv4_attn(**{**t, **kw}, Tq=1, H=4, Hkv=2, hd=hd), t, ("out",)))
    for call, args, names in calls:
        for name in names:
            view = off(args[name])
            assert view.is_contiguous() and view.data_ptr() % 16
            with pytest.raises(ValueError, match=rf"\b{name}\b.*16-byte"):
                call(**{name: view})


# ------------------------------------------------------------------ the whole path
def small(V=50, T=80, hd=32, H=2, L=2):
    g = GPT(Config(V=V, C=H * hd, L=L, H=H, I=48, T=T), 2, "cpu")
    g.init_weights(3)
    g.master.mul_(5)
    return g


def test_generate_from_the_cache_on_cpu():
    """The first token is the uncached one (the prompt's attention is over unrounded keys and values); pages of any size and batches give the same tokens."""
    g = small()
    torch.manual_seed(0)
    prompt = torch.randint(0, 50, (3, 21))
    assert torch.equal(g.generate(prompt[:2], 1), g.generate(prompt[:2], 1, kv="4bit"))
    a = g.generate(prompt, 20, kv="4bit", page=16)
    assert a.shape == (3, 41) and torch.equal(a, g.generate(prompt, 20, kv="4bit", page=64)) and torch.equal(a[2:], g.generate(prompt[2:], 20, kv="4bit"))
    s = [g.generate(prompt, 6, temperature=1.0, top_k=4, seed=5, kv="4bit") for _ in range(2)]
    assert torch.equal(s[0], s[1])


def test_a_step_from_the_cache_is_the_uncached_pass_over_what_the_cache_holds():
    """One layer: a step's logits against the model restated with the cached keys and values as they were read back."""
    g = small(L=1)
    c = g.cfg
    torch.manual_seed(1)
    P = 19
    ids = torch.randint(0, 50, (1, P + 1)).int()
    m = generation.CachedDecoder(g, 1, P + 1, 16)
    slots, _, _ = m.cache.grow(ints([P]), P)
    m.prompt(ids[:, :P].contiguous(), slots)
    logits = m.step(ids[:, P].contiguous())
    at = torch.arange(P + 1)
    k, v = torch.empty(P + 1, c.C), torch.empty(P + 1, c.C)
    ops.kv4_read(k, v, m.cache.pages[0], (m.cache.table[0][at // 16] * 16 + at % 16).int())
    o = g.layout.layer(0)
    x = g.P(g.layout.off_wte, c.V, c.C)[ids[0, P].long()]
    n = lambda t, w: t * torch.rsqrt(t.pow(2).mean() + c.eps) * w
    q = g.P(o.qkv, 3 * c.C, c.C)[:c.C] @ n(x, g.P(o.ln1, c.C))
    a, b = q.view(c.H, c.hd).chunk(2, -1)
    q = torch.cat([a * g.cos[P] - b * g.sin[P], b * g.cos[P] + a * g.sin[P]], -1)
    p = torch.softmax(torch.einsum("hd,thd->ht", q, k.view(-1, c.H, c.hd)) / math.sqrt(c.hd), -1)
    x = x + g.P(o.o, c.C, c.C) @ torch.einsum("ht,thd->hd", p, v.view(-1, c.H, c.hd)).reshape(-1)
    gu = g.P(o.gate, 2 * c.I, c.C) @ n(x, g.P(o.ln2, c.C))
    x = x + g.P(o.down, c.C, c.I) @ (torch.nn.functional.silu(gu[:c.I]) * gu[c.I:])
    want = g.P(g.layout.off_lm, c.V, c.C) @ n(x, g.P(g.layout.off_lnf, c.C))
    assert torch.allclose(logits[0], want, atol=1e-3 * float(want.abs().max()))


@pytest.mark.parametrize("page,P", [(16, 21), (16, 32), (64, 5)])
def test_beam_search_on_cpu(page, P):
    """Every beam's log-probability is the sum of those its own tokens get through a cache without beams, and one beam is greedy."""
    g = small()
    torch.manual_seed(P)
    prompt = torch.randint(0, 50, (2, P))
    n, K = 20, 3
    hist, scores = generation.beam_search(g, prompt, n, K, page=page)
    rows = hist.view(2 * K, -1)
    m = generation.CachedDecoder(g, 2 * K, P + n, 32)
    slots, _, _ = m.cache.grow(torch.full((2 * K,), P, dtype=I32), 2 * K * P)
    logits, total = m.prompt(rows[:, :P].int().contiguous(), slots), torch.zeros(2 * K)
    for t in range(P, P + n):
        total += torch.log_softmax(logits, -1).gather(1, rows[:, t:t + 1]).view(-1)
        if t + 1 < P + n:
            logits = m.step(rows[:, t].int().contiguous())
    assert torch.allclose(scores.view(-1), total, atol=1e-3) and (scores[:, :-1] >= scores[:, 1:]).all()
    assert torch.equal(generation.beam_search(g, prompt, n, 1, page=page)[0][:, 0], g.generate(prompt, n, kv="4bit", page=page))
    assert torch.equal(g.generate(prompt, n, kv="4bit", beams=K, page=page), hist[:, 0])


@pytest.mark.parametrize("V,K", [(3, 4), (4, 4), (8, 4), (2, 9)])
@pytest.mark.parametrize("P", [5, 16, 20, 48])
def test_beam_search_with_more_beams_than_continuations(V, K, P):
    """A first step that has fewer continuations than beams leaves rows on beams that are none: those hold the prompt as well, shorter than a page, as long as one
    and longer.  What is kept in the end are the best continuations; enough beams keep them all."""
    g = small(V=V)
    torch.manual_seed(V + P)
    prompt = torch.randint(0, V, (2, P))
    n = 3
    hist, scores = generation.beam_search(g, prompt, n, K, page=16)
    assert hist.shape == (2, K, P + n) and torch.equal(hist[:, :, :P], prompt[:, None].expand(2, K, P)) and not torch.isnan(scores).any()
    live = torch.isfinite(scores)
    assert live.sum(1).tolist() == [min(K, V ** n)] * 2
    m = generation.CachedDecoder(g, 2 * K, P + n, 32)
    rows = hist.view(2 * K, -1)
    slots, _, _ = m.cache.grow(torch.full((2 * K,), P, dtype=I32), 2 * K * P)
    logits, total = m.prompt(rows[:, :P].int().contiguous(), slots), torch.zeros(2 * K)
    for t in range(P, P + n):
        total += torch.log_softmax(logits, -1).gather(1, rows[:, t:t + 1]).view(-1)
        if t + 1 < P + n:
            logits = m.step(rows[:, t].int().contiguous())
    assert torch.allclose(scores.view(-1)[live.view(-1)], total[live.view(-1)], atol=1e-3)


@pytest.mark.parametrize("beams", [1, 3])
def test_generation_asks_for_the_kernels_errors_once_at_its_end(monkeypatch, beams):
    asked = []
    monkeypatch.setattr(generation.CachedDecoder, "check", lambda self: asked.append(len(steps)), raising=False)
    steps, step = [], generation.CachedDecoder.step
    monkeypatch.setattr(generation.CachedDecoder, "step", lambda self, ids: steps.append(1) or step(self, ids))
    g = small()
    g.generate(torch.zeros(1, 10, dtype=torch.long), 4, kv="4bit", beams=beams)
    assert asked == [3]


def test_an_error_word_is_raised_in_words_and_cleared(monkeypatch):
    from ml_b200.ops import native
    words = [3 << 24 | 0xC1]
    monkeypatch.setattr(native, "get_error", lambda: words[0])
    monkeypatch.setattr(native, "clear_error", lambda: words.__setitem__(0, 0))
    with pytest.raises(RuntimeError, match="page outside the pool"):
        native.raise_error("generation")
    native.raise_error("generation")


@pytest.mark.parametrize("kv", [None, "4bit"])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_eos_ends_a_single_continuation_too(kv, temperature):
    """What follows the first eos is eos, and what stands before it is what comes without one."""
    g = small()
    torch.manual_seed(4)
    prompt = torch.randint(0, 50, (2, 12))
    kw = dict(kv=kv, temperature=temperature, seed=6)
    free = g.generate(prompt, 20, **kw)
    eos = int(free[0, 16])
    ended = g.generate(prompt, 20, eos=eos, **kw)
    for r, (a, b) in enumerate(zip(free[:, 12:].tolist(), ended[:, 12:].tolist())):
        n = a.index(eos) if eos in a else 20
        assert b[:n] == a[:n] and set(b[n:]) <= {eos}, r
    assert not torch.equal(free, ended) or set(free[0, 16:].tolist()) == {eos}
    assert torch.equal(g.generate(prompt, 20, **kw), free)
    if kv and not temperature:
        assert torch.equal(generation.beam_search(g, prompt, 20, 1, eos=eos)[0][:, 0], ended)


def test_generate_refuses_what_the_cache_has_not():
    g = small()
    p = torch.zeros(1, 10, dtype=torch.long)
    for kw in (dict(kv="8bit"), dict(beams=2), dict(kv="4bit", beams=2, temperature=1.0), dict(kv="4bit", page=48), dict(kv="4bit", beams=33)):
        with pytest.raises(ValueError):
            g.generate(p, 4, **kw)
    with pytest.raises(ValueError):
        g.generate(p, 71, kv="4bit")
    odd = GPT(Config(V=50, C=32, L=1, H=2, I=48, T=40), 1, "cpu")      # head size 16
    odd.init_weights(1)
    with pytest.raises(ValueError, match="head size"):
        odd.generate(p, 2, kv="4bit")


@pytest.mark.parametrize("page", [-64, 0, 8, 24, 48, 100, 256])
def test_pages_of_other_sizes_are_refused_before_anything_is_laid_out(page):
    """A pool cut down to whole blocks would not be the one that slots are counted in."""
    with pytest.raises(ValueError, match="pages of"):
        generation.Cache4(1, 1, 100, 1, 64, page)
    with pytest.raises(ValueError, match="pages of"):
        small().generate(torch.zeros(1, 10, dtype=torch.long), 4, kv="4bit", page=page)


def test_no_beam_is_refused():
    for n in (0, 4):
        with pytest.raises(ValueError, match="0 beams"):
            small().generate(torch.zeros(1, 10, dtype=torch.long), n, kv="4bit", beams=0)


@pytest.mark.parametrize("B,K,V,eos", [(2, 5, 1, 0), (2, 32, 3, -1), (1, 4, 2, 7)])
def test_plain_selection_over_fewer_tokens_than_beams(B, K, V, eos):
    torch.manual_seed(K)
    z, prev, done = torch.randn(B * K, V), torch.randn(B, K), (torch.rand(B, K) < 0.5).int()
    z[0] = float("-inf")
    got = torch.empty(B, K), ints([[9] * K] * B), ints([[9] * K] * B), ints([[9] * K] * B)
    ops.beam_select(*got, z, prev, done, eos)
    assert ((0 <= got[1]) & (got[1] < V) & (0 <= got[2]) & (got[2] < K)).all() and not torch.isnan(got[0]).any()
    flat = got[2].long() * V + got[1]
    assert all(len(set(r)) == K for r in flat.tolist())


def test_generate_mode_reads_the_cache(tmp_path):
    import os
    import subprocess
    import sys
    env = dict(os.environ, ENTROPY_V="64", ENTROPY_C="64", ENTROPY_L="1", ENTROPY_H="2", ENTROPY_I="48", ENTROPY_T="32")
    from ml_b200.utils import ckpt as ck
    g = GPT(Config(V=64, C=64, L=1, H=2, I=48, T=32), 1, "cpu")
    g.init_weights(2)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    from ml_b200.trainer import Trainer
    t = Trainer(Config(V=64, C=64, L=1, H=2, I=48, T=32), B=1, device="cpu", lr=1e-3, wd=0.0)
    t.save_checkpoint(str(tmp_path / "ck"), step=1, loss=1.0)
    run = lambda *a: subprocess.run([sys.executable, "-m", "ml_b200.gpt", "generate", "--ckpt-dir", str(tmp_path / "ck"), "--prompt", "5 17 20", "--n", "6", *a],
                                    cwd=root, env=env, capture_output=True, text=True)
    for a in (("--kv", "4bit"), ("--kv", "4bit", "--beams", "3", "--eos", "2", "--page", "16")):
        r = run(*a)
        assert r.returncode == 0, r.stderr
        assert len(r.stdout.strip().splitlines()[-1].split()) == 9
