"""Kernels of generation (4-bit key / value cache, block tables, beams) against the definitions in 64 bits."""
import math

import numpy as np
import pytest
import torch

from ml_b200 import ops
from ml_b200.ops import ref
from tests import generation_oracle as oracle

pytestmark = pytest.mark.gpu
I32 = torch.int32


def dev():
    return torch.device("cuda:0")


def nat():
    from ml_b200.ops import native
    return native


@pytest.fixture(autouse=True)
def no_errors():
    yield
    torch.cuda.synchronize()
    err = nat().get_error()
    nat().clear_error()
    assert err == 0, nat().describe_error(err)


def raised(detail):
    """The error word says that an index was out of range, and where; it is cleared."""
    torch.cuda.synchronize()
    err = nat().get_error()
    nat().clear_error()
    assert err == 3 << 24 | detail, hex(err)


def ints(x):
    return torch.tensor(x, dtype=I32, device=dev())


def special_rows(x):
    """Groups that the 4 bits treat apart: zeros, ties of sign, values too small for a scale, infinities and NaN, one large value."""
    g = x.view(-1, 32)
    g[0] = 0
    if len(g) > 8:
        g[1, 3], g[1, 17] = 6.0, -6.0
        g[1].clamp_(-6, 6)
        g[2] = 1e-38
        g[3, 5] = math.inf
        g[4, 9] = math.nan
        g[5, 31] = -1e30
        g[6] = 2.0 ** -100
        g[7] = -0.0
    return x


# ------------------------------------------------------------------ append, read
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("N,H,Hkv,page,rope,wide", [(1, 1, 1, 16, True, 0), (7, 3, 1, 32, True, 8), (33, 4, 2, 64, False, 0), (150, 2, 2, 128, True, 0), (64, 0, 5, 16, False, 24)])
def test_append_and_read(hd, N, H, Hkv, page, rope, wide):
    """Codes and scales are those of the definition to the bit (without a rotation the values are exact; with one they are rounded to fp32 operation by
    operation, as the plain form does), other slots stay as they were, and reading gives (c - 8) s."""
    torch.manual_seed(hd + N)
    T, n_pages = 50, -(-N // page) + 2
    W = (H + 2 * Hkv) * hd
    x = torch.randn(N, W) * 3
    kv = special_rows(x[:, H * hd:].contiguous()) if not rope else x[:, H * hd:]
    x = torch.cat([x[:, :H * hd], kv], 1).bfloat16()
    buf = torch.zeros(N, W + wide, dtype=torch.bfloat16, device=dev())
    buf[:, :W] = x.to(dev())
    slots = torch.randperm(n_pages * page)[:N].int()
    if N > 5:
        slots[3] = -1
    pos = torch.randint(0, T, (N,)).int()
    cos, sin = ref.rope_tables(T, hd, 10000.0, "cpu")
    pages = torch.randint(0, 256, (n_pages, Hkv, page // 16, 18 * hd), dtype=torch.uint8)
    want, qw = pages.clone(), torch.zeros(N, H * hd, dtype=torch.bfloat16)
    args = (pos, cos, sin) if rope else (None, None, None)
    ref.kv4_append(want, qw, x, slots, *args, H, Hkv, hd)
    got, q = pages.to(dev()), torch.zeros(N, H * hd, dtype=torch.bfloat16, device=dev())
    ops.kv4_append(got, q if H else None, buf[:, :W], slots.to(dev()), *(a if a is None else a.to(dev()) for a in args), H, Hkv, hd)
    assert torch.equal(got.cpu(), want) and torch.equal(q.cpu(), qw)
    # the definition, apart from the plain form
    kc, vc, ks, vs = oracle.block_fields(got)
    v = x[:, (H + Hkv) * hd:].double().numpy().reshape(N, Hkv, hd)
    k = x[:, H * hd:(H + Hkv) * hd].double().numpy().reshape(N, Hkv, hd)
    for n in range(N):
        s = int(slots[n])
        if s < 0:
            continue
        at = (s // page, slice(None), s % page // 16, s % 16)
        for codes, scales, val in ((vc, vs, v),) if rope else ((vc, vs, v), (kc, ks, k)):
            c, sc = oracle.quantised(val[n])
            assert np.array_equal(codes[at], c) and np.array_equal(scales[at], sc, equal_nan=True)
        if rope:
            r = oracle.rotated(k[n:n + 1], cos[pos[n:n + 1].long()].double().numpy(), sin[pos[n:n + 1].long()].double().numpy())[0]
            held = oracle.values(kc[at], ks[at])
            step = np.abs(np.repeat(ks[at], 32, -1))
            assert (np.abs(held - r) <= step * (0.5 + 2.0 ** -7) + np.where(kc[at] == 15, step, 0)).all()      # (7 is the last step up; bf16 scale)
    rk, rv = (torch.empty(N, Hkv * hd, dtype=torch.bfloat16, device=dev()) for _ in range(2))
    ops.kv4_read(rk, rv, got, slots.to(dev()))
    for r, codes, scales in ((rk, kc, ks), (rv, vc, vs)):
        for n in range(N):
            s = int(slots[n])
            want_row = np.zeros((Hkv, hd)) if s < 0 else oracle.values(codes, scales)[s // page, :, s % page // 16, s % 16]
            assert torch.equal(r[n].cpu().nan_to_num(nan=7.0), torch.from_numpy(want_row).float().bfloat16().view(-1).nan_to_num(nan=7.0))


def test_append_skips_and_reports_what_lies_outside():
    hd, pages = 64, torch.zeros(2, 1, 1, 18 * 64, dtype=torch.uint8, device=dev())
    x = torch.randn(3, 3 * hd, device=dev()).bfloat16()
    cos, sin = ref.rope_tables(8, hd, 10000.0, dev())
    ops.kv4_append(pages, None, x, ints([-1, 32, -5]), ints([0, 1, 2]), cos, sin, 1, 1, hd)
    raised(0xC2)
    assert int(pages.sum()) == 0
    ops.kv4_append(pages, None, x, ints([0, -1, -1]), ints([8, 0, 0]), cos, sin, 1, 1, hd)
    raised(0xC3)
    k, v = (torch.ones(1, hd, dtype=torch.bfloat16, device=dev()) for _ in range(2))
    ops.kv4_read(k, v, pages, ints([32]))
    raised(0xC2)
    assert int(k.abs().sum()) == 0 and int(v.abs().sum()) == 0
    ops.kv4_append(pages, None, x[:0], ints([]), None, None, None, 1, 1, hd)
    ops.kv4_read(k[:0], v[:0], pages, ints([]))


# ------------------------------------------------------------------ attention
def attend(lens, Tq, H, Hkv, hd, page, seed, extra=0, spread=1.0, scale=None, wide=0, spoil=True):
    """Random cache and queries; (kernel's out, lse) and the oracle's with its bounds."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    width = max(1, max(-(-n // page) for n in lens)) + extra
    used = [-(-n // page) for n in lens]
    n_pages = sum(used) + 2
    pages = oracle.random_pages(n_pages, Hkv, page, hd, seed, spread)
    order = torch.randperm(n_pages, generator=g).tolist()
    table = np.full((B, width), -1, dtype=np.int64)
    for b in range(B):
        for p in range(used[b]):
            table[b, p] = order.pop()
    dirty = pages.clone()
    if spoil:      # what no query sees is anything: NaN scales behind every sequence's end
        for b in range(B):
            for t in range(lens[b], used[b] * page):
                blk = dirty[table[b, t // page], :, t % page // 16]
                ng = hd // 32
                for a in (16, 17):
                    blk[:, a * hd + t % 16 * 2 * ng:a * hd + (t % 16 + 1) * 2 * ng] = 0xFF
    q = torch.randn(B * Tq, H * hd, generator=g).bfloat16()
    buf = torch.zeros(B * Tq, H * hd + wide, dtype=torch.bfloat16, device=dev())
    buf[:, :H * hd] = q.to(dev())
    out = torch.full((B * Tq, H * hd), 7.0, dtype=torch.bfloat16, device=dev())
    lse = torch.full((B, H, Tq), 7.0, device=dev())
    args = (dirty.to(dev()), ints(table.tolist()), ints(lens), Tq, H, Hkv, hd)
    ops.kv4_attn(out, lse, buf[:, :H * hd], *args, scale)
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    ops.kv4_attn(again, lse2, buf[:, :H * hd], *args, scale)
    assert torch.equal(out, again) and torch.equal(lse, lse2)      # shares are put together in one order
    o, l, tol, ltol = oracle.attention(q, pages, table, lens, Tq, H, Hkv, hd, scale)
    return out.cpu().double().numpy().reshape(o.shape), lse.cpu().double().numpy(), o, l, tol, ltol


def close(got, lse, o, l, tol, ltol):
    assert (np.abs(got - o) <= tol).all(), np.max(np.abs(got - o) - tol)
    assert np.array_equal(np.isinf(lse), np.isinf(l))
    f = np.isfinite(l)
    assert (np.abs(lse[f] - l[f]) <= ltol[f]).all()


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("lens,Tq,H,Hkv,page", [
    ([1], 1, 1, 1, 16), ([0, 15, 16, 17, 0], 1, 2, 2, 16), ([100, 63, 64, 65], 1, 8, 1, 64), ([300], 1, 6, 2, 32), ([5, 130], 3, 4, 4, 128),
    ([2, 1, 0, 40], 4, 6, 2, 16), ([33, 200], 5, 8, 2, 32), ([70], 1, 17, 1, 64), ([48, 9], 9, 4, 2, 16)])
def test_attention(hd, lens, Tq, H, Hkv, page):
    """Empty sequences, fewer tokens than queries (their first rows see nothing), lengths around blocks and pages, one to 18 rows a key / value head."""
    close(*attend(lens, Tq, H, Hkv, hd, page, seed=hd + H))


@pytest.mark.parametrize("lens,Tq,H,Hkv,hd,page", [([6001], 1, 3, 3, 64, 64), ([2500, 1, 4003], 2, 8, 2, 128, 16), ([3000], 7, 4, 1, 96, 128)])
def test_attention_over_long_sequences(lens, Tq, H, Hkv, hd, page):
    """Heads whose blocks many thread blocks share."""
    close(*attend(lens, Tq, H, Hkv, hd, page, seed=3, extra=3))


def test_attention_of_strided_queries_with_a_scale():
    close(*attend([90, 31], 2, 4, 2, 64, 32, seed=5, wide=136, scale=0.3))
    close(*attend([90, 31], 1, 4, 2, 64, 32, seed=6, scale=-0.2))
    close(*attend([90, 31], 1, 4, 2, 64, 32, seed=6, scale=0.0))


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("size,scale", [(0.0, 1e-12), (1e-30, 1e-13), (1.0, 1e-30), (1.0, -1e-42), (0.0, 1e-45)])
def test_attention_with_scales_that_leave_nothing_of_scores(hd, size, scale):
    """Scores of 0 or next to it: seen tokens count alike, the others, in the last block and behind a query's own token, not at all."""
    lens, Tq, H, Hkv, page = [20, 37, 2], 3, 4, 2, 16
    pages = oracle.random_pages(6, Hkv, page, hd, 11)
    table = np.array([[0, 1, 0], [2, 3, 4], [5, 0, 0]])
    q = (torch.randn(len(lens) * Tq, H * hd, generator=torch.Generator().manual_seed(hd)) * size).bfloat16()
    out, lse = torch.empty_like(q, device=dev()), torch.empty(len(lens), H, Tq, device=dev())
    ops.kv4_attn(out, lse, q.to(dev()), pages.to(dev()), ints(table.tolist()), ints(lens), Tq, H, Hkv, hd, scale)
    o, l, tol, ltol = oracle.attention(q, pages, table, lens, Tq, H, Hkv, hd, scale)
    close(out.cpu().double().numpy().reshape(o.shape), lse.cpu().double().numpy(), o, l, tol, ltol)


def test_attention_with_large_scores():
    """Scores in the hundreds: most weights vanish, the running maximum moves block by block."""
    close(*attend([500, 37], 1, 4, 2, 64, 32, seed=8, spread=30.0))


@pytest.mark.parametrize("B", [2047, 2049, 5000])
def test_attention_of_more_sequences_than_a_launch_takes(B):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 20, (B,), generator=g).tolist()
    close(*attend(lens, 1, 1, 1, 32, 16, seed=1, spoil=False))


def test_attention_of_many_sequences_at_head_size_128():
    """More sequences than leave room for a third thread block's ring on an SM, short and long ones, empty ones among them."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 40, (700,), generator=g).tolist()
    lens[13], lens[500] = 1500, 900
    close(*attend(lens, 1, 2, 1, 128, 64, seed=2, spoil=False))


def test_attention_of_no_sequence_and_without_lse():
    pages = oracle.random_pages(1, 1, 16, 64, 0).to(dev())
    ops.kv4_attn(torch.empty(0, 64, dtype=torch.bfloat16, device=dev()), None, torch.empty(0, 64, dtype=torch.bfloat16, device=dev()), pages, ints([]).view(0, 1), ints([]), 1, 1, 1, 64)
    out = torch.empty(1, 64, dtype=torch.bfloat16, device=dev())
    ops.kv4_attn(out, None, torch.ones_like(out), pages, ints([[0]]), ints([1]), 1, 1, 1, 64)
    kc, vc, ks, vs = oracle.block_fields(pages)
    assert torch.equal(out.cpu().view(-1), torch.from_numpy(oracle.values(vc, vs)[0, 0, 0, 0]).float().bfloat16())


def test_attention_reports_pages_and_lengths_outside():
    """A page that is none of the pool's is left out, a length past the table's row is cut to it."""
    hd, page = 64, 16
    pages = oracle.random_pages(3, 1, page, hd, 2)
    q = torch.randn(1, hd).bfloat16()
    out, lse = torch.empty(1, hd, dtype=torch.bfloat16, device=dev()), torch.empty(1, 1, 1, device=dev())
    for bad in (-1, 3, 2 ** 31 - 1, -2 ** 31):
        ops.kv4_attn(out, lse, q.to(dev()), pages.to(dev()), ints([[0, bad, 2]]), ints([48]), 1, 1, 1, hd)
        raised(0xC1)
        o, l, tol, ltol = oracle.attention(q, pages, np.array([[0, 2]]), [32], 1, 1, 1, hd)
        close(out.cpu().double().numpy().reshape(o.shape), lse.cpu().double().numpy(), o, l, tol, ltol)
    ops.kv4_attn(out, lse, q.to(dev()), pages.to(dev()), ints([[0, 2]]), ints([33]), 1, 1, 1, hd)
    raised(0xC4)
    o, l, tol, ltol = oracle.attention(q, pages, np.array([[0, 2]]), [32], 1, 1, 1, hd)
    close(out.cpu().double().numpy().reshape(o.shape), lse.cpu().double().numpy(), o, l, tol, ltol)


def test_nan_and_infinity_reach_the_rows_that_see_them_and_no_others():
    hd, page, Tq = 64, 16, 3
    pages = oracle.random_pages(1, 1, page, hd, 4)
    ng, nan = hd // 32, 0x7FC0
    blk = pages[0, 0, 0]
    for a in (16, 17):      # token 9, seen by the last of three queries alone
        blk[a * hd + 9 * 2 * ng:a * hd + 10 * 2 * ng] = torch.tensor([nan & 255, nan >> 8] * ng, dtype=torch.uint8)
    q = torch.randn(Tq, hd).bfloat16()
    out, lse = torch.empty(Tq, hd, dtype=torch.bfloat16, device=dev()), torch.empty(1, 1, Tq, device=dev())
    ops.kv4_attn(out, lse, q.to(dev()), pages.to(dev()), ints([[0]]), ints([10]), Tq, 1, 1, hd)
    assert torch.isfinite(out[:2]).all() and torch.isfinite(lse[0, 0, :2]).all() and torch.isnan(out[2]).all() and torch.isnan(lse[0, 0, 2])
    o, l, tol, ltol = oracle.attention(q[:2], pages, np.array([[0]]), [9], 2, 1, 1, hd)
    close(out[:2].cpu().double().numpy().reshape(o.shape), lse[..., :2].cpu().double().numpy(), o, l, tol, ltol)


@pytest.mark.parametrize("lens,Tq,H,Hkv,hd,page", [([1000], 950, 8, 1, 32, 64), ([130, 0, 90], 120, 6, 2, 96, 16), ([300, 41], 40, 16, 2, 128, 32), ([200], 200, 3, 3, 64, 128)])
def test_attention_of_more_row_tiles_than_there_are_multiprocessors(lens, Tq, H, Hkv, hd, page):
    """Prompts' worth of new tokens: few thread blocks for each tile of rows, down to one."""
    close(*attend(lens, Tq, H, Hkv, hd, page, seed=7))


@pytest.mark.parametrize("B,T,Tq,H,Hkv,hd", [(1, 900, 1, 4, 4, 64), (16, 700, 1, 8, 4, 128), (3, 900, 40, 8, 2, 32), (2, 1300, 1300, 4, 2, 128), (2500, 20, 2, 2, 1, 64), (2049, 300, 9, 2, 1, 128)])
def test_attention_stays_in_its_workspace(B, T, Tq, H, Hkv, hd):
    """What the library says it wants is enough: nothing behind it is written, and the answer is the one of a call of the operator."""
    n, page = nat(), 64
    width = -(-T // page)
    pages = oracle.random_pages(width, Hkv, page, hd, 3).to(dev())
    table, lens = ints([list(range(width))]).repeat(B, 1), torch.randint(T // 2, T + 1, (B,), dtype=I32, device=dev())
    q = torch.randn(B * Tq, H * hd, device=dev()).bfloat16()
    want, got = torch.empty_like(q), torch.empty_like(q)
    ops.kv4_attn(want, None, q, pages, table, lens, Tq, H, Hkv, hd)
    e = n._entries()
    floats = e.mlb_kv4_attn_scratch(B, Tq, H, Hkv, hd, width, page)
    part = torch.full((floats + 65536,), 7.25, device=dev())
    count = torch.zeros(B * Hkv * (-(-H // Hkv * Tq // 8) + 1), dtype=I32, device=dev())
    n._chk(e.mlb_kv4_attn(got, n.NONE, q, pages, table, lens, part, count, width, q.stride(0), B, Tq, H, Hkv, hd, width, page, hd ** -0.5), "kv4_attn")
    torch.cuda.synchronize()
    assert bool((part[floats:] == 7.25).all()) and torch.equal(want, got) and int(count.abs().sum()) == 0


@pytest.mark.parametrize("hd,size", [(64, 1e9), (64, 3e10), (128, 1e11), (32, 1e20), (96, 1e36), (128, 1e36), (64, 1e-10), (128, 1e-20)])
@pytest.mark.parametrize("T,Tq,H", [(700, 1, 4), (90, 5, 8)])
def test_attention_over_values_of_any_size(hd, size, T, Tq, H):
    """Large ones, some tokens' among ordinary ones: weights times scales pass the range that the sums are kept in at first."""
    torch.manual_seed(hd)
    Hkv, page, n = 2, 32, -(-T // 32)
    pages, table, slots = torch.zeros(n, Hkv, page // 16, 18 * hd, dtype=torch.uint8, device=dev()), torch.randperm(n), torch.arange(T)
    qkv = torch.randn(T, 2 * Hkv * hd)
    v = qkv[:, Hkv * hd:]
    v *= size if size < 1 else torch.where(torch.rand(T, 1) < 0.1, size, 1.0)
    ops.kv4_append(pages, None, qkv.bfloat16().to(dev()), (table[slots // page] * page + slots % page).int().to(dev()), None, None, None, 0, Hkv, hd)
    q = torch.randn(Tq, H * hd).bfloat16()
    out, lse = torch.empty(Tq, H * hd, dtype=torch.bfloat16, device=dev()), torch.empty(1, H, Tq, device=dev())
    ops.kv4_attn(out, lse, q.to(dev()), pages, ints(table[None].tolist()), ints([T]), Tq, H, Hkv, hd)
    o, l, tol, ltol = oracle.attention(q, pages.cpu(), table[None].numpy(), [T], Tq, H, Hkv, hd)
    close(out.cpu().double().numpy().reshape(o.shape), lse.cpu().double().numpy(), o, l, tol, ltol)


@pytest.mark.parametrize("hd,size", [(32, 1e-22), (64, 1e-25), (96, 1e-30), (128, 1e-33), (64, 1e-33)])
@pytest.mark.parametrize("T,Tq,H", [(1, 1, 2), (16, 1, 4), (700, 1, 4), (90, 5, 8), (3000, 20, 4)])
@pytest.mark.parametrize("part", ["all", "group", "tokens"])
def test_attention_over_tiny_values(hd, size, T, Tq, H, part):
    """What the cache holds reaches the output, whatever its size: all values, those of one group of 32 beside ordinary ones, those of the first tokens.  (Held to the bound
    of the elements themselves; a scale's smallest number is 2^-120, half of what adding up may lose.)"""
    torch.manual_seed(hd + T)
    Hkv, page, n = 2, 32, -(-T // 32)
    pages, table, slots = torch.zeros(n, Hkv, page // 16, 18 * hd, dtype=torch.uint8, device=dev()), torch.randperm(n), torch.arange(T)
    qkv = torch.randn(T, 2 * Hkv * hd)
    v = qkv[:, Hkv * hd:].view(T, Hkv, hd)
    (v if part == "all" else v[:, 1, -32:] if part == "group" else v[:T // 3]).mul_(size)
    ops.kv4_append(pages, None, qkv.bfloat16().to(dev()), (table[slots // page] * page + slots % page).int().to(dev()), None, None, None, 0, Hkv, hd)
    q = torch.randn(Tq, H * hd).bfloat16()
    out, lse = torch.empty(Tq, H * hd, dtype=torch.bfloat16, device=dev()), torch.empty(1, H, Tq, device=dev())
    ops.kv4_attn(out, lse, q.to(dev()), pages, ints(table[None].tolist()), ints([T]), Tq, H, Hkv, hd)
    o, l, tol, ltol = oracle.attention(q, pages.cpu(), table[None].numpy(), [T], Tq, H, Hkv, hd)
    close(out.cpu().double().numpy().reshape(o.shape), lse.cpu().double().numpy(), o, l, tol, ltol)


def test_attention_over_values_that_are_zero():
    """Exact zeros stay zeros."""
    hd, T = 64, 90
    pages = torch.zeros(3, 1, 2, 18 * hd, dtype=torch.uint8, device=dev())
    kv = torch.randn(T, 2 * hd, device=dev()).bfloat16()
    kv[:, hd:] = 0
    ops.kv4_append(pages, None, kv, ints(list(range(T))), None, None, None, 0, 1, hd)
    out = torch.full((1, hd), 7.0, dtype=torch.bfloat16, device=dev())
    ops.kv4_attn(out, None, torch.randn(1, hd, device=dev()).bfloat16(), pages, ints([[0, 1, 2]]), ints([T]), 1, 1, 1, hd)
    assert bool((out == 0).all())


def test_cache_past_4_gigabytes():
    """Pages whose bytes lie past 2^32, written, read and attended to."""
    hd, page, Hkv = 128, 128, 8
    n = (1 << 32) // (Hkv * page // 16 * 18 * hd) + 20
    pages = torch.empty(n, Hkv, page // 16, 18 * hd, dtype=torch.uint8, device=dev())
    torch.manual_seed(0)
    N = 200
    x = torch.randn(N, 3 * Hkv * hd, device=dev()).bfloat16()
    slots = torch.cat([torch.arange(128) + (n - 1) * page, torch.arange(72) + (n - 2) * page]).int()
    ops.kv4_append(pages, None, x, slots.to(dev()), None, None, None, Hkv, Hkv, hd)
    k, v = (torch.empty(N, Hkv * hd, dtype=torch.bfloat16, device=dev()) for _ in range(2))
    ops.kv4_read(k, v, pages, slots.to(dev()))
    c, s = oracle.quantised(x[:, 2 * Hkv * hd:].double().cpu().numpy().reshape(N, Hkv, hd))
    assert torch.equal(v.cpu(), torch.from_numpy(oracle.values(c, s)).float().bfloat16().view(N, -1))
    q = torch.randn(1, Hkv * hd).bfloat16()
    out, lse = torch.empty(1, Hkv * hd, dtype=torch.bfloat16, device=dev()), torch.empty(1, Hkv, 1, device=dev())
    ops.kv4_attn(out, lse, q.to(dev()), pages, ints([[n - 1, n - 2]]), ints([N]), 1, Hkv, Hkv, hd)
    o, l, tol, ltol = oracle.attention(q, pages[n - 2:].cpu(), np.array([[1, 0]]), [N], 1, Hkv, Hkv, hd)
    close(out.cpu().double().numpy().reshape(o.shape), lse.cpu().double().numpy(), o, l, tol, ltol)


def test_attention_on_another_stream_and_in_a_graph():
    """Workspaces belong to the stream, replays read what the tensors hold then."""
    hd, page, lens = 64, 16, [700, 90]
    pages = oracle.random_pages(60, 2, page, hd, 9).to(dev())
    table = ints([list(range(44)), list(range(16, 60))])
    q = torch.randn(2, 4 * hd, device=dev()).bfloat16()
    n = ints(lens)
    run = lambda out: ops.kv4_attn(out, None, q, pages, table, n, 1, 4, 2, hd)
    a, b, c = (torch.empty(2, 4 * hd, dtype=torch.bfloat16, device=dev()) for _ in range(3))
    run(a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(b)
    side.synchronize()
    assert torch.equal(a, b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(c)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, c)
    q.mul_(2)
    n.copy_(ints([650, 91]))
    run(a)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, c)


# ------------------------------------------------------------------ block tables
@pytest.mark.parametrize("B,page,width,most_old,most_new,free,alias", [
    (1, 16, 4, 0, 5, 10, False), (3, 16, 4, 60, 9, 10, True), (64, 64, 20, 1000, 1, 64, False), (300, 16, 30, 0, 200, 900, True), (257, 5, 9, 40, 12, 300, False),
    (4096, 16, 3, 40, 3, 4000, True), (40, 128, 3, 380, 40, 0, False)])
def test_block_tables(B, page, width, most_old, most_new, free, alias):
    """Requests without new tokens, that outgrow their row, or that find no page any more; outputs that are inputs; pages of any size."""
    rng = np.random.default_rng(B + page)
    lens = rng.integers(0, most_old + 1, B).tolist()
    new = rng.integers(0, most_new + 1, B).tolist()
    held = [-(-n // page) for n in lens]
    ids = rng.permutation(sum(held) + free).tolist()
    stack = [ids.pop() for _ in range(free)]
    table = [[ids.pop() for _ in range(h)] + [-1] * (width - h) for h in held]
    rows = sum(new) + 3
    want = oracle.tables(table, lens, new, stack, free, page, rows)
    t, l, nf = ints(table), ints(lens), ints([free])
    slots, pos, starts = (torch.full((n,), 77, dtype=I32, device=dev()) for n in (rows, rows, B + 1))
    new_lens, left = (l, nf) if alias else (torch.empty_like(l), torch.empty_like(nf))
    stack_t = ints(stack + [5] * 3)      # more room than what is on the stack
    ops.block_tables(t, slots, pos, starts, new_lens, left, l, ints(new), stack_t, nf, page)
    got = (t.tolist(), slots.tolist(), pos.tolist(), starts.tolist(), new_lens.tolist(), int(left))
    for g, w, name in zip(got, want, ("table", "slots", "pos", "starts", "new_lens", "left")):
        assert g == w, name


def test_a_page_number_whose_slot_passes_32_bits_gets_a_slot_of_no_pool():
    """... and not another page's."""
    table, slots, pos = ints([[-1, -1]]), ints([0] * 70), ints([0] * 70)
    ops.block_tables(table, slots, pos, ints([0, 0]), ints([0]), ints([0]), ints([0]), ints([70]), ints([1 << 26, 1 << 24]), ints([2]), 64)
    assert table.tolist() == [[1 << 24, 1 << 26]]
    assert slots.tolist() == [(1 << 30) + t for t in range(64)] + [(1 << 31) - 1] * 6


def test_tables_past_32_bits_are_refused():
    x = torch.zeros(1, 64, dtype=torch.bfloat16, device=dev())
    pages = torch.zeros(4, 1, 8, 18 * 64, dtype=torch.uint8, device=dev())
    wide, other = (torch.zeros(1, 1 << 24, dtype=I32, device=dev()) for _ in range(2))
    calls = [lambda t: ops.kv4_attn(torch.empty_like(x), None, x, pages, t, ints([0]), 1, 1, 1, 64),
             lambda t: ops.block_tables(t, ints([0]), ints([0]), ints([0, 0]), ints([0]), ints([0]), ints([0]), ints([0]), ints([0]), ints([1]), 128),
             lambda t: ops.beam_reorder(pages[None], other[:, :t.shape[1]], ints([0]), ints([[0]]), t, ints([0]), ints([0]), ints([[0]]), ints([[0]]), ints([[0]]))]
    for f in calls:
        f(wide[:, :-1])
        with pytest.raises(ValueError, match="32-bit"):
            f(wide)


def test_block_tables_report_what_does_not_fit():
    def call(lens, new, places, n_free=4):
        t, s, p, st = torch.full((len(lens), 3), -1, dtype=I32, device=dev()), torch.zeros(places, dtype=I32, device=dev()), torch.zeros(places, dtype=I32, device=dev()), torch.zeros(len(lens) + 1, dtype=I32, device=dev())
        nl, left = torch.zeros(len(lens), dtype=I32, device=dev()), ints([0])
        ops.block_tables(t, s, p, st, nl, left, ints(lens), ints(new), ints([9, 8, 7, 6]), ints([n_free]), 16)
        return s.tolist(), nl.tolist(), int(left)

    assert call([-1, 0], [1, 2], 3) == ([96, 97, -1], [-1, 2], 3)
    raised(0xB1)
    assert call([0, 0], [-3, 2], 3) == ([96, 97, -1], [0, 2], 3)
    raised(0xB1)
    assert call([0, 0], [2 ** 31 - 1, 2], 3) == ([96, 97, -1], [0, 2], 3)
    raised(0xB1)
    assert call([0, 0], [2, 2], 3) == ([96, 97, -1], [2, 0], 3)
    raised(0xB2)
    assert call([0], [2], 2, n_free=5) == ([96, 97], [2], 3)
    raised(0xB1)


# ------------------------------------------------------------------ beam selection
def choose(logits, prev, done, eos, alias=False, stride=0):
    B, K = prev.shape
    buf = torch.zeros(B * K, logits.shape[1] + stride, dtype=logits.dtype, device=dev())
    buf[:, :logits.shape[1]] = logits.to(dev())
    p, d = prev.to(dev()), done.to(dev())
    scores, tokens, parents, ended = (p if alias else torch.empty_like(p)), torch.empty_like(d), torch.empty_like(d), (d if alias else torch.empty_like(d))
    ops.beam_select(scores, tokens, parents, ended, buf[:, :logits.shape[1]], p, d, eos)
    return scores.cpu(), tokens.cpu(), parents.cpu(), ended.cpu()


def check_choice(logits, prev, done, eos, **kw):
    """The 64-bit scores of what was chosen are the best ones, in order, up to the rounding of a 32-bit score (its magnitude times 2^-22: three roundings, a
    sum of exponentials off by 2^-21 and its logarithm); equal ones by index."""
    B, K = prev.shape
    V = logits.shape[1]
    scores, tokens, parents, ended = choose(logits, prev, done, eos, **kw)
    all_ = oracle.selected(logits, prev, done, eos)
    n = min(K, K * V)
    best, at = torch.sort(all_, dim=1, descending=True, stable=True)
    for b in range(B):
        flat = parents[b, :n].long() * V + tokens[b, :n].long()
        assert len(set(flat.tolist())) == n and int(flat.min()) >= 0 and int(flat.max()) < K * V
        for k in range(n):
            w, g = float(best[b, k]), float(all_[b, flat[k]])
            tol = 2.0 ** -20 * (abs(float(prev[b][torch.isfinite(prev[b])].abs().max() if torch.isfinite(prev[b]).any() else 0)) + 30 + abs(w)) if math.isfinite(w) else 0.0
            assert g == w or abs(g - w) <= tol, (b, k, g, w)
            assert float(scores[b, k]) == w or abs(float(scores[b, k]) - w) <= tol
            near = (all_[b] - w).abs() <= tol if math.isfinite(w) else all_[b] == w
            if int(near.sum()) == 1 or not math.isfinite(w):
                assert int(flat[k]) == int(at[b, k]), (b, k)
            assert int(ended[b, k]) == int(bool(done[b, parents[b, k]]) or int(tokens[b, k]) == eos)
        for k in range(n, K):
            assert float(scores[b, k]) == -math.inf and int(ended[b, k]) == 1
    return scores, tokens, parents, ended


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K,V,stride", [(1, 1, 1, 0), (1, 4, 3, 0), (2, 3, 50, 0), (3, 8, 1000, 8), (1, 4, 50304, 0), (5, 5, 12345, 1), (2, 32, 9001, 0), (9, 9, 777, 0), (1, 1, 100001, 3)])
def test_beam_select(dtype, B, K, V, stride):
    torch.manual_seed(V + K)
    logits = (torch.randn(B * K, V) * 3).to(dtype)
    prev = -10 * torch.rand(B, K)
    done = torch.zeros(B, K, dtype=I32)
    check_choice(logits, prev, done, V // 2, stride=stride)
    if K > 1:
        done[:, 1] = 1
        prev[0, 0] = -math.inf
        check_choice(logits, prev, done, V - 1, alias=True, stride=stride)
        first = torch.full((B, K), -math.inf)
        first[:, 0] = 0
        check_choice(logits, first, torch.zeros_like(done), -1, stride=stride)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_beam_select_of_equal_logits_masks_and_nan(dtype):
    """Ties by the lowest index, however many; masked tokens (-inf or the type's lowest value); rows that are masked whole; NaN; +inf."""
    low = torch.finfo(dtype).min
    V, K = 3000, 4
    prev, done = torch.tensor([[0.0, 0.0, -1.0, -2.0]]), torch.zeros(1, K, dtype=I32)
    same = torch.zeros(K, V).to(dtype)
    s, t, p, _ = choose(same, prev, done, -1)
    assert t.tolist() == [[0, 1, 2, 3]] and p.tolist() == [[0] * 4] and torch.allclose(s, torch.full((1, 4), -math.log(V)), atol=1e-6)
    z = torch.randn(K, V).to(dtype)
    z[:, 10:] = low
    check_choice(z, prev, done, 5)
    z[:, 10:] = -math.inf
    check_choice(z, prev, done, 5)
    z[:, 2:] = -math.inf      # fewer continuations than beams in a row
    check_choice(z, prev, done, 5)
    z[0] = -math.inf
    check_choice(z, prev, done, 5)
    z[1, 0] = math.nan
    check_choice(z, prev, done, 5)
    z[:] = -math.inf      # nothing at all: the first indices
    s, t, p, e = check_choice(z, prev, done, 2)
    assert t.tolist() == [[0, 1, 2, 3]] and e.tolist() == [[0, 0, 1, 0]]
    z = torch.randn(K, V).to(dtype)
    z[2, 7] = math.inf      # no logarithm of a sum: the beam has no continuation
    s, t, p, _ = check_choice(z, prev, done, 5)
    assert 2 not in p.tolist()[0]
    check_choice(z, torch.full((1, K), -math.inf), done, 5)
    check_choice(z, prev, torch.ones_like(done), 5)


@pytest.mark.parametrize("B,K,V,eos", [(2, 5, 1, 0), (2, 32, 3, -1), (1, 4, 2, 7), (3, 17, 16, 15)])
def test_beam_select_over_fewer_tokens_than_beams(B, K, V, eos):
    torch.manual_seed(K)
    logits, prev, done = torch.randn(B * K, V).bfloat16(), -10 * torch.rand(B, K), (torch.rand(B, K) < 0.5).int()
    logits[0] = -math.inf
    check_choice(logits, prev, done, eos)
    prev[:, 1:] = -math.inf
    check_choice(logits, prev, torch.zeros_like(done), eos)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K,V,stride", [(1, 32, 50304, 0), (2, 16, 70001, 7), (1000, 1, 300, 0), (3, 24, 40000, 0)])
def test_beam_select_of_pieces_that_are_fetched_in_parts(dtype, B, K, V, stride):
    """Many beams: few pieces, several fetches each, the bound moving from one to the next; and logits all alike in the second half, which leave no room for
    candidates there."""
    torch.manual_seed(V)
    logits = (torch.randn(B * K, V) * 3).to(dtype)
    prev, done = -10 * torch.rand(B, K), torch.zeros(B, K, dtype=I32)
    check_choice(logits, prev, done, 7, stride=stride)
    logits[:, V // 2:] = 20.0
    check_choice(logits, prev, done, 7, stride=stride)
    logits[:, -1] = 21.0
    check_choice(logits, prev, done, 7, stride=stride)


def rounded_scores(logits, prev, done, eos, lse_by=1.0):
    """Scores as 32-bit numbers, prev + (logit - lse) rounded operation by operation; lse from 64 bits, off by a factor."""
    B, K = prev.shape
    z = logits.float().view(B, K, -1)
    lse = torch.logsumexp(z.double(), -1, keepdim=True)
    s = prev[..., None] + (z - (lse * lse_by).float())
    s = torch.where((done != 0)[..., None], torch.where(torch.arange(z.shape[-1]) == eos, prev[..., None], -math.inf), s)
    return s.view(B, -1)


def check_ties(logits, prev, done, eos, stride=0):
    """The choice is that of the plain form, to the index: the largest 32-bit scores, equal ones by the lowest index.  (Inputs whose choice does not hang on a logarithm
    that is off by a few of its last bits.)"""
    B, K = prev.shape
    V = logits.shape[1]
    order = [torch.sort(rounded_scores(logits, prev, done, eos, 1 + e * 2.0 ** -22), dim=1, descending=True, stable=True).indices[:, :K] for e in (0, -2, -1, 1, 2)]
    assert all(torch.equal(order[0], o) for o in order[1:])
    plain = torch.empty(B, K), *(torch.empty(B, K, dtype=I32) for _ in range(3))
    ref.beam_select(*plain, logits, prev, done, eos)
    s, t, p, e = choose(logits, prev, done, eos, stride=stride)
    assert torch.equal(plain[2].long() * V + plain[1], order[0])
    assert torch.equal(p.long() * V + t, order[0]) and torch.equal(e, plain[3])


@pytest.mark.parametrize("B,K,V,stride", [(1, 1, 1000, 0), (2, 4, 3000, 0), (1, 4, 50304, 0), (3, 20, 9001, 1), (1, 32, 50304, 0), (40, 3, 20000, 0), (2, 16, 70001, 7)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("near", [3, 40, 900])
def test_beam_select_of_scores_that_rounding_makes_equal(dtype, B, K, V, stride, near):
    """Logits that differ, `near` of them so little beside a beam's large score that theirs are equal: the lowest indices, not the largest logits."""
    g = torch.Generator().manual_seed(V + K + near)
    logits = torch.full((B * K, V), -5.0)
    for r in range(B * K):
        at = torch.randperm(V, generator=g)[:near]
        step = 2.0 ** -26 if dtype == torch.bfloat16 else 2.0 ** -23
        logits[r, at] = (2.0 ** -12 if dtype == torch.bfloat16 else 1.0) + step * (128 // 8 if dtype == torch.bfloat16 else 1) * torch.randperm(near, generator=g) % 2.0 ** -11
    logits = logits.to(dtype)
    prev, done = torch.full((B, K), -20000.0), torch.zeros(B, K, dtype=I32)
    check_ties(logits, prev, done, 7, stride)
    prev[:, 1:] = -math.inf
    check_ties(logits, prev, done, 7, stride)
    prev[:, 1:] = -20000.0
    done[:, K // 2:] = 1
    check_ties(logits, prev, done, V - 1, stride)


@pytest.mark.parametrize("K,V", [(16, 70001), (9, 150000), (32, 70001), (4, 400000)])
@pytest.mark.parametrize("live", [1, 4])
def test_beam_select_of_two_logits_with_one_score(K, V, live):
    """A few of the larger logit behind many of the smaller one, all in what is fetched first: candidates that go when room is made for the next part are as good as what stays.
    (The next smaller bf16 number has another score: the counts of logits at 0 put a boundary of rounding below the two.)"""
    hi, lo, unit = 1 + 2.0 ** -7, 1.0, 2.0 ** -6      # (scores of 2^17 ... 2^18 are multiples of 2^-6)
    lse = lambda m: math.log(10 * math.exp(hi) + 60 * math.exp(lo) + m + (V - 70 - m) * math.exp(-5))
    m = next(m for m in range(1000) if 0.55 < (lo - lse(m)) / unit % 1 < 0.65)
    z = torch.full((K, V), -5.0)
    z[:, V - m:] = 0.0
    at = torch.randperm(4000, generator=torch.Generator().manual_seed(K))[:70].sort().values
    z[:, at[:60]], z[:, at[60:]] = lo, hi
    prev = torch.full((1, K), -math.inf)
    prev[0, :live] = -150000.0
    check_ties(z.bfloat16(), prev, torch.zeros(1, K, dtype=I32), 7)


@pytest.mark.parametrize("B,K,V", [(2, 4, 50304), (1, 32, 50304), (4, 1, 30000), (2, 9, 12345)])
def test_beam_select_of_random_logits_behind_large_scores(B, K, V):
    """Random fp32 logits, scores some ten of which are equal at the top."""
    torch.manual_seed(V + K)
    logits = torch.randn(B * K, V) * 3
    check_ties(logits, torch.full((B, K), -300000.0) - 0.25 * torch.arange(K), torch.zeros(B, K, dtype=I32), 3)


def test_beam_select_in_a_graph():
    torch.manual_seed(1)
    z = torch.randn(8, 5000, device=dev()).bfloat16()
    prev, done = torch.zeros(2, 4, device=dev()), torch.zeros(2, 4, dtype=I32, device=dev())
    out = lambda: (torch.empty_like(prev), torch.empty_like(done), torch.empty_like(done), torch.empty_like(done))
    a, b = out(), out()
    ops.beam_select(*a, z, prev, done, 3)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.beam_select(*b, z, prev, done, 3)
    for _ in range(3):
        z.copy_(torch.randn(8, 5000, device=dev()))
        ops.beam_select(*a, z, prev, done, 3)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------ beams in order
@pytest.mark.parametrize("B,K,L,Hkv,hd,page,width,lens,T", [
    (1, 1, 1, 1, 32, 16, 2, [5], 40), (2, 4, 3, 2, 64, 32, 4, [64, 70], 100), (3, 5, 2, 3, 96, 16, 3, [47, 0, 48], 48), (1, 8, 4, 2, 128, 128, 3, [257], 300), (2, 3, 0, 1, 32, 64, 2, [1, 63], 10)])
@pytest.mark.parametrize("cached", [True, False])
def test_beam_reorder(B, K, L, Hkv, hd, page, width, lens, T, cached):
    g = torch.Generator().manual_seed(B * K + page)
    rows = B * K
    n = rows * (width + 1)
    ids = torch.randperm(n, generator=g).int()
    table, spare = ids[:rows * width].view(rows, width).contiguous(), ids[rows * width:].contiguous()
    pages = torch.randint(0, 256, (L, n, Hkv, page // 16, 18 * hd), generator=g, dtype=torch.uint8)
    ln = torch.tensor(lens, dtype=I32).repeat_interleave(K)
    hist = torch.randint(0, 1000, (rows, T), generator=g, dtype=I32)
    parents, tokens = torch.randint(0, K, (B, K), generator=g, dtype=I32), torch.randint(0, 1000, (B, K), generator=g, dtype=I32)
    outs = lambda d: [torch.full_like(t, -9, device=d) for t in (table, spare, hist)]
    want, wp = outs("cpu"), pages.clone()
    ref.beam_reorder(wp if cached else None, *want, table, spare, ln, hist, parents, tokens, page)
    got, gp = outs(dev()), pages.to(dev())
    ops.beam_reorder(gp if cached else None, *got, *(t.to(dev()) for t in (table, spare, ln, hist, parents, tokens)), page)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    assert torch.equal(gp.cpu(), wp)
    # the definition: each row holds what its parent held, then its token
    for r in range(rows):
        t, src = int(ln[r]), r // K * K + int(parents.view(-1)[r])
        h = min(t, T)
        assert got[2][r, :h].tolist() == hist[src, :h].tolist() and (t >= T or int(got[2][r, t]) == int(tokens.view(-1)[r]))
        for tok in range(t) if cached else ():
            a, b = int(table[src, tok // page]), int(got[0][r, tok // page])
            assert torch.equal(pages[:, a, :, tok % page // 16], gp[:, b, :, tok % page // 16].cpu())
    if cached:
        full = torch.cat([got[0].cpu()[torch.arange(rows), (ln // page).clamp(max=width - 1).long()], got[1].cpu()])
        held = torch.cat([ln % page > 0, torch.ones(rows, dtype=torch.bool)])
        assert len(set(full[held].tolist())) == int(held.sum())      # pages that are being filled and spare ones belong to one row


def test_beam_reorder_reports_what_lies_outside():
    table, spare, hist = ints([[0, 1], [2, 3]]), ints([4, 9]), ints([[1, 2, 3], [4, 5, 6]])
    pages = torch.zeros(1, 5, 1, 1, 18 * 32, dtype=torch.uint8, device=dev())
    out = [torch.zeros_like(t) for t in (table, spare, hist)]
    ops.beam_reorder(pages, *out, table, spare, ints([2, 2]), hist, ints([[0, 2]]), ints([[7, 8]]))
    raised(0xB3)
    assert out[0].tolist() == table.tolist() and out[2].tolist() == [[1, 2, 7], [4, 5, 8]]
    ops.beam_reorder(pages, *out, table, spare, ints([2, 2]), hist, ints([[0, 0]]), ints([[7, 8]]))
    raised(0xB4)


# ------------------------------------------------------------------ refusals, entry points
def test_refusals():
    """Before anything is launched, with the argument's name."""
    hd, bf = 64, torch.bfloat16
    pages = torch.zeros(4, 2, 1, 18 * hd, dtype=torch.uint8, device=dev())
    x = torch.zeros(3, 8 * hd, dtype=bf, device=dev())
    s = ints([0, 1, 2])
    bad = [
        lambda: ops.kv4_append(pages, None, x, s, None, None, None, 4, 2, 128),
        lambda: ops.kv4_append(pages, None, x, s, None, None, None, 3, 2, hd),
        lambda: ops.kv4_append(pages, None, x, s.long(), None, None, None, 4, 2, hd),
        lambda: ops.kv4_append(pages, None, x.float(), s, None, None, None, 4, 2, hd),
        lambda: ops.kv4_append(pages[:, :, :, :-18], None, x, s, None, None, None, 4, 2, hd),
        lambda: ops.kv4_append(pages[:, :1], None, x[:, :6 * hd], s, None, None, None, 4, 1, hd),      # (not contiguous)
        lambda: ops.kv4_append(pages, None, torch.zeros(3, 8 * hd + 1, dtype=bf, device=dev())[:, :8 * hd], s, None, None, None, 4, 2, hd),
        lambda: ops.kv4_append(pages, None, x.cpu(), s, None, None, None, 4, 2, hd),
        lambda: ops.kv4_read(x[:, :hd], x[:, :hd], pages, s),
        lambda: ops.kv4_attn(x[:1, :4 * hd], None, x[:1, :4 * hd], pages, ints([[0]]), ints([1]), 1, 4, 4, hd),
        lambda: ops.kv4_attn(x[:1, :3 * hd], None, x[:1, :3 * hd], pages, ints([[0]]), ints([1]), 1, 3, 2, hd),
        lambda: ops.kv4_attn(x[:1, :4 * hd], None, x[:1, :4 * hd], pages, ints([[0], [1]]), ints([1]), 1, 4, 2, hd),
        lambda: ops.kv4_attn(x[:1, :4 * hd], None, x[:1, :4 * hd], pages, ints([[0]]).long(), ints([1]), 1, 4, 2, hd),
        lambda: ops.kv4_attn(x[:1, :4 * hd], torch.zeros(1, 4, device=dev()), x[:1, :4 * hd], pages, ints([[0]]), ints([1]), 1, 4, 2, hd),
        lambda: ops.beam_select(*[torch.zeros(1, 33, device=dev())] * 1, *[torch.zeros(1, 33, dtype=I32, device=dev())] * 3, torch.zeros(33, 9, dtype=bf, device=dev()), torch.zeros(1, 33, device=dev()), torch.zeros(1, 33, dtype=I32, device=dev()), 0),
        lambda: ops.beam_select(torch.zeros(1, 2, device=dev()), *[torch.zeros(1, 2, dtype=I32, device=dev())] * 3, torch.zeros(2, 9, dtype=torch.float16, device=dev()), torch.zeros(1, 2, device=dev()), torch.zeros(1, 2, dtype=I32, device=dev()), 0),
        lambda: ops.beam_select(torch.zeros(1, 2, device=dev()), *[torch.zeros(1, 2, dtype=I32, device=dev())] * 3, torch.zeros(9, 2, dtype=bf, device=dev()).t(), torch.zeros(1, 2, device=dev()), torch.zeros(1, 2, dtype=I32, device=dev()), 0),
        lambda: ops.block_tables(ints([[0]]), s, s, ints([0]), ints([0]), ints([0]), ints([0]), ints([0]), s, ints([1]), 16),
        lambda: ops.block_tables(ints([[0]]), s, s, ints([0, 0]), ints([0]), ints([0]), ints([0]), ints([0]), s, ints([1]), 0),
        lambda: ops.beam_reorder(None, ints([[0]]), ints([0]), ints([[0]]), ints([[0]]), ints([0]), ints([1]), ints([[0]]), ints([[0]]), ints([[0]])),
        lambda: (lambda t: ops.beam_reorder(None, t, ints([0]), ints([[0]]), t, ints([0]), ints([1]), ints([[0]]), ints([[0]]), ints([[0]]), 16))(ints([[0]])),
    ]
    for k, f in enumerate(bad):
        with pytest.raises((ValueError, AssertionError)):
            f()
            pytest.fail(f"call {k} was taken")


@pytest.mark.parametrize("scale", [2e38, -1e300, math.inf, math.nan])
def test_scales_past_32_bits_are_refused(scale):
    x, pages = torch.zeros(1, 64, dtype=torch.bfloat16, device=dev()), torch.zeros(4, 1, 1, 18 * 64, dtype=torch.uint8, device=dev())
    with pytest.raises(ValueError, match="scale"):
        ops.kv4_attn(torch.empty_like(x), None, x, pages, ints([[0]]), ints([1]), 1, 1, 1, 64, scale)


@pytest.mark.parametrize("module", [True, False])
def test_views_that_begin_off_16_bytes_are_refused(monkeypatch, module):
    """Contiguous ones too, by the argument's name, on both ways into the library; nothing is launched."""
    n, bf, hd = nat(), torch.bfloat16, 64
    if not module:
        monkeypatch.setattr(n, "_E", n._Ctypes())
    new = lambda *s, dtype=bf: torch.zeros(*s, dtype=dtype, device=dev())
    off = lambda t: torch.zeros(t.numel() + 1, dtype=t.dtype, device=dev())[1:].view(t.shape)
    pages, s = new(4, 2, 1, 18 * hd, dtype=torch.uint8), ints([0, 1, 2])
    q, x, a, k, o = new(3, 4 * hd), new(3, 8 * hd), new(9, hd // 2, dtype=torch.float32), new(3, 2 * hd), new(1, 4 * hd)
    calls = {
        "q_out": lambda: ops.kv4_append(pages, off(q), x, s, None, None, None, 4, 2, hd),
        "qkv": lambda: ops.kv4_append(pages, q, off(x), s, None, None, None, 4, 2, hd),
        "cos": lambda: ops.kv4_append(pages, q, x, s, s, off(a), a, 4, 2, hd),
        "sin": lambda: ops.kv4_append(pages, q, x, s, s, a, off(a), 4, 2, hd),
        "k": lambda: ops.kv4_read(off(k), k, pages, s),
        "v": lambda: ops.kv4_read(k, off(k), pages, s),
        "pages": lambda: ops.kv4_read(k, k, off(pages), s),
        "out": lambda: ops.kv4_attn(off(o), None, o, pages, ints([[0]]), ints([1]), 1, 4, 2, hd),
        "q": lambda: ops.kv4_attn(o, None, off(o), pages, ints([[0]]), ints([1]), 1, 4, 2, hd),
    }
    for name, call in calls.items():
        with pytest.raises(ValueError, match=rf"\b{name}\b.*16-byte"):
            call()


def test_generation_entry_points_through_ctypes_and_through_the_module(monkeypatch):
    """The same bits through the extension module and through ctypes."""
    n, seen = nat(), set()

    class Spy:
        def __init__(self, entries):
            self.entries = entries

        def __getattr__(self, name):
            seen.add(name)
            return getattr(self.entries, name)

    def work():
        torch.manual_seed(0)
        hd, H, made = 64, 4, []
        e = lambda *s, dtype=torch.bfloat16: made.append(torch.zeros(s, dtype=dtype, device=dev())) or made[-1]
        cos, sin = ref.rope_tables(64, hd, 10000.0, dev())
        pages, x = e(1, 6, 2, 1, 18 * hd, dtype=torch.uint8), torch.randn(20, 8 * hd, device=dev()).bfloat16()
        table, slots, pos = e(2, 2, dtype=I32), e(20, dtype=I32), e(20, dtype=I32)
        lens = e(2, dtype=I32)
        n.block_tables(table, slots, pos, e(3, dtype=I32), lens, e(1, dtype=I32), lens, ints([11, 9]), ints([0, 1, 2, 3]), ints([4]), 16)
        n.kv4_append(pages[0], q := e(20, 4 * hd), x, slots, pos, cos, sin, H, 2, hd)
        n.kv4_read(e(20, 2 * hd), e(20, 2 * hd), pages[0], slots)
        n.kv4_attn(e(2, 4 * hd), e(2, H, 1, dtype=torch.float32), q[:2], pages[0], table, lens, 1, H, 2, hd)
        par, tok = e(1, 2, dtype=I32), e(1, 2, dtype=I32)
        n.beam_select(e(1, 2, dtype=torch.float32), tok, par, e(1, 2, dtype=I32), torch.randn(2, 300, device=dev()), torch.zeros(1, 2, device=dev()), torch.zeros(1, 2, dtype=I32, device=dev()), 0)
        hist = torch.randint(0, 9, (2, 12), dtype=I32, device=dev())
        n.beam_reorder(pages, e(2, 2, dtype=I32), e(2, dtype=I32), e(2, 12, dtype=I32), table, ints([4, 5]), ints([9, 9]), hist, par, tok)
        return made

    outs = []
    for entries in (n._Ctypes(), n.bridge()):
        seen.clear()
        monkeypatch.setattr(n, "_E", Spy(entries))
        outs.append(work())
        assert seen == {"mlb_" + k for k in n._GEN_KINDS}
    for a, b in zip(*outs):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ the whole path
def small(T=160, V=500, hd=64, H=2, L=2, seed=0):
    from ml_b200 import Config
    from ml_b200.models import GPT
    g = GPT(Config(V=V, C=H * hd, L=L, H=H, I=192, T=T), 2, "cuda:0")
    g.init_weights(7 + seed)
    return g


def test_generate_from_the_cache_follows_the_uncached_pass():
    """With weights as they are initialised the logits of the first token equal the uncached ones (the prompt's attention is over unrounded keys); later ones are
    those of a model with keys and values rounded to 4 bits: checked against a plain restatement by the oracle of a step's attention in test_attention."""
    g = small()
    torch.manual_seed(1)
    prompt = torch.randint(0, 500, (2, 37))
    a, b = g.generate(prompt, 1), g.generate(prompt, 1, kv="4bit")
    assert torch.equal(a, b)
    c = g.generate(prompt, 30, kv="4bit", page=16)
    assert c.shape == (2, 67) and torch.equal(c[:, :37].cpu(), prompt) and torch.equal(c, g.generate(prompt, 30, kv="4bit", page=64))
    assert torch.equal(c[:1], g.generate(prompt[:1], 30, kv="4bit", page=32))
    s = [g.generate(prompt, 8, temperature=1.0, top_k=5, seed=3, kv="4bit") for _ in range(2)]
    assert torch.equal(s[0], s[1])


@pytest.mark.parametrize("page,P", [(16, 37), (64, 64), (32, 5)])
def test_beam_search_scores_are_those_of_its_tokens(page, P):
    """Every beam's log-probability is the sum of those its own tokens get when they are fed one by one through a cache without beams: tables, shared pages,
    copies and spare pages give each beam its own past."""
    from ml_b200.models import generation
    g = small()
    g.master.mul_(6)      # sharper distributions than those of fresh weights
    g.sync_params()
    torch.manual_seed(P)
    prompt = torch.randint(0, 500, (2, P))
    n, K = 20, 4
    hist, scores = generation.beam_search(g, prompt, n, K, page=page)
    assert hist.shape == (2, K, P + n) and (scores[:, :-1] >= scores[:, 1:]).all()
    assert len({tuple(h) for h in hist[0].tolist()}) == K
    rows = hist.view(2 * K, -1)
    m = generation.CachedDecoder(g, 2 * K, P + n, 16)
    slots, _, _ = m.cache.grow(torch.full((2 * K,), P, dtype=I32, device=dev()), 2 * K * P)
    logits, total = m.prompt(rows[:, :P].int().contiguous(), slots), torch.zeros(2 * K, device=dev(), dtype=torch.float64)
    for t in range(P, P + n):
        total += torch.log_softmax(logits.double(), -1).gather(1, rows[:, t:t + 1]).view(-1)
        if t + 1 < P + n:
            logits = m.step(rows[:, t].int().contiguous())
    # (bf16 products of another number of rows may take another kernel: logits of magnitude up to 20 differ by their rounding)
    assert (scores.view(-1).double() - total).abs().max() <= n * 20 * 2.0 ** -8
    top = g.generate(prompt, n, kv="4bit", beams=K, page=page)
    assert torch.equal(top, hist[:, 0])


@pytest.mark.parametrize("V,K,P,page", [(3, 4, 20, 16), (3, 4, 16, 16), (8, 4, 48, 16), (2, 9, 70, 32), (3, 4, 5, 16)])
def test_beam_search_with_more_beams_than_continuations(V, K, P, page):
    """Rows on beams that are none hold the prompt too; the kernels find no page outside the pool (asked after every test)."""
    from ml_b200 import Config
    from ml_b200.models import GPT, generation
    g = GPT(Config(V=V, C=128, L=2, H=2, I=192, T=160), 2, "cuda:0")
    g.init_weights(7)
    torch.manual_seed(V + P)
    prompt, n = torch.randint(0, V, (2, P)), 4
    hist, scores = generation.beam_search(g, prompt, n, K, page=page)
    assert torch.equal(hist[:, :, :P].cpu(), prompt[:, None].expand(2, K, P)) and torch.isfinite(scores).all()
    assert all(len({tuple(r) for r in h}) == K for h in hist.tolist())


@pytest.mark.parametrize("beams", [1, 3])
def test_generation_raises_what_its_kernels_report(beams):
    """A token outside the vocabulary: an error in words, as CPU tensors give one, and no word left for whoever looks next."""
    g = small()
    prompt = torch.randint(0, 500, (2, 20))
    prompt[1, 7] = 500
    with pytest.raises(RuntimeError, match="token id outside the vocabulary"):
        g.generate(prompt, 5, kv="4bit", beams=beams)
    assert nat().get_error() == 0
    assert g.generate(prompt[:1], 5, kv="4bit", beams=beams).shape == (1, 25)


def test_a_step_outside_the_pool_is_reported():
    """A block table that names no page, which the kernels leave out: generation does not hand on what came of it."""
    from ml_b200.models import generation
    g = small()
    m = generation.CachedDecoder(g, 2, 30, 16)
    ids = torch.randint(0, 500, (2, 20), dtype=I32, device=dev())
    slots, _, _ = m.cache.grow(ints([20, 20]), 40)
    m.prompt(ids, slots)
    m.cache.table[1, 0] = -1
    m.step(ids[:, 0].contiguous())
    with pytest.raises(RuntimeError, match="page outside the pool"):
        m.check()
    assert nat().get_error() == 0
    m.check()


def test_beams_end():
    from ml_b200.models import generation
    g = small()
    torch.manual_seed(3)
    prompt = torch.randint(0, 500, (1, 9))
    free, _ = generation.beam_search(g, prompt, 6, 3)
    eos = int(free[0, 0, 11])      # a token that the best beam chooses on its way
    hist, scores = generation.beam_search(g, prompt, 12, 3, eos=eos)
    for h in hist[0, :, 9:].tolist():
        if eos in h:
            assert set(h[h.index(eos):]) == {eos}
    assert any(eos in h for h in hist[0, :, 9:].tolist())
    long, ls = generation.beam_search(g, prompt, 12, 3, eos=eos, length_penalty=1.0)
    assert sorted(map(tuple, long[0].tolist())) == sorted(map(tuple, hist[0].tolist()))
