"""The operators of generation on the kernels of csrc/kernels/kv4.cu and beam.cu: arguments looked at, workspace fetched, one launch each on the current
stream, nothing read back.  What they do stands with their plain forms in `ops.ref_gen`.  The extension module takes plain calls whole and hands back the
others (ops/autograd.py has its operators the same way); a step of generation is bound by what its launches cost the host."""
from __future__ import annotations

import math

import torch

from . import native as _n
from .ref_gen import check_append, check_attn, check_read, check_reorder, check_select, check_tables

NONE, Address = _n.NONE, _n.Address
F32, I32 = torch.float32, torch.int32


def _rows(t, what):
    """Address of a bf16 matrix whose rows may be apart (a part of a wider one), for kernels that read 16 bytes at a time."""
    if t.dtype != torch.bfloat16 or not t.is_cuda or (t.shape[1] > 1 and t.stride(1) != 1) or t.stride(0) % 8 or t.data_ptr() % 16:
        raise ValueError(f"{what}: need CUDA bf16 rows that begin on 16-byte boundaries")
    return Address(t.data_ptr())


def _on_16_bytes(**tensors):
    """Other tensors that a kernel reads or writes 16 bytes at a time."""
    for what, t in tensors.items():
        if t is not None and t.data_ptr() % 16:
            raise ValueError(f"{what}: need memory that begins on a 16-byte boundary")


def _pool(pages):
    if not pages.is_cuda or not pages.is_contiguous() or pages.data_ptr() % 16:
        raise ValueError("pages: need contiguous CUDA memory on a 16-byte boundary")
    return pages


def _took(rc, name):
    if rc == -7:
        raise ValueError(f"{name}: sizes past what the kernel counts in 32 bits, or memory off a 16-byte boundary")
    _n._chk(rc, name)


def _here(*ts):
    dev = torch._C._cuda_getDevice()
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"a tensor is on device {t.get_device()}, the current one is {dev}")


def _plain(name, *args):
    e = _n._entries()
    if e is not _n.bridge() or getattr(e, name)(*args) is NotImplemented:
        return False
    _n.LAUNCHES += 1
    return True


def kv4_append(pages, q_out, qkv, slots, pos, cos, sin, H, Hkv, hd):
    if _plain('kv4_append', pages, q_out, qkv, slots, pos, cos, sin, H, Hkv, hd):
        return
    n, page, N = check_append(pages, q_out, qkv, slots, pos, cos, sin, H, Hkv, hd)
    _on_16_bytes(q_out=q_out, cos=cos, sin=sin)
    _here(pages, q_out, qkv, slots, pos, cos, sin)
    if N == 0:
        return
    rope = cos is not None
    _took(_n._entries().mlb_kv4_append(_pool(pages), NONE if q_out is None else q_out, _rows(qkv, "qkv"), slots, pos if rope else NONE, cos if rope else NONE,
                                         sin if rope else NONE, n, page, N, qkv.stride(0), H, Hkv, hd, cos.shape[0] if rope else 0), "kv4_append")


def kv4_read(k, v, pages, slots):
    if _plain('kv4_read', k, v, pages, slots):
        return
    n, Hkv, page, hd, N = check_read(k, v, pages, slots)
    _on_16_bytes(k=k, v=v)
    _here(k, v, pages, slots)
    if N:
        _took(_n._entries().mlb_kv4_read(k, v, _pool(pages), slots, n, page, N, Hkv, hd), "kv4_read")


def kv4_attn(out, lse, q, pages, table, lens, Tq, H, Hkv, hd, scale=None):
    if _plain('kv4_attn', out, lse, q, pages, table, lens, Tq, H, Hkv, hd, scale):
        return
    n, page, B = check_attn(out, lse, q, pages, table, lens, Tq, H, Hkv, hd, scale)
    _on_16_bytes(out=out)
    _here(out, lse, q, pages, table, lens)
    if B == 0:
        return
    e, dev, width = _n._entries(), q.device, table.shape[1]
    part = _n.scratch("kv4_part", max(0, e.mlb_kv4_attn_scratch(B, Tq, H, Hkv, hd, width, page)), F32, dev)
    count = _n.scratch("kv4_count", B * Hkv * -(-H // Hkv * Tq // 8), I32, dev, zero=True)
    _took(e.mlb_kv4_attn(out, NONE if lse is None else lse, _rows(q, "q"), _pool(pages), table, lens, part, count, n, q.stride(0), B, Tq, H, Hkv, hd, width, page,
                           1.0 / math.sqrt(hd) if scale is None else scale), "kv4_attn")


def block_tables(table, slots, pos, starts, new_lens, left, lens, new, free, n_free, page):
    if _plain('block_tables', table, slots, pos, starts, new_lens, left, lens, new, free, n_free, page):
        return
    B = check_tables(table, slots, pos, starts, new_lens, left, lens, new, free, n_free, page)
    _here(table, slots, pos, starts, new_lens, left, lens, new, free, n_free)
    ticket = _n.scratch("tables_ticket", 1, I32, table.device, zero=True)
    _took(_n._entries().mlb_block_tables(table, slots, pos, starts, new_lens, left, ticket, lens, new, free, n_free, B, table.shape[1], page, slots.numel(),
                                           free.numel()), "block_tables")


def beam_select(scores, tokens, parents, done_out, logits, prev, done, eos):
    if _plain('beam_select', scores, tokens, parents, done_out, logits, prev, done, eos):
        return
    B, K, V = check_select(scores, tokens, parents, done_out, logits, prev, done)
    _here(scores, tokens, parents, done_out, logits, prev, done)
    if B == 0:
        return
    if V > 1 and logits.stride(1) != 1:
        raise ValueError("logits: need rows of neighbouring elements")
    e, dev, rows, bits = _n._entries(), logits.device, B * K, 16 if logits.dtype == torch.bfloat16 else 32
    pieces = e.mlb_beam_select_pieces(rows, K, V, bits)
    if pieces < 0:
        raise ValueError(f"{B} x {K} beams: at most 65535 rows")
    part = _n.scratch("select_part", rows * pieces * (4 + 4 * K), F32, dev)
    ticket = _n.scratch("select_ticket", B, I32, dev, zero=True)
    base, n = part.data_ptr(), rows * pieces
    _took(e.mlb_beam_select(scores, tokens, parents, done_out, Address(logits.data_ptr()), prev, done, part, Address(base + 8 * n), Address(base + 8 * n + 4 * n * (2 * K + 1)),
                              ticket, rows, K, V, logits.stride(0), eos, bits), "beam_select")


def beam_reorder(pages, table_out, spare_out, hist_out, table, spare, lens, hist, parents, tokens, page=None):
    if _plain('beam_reorder', pages, table_out, spare_out, hist_out, table, spare, lens, hist, parents, tokens, page):
        return
    layers, n, Hkv, page, block, B, K = check_reorder(pages, table_out, spare_out, hist_out, table, spare, lens, hist, parents, tokens, page)
    _here(pages, table_out, spare_out, hist_out, table, spare, lens, hist, parents, tokens)
    if B * K == 0:
        return
    _took(_n._entries().mlb_beam_reorder(NONE if pages is None else _pool(pages), table_out, spare_out, hist_out, table, spare, lens, hist, parents, tokens, layers, n,
                                           Hkv, page, block, B, K, table.shape[1], hist.shape[1]), "beam_reorder")
