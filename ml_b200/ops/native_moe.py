"""The operators of a mixture of experts on the kernels of csrc/kernels/moe.cu and moe_route.cuh: arguments looked at, workspace fetched, launches on the current
stream, nothing read back.  What they do stands with their plain forms in `ops.ref_moe`."""
from __future__ import annotations

import torch

from . import native as _n
from .ref_moe import check_mlp, check_plan, check_route, check_route_bwd, _need

NONE, Address = _n.NONE, _n.Address
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def _took(rc, name):
    if rc == -7:
        raise ValueError(f"{name}: sizes past what the kernels count in 32 bits, or memory off a 16-byte boundary")
    _n._chk(rc, name)


def _here(*ts):
    dev = torch._C._cuda_getDevice()
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"a tensor is on device {t.get_device()}, the current one is {dev}")


def _dense(**tensors):
    for what, t in tensors.items():
        if t is not None and not t.is_contiguous():
            raise ValueError(f"{what}: need contiguous memory")


def _at(t):
    return NONE if t is None else Address(t.data_ptr())


def _bits(t):
    return 16 if t.dtype == BF16 else 32


def _rows(t, what, eights=True):
    """Elements between the rows of a matrix of which they may be a part."""
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{what}: need rows of neighbouring elements")
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if ld < t.shape[1] and t.shape[0] > 1:
        raise ValueError(f"{what}: rows lie over one another")
    if eights and (ld % 8 or t.data_ptr() % 16):
        raise ValueError(f"{what}: need rows that begin on 16-byte boundaries")
    return ld


def _plain(name, *args):
    e = _n._entries()
    if e is not _n.bridge() or getattr(e, name)(*args) is NotImplemented:
        return False
    _n.LAUNCHES += 1
    return True


# ------------------------------------------------------------------ routing
def moe_route(weights, idx, mean, logits, bias=None, score="softmax", groups=1, top_groups=1, renorm=True, scale=1.0):
    if mean is None and _plain("moe_route_out", weights, idx, logits, bias, score, groups, top_groups, renorm, scale):
        return
    N, E, k = check_route(weights, idx, mean, logits, bias, score, groups, top_groups)
    _here(weights, idx, mean, logits, bias)
    _dense(weights=weights, idx=idx, mean=mean, bias=bias)
    if N == 0:
        if mean is not None:
            mean.zero_()
        return
    e = _n._entries()
    part = NONE if mean is None else _n.scratch("route_part", e.mlb_moe_route_part(N, E), F32, logits.device)
    _took(e.mlb_moe_route(_at(weights), idx, NONE if mean is None else mean, part, _at(logits), NONE if bias is None else bias, N, _rows(logits, "logits", False), E, k,
                          int(score == "sigmoid"), groups, top_groups, int(renorm), float(scale), _bits(logits), _bits(weights)), "moe_route")


def moe_route_bwd(dlogits, dweights, dmean, logits, idx, score="softmax", renorm=True, scale=1.0):
    N, E, k = check_route_bwd(dlogits, dweights, dmean, logits, idx, score)
    _here(dlogits, dweights, dmean, logits, idx)
    _dense(dlogits=dlogits, dweights=dweights, dmean=dmean, idx=idx)
    if N == 0:
        return
    _took(_n._entries().mlb_moe_route_bwd(_at(dlogits), _at(dweights), NONE if dmean is None else dmean, _at(logits), idx, N, _rows(logits, "logits", False), E, k,
                                          int(score == "sigmoid"), int(renorm), float(scale), _bits(logits), _bits(dweights)), "moe_route_bwd")


# ------------------------------------------------------------------ the experts
def _plan(idx, E):
    """(plan, rows of the buffers in which the copies of the tokens are sorted by expert)"""
    N, k = check_plan(idx, E)
    e = _n._entries()
    plan = torch.empty(e.mlb_moe_plan_ints(N, k, E), dtype=I32, device=idx.device)
    _took(e.mlb_moe_plan(plan, idx, N, k, E), "moe_plan")
    return plan, e.mlb_moe_plan_rows(N, k, E)


def _check(x, weights, idx, gate_up, down):
    N, k, E, C, I = check_mlp(x, weights, idx, gate_up, down)
    if x.dtype != BF16:
        raise ValueError(f"x {x.dtype}: the kernels take bfloat16")
    if C % 16 or I % 16:
        raise ValueError(f"{C} columns, experts of {I}: need multiples of 16")
    _dense(weights=weights, idx=idx, gate_up=gate_up, down=down)
    return N, k, E, C, I


def _fwd(out, x, weights, idx, gate_up, down, keep):
    N, k, E, C, I = _check(x, weights, idx, gate_up, down)
    _need(out, (N, C), "out", (BF16,))
    _here(out, x, weights, idx, gate_up, down)
    _dense(out=out)
    ldx = _rows(x, "x")
    if N == 0:
        return None
    e = _n._entries()
    few = 0 if keep else e.mlb_moe_few_floats(N, k, E, C, I)
    if few:
        part = _n.scratch("moe_few", few, F32, x.device)
        _took(e.mlb_moe_few(out, _at(x), _at(weights), idx, gate_up, down, part, N, ldx, k, E, C, I, _bits(weights)), "moe_mlp")
        return None
    plan, R = _plan(idx, E)
    new = lambda c: torch.empty(R, c, dtype=BF16, device=x.device)
    xs, gu, h, y = new(C), new(2 * I) if keep else None, new(I), new(C)
    _took(e.mlb_moe_fwd(out, xs, _at(gu), h, y, _at(x), _at(weights), gate_up, down, plan, N, ldx, k, E, C, I, _bits(weights)), "moe_mlp")
    return plan, xs, gu, h, y


def moe_mlp(out, x, weights, idx, gate_up, down):
    if _plain("moe_mlp_out", out, x, weights, idx, gate_up, down):
        return
    _fwd(out, x, weights, idx, gate_up, down, False)


def moe_mlp_fwd(out, x, weights, idx, gate_up, down):
    return _fwd(out, x, weights, idx, gate_up, down, True) or ()


def moe_mlp_bwd(dx, dweights, dgate_up, ddown, dout, x, weights, idx, gate_up, down, saved):
    N, k, E, C, I = _check(x, weights, idx, gate_up, down)
    _need(dout, (N, C), "dout", (BF16,))
    _need(dweights, (N, k), "dweights", (weights.dtype,))
    for t, like, what in ((dx, x, "dx"), (dgate_up, gate_up, "dgate_up"), (ddown, down, "ddown")):
        if t is not None:
            _need(t, like.shape, what, (BF16,))
    _here(dx, dweights, dgate_up, ddown, dout, x, weights, idx, gate_up, down, *saved)
    _dense(dx=dx, dweights=dweights, dgate_up=dgate_up, ddown=ddown)
    if N == 0:
        for t in (dgate_up, ddown):
            if t is not None:
                t.zero_()
        return
    plan, xs, gu, h, y = saved
    e = _n._entries()
    R = e.mlb_moe_plan_rows(N, k, E)
    _need(plan, (e.mlb_moe_plan_ints(N, k, E),), "saved plan", (I32,))
    for t, c in ((xs, C), (gu, 2 * I), (h, I), (y, C)):
        _need(t, (R, c), "saved rows", (BF16,))
    new = lambda c: torch.empty(R, c, dtype=BF16, device=x.device)
    ys, dgu, dxs = new(C), new(2 * I), new(C)
    _took(e.mlb_moe_bwd(_at(dx), _at(dweights), _at(dgate_up), _at(ddown), ys, dgu, dxs, _at(dout), xs, gu, h, y, _at(weights), gate_up, down, plan, N, _rows(dout, "dout"), k, E, C, I,
                        _bits(weights)), "moe_mlp_bwd")
