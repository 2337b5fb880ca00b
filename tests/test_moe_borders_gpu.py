"""Routing on the GPU against its definition in 64 bits, all tokens at once: many tokens, and choices that lie next to a border."""
import math

import pytest
import torch

from ml_b200 import ops
from ml_b200.ops import autograd as F

pytestmark = pytest.mark.gpu
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
NEG = -math.inf
STEP = 2.0 ** -24      # half a step of fp32, relative


def dev():
    return torch.device("cuda:0")


@pytest.fixture(autouse=True)
def no_errors():
    from ml_b200.ops import native
    yield
    torch.cuda.synchronize()
    err = native.get_error()
    native.clear_error()
    assert err == 0, native.describe_error(err)


def scores(z, score):
    there = z > NEG
    if score == "sigmoid":
        return torch.where(there, 1 / (1 + torch.exp(-z)), 0.0)
    m = z.amax(1, keepdim=True)
    e = torch.where(there, torch.exp(z - torch.where(m > NEG, m, 0.0)), 0.0)
    return e / e.sum(1, keepdim=True).clamp(min=1e-300)


def chosen(z, k, bias=None, score="softmax", groups=1, top_groups=1):
    """idx of logits in 64 bits without NaN"""
    N, E = z.shape
    t = z if bias is None and groups == 1 else scores(z, score) + (0.0 if bias is None else bias.double())
    t = torch.where(z > NEG, t, NEG)
    if groups > 1:
        parts = t.view(N, groups, E // groups)
        best = parts.sort(dim=2, descending=True).values[..., :2]
        second = best[..., 1] if best.shape[2] > 1 else torch.full_like(best[..., 0], NEG)
        of = best[..., 0] + torch.where(second > NEG, second, 0.0)
        at = of.sort(dim=1, descending=True, stable=True).indices[:, :top_groups]
        t = torch.where(torch.zeros_like(of, dtype=torch.bool).scatter_(1, at, True)[..., None], parts, NEG).view(N, E)
    best, at = t.sort(dim=1, descending=True, stable=True)
    return torch.where(best[:, :k] > NEG, at[:, :k], -1).to(I32)


def routed(z, k, **how):
    w, idx = torch.empty(len(z), k, device=dev()), torch.empty(len(z), k, dtype=I32, device=dev())
    ops.moe_route(w, idx, None, z, **how)
    return idx


def same(idx, want):
    wrong = (idx != want).any(1)
    assert not bool(wrong.any()), (int(wrong.sum()), idx[wrong][:4].tolist(), want[wrong][:4].tolist())


# ------------------------------------------------------------------ borders
@pytest.mark.parametrize("level", [-2.0, -10.0, -30.0, -50.0, -80.0, -87.6, -95.0])
@pytest.mark.parametrize("biased", [False, True])
def test_groups_whose_sums_are_nearly_equal(level, biased):
    """Sigmoids far below 0: a rounding of the logit's product with log2 e is |z| 2^-24 of the score, and below e^-87 there are no normal numbers.  Four groups' sums of two, a few 1e-6 apart."""
    g = torch.Generator(device="cuda").manual_seed(int(-10 * level))
    N, groups, size = 40000, 4, 4
    a = level + 0.6 * torch.rand(N, groups, generator=g, device=dev(), dtype=F64)
    both = 2.2 * math.exp(level + 0.6) * (1 + 3e-6 * torch.randn(N, groups, generator=g, device=dev(), dtype=F64))
    z = torch.full((N, groups, size), level - 4.0, device=dev())
    s = torch.sigmoid(a.float().double())
    rest = (both - s).clamp(min=0.2 * both.min())
    z[..., 1], z[..., 2] = a.float(), (torch.log(rest) - torch.log1p(-rest)).float()
    z = z.view(N, groups * size)
    bias = torch.zeros(groups * size, device=dev()) if biased else None
    for top in (1, 2, 3):
        how = dict(score="sigmoid", groups=groups, top_groups=top, bias=bias)
        same(routed(z, 2, **how), chosen(z.double(), 2, **how))


@pytest.mark.parametrize("level", [-30.0, -50.0, -87.6])
def test_sigmoids_that_are_nearly_equal(level):
    g = torch.Generator(device="cuda").manual_seed(1)
    z = level + 1e-4 * torch.randint(0, 3, (20000, 64), generator=g, device=dev()) + torch.randint(-2, 2, (20000, 64), generator=g, device=dev()).float() * abs(level) * 2.0 ** -23
    how = dict(score="sigmoid", bias=torch.zeros(64, device=dev()))
    same(routed(z, 6, **how), chosen(z.double(), 6, **how))


@pytest.mark.parametrize("E", [512, 1024])
@pytest.mark.parametrize("groups", [1, 4])
def test_softmax_with_a_bias_next_to_a_border(E, groups):
    """An expert's number is all score and another's all but all bias, by one step of fp32 the larger, so that what a sum of exponentials has lost in 32 bits does not cancel: a lane's first
    terms add up to a little over 1, and each of the others is less than half a step of that."""
    g = torch.Generator().manual_seed(E + groups)
    tiny, size = -16.64, E // groups
    for v in (math.log(0.5) + 1e-4 + 2e-3 * torch.rand(1500, generator=g)).tolist():
        z = torch.full((1, E), tiny)
        z[0, 1:64], z[0, 0], z[0, 32] = v, 0.0, tiny
        if groups > 1:                                                # the group's second as good as its first
            z[0, 1], z[0, 33] = 0.0, tiny
        p = torch.softmax(z.double(), 1)[0]
        bias = torch.zeros(E)
        if groups == 1:
            bias[E - 1] = p[0] - p[E - 1]
            at = [E - 1]
        else:
            bias[E - 1] = (p[0] + p[1] - p[E - 1] - p[E - 2]) / 2
            bias[E - 2] = p[0] + p[1] - p[E - 1] - p[E - 2] - bias[E - 1].double()
            at = [E - 2]
        bias[at] = torch.nextafter(bias[at], torch.ones(1))
        t = p + bias.double()
        group = int(t.view(groups, size).sort(1, descending=True).values[:, :2].sum(1).argmax())
        want = group * size + int(t.view(groups, size)[group].argmax()) if groups > 1 else int(t.argmax())
        got = routed(z.to(dev()), 1, bias=bias.to(dev()), groups=groups, top_groups=1)
        assert int(got) == want, (v, int(got), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logits_and_biases_below_the_normal_numbers(dtype):
    z = torch.zeros(3, 40, device=dev())
    z[0, 7], z[0, 30], z[0, 3] = 3e-39, 2e-39, -1e-39
    z[1], z[1, 5], z[1, 20] = -2e-39, -1e-39, 1e-39
    z[2, ::2] = -0.0
    z = z.to(dtype)
    same(routed(z, 3), chosen(z.double(), 3))
    z = torch.full((2, 40), -95.0, device=dev(), dtype=dtype)
    bias = torch.zeros(40, device=dev())
    bias[9], bias[4], bias[30] = 3e-40, 2e-40, -1e-40
    how = dict(score="sigmoid", bias=bias)
    same(routed(z, 4, **how), chosen(z.double(), 4, **how))
    how = dict(score="sigmoid", bias=bias, groups=5, top_groups=2)
    same(routed(z, 4, **how), chosen(z.double(), 4, **how))


# ------------------------------------------------------------------ several tokens to a warp
MANY = [(5001, 8, 2, 1, 1), (5001, 60, 4, 1, 1), (20000, 60, 4, 6, 3), (9600, 256, 8, 8, 4), (20000, 256, 8, 1, 1), (5001, 1000, 5, 1, 1), (530001, 8, 2, 1, 1)]      # (the last: several in the backward pass, too)


@pytest.mark.parametrize("N,E,k,groups,top", MANY)
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("biased", [False, True])
def test_more_tokens_than_warps(N, E, k, groups, top, score, renorm, biased):
    """Indices, weights, means and gradient of as many tokens as give every warp several, rows of NaN, -inf and equal logits between ordinary ones."""
    dtype = BF16 if N == 5001 else F32
    g = torch.Generator(device="cuda").manual_seed(N + E)
    z = (2 * torch.randn(N, E, generator=g, device=dev())).to(dtype)
    kind = torch.randint(0, 12, (N,), generator=g, device=dev())
    z[kind == 0] = NEG
    z[kind == 1] = torch.where(torch.rand(int((kind == 1).sum()), E, generator=g, device=dev()) < 0.5, math.nan, z[kind == 1].float()).to(dtype)
    z[kind == 2] = 0.5
    z[kind == 3, 1:] = NEG
    z[kind == 4] = z[kind == 4].clamp(min=-1, max=1).round()
    bias = 0.1 * torch.randn(E, generator=g, device=dev()) if biased else None
    how = dict(bias=bias, score=score, groups=groups, top_groups=top)
    scale = 1.5
    zr = z.clone().requires_grad_()
    w, idx, mean = F.moe_route(zr, k, renorm=renorm, scale=scale, dtype=F32, **how)
    dw, dm = torch.randn(N, k, generator=g, device=dev()), torch.randn(E, generator=g, device=dev()) * E
    dz, = torch.autograd.grad([w, mean], [zr], [dw, dm])

    zd = torch.where(torch.isnan(z), NEG, z.double())
    want = chosen(zd, k, **how)
    same(idx, want)
    s, has, at = scores(zd, score), want >= 0, want.clamp(min=0).long()
    sj = torch.where(has, s.gather(1, at), 0.0)
    q = sj / sj.sum(1, keepdim=True).clamp(min=1e-300)
    p = s / s.sum(1, keepdim=True).clamp(min=1e-300)
    # exp and a division 10 half steps; sums of E terms 5 + E / 32 additions and its terms; the difference of a logit and the largest, rounded, |z| + |m| half steps of an exponential
    span = torch.where(zd > NEG, zd.abs() + zd.amax(1, keepdim=True).abs(), 0.0)
    tol = STEP * (10 + 2 * (5 + E / 32) + 4)
    ew = scale * (q if renorm else sj)
    spread = span.amax(1, keepdim=True)
    assert torch.all((w.double() - ew).abs() <= (tol + 2 * STEP * spread) * ew + 1e-37)
    # a warp's running sum, those of 8 warps, and 32 threads' of the blocks'
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    adds = N / (32 * sms) + 1 + 8 + sms / 8 + 1 + 5 + 2
    assert torch.all((mean.double() - p.mean(0)).abs() <= STEP * (adds * p.mean(0)) + tol * p.mean(0) + 2 * STEP * (p * spread).mean(0) + 1e-37)

    gw = torch.zeros_like(s).scatter_add_(1, at, torch.where(has, dw.double() * scale, 0.0))
    qf = torch.zeros_like(s).scatter_add_(1, at, q)
    h, rest = dm.double() / N, (1.0 if score == "softmax" else 1 - s)
    if renorm:
        ez = qf * (gw - (qf * gw).sum(1, keepdim=True)) * rest
    elif score == "softmax":
        ez = s * (gw - (s * gw).sum(1, keepdim=True))
    else:
        ez = s * rest * gw
    ez = ez + p * (h - (p * h).sum(1, keepdim=True)) * rest
    # two differences p (g - sum p g), whose terms are off by as much as a weight is, relative to the largest g of the row; then the rounding to the logits' type
    size = scale * dw.abs().amax(1, keepdim=True).double() + dm.abs().max().double() / N
    half = 2.0 ** -8 if dtype == BF16 else STEP
    assert torch.all((dz.double() - ez).abs() <= half * ez.abs() + 3 * (tol + 4 * STEP + 2 * STEP * spread) * size + 1e-37)


def test_routing_gives_the_same_bits_on_every_run():
    z = torch.randn(20000, 60, device=dev()).requires_grad_()
    bias = torch.randn(60, device=dev()) * 0.1
    dw, dm = torch.randn(20000, 4, device=dev()), torch.randn(60, device=dev())

    def step():
        w, idx, mean = F.moe_route(z, 4, bias=bias, score="sigmoid")
        return [w.detach(), idx, mean.detach(), *torch.autograd.grad([w, mean], [z], [dw, dm])]

    first = step()
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
