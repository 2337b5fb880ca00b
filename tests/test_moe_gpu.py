"""Kernels of a mixture of experts (routing, the experts' products and their gradients) against the definitions in 64 bits."""
import math

import pytest
import torch

from ml_b200 import ops
from ml_b200.ops import autograd as F
from tests import moe_oracle as oracle

pytestmark = pytest.mark.gpu
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}      # half a step, relative: what one rounding is off by at most


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
    torch.cuda.synchronize()
    err = nat().get_error()
    nat().clear_error()
    assert err == 3 << 24 | detail, hex(err)


# ------------------------------------------------------------------ routing
def logits_of(N, E, dtype, seed=0, special=True):
    g = torch.Generator().manual_seed(1000 * N + E + seed)
    z = (torch.randn(N, E, generator=g) * 2).to(dtype)
    if special and N > 12:
        z[1] = -math.inf                       # a token that goes nowhere
        z[2, ::2] = math.nan                   # NaN is no expert
        z[3, 1:] = -math.inf                   # one expert left
        z[4] = 0.5                             # all equal
        z[5, :E // 2] = z[5, E - E // 2:].clone()
        z[6] = -90 - torch.arange(E, dtype=F32).to(dtype) / 8      # scores that vanish in 32 bits
        z[7] = torch.where(torch.arange(E) % 3 == 0, 40.0, -40.0).to(dtype)
        z[8] = torch.where(torch.arange(E) % 2 == 0, 0.0, -0.0).to(dtype)
    return z


def routed(z, k, wdtype=F32, mean=True, **how):
    N, E = z.shape
    w = torch.full((N, k), 7.0, dtype=wdtype, device=dev())
    idx, m = torch.full((N, k), 77, dtype=I32, device=dev()), torch.full((E,), 7.0, device=dev()) if mean else None
    b = how.pop("bias", None)
    ops.moe_route(w, idx, m, z.to(dev()), None if b is None else b.to(dev()), **how)
    return w, idx, m


ROUTES = [(1, 1, 1), (1, 2, 2), (7, 8, 2), (40, 33, 5), (100, 64, 6), (33, 128, 8), (20, 200, 8), (70, 256, 8), (16, 500, 3), (16, 1024, 32)]


@pytest.mark.parametrize("N,E,k", ROUTES)
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("biased", [False, True])
def test_routing(N, E, k, score, renorm, dtype, biased):
    z = logits_of(N, E, dtype)
    bias = torch.randn(E, generator=torch.Generator().manual_seed(E)) * 0.1 if biased else None
    how = dict(score=score, renorm=renorm, scale=1.5)
    w, idx, mean = routed(z, k, bias=bias, **how)
    ew, eidx, emean = oracle.route(z.double(), k, bias, **how)
    assert torch.equal(idx.cpu(), eidx)
    # exp: 3 steps of 2^-23 (its own 2, the split product 1); sums of E terms in a tree of 5 + E / 32 additions; a division, a product with the scale
    tol = (6 + 2 * (5 + E / 32) + 4) * HALF[F32]
    assert torch.all((w.cpu().double() - ew).abs() <= tol * ew.abs() + 1e-37)
    # and N of them added up, N / 8 and more in each of some running sums
    assert torch.all((mean.cpu().double() - emean).abs() <= (tol + (N / 8 + 16) * HALF[F32]) * emean + 1e-37)


@pytest.mark.parametrize("N,E,k,groups,top", [(5, 4, 1, 4, 1), (40, 12, 3, 4, 2), (60, 64, 4, 8, 4), (30, 256, 8, 8, 4), (20, 60, 5, 6, 5), (20, 32, 2, 32, 3), (9, 1024, 8, 32, 7)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_routing_in_groups(N, E, k, groups, top, score, biased):
    z = logits_of(N, E, F32, seed=3)
    if N > 12:
        z[9, E // groups:] = -math.inf                      # one group has experts
        z[10, :E - 1] = -math.inf                           # and the last one a single one
        z[11] = z[11, :E // groups].repeat(groups)          # equal groups
    bias = torch.randn(E, generator=torch.Generator().manual_seed(E)) * 0.1 if biased else None
    how = dict(score=score, groups=groups, top_groups=top)
    w, idx, _ = routed(z, k, bias=bias, mean=False, **how)
    ew, eidx, _ = oracle.route(z.double(), k, bias, **how)
    assert torch.equal(idx.cpu(), eidx)
    assert torch.all((w.cpu().double() - ew).abs() <= (6 + 2 * (5 + E / 32) + 4) * HALF[F32] * ew + 1e-37)


def test_routing_next_to_a_border():
    """Scores that 32 bits cannot tell apart are told apart, and equal ones go to the lowest index."""
    E = 64
    z = torch.zeros(3, E)
    bias = torch.zeros(E)
    bias[40], bias[3] = 1e-9, 5e-10                # beside scores of 0.5: one rounding of fp32 there is 3e-8
    z[1, 50] = 2.0 ** -30
    _, idx, _ = routed(z, 3, bias=bias, score="sigmoid")
    assert idx.tolist() == [[40, 3, 0], [40, 3, 50], [40, 3, 0]]


def test_routing_infinite_logits():
    z = torch.randn(4, 40)
    z[0, [7, 30]] = math.inf
    z[1, 5] = math.inf
    w, idx, _ = routed(z, 2)
    assert idx[0].tolist() == [7, 30] and w[0].tolist() == [0.5, 0.5] and idx[1, 0] == 5 and w[1].tolist() == [1.0, 0.0]
    w, _, mean = routed(z, 2, score="sigmoid", renorm=False)
    assert w[0].tolist() == [1.0, 1.0] and bool(torch.isfinite(mean).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_routing_of_strided_logits_and_bf16_weights(dtype):
    wide = logits_of(50, 90, dtype).to(dev())
    z = wide[:, 11:71]
    w, idx, mean = routed(z, 4, wdtype=BF16)
    ew, eidx, emean = oracle.route(z.cpu().double(), 4)
    assert torch.equal(idx.cpu(), eidx)
    assert torch.all((w.cpu().double() - ew).abs() <= (HALF[BF16] + 1e-5) * ew)
    d = torch.empty(50, 60, dtype=dtype, device=dev())
    g = torch.randn(50, 4, device=dev())
    ops.moe_route_bwd(d, g, None, z, idx)
    e = torch.empty_like(d)
    ops.moe_route_bwd(e, g, None, z.contiguous(), idx)
    assert torch.equal(d, e)


@pytest.mark.parametrize("N,E,k", ROUTES)
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradient_of_routing(N, E, k, score, renorm, dtype):
    z = logits_of(N, E, dtype)
    how = dict(score=score, renorm=renorm, scale=1.5)
    zc = z.to(dev()).requires_grad_()
    w, idx, mean = F.moe_route(zc, k, dtype=F32, **how)
    dw, dm = torch.randn(N, k, device=dev()), torch.randn(E, device=dev()) * E
    dz, = torch.autograd.grad([w, mean], [zc], [dw, dm])
    zd = torch.where(torch.isfinite(z), z.double(), -math.inf).requires_grad_()
    ew, eidx, emean = oracle.route(zd, k, **how)
    ez, = torch.autograd.grad([ew, emean], [zd], [dw.cpu().double(), dm.cpu().double()])
    ez = torch.nan_to_num(ez)
    assert torch.equal(idx.cpu(), eidx)
    # every gradient is a sum of two differences p (g - sum p g), whose terms are off by as much as a weight is: relative to the largest g of the row
    p_tol = (6 + 2 * (5 + E / 32) + 8) * HALF[F32]
    size = 1.5 * dw.abs().amax(1).cpu().double() + dm.abs().max().cpu().double() / N
    err = (dz.cpu().double() - ez).abs()
    assert torch.all(err <= HALF[dtype] * ez.abs() + 3 * p_tol * size[:, None] + 1e-37)


def test_gradient_of_routing_of_one_output():
    z = logits_of(30, 20, F32, special=False).to(dev()).requires_grad_()
    for pick in (0, 2):
        out = F.moe_route(z, 3)
        g = torch.randn_like(out[pick])
        dz, = torch.autograd.grad(out[pick], z, g)
        zd = z.detach().cpu().double().requires_grad_()
        ez, = torch.autograd.grad(oracle.route(zd, 3)[pick], zd, g.cpu().double())
        assert torch.allclose(dz.cpu().double(), ez, atol=1e-6, rtol=1e-5)


@pytest.mark.parametrize("groups", [1, 4])
def test_bias_that_is_no_number(groups):
    z = torch.randn(6, 64, generator=torch.Generator().manual_seed(1)).to(dev())
    bias = torch.zeros(64, device=dev())
    bias[3], bias[40], bias[50], bias[20] = math.nan, -math.inf, math.inf, math.inf
    w, idx = torch.empty(6, 4, device=dev()), torch.empty(6, 4, dtype=I32, device=dev())
    ops.moe_route(w, idx, None, z, bias, "sigmoid", groups, groups, False)
    free = torch.sigmoid(z.double())
    free[:, [3, 40]] = -1
    free[:, [20, 50]] = 2
    at = free.sort(dim=1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(idx.long(), at) and torch.allclose(w, torch.sigmoid(z).gather(1, at), rtol=1e-5)


def test_routing_of_no_tokens():
    w, idx, mean = routed(torch.empty(0, 8), 2)
    assert w.shape == (0, 2) and mean.abs().sum() == 0
    z = torch.empty(0, 8, device=dev(), requires_grad=True)
    out = F.moe_route(z, 2)
    assert torch.autograd.grad(out[0].sum() + out[2].sum(), z)[0].shape == (0, 8)


def test_gradient_of_an_expert_that_there_is_not():
    z = torch.zeros(2, 4, device=dev())
    d = torch.empty_like(z)
    ops.moe_route_bwd(d, torch.ones(2, 1, device=dev()), None, z, torch.tensor([[4], [-1]], dtype=I32, device=dev()))
    raised(0xD2)
    assert d.abs().sum() == 0


# ------------------------------------------------------------------ the experts
def experts(N, E, k, C, I, gates=BF16, seed=0, route="even", drop=0):
    g = torch.Generator().manual_seed(seed + N + 10 * E + 100 * C + I)
    r = lambda *s: torch.randn(*s, generator=g)
    if route == "even":
        idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(N)]) if N else torch.zeros(0, k)
    else:                                        # most tokens to the first experts
        idx = torch.topk(r(N, E) - 0.8 * torch.arange(E), k, 1).indices
    idx = idx.to(I32)
    w = torch.softmax(r(N, k), 1)
    if drop:
        lost = torch.randperm(N, generator=g)[:drop]
        idx[lost, :(k + 1) // 2] = -1
    to = lambda t: t.to(dev())
    return to(r(N, C).to(BF16)), to(w.to(gates)), to(idx), to((r(E, 2 * I, C) * C ** -0.5).to(BF16)), to((r(E, C, I) * I ** -0.5).to(BF16))


WHAT = ("out", "dx", "dweights", "dgate_up", "ddown")
# roundings to bf16 between the inputs and each:  h, y, out;  w dout, dh, g and u 2, dgu, dxs, dx;  h, y, the result;  w dout, dh, g and u 2, dgu, the result;  w dout, h, the result
ROUNDINGS = (3, 7, 3, 6, 3)


def close(got, want, sizes, names=WHAT):
    """Each rounding is off by half a step at most, relative to the terms that it is part of.  So row by row against the sums of the terms' absolute values (fp32 accumulation of up to
    2000 terms adds less than a tenth of a step); and all in all, where independent errors do not add up in size but in squares, against the norm itself."""
    for name, g in zip(names, got):
        i = WHAT.index(name)
        tol, w, s = ROUNDINGS[i] * HALF[BF16], want[i], sizes[i]
        d = g.detach().double() - w
        assert bool(torch.isfinite(d).all()), name
        if d.numel():
            assert float(d.norm()) <= tol * float(w.norm()) + 1e-30, (name, float(d.norm() / w.norm()), tol)
            rows, size = d.flatten(0, -2).norm(dim=1), s.flatten(0, -2).norm(dim=1)
            assert bool((rows <= 1.1 * tol * size + 1e-30).all()), name


MLPS = [(1, 1, 1, 16, 16), (1, 4, 2, 64, 48), (3, 5, 2, 48, 80), (31, 2, 1, 64, 64), (33, 4, 2, 256, 128), (64, 3, 3, 128, 256), (257, 64, 8, 64, 96), (301, 8, 3, 336, 208),
        (520, 2, 2, 272, 144), (700, 3, 1, 128, 272), (1500, 16, 4, 192, 160), (2500, 7, 2, 512, 320)]


@pytest.mark.parametrize("N,E,k,C,I", MLPS)
@pytest.mark.parametrize("gates", [BF16, F32])
@pytest.mark.parametrize("route", ["even", "crowded"])
def test_experts(N, E, k, C, I, gates, route):
    x, w, idx, gate_up, down = experts(N, E, k, C, I, gates, route=route, drop=N // 9)
    out = torch.full((N, C), 7.0, dtype=BF16, device=dev())
    ops.moe_mlp(out, x, w, idx, gate_up, down)
    close([out], [oracle.mlp(x.double(), w.double(), idx, gate_up.double(), down.double())], oracle.mlp_sizes(out, x, w, idx, gate_up, down))
    gone = (idx < 0).all(1)
    assert out[gone].abs().sum() == 0


@pytest.mark.parametrize("N,E,k,C,I", MLPS)
@pytest.mark.parametrize("gates", [BF16, F32])
@pytest.mark.parametrize("route", ["even", "crowded"])
def test_gradients_of_experts(N, E, k, C, I, gates, route):
    x, w, idx, gate_up, down = leaves = experts(N, E, k, C, I, gates, route=route, drop=N // 9)
    for t in (x, w, gate_up, down):
        t.requires_grad_()
    dout = torch.randn(N, C, generator=torch.Generator().manual_seed(N)).to(BF16).to(dev())
    out = F.moe_mlp(*leaves)
    grads = torch.autograd.grad(out, [x, w, gate_up, down], dout)
    close((out, *grads), oracle.mlp_grads(dout, x, w, idx, gate_up, down), oracle.mlp_sizes(dout, x, w, idx, gate_up, down))
    assert grads[1][idx < 0].abs().sum() == 0
    unused = [e for e in range(E) if not bool((idx == e).any())]
    assert grads[2][unused].abs().sum() == 0 and grads[3][unused].abs().sum() == 0


@pytest.mark.parametrize("N,E,k", [(5000, 300, 2), (20000, 6, 1), (3000, 1024, 4)])
def test_experts_of_many_copies(N, E, k):
    """Copies enough for several thread blocks of the plan, and more experts than it has threads."""
    x, w, idx, gate_up, down = leaves = experts(N, E, k, 32, 16, F32, route="even", drop=100)
    for t in (x, w, gate_up, down):
        t.requires_grad_()
    out = F.moe_mlp(*leaves)
    grads = torch.autograd.grad(out, [x, w, gate_up, down], dout := torch.randn(N, 32, device=dev()).to(BF16))
    close((out, *grads), oracle.mlp_grads(dout, x, w, idx, gate_up, down), oracle.mlp_sizes(dout, x, w, idx, gate_up, down))


@pytest.mark.parametrize("N,E,k", [(8, 3, 3), (6, 4, 8), (8, 2, 20), (8, 1, 32)])
def test_few_tokens_with_an_expert_many_times(N, E, k):
    x, w, idx, gate_up, down = experts(N, max(E, k), k, 96, 48, F32)
    idx.copy_(torch.randint(-1, E, idx.shape, generator=torch.Generator().manual_seed(N), dtype=I32))
    out = torch.empty_like(x)
    ops.moe_mlp(out, x, w, idx, gate_up[:E].contiguous(), down[:E].contiguous())
    close([out], [oracle.mlp(x.double(), w.double(), idx, gate_up.double(), down.double())], oracle.mlp_sizes(out, x, w, idx, gate_up, down))


@pytest.mark.parametrize("N", [1, 2, 7, 8, 9, 33])
@pytest.mark.parametrize("C,I,E,k", [(16, 16, 4, 2), (80, 528, 12, 3), (1040, 96, 6, 1), (2048, 1376, 16, 6), (256, 2816, 2, 2), (4112, 64, 9, 4)])
def test_few_tokens(N, C, I, E, k):
    """The form for few tokens, and the first number of tokens for the other one: sizes that end inside a stage, a warp's and a thread block's share, and leave some without any."""
    x, w, idx, gate_up, down = experts(N, E, k, C, I, F32, drop=N // 4)
    want, sizes = [oracle.mlp(x.double(), w.double(), idx, gate_up.double(), down.double())], oracle.mlp_sizes(x, x, w, idx, gate_up, down)
    for _ in range(2):
        out = torch.full_like(x, 7.0)
        ops.moe_mlp(out, x, w, idx, gate_up, down)
        close([out], want, sizes)


def test_the_same_expert_twice():
    x, w, idx, gate_up, down = leaves = experts(40, 4, 2, 64, 64)
    idx[:, 1] = idx[:, 0]
    for t in (x, w, gate_up, down):
        t.requires_grad_()
    out = F.moe_mlp(*leaves)
    grads = torch.autograd.grad(out, [x, w, gate_up, down], dout := torch.randn(40, 64, device=dev()).to(BF16))
    close((out, *grads), oracle.mlp_grads(dout, x, w, idx, gate_up, down), oracle.mlp_sizes(dout, x, w, idx, gate_up, down))


def test_tokens_that_all_go_nowhere():
    x, w, idx, gate_up, down = leaves = experts(20, 4, 2, 64, 64)
    idx.fill_(-1)
    for t in (x, w, gate_up, down):
        t.requires_grad_()
    out = F.moe_mlp(*leaves)
    grads = torch.autograd.grad(out, [x, w, gate_up, down], torch.ones_like(out))
    assert out.abs().sum() == 0 and all(g.abs().sum() == 0 for g in grads)


def test_no_tokens():
    leaves = experts(0, 4, 2, 64, 64)
    for t in (leaves[0], leaves[1], leaves[3], leaves[4]):
        t.requires_grad_()
    out = F.moe_mlp(*leaves)
    grads = torch.autograd.grad(out.sum(), [leaves[0], leaves[1], leaves[3], leaves[4]])
    assert out.shape == (0, 64) and all(g.abs().sum() == 0 for g in grads)


def test_an_expert_that_there_is_not():
    x, w, idx, gate_up, down = experts(20, 4, 2, 64, 64)
    out, clean = torch.empty_like(x), torch.empty_like(x)
    bad = idx.clone()
    bad[3, 1] = 4
    ops.moe_mlp(out, x, w, bad, gate_up, down)
    raised(0xD1)
    idx[3, 1] = -1
    ops.moe_mlp(clean, x, w, idx, gate_up, down)
    assert torch.equal(out, clean)


@pytest.mark.parametrize("N", [6, 200])
def test_values_that_are_not_numbers_stay_with_their_token(N):
    """NaN and infinities in a token reach its own row, and the gradients of the experts that it went to."""
    x, w, idx, gate_up, down = experts(N, 6, 2, 64, 64)
    idx[2], idx[4] = torch.tensor([0, 1]), torch.tensor([0, -1])
    idx[idx[:, 0] != 0, :] = idx[idx[:, 0] != 0, :].clamp(min=2)
    ref = torch.empty_like(x)
    ops.moe_mlp(ref, x, w, idx, gate_up, down)
    bad = x.clone()
    bad[2], bad[4, 5] = math.nan, math.inf
    out = torch.empty_like(x)
    ops.moe_mlp(out, bad, w, idx, gate_up, down)
    rest = [n for n in range(N) if n not in (2, 4)]
    assert torch.equal(out[rest], ref[rest]) and bool(out[2].isnan().all())
    leaves = [bad.requires_grad_(), w, gate_up.requires_grad_(), down.requires_grad_()]
    y = F.moe_mlp(leaves[0], w, idx, gate_up, down)
    dx, dgu, dd = torch.autograd.grad(y, [leaves[0], gate_up, down], torch.randn_like(y))
    assert torch.isfinite(dx[rest]).all() and torch.isfinite(dgu[2:]).all() and torch.isfinite(dd[2:]).all()


def test_rows_of_a_wider_tensor_and_frozen_weights():
    x, w, idx, gate_up, down = experts(70, 4, 2, 64, 48)
    wide = torch.zeros(70, 96, dtype=BF16, device=dev())
    wide[:, 16:80] = x
    part = wide[:, 16:80].requires_grad_()
    out, ref = torch.empty_like(x), torch.empty_like(x)
    ops.moe_mlp(out, part.detach(), w, idx, gate_up, down)
    ops.moe_mlp(ref, x, w, idx, gate_up, down)
    assert torch.equal(out, ref)
    y = F.moe_mlp(part, w, idx, gate_up, down)      # only the tokens are trained
    dx, = torch.autograd.grad(y, part, torch.ones_like(y[:1]).expand_as(y))
    want, sizes = (f(torch.ones_like(y), x, w, idx, gate_up, down) for f in (oracle.mlp_grads, oracle.mlp_sizes))
    close([dx], want, sizes, ["dx"])
    y = F.moe_mlp(x, w, idx, gate_up, down.requires_grad_())
    close(torch.autograd.grad(y, down, torch.ones_like(y)), want, sizes, ["ddown"])


def test_inputs_of_any_layout():
    """Broadcast, transposed and unaligned tensors, through the differentiable operators."""
    x, w, idx, gate_up, down = experts(40, 4, 2, 64, 48)
    one = x[:1].clone().requires_grad_()
    y = F.moe_mlp(one.expand(40, 64), w, idx, gate_up, down)
    d, = torch.autograd.grad(y, one, dout := torch.randn(40, 64, device=dev()).to(BF16))
    want = oracle.mlp_grads(dout, one.detach().expand(40, 64), w, idx, gate_up, down)
    assert float((d.double() - want[1].sum(0, keepdim=True)).norm()) <= 8 * HALF[BF16] * float(want[1].sum(0).norm())
    for t in (x.T.contiguous().T, torch.cat([x.flatten()[:1], x.flatten()])[1:].view(40, 64)):
        with torch.no_grad():
            assert torch.equal(F.moe_mlp(t, w, idx, gate_up, down), F.moe_mlp(x, w, idx, gate_up, down))
        g, = torch.autograd.grad(F.moe_mlp(t.requires_grad_(), w.T.contiguous().T, idx.T.contiguous().T, gate_up.transpose(1, 2).contiguous().transpose(1, 2), down), t, dout)
        assert torch.equal(g, torch.autograd.grad(F.moe_mlp(xr := x.clone().requires_grad_(), w, idx, gate_up, down), xr, dout)[0])
    z = torch.randn(8, 40, device=dev()).T.requires_grad_()
    a, b = F.moe_route(z, 2), F.moe_route(zc := z.detach().contiguous().requires_grad_(), 2)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert torch.equal(torch.autograd.grad(a[0].sum() + a[2][0], z)[0], torch.autograd.grad(b[0].sum() + b[2][0], zc)[0])


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (3,), (0, 2), (1, 3)])
def test_any_of_the_gradients(which):
    x, w, idx, gate_up, down = experts(70, 5, 2, 128, 80)
    leaves = [x, w, gate_up, down]
    for i in which:
        leaves[i].requires_grad_()
    y = F.moe_mlp(x, w, idx, gate_up, down)
    wanted = [leaves[i] for i in which]
    first = torch.autograd.grad(y, wanted, dout := torch.randn(70, 128, device=dev()).to(BF16), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, wanted, dout)))      # (nothing kept for it has changed)
    want, sizes = (f(dout, x, w, idx, gate_up, down) for f in (oracle.mlp_grads, oracle.mlp_sizes))
    close(first, want, sizes, [WHAT[1 + i] for i in which])


@pytest.mark.parametrize("extension", [True, False])
def test_there_is_no_second_derivative(extension):
    x, w, idx, gate_up, down = experts(20, 4, 2, 64, 48)
    z = torch.randn(20, 4, device=dev()).requires_grad_()
    x.requires_grad_(), down.requires_grad_()
    y = F.moe_mlp(x, w, idx, gate_up, down) if extension else F.MoEMLP.apply(x, w, idx, gate_up, down)
    p = F.moe_route(z, 2)[0] if extension else F.MoERoute.apply(z, 2, None, "softmax", 1, 1, True, 1.0, F32)[0]
    for out, of in ((y, [x, down]), (y, [x]), (p, [z])):
        dout = torch.randn_like(out)
        plain, grads = (torch.autograd.grad(out, of, dout, retain_graph=True, create_graph=c) for c in (False, True))
        assert all(torch.equal(a, b) for a, b in zip(plain, grads))
        with pytest.raises(RuntimeError, match="no second derivative"):
            sum(g.float().square().sum() for g in grads).backward()


@pytest.mark.parametrize("N", [3, 60])
def test_negative_indices_of_any_size_are_none(N):
    x, w, idx, gate_up, down = experts(N, 4, 2, 64, 48, drop=2)
    a, b = torch.empty_like(x), torch.empty_like(x)
    ops.moe_mlp(a, x, w, idx, gate_up, down)
    ops.moe_mlp(b, x, w, torch.where(idx < 0, -(1 << 31), idx.long()).to(I32), gate_up, down)
    assert torch.equal(a, b)


@pytest.mark.parametrize("N,E,k,C,I", [(1, 8, 2, 256, 128), (16, 8, 2, 256, 128), (900, 8, 3, 128, 256), (257, 64, 8, 64, 96)])
def test_the_same_bits_on_every_run_and_from_a_graph(N, E, k, C, I):
    x, w, idx, gate_up, down = leaves = experts(N, E, k, C, I, F32)
    for t in (x, w, gate_up, down):
        t.requires_grad_()
    dout = torch.randn(N, C, device=dev()).to(BF16)

    def step():
        out = F.moe_mlp(*leaves)
        return [out.detach(), *torch.autograd.grad(out, [x, w, gate_up, down], dout)]

    def serve():
        with torch.no_grad():
            return F.moe_mlp(*leaves)

    first, one = step(), serve()
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(first, step())) and torch.equal(one, serve())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), serve()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, out = step(), serve()
    for t in (*got, out):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, got)) and torch.equal(one, out)


def test_experts_on_another_stream():
    x, w, idx, gate_up, down = experts(300, 8, 2, 256, 128)
    ref, out = torch.empty_like(x), torch.empty_like(x)
    ops.moe_mlp(ref, x, w, idx, gate_up, down)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            ops.moe_mlp(out, x, w, idx, gate_up, down)
    ops.moe_mlp(ref, x, w, idx, gate_up, down)      # at the same time
    torch.cuda.synchronize()
    assert torch.equal(ref, out)


@pytest.mark.parametrize("N", [1, 6, 200])
def test_two_graphs_at_once(N):
    """Two captured calls, each with its own inputs, replayed on two streams beside one another and an uncaptured call: no workspace is another's."""
    calls = []
    for seed in range(2):
        torch.manual_seed(seed)
        x, w, idx, gate_up, down = experts(N, 8, 2, 512, 768)
        idx = (idx + seed) % 8
        z = torch.randn(N, 8, device=dev())
        outs = [torch.zeros_like(x), torch.zeros(N, 2, device=dev()), torch.zeros(N, 2, dtype=I32, device=dev()), torch.zeros(8, device=dev())]

        def work(outs=outs, x=x, w=w, idx=idx, gate_up=gate_up, down=down, z=z):
            ops.moe_mlp(outs[0], x, w, idx, gate_up, down)
            ops.moe_route(outs[1], outs[2], outs[3], z, score="sigmoid", groups=4, top_groups=2)

        work()
        want = [t.clone() for t in outs]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(8):
                work()
        calls.append((work, graph, outs, want, torch.cuda.Stream()))
    for _, _, outs, _, _ in calls:
        for t in outs:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(10):
        for _, graph, _, _, stream in calls:
            with torch.cuda.stream(stream):
                graph.replay()
        mine = [torch.zeros_like(t) for t in calls[0][2]]
        calls[0][0](mine)
        assert all(torch.equal(a, b) for a, b in zip(mine, calls[0][3]))
    torch.cuda.synchronize()
    for _, _, outs, want, _ in calls:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("N", [1, 8, 100])
def test_the_output_in_the_tokens_place(N):
    x, w, idx, gate_up, down = experts(N, 4, 2, 320, 64)
    out = torch.empty_like(x)
    ops.moe_mlp(out, x, w, idx, gate_up, down)
    ops.moe_mlp(x, x, w, idx, gate_up, down)
    assert torch.equal(out, x)


def test_a_token_costs_the_same_bits_in_any_batch_of_the_kind():
    """What a token's experts give does not depend on who else is there (in the same form of the kernels)."""
    x, w, idx, gate_up, down = experts(900, 8, 2, 128, 128)
    all_, some = torch.empty_like(x), torch.empty_like(x[:700])
    ops.moe_mlp(all_, x, w, idx, gate_up, down)
    ops.moe_mlp(some, x[:700], w[:700], idx[:700], gate_up, down)
    assert torch.equal(all_[:700], some)


def test_refusals():
    x, w, idx, gate_up, down = experts(20, 4, 2, 64, 64)
    out = torch.empty_like(x)
    ops_args = ("out", "x", "weights", "idx", "gate_up", "down")
    def refused(**kw):
        a = {**dict(zip(ops_args, (out, x, w, idx, gate_up, down))), **kw}
        with pytest.raises(ValueError):
            ops.moe_mlp(*(a[n] for n in ops_args))
    refused(x=x.float()), refused(out=out.float()), refused(idx=idx.long()), refused(gate_up=gate_up[:, :-2]), refused(down=down.transpose(1, 2))
    refused(weights=w[:, :1]), refused(out=torch.empty(64, 20, dtype=BF16, device=dev()).T), refused(x=torch.empty(64, 20, dtype=BF16, device=dev()).T)
    refused(x=torch.empty(20 * 64 + 1, dtype=BF16, device=dev())[1:].view(20, 64))
    refused(gate_up=torch.empty(4 * 128 * 64 + 1, dtype=BF16, device=dev())[1:].view(4, 128, 64))
    odd = experts(20, 4, 2, 64, 64)
    refused(gate_up=odd[3][:, :80].contiguous(), down=odd[4][:, :, :40].contiguous())      # 40 is no multiple of 16
    refused(x=x[:, :56].contiguous(), out=out[:, :56].contiguous(), gate_up=gate_up[:, :, :56].contiguous(), down=down[:, :56].contiguous())
    z = torch.zeros(4, 8, device=dev())
    w8, i8 = torch.empty(4, 2, device=dev()), torch.empty(4, 2, dtype=I32, device=dev())
    for bad in (dict(score="other"), dict(groups=3), dict(groups=4, top_groups=5), dict(groups=8, top_groups=1), dict(groups=0)):
        with pytest.raises(ValueError):
            ops.moe_route(w8, i8, None, z, **bad)
    for a in ((w8.double(), i8, None, z), (w8, i8.long(), None, z), (w8, i8, torch.empty(7, device=dev()), z), (w8, i8, None, z.half()), (w8, i8, None, z, torch.zeros(9, device=dev())),
              (w8, i8, None, torch.zeros(8, 4, device=dev()).T), (w8, i8, None, torch.zeros(4, 2000, device=dev()))):
        with pytest.raises(ValueError):
            ops.moe_route(*a)


def test_entry_points_are_called_alike_through_python_and_the_extension_module(monkeypatch):
    n = nat()
    x, w, idx, gate_up, down = leaves = experts(50, 8, 2, 64, 64)
    z = torch.randn(50, 8, device=dev()).requires_grad_()
    for t in (x, w, gate_up, down):
        t.requires_grad_()

    def work():
        rw, ridx, mean = F.moe_route(z, 2)
        out = F.moe_mlp(*leaves)
        served = torch.empty_like(x)
        ops.moe_mlp(served, *(t.detach() for t in leaves))
        return [rw.detach(), ridx, mean.detach(), out.detach(), served, *torch.autograd.grad([rw, mean], z, [torch.ones_like(rw), torch.ones_like(mean)]),
                *torch.autograd.grad(out, [x, w, gate_up, down], torch.ones_like(out))]

    outs = []
    for entries in (n._Ctypes(), n.bridge()):
        monkeypatch.setattr(n, "_E", entries)
        outs.append(work())
    assert all(torch.equal(a, b) for a, b in zip(*outs))


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("how", [dict(), dict(score="sigmoid", balanced=True, groups=4, top_groups=2, scale=2.5), dict(renorm=False)])
@pytest.mark.parametrize("N", [1, 5, 300])
def test_block_of_experts(how, N):
    """Router, experts and balancing loss together, forward and backward, against the definitions with the logits and weights that the block has."""
    from ml_b200.models.moe import MoE
    torch.manual_seed(N)
    m = MoE(128, 96, 8, 2, device=dev(), dtype=BF16, std=0.1, **how)
    if m.bias is not None:
        m.bias.normal_(std=0.05)
    x = torch.randn(N, 128, device=dev()).to(BF16).requires_grad_()
    y, aux = m(x)
    dout = torch.randn(N, 128, device=dev()).to(BF16)
    grads = torch.autograd.grad([y, aux], [x, m.gate_up, m.down, m.router], [dout, torch.ones_like(aux)])
    z = (x.detach() @ m.router.detach().T)      # what the block's product gives, to a rounding: the choice is compared where it is clear
    logits = F.linear(x.detach(), m.router.detach())
    assert torch.allclose(z.float(), logits.float(), atol=0.05, rtol=0.02)
    kw = {k: v for k, v in m.how.items()}
    zd = logits.double().cpu().requires_grad_()
    w, idx, mean = oracle.route(zd, 2, None if m.bias is None else m.bias.cpu(), **kw)
    wb = w.detach().to(BF16).to(dev())
    want, sizes = (f(dout, x, wb, idx.to(dev()), m.gate_up, m.down) for f in (oracle.mlp_grads, oracle.mlp_sizes))
    close([y, grads[1], grads[2]], want, sizes, ["out", "dgate_up", "ddown"])
    load = torch.bincount(idx[idx >= 0].long().flatten(), minlength=8).double()
    assert torch.equal(m.load.cpu().double(), load)
    want_aux = float(8 * (mean.detach() * load).sum() / idx.numel())
    assert abs(float(aux.detach()) - want_aux) < 1e-4 * max(1.0, want_aux)
    # the router: the weights' and the loss's gradients through the logits, rounded to bf16 on their way (5 roundings: weights', logits', a product's each)
    back = 8 * (mean * load).sum() / idx.numel()
    dz, = torch.autograd.grad([w, back], zd, [want[2].cpu(), torch.ones_like(back)])
    dr = dz.T @ x.detach().double().cpu()
    assert float((grads[3].double().cpu() - dr).norm()) <= 8 * HALF[BF16] * float(dr.norm()) + 1e-6
    m.eval()
    with torch.no_grad():
        served, _ = m(x.detach())
    close([served], want[:1], sizes, ["out"])


def test_decoder_with_experts_trains_and_is_captured():
    from ml_b200 import Config
    from ml_b200.models.modules import Decoder
    cfg = Config(V=512, C=128, L=2, H=2, I=192, T=64)
    torch.manual_seed(0)
    m = Decoder(cfg, device="cuda:0", experts=dict(n_experts=8, top_k=2, std=0.05))
    for n, p in m.named_parameters():
        if "moe" not in n:
            torch.nn.init.normal_(p, std=0.05)
    ids = torch.randint(0, 512, (2, 64), dtype=I32, device=dev())
    tgt = torch.roll(ids, -1).contiguous()
    ps = list(m.parameters())

    def step():
        loss = m(ids, tgt)
        return [loss.detach(), *torch.autograd.grad(loss, ps)]

    first = step()
    assert all(bool(torch.isfinite(t).all()) for t in first) and all(float(t.float().abs().sum()) > 0 for t in first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    for (n, _), a, b in zip([("loss", None), *m.named_parameters()], first, got):      # (products whose sums are split add up in the order of arrival: equal to a rounding)
        assert torch.allclose(a.float(), b.float(), atol=2e-2 * float(a.float().abs().max()), rtol=2e-2), n
