"""Experts on the GPU: how far roundings add up, and the block with any number of experts and tokens."""
import pytest
import torch

from ml_b200.ops import autograd as F
from tests import moe_oracle as oracle

pytestmark = pytest.mark.gpu
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
HALF = 2.0 ** -8      # half a step of bf16, relative


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


# What is rounded to bf16 on the way to each, fp32 gates:  h, y, out;  w dout, dh's two factors g and u, dgu, dxs, dx;  h, y;  w dout, g and u, dgu, the result;  w dout, h, the result
ROUNDINGS = {"out": 3, "dx": 6, "dweights": 2, "dgate_up": 5, "ddown": 3}


@pytest.mark.parametrize("N,E,k,C,I", [(1500, 16, 4, 192, 160), (2500, 7, 2, 512, 320), (4000, 8, 2, 768, 256)])
def test_roundings_add_up_in_squares(N, E, k, C, I):
    """A rounding is off by half a step at most, a value's mantissa anywhere in its binade: the error's square is on average a third of the largest's, the value's about twice its least, so that
    0.41 half steps of the norm are lost.  Independent roundings add up in squares, over 10^5 values and more to a fraction of a per cent.  Some go through factors above 1 (SwiGLU's gradient
    moves by |g silu''| of a step of g beside |silu'|, in squares within 1.5 of its own size for normal g), so 0.6 half steps are allowed for each: half as much error again is over it."""
    g = torch.Generator().manual_seed(N)
    r = lambda *s: torch.randn(*s, generator=g)
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(N)]).to(dev(), I32)
    to = lambda t, s=1.0: (t * s).to(dev(), BF16).requires_grad_()
    x, gate_up, down = to(r(N, C)), to(r(E, 2 * I, C), C ** -0.5), to(r(E, C, I), I ** -0.5)
    w = torch.softmax(r(N, k), 1).to(dev()).requires_grad_()
    dout = r(N, C).to(dev(), BF16)
    y = F.moe_mlp(x, w, idx, gate_up, down)
    got = (y, *torch.autograd.grad(y, [x, w, gate_up, down], dout))
    want = oracle.mlp_grads(dout, x, w, idx, gate_up, down)
    for (name, n), a, b in zip(ROUNDINGS.items(), got, want):
        err = float((a.detach().double() - b).norm() / b.norm())
        assert err <= 0.6 * HALF * n ** 0.5, (name, err, err / HALF / n ** 0.5)


@pytest.mark.parametrize("E,k", [(1, 1), (2, 1), (6, 2), (60, 4), (100, 3)])
@pytest.mark.parametrize("N", [1, 7, 33, 130])
def test_block_of_any_number_of_experts(E, k, N):
    """Router products of any width, forward and backward, in training and without a gradient."""
    from ml_b200.models.moe import MoE
    torch.manual_seed(E + N)
    m = MoE(64, 48, E, k, score="sigmoid", balanced=True, device=dev(), dtype=BF16, std=0.1)
    x = torch.randn(N, 64, device=dev()).to(BF16).requires_grad_()
    y, aux = m(x)
    logits = F.linear(x.detach(), m.router.detach())
    exact = x.detach().double() @ m.router.detach().double().T
    assert float((logits.double() - exact).norm()) <= 1.01 * HALF * float(exact.norm())
    w, idx, mean = F.moe_route(logits, k, bias=m.bias, **m.how)
    want = oracle.mlp(x.detach().double(), w.double(), idx, m.gate_up.detach().double(), m.down.detach().double())
    assert float((y.detach().double() - want).norm()) <= 3 * HALF * float(want.norm())
    assert m.load.tolist() == torch.bincount(idx.flatten().long(), minlength=E).tolist()
    grads = torch.autograd.grad([y, aux], [x, *m.parameters()], [torch.randn_like(y), torch.ones_like(aux)])
    assert all(bool(torch.isfinite(t).all()) for t in grads)
    m.eval()
    with torch.no_grad():
        served, _ = m(x.detach())
    assert float((served.double() - want).norm()) <= 3 * HALF * float(want.norm())


@pytest.mark.parametrize("device,dtype", [("cpu", F32), ("cuda:0", BF16)])
def test_block_of_no_tokens(device, dtype):
    from ml_b200.models.moe import MoE
    m = MoE(64, 48, 6, 2, score="sigmoid", balanced=True, device=device, dtype=dtype)
    x = torch.empty(0, 64, device=device, dtype=dtype, requires_grad=True)
    y, aux = m(x)
    assert y.shape == (0, 64) and float(aux.detach()) == 0 and m.load.sum() == 0
    grads = torch.autograd.grad(y.sum() + aux, [x, *m.parameters()])
    assert all(bool((t == 0).all()) for t in grads)
    with torch.no_grad():
        assert m.eval()(x)[0].shape == (0, 64)
