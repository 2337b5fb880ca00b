"""The autograd nodes of routing and experts: what transforms, modes and traces get, and saved tensors that come back in another form."""
import pytest
import torch

from ml_b200 import ops
from ml_b200.ops import autograd as F

pytestmark = pytest.mark.gpu
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
NODES = ["route", "route_grouped", "experts", "experts_few"]


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


def node(name):
    """(operands, call): each a plain call of the extension module with one result"""
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g).to(dev())
    if name.startswith("route"):
        how = dict(score="sigmoid", groups=4, top_groups=2, renorm=False) if name == "route_grouped" else {}
        return [r(50, 24).to(BF16)], lambda z: F.moe_route(z, 3, **how)[0]
    N = 5 if name == "experts_few" else 70
    idx = torch.stack([torch.randperm(6, generator=g)[:2] for _ in range(N)]).to(dev(), I32)
    idx[1, 0] = -1
    return [r(N, 96).to(BF16), torch.softmax(r(N, 2), 1), (r(6, 160, 96) / 10).to(BF16), (r(6, 96, 80) / 9).to(BF16)], lambda x, w, gate_up, down: F.moe_mlp(x, w, idx, gate_up, down)


def strided(t):
    u = torch.empty(*t.shape[::-1], 2, dtype=t.dtype, device=t.device)[..., 0]
    return u.permute(*reversed(range(t.dim()))).copy_(t)


def offset(t):
    return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)


@pytest.mark.parametrize("name", NODES)
def test_saved_tensors_come_back_in_another_form(name):
    """The same values in another layout or off a 16-byte boundary give the same gradients; another type, device or size is refused in front of the launches."""
    from torch.autograd.graph import saved_tensors_hooks
    operands, call = node(name)
    leaves = [t.requires_grad_() for t in operands]

    def grads(change):
        with saved_tensors_hooks(lambda t: t, change):
            y = call(*leaves)
        assert "CppNode" in y.grad_fn.name()
        torch.manual_seed(4)
        return torch.autograd.grad(y, leaves, torch.randn(y.shape, device=dev()).to(y.dtype))

    want = grads(lambda t: t)
    for same in (strided, offset, lambda t: strided(offset(t)), lambda t: t.cpu().cuda()):
        assert all(torch.equal(a, b) for a, b in zip(want, grads(same)))
    for other in (torch.Tensor.float, torch.Tensor.double, torch.Tensor.half, torch.Tensor.cpu, lambda t: t[:-1], lambda t: t.view(-1), lambda t: t[None]):
        changed = lambda t: other(t).dtype != t.dtype or other(t).device != t.device or other(t).shape != t.shape
        with pytest.raises(AssertionError, match="saved tensor"):
            grads(lambda t: other(t) if changed(t) else t)
    assert all(torch.equal(a, b) for a, b in zip(want, grads(lambda t: t)))


@pytest.mark.parametrize("name", NODES)
def test_transforms_and_modes_take_the_functions(name):
    """Whether or not a gradient is asked for: under a transform, a trace, a dispatch mode or with a tangent the Python Function runs, with its results and its errors."""
    import torch.autograd.forward_ad as fwAD
    from torch.utils._python_dispatch import TorchDispatchMode
    operands, call = node(name)
    assert "CppNode" in call(*(t.requires_grad_() for t in operands)).grad_fn.name()
    operands = [t.detach() for t in operands]
    want = call(*operands)
    assert not want.requires_grad
    with pytest.raises(RuntimeError, match="autograd.Function with functorch"):
        torch.func.grad(lambda x: call(x, *operands[1:]).float().sum())(operands[0])
    with pytest.raises(RuntimeError, match="autograd.Function with functorch"):
        torch.vmap(lambda x: call(x, *operands[1:]))(torch.stack([operands[0], operands[0]]))
    with pytest.raises(RuntimeError, match="autograd.Function with functorch"):
        torch.func.grad(lambda s: (call(*operands).float() * s).sum())(torch.ones(1, device=dev()))
    for i in range(len(operands)):
        with fwAD.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError):
            call(*(fwAD.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(operands)))

    class Seen(TorchDispatchMode):
        ops = []

        def __torch_dispatch__(self, fn, types, args=(), kwargs=None):
            self.ops.append(str(fn))
            return fn(*args, **(kwargs or {}))

    with Seen() as seen:
        got = call(*operands)
    assert torch.equal(got, want) and any("new_empty" in o for o in seen.ops)
    graph = torch.jit.trace(lambda *a: call(*a), tuple(operands), check_trace=False).graph
    assert any(n.kind() == "prim::PythonOp" for n in graph.nodes()), graph


@pytest.mark.parametrize("N", [1, 8, 9, 200])
def test_without_a_gradient_the_operator_is_the_entry_point(N):
    """Weights that take gradients, none asked for: the bits of `ops.moe_mlp`, eagerly, in inference mode and from a graph."""
    g = torch.Generator().manual_seed(N)
    r = lambda *s: torch.randn(*s, generator=g).to(dev())
    x, w, gate_up, down = r(N, 96).to(BF16), torch.softmax(r(N, 2), 1), (r(6, 160, 96) / 10).to(BF16).requires_grad_(), (r(6, 96, 80) / 9).to(BF16).requires_grad_()
    idx = torch.stack([torch.randperm(6, generator=g)[:2] for _ in range(N)]).to(dev(), I32)
    want = torch.empty_like(x)
    ops.moe_mlp(want, x, w, idx, gate_up, down)
    with torch.no_grad():
        assert torch.equal(F.moe_mlp(x, w, idx, gate_up, down), want)
        wide = torch.zeros(N, 104, dtype=BF16, device=dev())
        wide[:, :96] = x
        assert torch.equal(F.moe_mlp(wide[:, :96], w, idx, gate_up, down), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = F.moe_mlp(x, w, idx, gate_up, down)
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    with torch.inference_mode():
        assert torch.equal(F.moe_mlp(x * 1, w, idx, gate_up, down), want)
        assert torch.equal(F.moe_mlp(x, w, idx, gate_up, down), want)


@pytest.mark.parametrize("form", [offset, strided, lambda t: t[:1].expand_as(t)], ids=["offset", "strided", "broadcast"])
@pytest.mark.parametrize("extension", [True, False])
def test_gradients_that_arrive_in_any_layout(form, extension):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).to(dev())
    N = 40
    x, w, gate_up, down = r(N, 96).to(BF16), torch.softmax(r(N, 2), 1), (r(6, 160, 96) / 10).to(BF16), (r(6, 96, 80) / 9).to(BF16)
    idx = torch.stack([torch.randperm(6, generator=g)[:2] for _ in range(N)]).to(dev(), I32)
    dout = form(r(N, 96).to(BF16))
    leaves = [t.requires_grad_() for t in (x, w, gate_up, down)]
    # (tokens off a 16-byte boundary are no plain call)
    y = F.moe_mlp(x if extension else offset(x), w, idx, gate_up, down)
    assert ("CppNode" in y.grad_fn.name()) == extension
    want = torch.autograd.grad(F.moe_mlp(x, w, idx, gate_up, down), leaves, dout.contiguous().clone())
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dout), want))
    z = r(N, 6).requires_grad_()
    p = F.moe_route(z, 2)[0] if extension else F.MoERoute.apply(z, 2, None, "softmax", 1, 1, True, 1.0, F32)[0]
    dp = form(r(N, 2))
    assert torch.equal(*(torch.autograd.grad(p, z, d, retain_graph=True)[0] for d in (dp, dp.contiguous().clone())))
