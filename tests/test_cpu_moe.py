"""A mixture of experts on the CPU: the plain forms of routing and experts against the definitions in 64 bits, the block and the decoder with experts."""
import math
import re

import pytest
import torch

from ml_b200 import ops
from ml_b200.ops import autograd as F
from tests import moe_oracle as oracle

I32 = torch.int32


def logits_of(N, E):
    z = torch.randn(N, E, generator=torch.Generator().manual_seed(N + E)) * 2
    if N > 5:
        z[1], z[2, ::2], z[3, 1:], z[4] = -math.inf, math.nan, -math.inf, 0.5
        z[5] = -95 - torch.arange(E) / 8
    return z


@pytest.mark.parametrize("N,E,k,groups,top", [(1, 1, 1, 1, 1), (9, 6, 2, 1, 1), (20, 33, 4, 1, 1), (12, 12, 3, 4, 2), (10, 64, 8, 8, 3), (8, 4, 1, 4, 1)])
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("biased", [False, True])
def test_plain_routing(N, E, k, groups, top, score, renorm, biased):
    z = logits_of(N, E).requires_grad_()
    bias = torch.randn(E) * 0.1 if biased else None
    how = dict(score=score, groups=groups, top_groups=top, renorm=renorm, scale=1.5)
    w, idx, mean = F.moe_route(z, k, bias=bias, **how)
    zd = torch.where(torch.isfinite(z.detach()), z.detach().double(), -math.inf).requires_grad_()
    ew, eidx, emean = oracle.route(zd, k, bias, **how)
    assert torch.equal(idx, eidx)
    assert torch.allclose(w.double(), ew, atol=1e-6) and torch.allclose(mean.double(), emean, atol=1e-6)
    dw, dm = torch.randn(N, k), torch.randn(E)
    dz, = torch.autograd.grad([w, mean], z, [dw, dm])
    ez, = torch.autograd.grad([ew, emean], zd, [dw.double(), dm.double()])
    assert torch.allclose(dz.double(), torch.nan_to_num(ez), atol=2e-6, rtol=1e-5)


@pytest.mark.parametrize("groups", [1, 4])
def test_bias_that_is_no_number(groups):
    z = torch.randn(6, 64, generator=torch.Generator().manual_seed(1))
    bias = torch.zeros(64)
    bias[3], bias[40], bias[50], bias[20] = math.nan, -math.inf, math.inf, math.inf
    w, idx = torch.empty(6, 4), torch.empty(6, 4, dtype=I32)
    ops.moe_route(w, idx, None, z, bias, "sigmoid", groups, groups, False)
    free = torch.sigmoid(z.double())
    free[:, [3, 40]] = -1
    free[:, [20, 50]] = 2
    at = free.sort(dim=1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(idx.long(), at) and torch.allclose(w, torch.sigmoid(z).gather(1, at), rtol=1e-5)


def test_routing_gradient_against_differences():
    torch.manual_seed(3)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            z = torch.randn(4, 7, dtype=torch.float64)
            dw, dm = torch.randn(4, 3, dtype=torch.float64), torch.randn(7, dtype=torch.float64)
            f = lambda t: (lambda w, i, m: float((w * dw).sum() + (m * dm).sum()))(*oracle.route(t, 3, score=score, renorm=renorm))
            zf = z.float().requires_grad_()
            w, _, mean = F.moe_route(zf, 3, score=score, renorm=renorm)
            dz, = torch.autograd.grad([w, mean], zf, [dw.float(), dm.float()])
            for n, e in ((0, 0), (1, 3), (2, 6), (3, 1), (3, 5)):
                up, lo = z.clone(), z.clone()
                up[n, e] += 1e-5
                lo[n, e] -= 1e-5
                assert abs((f(up) - f(lo)) / 2e-5 - float(dz[n, e])) < 1e-5


def case(N, E, k, C, I, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(N)]).to(I32)
    if N > 3:
        idx[1], idx[2, 0] = -1, -1
    return r(N, C), torch.softmax(r(N, k), 1), idx, r(E, 2 * I, C) * C ** -0.5, r(E, C, I) * I ** -0.5


@pytest.mark.parametrize("N,E,k,C,I", [(1, 1, 1, 16, 16), (7, 5, 2, 24, 40), (30, 4, 3, 16, 32)])
def test_plain_experts(N, E, k, C, I):
    x, w, idx, gate_up, down = leaves = case(N, E, k, C, I)
    with torch.no_grad():
        served = F.moe_mlp(*leaves)
    for t in (x, w, gate_up, down):
        t.requires_grad_()
    dout = torch.randn(N, C)
    out = F.moe_mlp(*leaves)
    got = [out.detach(), *torch.autograd.grad(out, [x, w, gate_up, down], dout)]
    assert torch.equal(served, got[0])
    for a, b in zip(got, oracle.mlp_grads(dout, x, w, idx, gate_up, down)):
        assert torch.allclose(a.double(), b, atol=1e-5, rtol=1e-4)


def test_frozen_parts_get_no_gradient():
    x, w, idx, gate_up, down = case(9, 4, 2, 16, 16)
    y = F.moe_mlp(x, w, idx, gate_up.requires_grad_(), down)
    want = oracle.mlp_grads(torch.ones_like(y), x, w, idx, gate_up, down)
    assert torch.allclose(torch.autograd.grad(y.sum(), gate_up)[0].double(), want[3], atol=1e-5)


def test_refusals():
    x, w, idx, gate_up, down = case(9, 4, 2, 16, 16)
    out = torch.empty_like(x)
    for bad in (dict(x=x[:, :8]), dict(out=out[:5]), dict(idx=idx.long()), dict(idx=idx[:, 0]), dict(weights=w[:, :1]), dict(gate_up=gate_up[:, :-1]), dict(down=down.transpose(1, 2)[:, :8]),
                dict(gate_up=gate_up.double()), dict(idx=idx + 4)):
        a = {**dict(out=out, x=x, weights=w, idx=idx, gate_up=gate_up, down=down), **bad}
        with pytest.raises(ValueError):
            ops.moe_mlp(a["out"], a["x"], a["weights"], a["idx"], a["gate_up"], a["down"])
    z, w, i = torch.zeros(4, 8), torch.empty(4, 2), torch.empty(4, 2, dtype=I32)
    for bad in (dict(score="other"), dict(groups=3), dict(groups=4, top_groups=5), dict(groups=8, top_groups=1), dict(groups=0), dict(bias=torch.zeros(7)), dict(bias=torch.zeros(8).double())):
        with pytest.raises(ValueError):
            ops.moe_route(w, i, None, z, **bad)
    for a in ((w.double(), i, None, z), (w, i.long(), None, z), (w, i, torch.empty(7), z), (w, i, None, z.double()), (w, i, None, torch.zeros(4, 2000)), (w, i, None, torch.zeros(8))):
        with pytest.raises(ValueError):
            ops.moe_route(*a)
    for a in ((torch.empty(4, 7), w, None, z, i), (torch.empty(4, 8), w.double(), None, z, i), (torch.empty(4, 8), w, torch.empty(7), z, i), (torch.empty(4, 8), w, None, z, i.long())):
        with pytest.raises(ValueError):
            ops.moe_route_bwd(*a)


def test_entry_points_have_one_signature():
    """What ctypes declares, what the extension module calls and what the kernel library's sources define are the same, parameter by parameter."""
    from ml_b200 import build
    from ml_b200.ops import native
    assert native.bridge().moe_signatures() == {"mlb_" + k: v for k, v in native._MOE_KINDS.items()}
    letter = {"void*": "p", "float*": "f", "int*": "i", "uint8_t*": "u", "int": "n", "long": "l", "float": "d", "cudaStream_t": "s"}
    defined = {}
    for src in (build.CSRC / "kernels").glob("moe*.cu*"):
        for name, args in re.findall(r"^MLB_API [\w ]+? (mlb_\w+)\(([^)]*)\)", src.read_text(), re.M):
            types = [re.sub(r"\s*\w+$", "", a.replace("const ", "").strip()).replace(" *", "*") for a in args.split(",")]
            defined[name] = "".join(letter.get(t, "?") for t in types)
    assert set(defined) == {"mlb_" + k for k in native._MOE_KINDS}
    for name, kinds in native._MOE_KINDS.items():
        assert len(defined["mlb_" + name]) == len(kinds), name
        assert all(d == k or (d == "p" and k in "bfiu") for d, k in zip(defined["mlb_" + name], kinds)), name


def test_entries_refuse_what_they_cannot_address():
    """-7, before anything is launched: memory off 16 bytes, rows apart by no multiple of 8, sizes out of range."""
    from ml_b200.ops import native
    if torch.cuda.is_available():
        pytest.skip("the addresses are nobody's memory: asked only where no kernel can run")
    L, ok, off = native.lib(), 1 << 20, (1 << 20) + 2
    sizes = dict(N=40, ld=64, k=2, E=4, C=64, I=48, bits=16)
    fwd = lambda **kw: L.mlb_moe_fwd(*{**{n: ok for n in ("out", "xs", "gu", "h", "y", "x", "weights", "gate_up", "down", "plan")}, **sizes, **kw}.values(), None)
    bwd = lambda **kw: L.mlb_moe_bwd(*{**{n: ok for n in ("dx", "dweights", "dgate_up", "ddown", "ys", "dgu", "dxs", "dout", "xs", "gu", "h", "y", "weights", "gate_up", "down", "plan")}, **sizes,
                                       **kw}.values(), None)
    few = lambda **kw: L.mlb_moe_few(*{**{n: ok for n in ("out", "x", "weights", "idx", "gate_up", "down", "part")}, **sizes, "N": 4, **kw}.values(), None)
    for call, names in ((fwd, ("out", "xs", "gu", "h", "y", "x", "gate_up", "down", "plan")),
                        (bwd, ("dx", "dgate_up", "ddown", "ys", "dgu", "dxs", "dout", "xs", "gu", "h", "y", "gate_up", "down", "plan")), (few, ("out", "x", "gate_up", "down", "part"))):
        for bad in [{n: off} for n in names] + [dict(ld=68), dict(C=72), dict(I=40), dict(E=1025), dict(E=0), dict(k=0), dict(bits=8), dict(N=1 << 31)]:
            assert call(**bad) == -7, (names, bad)
    assert few(N=9) == -7 and few(N=8, k=33) == -7
    assert L.mlb_moe_plan_ints(1 << 31, 2, 4) == L.mlb_moe_plan_rows(1 << 31, 2, 4) == -7
    assert L.mlb_moe_plan(off, ok, 40, 2, 4, None) == -7
    route = lambda **kw: L.mlb_moe_route(*{**dict(w=ok, idx=ok, mean=None, part=None, z=ok, bias=None, N=4, ld=64, E=64, k=2, sigmoid=0, groups=1, top=1, renorm=1, scale=1.0, zb=32, wb=32), **kw}.values(),
                                         None)
    for bad in (dict(E=1025), dict(k=0), dict(k=33), dict(E=1), dict(groups=3), dict(groups=64), dict(top=2), dict(zb=64), dict(N=-1)):
        assert route(**bad) == -7, bad


def test_a_plan_has_room_for_every_distribution():
    """Rows and tiles that the plan's buffers have, against the worst distributions of copies over experts."""
    from ml_b200.ops import native
    L = native.lib()
    for NK in (1, 2, 31, 32, 33, 255, 256, 257, 2048, 2049, 5000, 131073):
        for E in (1, 2, 7, 64, 1024):
            rows = L.mlb_moe_plan_rows(NK, 1, E)
            spread = [NK // E + (i < NK % E) for i in range(E)]
            ones = [1] * min(E - 1, NK - 1) + [NK - min(E - 1, NK - 1)]
            odd = [33] * min(E - 1, (NK - 1) // 33) + [NK - 33 * min(E - 1, (NK - 1) // 33)]
            tiles = NK // 256 + min(NK, E)
            for d in (spread, ones, odd):
                assert sum(-(-n // 32) * 32 for n in d) <= rows and rows % 32 == 0
                assert sum(-(-n // 256) for n in d) <= tiles
            assert L.mlb_moe_plan_ints(NK, 1, E) >= 2 * E + 2 + 4 * tiles + NK + rows


# ------------------------------------------------------------------ the block, the decoder
def test_block_gives_what_the_loop_over_experts_gives():
    from ml_b200.models.moe import MoE, MoEBlock
    torch.manual_seed(0)
    loop, block = MoEBlock(24, 32, 5, 2, std=0.3), MoE(24, 32, 5, 2, std=0.3)
    with torch.no_grad():
        block.router.copy_(loop.router)
        for e in range(5):
            block.gate_up[e].copy_(loop.gate_up[e])
            block.down[e].copy_(loop.down[e])
    x = torch.randn(40, 24)
    (a, la), (b, lb) = loop(x), block(x)
    assert torch.allclose(a, b, atol=1e-5) and torch.allclose(la, lb, atol=1e-6)
    (a.square().sum() + la).backward()
    (b.square().sum() + lb).backward()
    assert torch.allclose(loop.router.grad, block.router.grad, atol=1e-4)
    assert torch.allclose(torch.stack([p.grad for p in loop.down]), block.down.grad, atol=1e-4)


def test_balance_moves_the_choice():
    from ml_b200.models.moe import MoE
    torch.manual_seed(0)
    m = MoE(16, 16, 4, 1, score="sigmoid", balanced=True)
    with torch.no_grad():
        m.router.zero_()
    x = torch.randn(10, 16)
    m(x)
    assert m.load.tolist() == [10, 0, 0, 0]      # equal scores: the lowest index
    m.balance(0.1)
    assert m.bias.tolist() == pytest.approx([-0.1, 0.1, 0.1, 0.1])
    m(x)
    assert m.load.tolist() == [0, 10, 0, 0]
    m.eval()
    m(x[:2])
    assert m.load.tolist() == [0, 10, 0, 0]
    assert m.bfloat16().bias.dtype == torch.float32 and m.load.dtype == torch.float32
    with pytest.raises(ValueError):
        MoE(16, 16, 4, 1).balance()


def test_decoder_with_experts_trains():
    from ml_b200 import Config
    from ml_b200.models.modules import Decoder
    cfg = Config(V=61, C=32, L=2, H=2, I=48, T=16)
    torch.manual_seed(0)
    m = Decoder(cfg, experts=dict(n_experts=4, top_k=2, std=0.1))
    for n, p in m.named_parameters():
        if "moe" not in n:
            torch.nn.init.normal_(p, std=0.1)
    ids = torch.randint(0, 61, (2, 16), dtype=I32)
    loss = m(ids, torch.roll(ids, -1))
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    assert all(b.moe.router.grad.abs().sum() > 0 for b in m.blocks)
    with pytest.raises(ValueError):
        m.load_flat(torch.zeros(1))
    # the gradient of one weight against a difference
    p, at = m.blocks[1].moe.gate_up, (int(m.blocks[1].moe.load.argmax()), 5, 7)
    with torch.no_grad():
        both = []
        for d in (1e-2, -2e-2):
            p[at] += d
            both.append(float(m(ids, torch.roll(ids, -1))))
    assert abs((both[0] - both[1]) / 2e-2 - float(p.grad[at])) < 1e-3


def test_there_is_no_second_derivative():
    torch.manual_seed(0)
    x, w, idx = torch.randn(6, 8, requires_grad=True), torch.rand(6, 2, requires_grad=True), torch.randint(0, 3, (6, 2), dtype=torch.int32)
    gate_up, down, z = torch.randn(3, 8, 8, requires_grad=True), torch.randn(3, 8, 4, requires_grad=True), torch.randn(6, 3, requires_grad=True)
    for out, of in ((F.moe_mlp(x, w, idx, gate_up, down), [x, w, gate_up, down]), (F.moe_mlp(x, w, idx, gate_up, down), [x]), (F.moe_route(z, 2)[0], [z])):
        dout = torch.randn_like(out)
        plain, grads = (torch.autograd.grad(out, of, dout, retain_graph=True, create_graph=c) for c in (False, True))
        assert all(torch.equal(a, b) for a, b in zip(plain, grads)) and not any(g.requires_grad for g in plain)
        with pytest.raises(RuntimeError, match="no second derivative"):
            sum(g.square().sum() for g in grads).backward()


def test_tangents_and_traces_meet_the_functions():
    """Where nothing asks for a gradient, too: a tangent is refused as the other operators refuse it, and a trace holds the operator."""
    import torch.autograd.forward_ad as fwAD
    x, w, idx, gate_up, down = case(9, 4, 2, 16, 16)
    z = torch.randn(9, 4)
    for grad in (False, True):
        with torch.set_grad_enabled(grad), fwAD.dual_level():
            dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))
            for call in (lambda: F.moe_mlp(dual(x), w, idx, gate_up, down), lambda: F.moe_mlp(x, dual(w), idx, gate_up, down), lambda: F.moe_mlp(x, w, idx, gate_up, dual(down)),
                         lambda: F.moe_route(dual(z), 2)):
                with pytest.raises(NotImplementedError):
                    call()
    for call, args in ((F.moe_mlp, (x, w, idx, gate_up, down)), (lambda t: F.moe_route(t, 2)[0], (z,))):
        graph = torch.jit.trace(call, args, check_trace=False).graph
        assert any(n.kind() == "prim::PythonOp" for n in graph.nodes()), graph
    with torch.inference_mode():
        served = F.moe_mlp(x * 1, w, idx, gate_up, down)
    assert torch.equal(served, F.moe_mlp(x, w, idx, gate_up.requires_grad_(), down).detach())


def test_another_type_of_weights_leaves_the_balance_as_it_is():
    from ml_b200.models.moe import MoE
    m = MoE(16, 16, 8, 2, score="sigmoid", balanced=True)
    m.bias.copy_(0.5 + 1e-3 * torch.arange(8))
    m.load.copy_(70001.0 + torch.arange(8))
    bias, load = m.bias.clone(), m.load.clone()
    outer = torch.nn.Sequential(torch.nn.Sequential(m))
    for change in (torch.nn.Module.bfloat16, torch.nn.Module.half, torch.nn.Module.double, torch.nn.Module.float, lambda t: t.to(torch.bfloat16), lambda t: t.to("cpu", torch.float16),
                   lambda t: t.to(torch.device("cpu"))):
        change(outer)
        assert torch.equal(m.bias, bias) and torch.equal(m.load, load) and m.bias.dtype == m.load.dtype == torch.float32
    m.to("meta", torch.bfloat16)
    assert m.bias.is_meta and m.bias.dtype == torch.float32 and m.router.dtype == torch.bfloat16
    m.to_empty(device="cpu")
    assert m.bias.device.type == "cpu" and m.bias.dtype == torch.float32
    assert {n for n, _ in m.named_buffers()} == {"bias", "load"} and "load" not in m.state_dict()


@pytest.mark.parametrize("first", ["native_moe", "native_gen", "native"])
def test_modules_of_operators_are_imported_in_any_order(first):
    import subprocess
    import sys
    from pathlib import Path
    code = f"from ml_b200.ops import {first}; from ml_b200.ops import native as n, native_moe as m, native_gen as g; assert n.moe_mlp is m.moe_mlp and n.kv4_attn is g.kv4_attn and not hasattr(n, 'none')"
    subprocess.run([sys.executable, "-c", code], check=True, cwd=Path(__file__).resolve().parent.parent, timeout=300)
