"""Top-k mixture-of-experts SwiGLU block.

The reference's prototype has router / gating / expert kernels that nothing calls and a forward that hard-codes expert 0
(csrc/kernels/moe_kernels.cu:18-194, csrc/src/model.cu:829-861).  This block is functional: softmax router, top-k
selection with renormalised gates, tokens grouped per expert, each expert a SwiGLU MLP on the fused ops (tcgen05 GEMMs on
GPU), results combined by gate weight.  Single-process; `ml_b200.parallel.ep.EPMoEBlock` is the expert-parallel form
(experts split over ranks, tokens exchanged by all-to-all).

`MoE` is the block whose routing and experts are operators of the framework (`ops.autograd.moe_route`, `moe_mlp`): the experts' weights lie in one tensor
each, no step waits for the host, and the routing has sigmoid scores, a bias for balance and groups as options.  `ml_b200.models.modules.Decoder` takes it as its
feed-forward part (`Decoder(cfg, experts=dict(n_experts=8, top_k=2))`).
"""
from __future__ import annotations

import torch
import torch.nn as nn

from ..ops import autograd as F


class MoEBlock(nn.Module):
    def __init__(self, C: int, I: int, n_experts: int, top_k: int = 2, device="cpu", dtype=torch.float32, std: float = 0.02):
        super().__init__()
        self.C, self.I, self.E, self.k = C, I, n_experts, top_k
        mk = lambda *s: nn.Parameter(torch.randn(*s, device=device, dtype=dtype) * std)
        self.router = mk(n_experts, C)
        self.gate_up = nn.ParameterList([mk(2 * I, C) for _ in range(n_experts)])
        self.down = nn.ParameterList([mk(C, I) for _ in range(n_experts)])

    def forward(self, x):
        """x: [N, C] -> [N, C]; also returns the load-balancing auxiliary loss (mean prob * mean assignment per expert)."""
        N = x.shape[0]
        probs = torch.softmax(F.linear(x, self.router).float(), dim=-1)           # [N, E]
        gate, idx = probs.topk(self.k, dim=-1)
        gate = (gate / gate.sum(-1, keepdim=True)).to(x.dtype)
        out = torch.zeros_like(x)
        for e in range(self.E):
            tok, slot = (idx == e).nonzero(as_tuple=True)
            if tok.numel() == 0:
                continue
            h = F.linear(F.swiglu(F.linear(x[tok].contiguous(), self.gate_up[e])), self.down[e])
            out = out.index_add(0, tok, h * gate[tok, slot].unsqueeze(1))
        assign = torch.zeros(self.E, device=x.device).index_add_(0, idx.flatten(), torch.ones(idx.numel(), device=x.device)) / (N * self.k)
        aux = self.E * (probs.mean(0) * assign).sum()
        return out, aux


class MoE(nn.Module):
    """n_experts SwiGLU experts of width I behind a router that sends each token to top_k of them.

    score, groups, top_groups, renorm and scale are those of `ops.autograd.moe_route`.  With `balanced` the choice (not the weights) goes by score + `bias`, a buffer that
    `balance(rate)` moves towards the experts that had too few tokens in the last pass in training.  On CUDA C and I are multiples of 16 and tensors bf16."""

    def __init__(self, C: int, I: int, n_experts: int, top_k: int = 2, score: str = "softmax", balanced: bool = False, groups: int = 1, top_groups: int = 1, renorm: bool = True,
                 scale: float = 1.0, device="cpu", dtype=torch.float32, std: float = 0.02):
        super().__init__()
        self.C, self.I, self.E, self.k = C, I, n_experts, top_k
        self.how = dict(score=score, groups=groups, top_groups=top_groups, renorm=renorm, scale=scale)
        mk = lambda *s: nn.Parameter(torch.randn(*s, device=device, dtype=dtype) * std)
        self.router, self.gate_up, self.down = mk(n_experts, C), mk(n_experts, 2 * I, C), mk(n_experts, C, I)
        self.register_buffer("bias", torch.zeros(n_experts, device=device) if balanced else None)
        self.register_buffer("load", torch.zeros(n_experts, device=device), persistent=False)

    def _apply(self, fn, recurse=True):
        held = {n: t for n in ("bias", "load") if (t := getattr(self, n)) is not None}
        super()._apply(fn, recurse)
        for n, t in held.items():      # (a change of the weights' type leaves these as they are, in 32 bits)
            if getattr(self, n).dtype != torch.float32:
                setattr(self, n, t.to(getattr(self, n).device))
        return self

    def forward(self, x):
        """x: [N, C] -> [N, C]; also returns the load-balancing auxiliary loss (mean prob * mean assignment per expert)."""
        logits = F.linear(x, self.router) if len(x) else x @ self.router.T      # (the kernels' product takes one row at least)
        weights, idx, mean = F.moe_route(logits, self.k, bias=self.bias, **self.how)
        out = F.moe_mlp(x, weights, idx, self.gate_up, self.down)
        chosen = idx.flatten()
        load = torch.zeros_like(self.load).scatter_add_(0, chosen.clamp(min=0).long(), (chosen >= 0).float())
        if self.training:
            self.load.copy_(load)
        return out, self.E * (mean * load).sum() / max(1, chosen.numel())

    @torch.no_grad()
    def balance(self, rate: float = 1e-3):
        """Moves the bias of each expert by `rate`: up where its load is below the mean, down where it is above."""
        if self.bias is None:
            raise ValueError("a block that is not balanced has no bias")
        self.bias.add_(rate * torch.sign(self.load.mean() - self.load))
