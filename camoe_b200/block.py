"""One CaMoE block from this package's parts: time mix, router, experts.

    x = x + time_mix(ln1(x));   x = x + sum over the top-k experts of weight * expert(ln2(x))

(camoe/system.py:304-355 without its market, critic and bridge: the router here
is a linear map with a softmax over the chosen logits).  ``ExpertBlock`` trains
with ``forward`` and generates with ``forward_state``, in which the sequences of
a batch may belong to different requests with their own low-rank adapters on
the time mix's projections.

    python -m camoe_b200.block      # a few training steps, then generation, on cuda:0
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .experts import ExpertLayer
from .timemix import RWKV7TimeMix


class ExpertBlock(nn.Module):
    def __init__(self, n_embd: int, n_layer: int, layer_id: int, n_experts: int = 8, top_k: int = 2,
                 hidden: int | None = None):
        super().__init__()
        if not 1 <= top_k <= n_experts:
            raise ValueError(f"top_k must be from 1 to the number of experts, got {top_k} of {n_experts}")
        self.top_k = top_k
        self.ln1, self.ln2 = nn.LayerNorm(n_embd), nn.LayerNorm(n_embd)
        self.att = RWKV7TimeMix(n_embd, n_layer, layer_id)
        self.router = nn.Linear(n_embd, n_experts, bias=False)
        self.experts = ExpertLayer(n_embd, n_experts, hidden)

    def _experts(self, x):
        h = self.ln2(x.to(self.ln2.weight.dtype))
        value, index = torch.topk(self.router(h).float(), self.top_k, dim=-1)
        return self.experts(h, index, torch.softmax(value, dim=-1))

    def forward(self, x: torch.Tensor, v_first: torch.Tensor | None = None):
        """x [B, T, C] fp32 or bf16, whose dtype the result has.  Returns (x, v_first,
        state_representation)."""
        y, v_first, srep = self.att(self.ln1(x.to(self.ln1.weight.dtype)), v_first)
        x = x + y.to(x.dtype)
        return x + self._experts(x).to(x.dtype), v_first, srep

    @torch.no_grad()
    def forward_state(self, x: torch.Tensor, v_first: torch.Tensor | None = None, state=None, adapters=None,
                      adapter: torch.Tensor | None = None):
        """The block over the next steps of each sequence (``RWKV7TimeMix.forward_state``,
        whose state, adapters and adapter these are).  Returns (x, v_first, new_state)."""
        y, v_first, _, state = self.att.forward_state(self.ln1(x.to(self.ln1.weight.dtype)), v_first, state, adapters,
                                                      adapter)
        x = x + y.to(x.dtype)
        return x + self._experts(x).to(x.dtype), v_first, state


def main():
    from .adapters import AdapterSet

    torch.manual_seed(0)
    C, L, B, T = 256, 2, 4, 64
    blocks = nn.ModuleList(ExpertBlock(C, L, i) for i in range(L)).cuda()
    optimizer = torch.optim.AdamW(blocks.parameters(), lr=1e-3)
    data, target = torch.randn(2, B, T, C, device="cuda")
    for step in range(5):
        x, v_first = data, None
        for block in blocks:
            x, v_first, _ = block(x, v_first)
        loss = (x - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        print(f"step {step}: loss {loss.item():.4f}")
    adapters = [AdapterSet().add("key", torch.randn(3, 16, C, device="cuda") * C ** -0.5,
                                 torch.randn(3, C, 16, device="cuda") * 0.1) for _ in range(L)]
    request = torch.tensor([0, 2, -1, 1], dtype=torch.int32, device="cuda")  # the third sequence has none
    state, x = [None] * L, data
    for token in range(4):
        v_first = None
        for i, block in enumerate(blocks):
            x, v_first, state[i] = block.forward_state(x, v_first, state[i], adapters[i], request)
        x = x[:, -1:]
        print(f"token {token}: norm {float(x.norm()):.4f}")


if __name__ == "__main__":
    main()
